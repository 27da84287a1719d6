// Gated linear recurrence over time, forward and backward: the member of the Elman family whose
// state enters linearly, so that it is elementwise over channels.  Per channel (b, i), state in fp32:
//   u_t = sigmoid(-f_t);  p_t = reset[t,b] ? 0 : h_{t-1};  h_t = p_t + u_t (c_t - p_t);  y_t = h_t silu(z_t)
// and backwards, with g_t = dL/dh_t and D_t the part of it that comes from later steps,
//   g_t = dy_t silu(z_t) + D_t;  dc_t = g_t u_t;  df_t = g_t (p_t - c_t) u_t (1 - u_t);
//   dz_t = dy_t h_t silu'(z_t);  D_{t-1} = reset[t,b] ? 0 : (1 - u_t) g_t.
// The state moves by u (c - p) rather than being rebuilt as (1-u) p + u c: a gate that keeps almost
// everything has u below the spacing of floats near 1, where 1 - u cannot hold it.
//
// Bound by HBM: forward 4 values an element, backward 7 (each of f, c, z, dy read once, each result
// written once); the backward pass recomputes the states from one in GL_CHUNK that the forward saved.
// Measured, calls on bf16, the same inputs again and again: T4096 B64 d1536 562 us forward (5.7 TB/s; 634 among other calls
// with inputs that change), 1120 backward (5.0; instruction issue is next); T65536 B1 d1280, where the columns are few and the
// tiles wait for the chain of states, 188 (3.6) and 340 (3.5).
#include <string.h>

#include <mutex>

#include "common.cuh"
#include "sm100_ptx.cuh"
#include "tc_helpers.cuh"

namespace elman {

namespace {

struct Strides { long t, b; };          // element strides of a [T, B, d] tensor whose channels are dense

struct GlParams {
  int T, B, d;
  const void *f, *c, *z, *dy;
  Strides sf, sc, sz, sy, sdf, sdc, sdz;   // sy: y (forward) or dy (backward)
  const float* h0;                      // [B, d] or null: zeros
  const unsigned char* reset;           // [T, B] or null
  float* saved;                         // [ceil(T / GL_CHUNK), B, d]: state before step k GL_CHUNK; null: not kept
  void* y;
  float* h_last;                        // [B, d]
  const float* dh_last;                 // [B, d] or null: zeros
  void *df, *dc, *dz;
  float* dh0;                           // [B, d]
};

// u = sigmoid(-f) and e = exp(f): 1 - u = e u to full relative precision.  f is held at 80 so that e
// stays finite (u = 1.8e-35 there); NaN passes.
__device__ __forceinline__ float keep_gate(float f, float& e) {
  e = __expf(f > 80.f ? 80.f : f);
  return __fdividef(1.f, 1.f + e);
}

// Up to SEQ_STEPS steps (the generation step is T = 1) one thread walks a channel: the warps of a tile
// would mostly idle.
constexpr int SEQ_STEPS = 8;

template <typename T>
__global__ void __launch_bounds__(128) gl_forward_seq_kernel(GlParams p) {
  const long col = (long)blockIdx.x * blockDim.x + threadIdx.x;
  if (col >= (long)p.B * p.d) return;
  const int b = (int)(col / p.d), i = (int)(col - (long)b * p.d);
  const T* f = (const T*)p.f + b * p.sf.b + i;
  const T* c = (const T*)p.c + b * p.sc.b + i;
  const T* z = (const T*)p.z + b * p.sz.b + i;
  T* y = (T*)p.y + b * p.sy.b + i;
  float h = p.h0 != nullptr ? p.h0[col] : 0.f;
#pragma unroll 8
  for (int t = 0; t < p.T; ++t) {
    if (p.saved != nullptr && t % GL_CHUNK == 0) p.saved[(long)(t / GL_CHUNK) * p.B * p.d + col] = h;
    if (p.reset != nullptr && p.reset[(long)t * p.B + b] != 0) h = 0.f;
    float e;
    const float u = keep_gate(to_f(f[t * p.sf.t]), e);
    h = fmaf(u, to_f(c[t * p.sc.t]) - h, h);
    y[t * p.sy.t] = from_f<T>(h * siluf_(to_f(z[t * p.sz.t])));
  }
  p.h_last[col] = h;
}

template <typename T>
__global__ void __launch_bounds__(128) gl_backward_seq_kernel(GlParams p) {
  const long col = (long)blockIdx.x * blockDim.x + threadIdx.x;
  const long cols = (long)p.B * p.d;
  if (col >= cols) return;
  const int b = (int)(col / p.d), i = (int)(col - (long)b * p.d);
  const T* f = (const T*)p.f + b * p.sf.b + i;
  const T* c = (const T*)p.c + b * p.sc.b + i;
  const T* z = (const T*)p.z + b * p.sz.b + i;
  const T* dy = (const T*)p.dy + b * p.sy.b + i;
  T* df = (T*)p.df + b * p.sdf.b + i;
  T* dc = (T*)p.dc + b * p.sdc.b + i;
  T* dz = (T*)p.dz + b * p.sdz.b + i;
  float D = p.dh_last != nullptr ? p.dh_last[col] : 0.f;
  float before[SEQ_STEPS], h = p.T > 0 ? p.saved[col] : 0.f;
#pragma unroll
  for (int t = 0; t < SEQ_STEPS; ++t) {
    if (t >= p.T) break;
    if (p.reset != nullptr && p.reset[(long)t * p.B + b] != 0) h = 0.f;
    before[t] = h;
    float e;
    const float u = keep_gate(to_f(f[t * p.sf.t]), e);
    h = fmaf(u, to_f(c[t * p.sc.t]) - h, h);
  }
#pragma unroll
  for (int t = SEQ_STEPS - 1; t >= 0; --t) {
    if (t >= p.T) continue;
    float e;
    const float u = keep_gate(to_f(f[t * p.sf.t]), e), cv = to_f(c[t * p.sc.t]), zv = to_f(z[t * p.sz.t]);
    const float g0 = to_f(dy[t * p.sy.t]), prev = before[t];
    const float now = fmaf(u, cv - prev, prev);
    const float g = fmaf(g0, siluf_(zv), D);
    dz[t * p.sdz.t] = from_f<T>(g0 * now * dsiluf_(zv));
    dc[t * p.sdc.t] = from_f<T>(g * u);
    df[t * p.sdf.t] = from_f<T>(g * (prev - cv) * u * (e * u));
    D = p.reset != nullptr && p.reset[(long)t * p.B + b] != 0 ? 0.f : fmaf(-u, g, g);
  }
  p.dh0[col] = D;
}

// ---------------------------------------------------------------------------
// Sequences of more than a few steps: tiles of (W warps x L steps) x (32 V channels), each read once.  The kernels
// of this section take the rows whose last 128 bytes would be mostly empty (whole_width below) and count channels through
// batch rows; the next section's take all others.
//
// A warp holds L steps of 32 lanes x V channels in registers and scans them from a zero state: h_out = P h_in + H with
// P = prod(1 - u).  Where P is near one its distance from one has to be exact, or what the steps add is lost; where it
// is small P itself, or a state that has long been forgotten leaves 2^-24 of itself behind.  So both are scanned, and
// the pair (K, H) keeps the one that counts: K = P where P < 1/2, else P - 1 (kept() below).  K = -1 says that a reset lies
// inside: h_out = H, and h_in (which may be anything) is not read.  The tile's own pair goes to the tiles that follow in time through L2;
// they fold the pairs of their group of GROUP tiles onto the state at the group's start, which the last
// tile of the group before has published.  The association is fixed, so results do not depend on
// timing; the chain of dependent exchanges is one per GROUP tiles.  Backwards the same with time
// reversed, D in place of h, and the states recomputed from `saved`.
//
// Pairs and states are their own flags: the workspace starts as all ones, which no published value is
// (NaN goes out as 0x7fffffff), so an exchange is one store and one load.  Tiles are handed out in time
// order by a counter: whoever a tile waits for has started before it and waits for nobody behind it.
// ---------------------------------------------------------------------------
// Long groups make the chain of states short, short ones leave fewer pairs to fold and registers to hold them.  Forward and
// backward, us, with 8 / 10 / 16: T65536 B1 d1280 bf16 518 / 527 / 540, T65536 B1 d256 168 / 162 / 157, T4096 B64 d1536
// 1670 / 1690 / 1736.
constexpr int GROUP = 10;
constexpr uint32_t NOT_YET = 0xFFFFFFFFu;

struct GlChain {             // workspace; all of it starts as NOT_YET
  uint32_t* ctrl;            // [0]: tiles handed out - 1; [1]: 0 once a wait has given up
  float2* pairs;             // [tiles in time][columns]
  float* states;             // [groups][columns]
  int* status;
  long spin_limit;
  int stall;                 // test hook: this tile publishes nothing
  int leave;                 // test hook: 32 k + w: at a block's tile k its warp w gives up the wait for the stage
};

struct Pair { float K, H; };
// K from P and P - 1: P only above zero (2^-149 stands for less), P - 1 from -1/2 up to zero.
__device__ __forceinline__ float kept(float P, float P_1) { return P_1 >= -0.5f ? P_1 : fmaxf(P, 1.4e-45f); }
template <bool RESET> __device__ __forceinline__ float pass(float S, Pair a) {
  const float rest = a.K > 0.f ? 0.f : 1.f;      // (known before S is: two dependent instructions a pair)
  const float t = fmaf(rest, S, fmaf(a.K, S, a.H));
  return RESET && a.K == -1.f ? a.H : t;
}
template <bool RESET> __device__ __forceinline__ Pair join(Pair a, Pair b) {       // a, then b
  const float Pa = a.K > 0.f ? a.K : 1.f + a.K, Pa_1 = a.K > 0.f ? a.K - 1.f : a.K;
  const float Pb = b.K > 0.f ? b.K : 1.f + b.K, Pb_1 = b.K > 0.f ? b.K - 1.f : b.K;
  const Pair ab = Pair{RESET && a.K == -1.f ? -1.f : kept(Pa * Pb, fmaf(Pa, Pb_1, Pa_1)), pass<false>(a.H, b)};
  return RESET && b.K == -1.f ? b : ab;
}

// The same with P and P - 1 both at hand, as a warp has them.  P - 1 = -2 says that a reset lies inside.
struct Stretch { float P, P_1, H; };
template <bool RESET> __device__ __forceinline__ float pass(float S, Stretch a) {
  const bool near = a.P_1 >= -0.5f;
  const float t = fmaf(near ? 1.f : 0.f, S, fmaf(near ? a.P_1 : a.P, S, a.H));
  return RESET && a.P_1 < -1.5f ? a.H : t;
}
template <bool RESET> __device__ __forceinline__ Stretch join(Stretch a, Stretch b) {
  const Stretch ab = Stretch{a.P * b.P, RESET && a.P_1 < -1.5f ? -2.f : fmaf(a.P, b.P_1, a.P_1), pass<false>(a.H, b)};
  return RESET && b.P_1 < -1.5f ? b : ab;
}
template <bool RESET> __device__ __forceinline__ Pair pair_of(Stretch a) {
  return Pair{RESET && a.P_1 < -1.5f ? -1.f : kept(a.P, a.P_1), a.H};
}

// The V channels of a lane; two of them are one packed fp32x2 operand (half the instructions: at HBM
// speed the forward kernel has 44 issue slots for a warp's 32 elements, the backward kernel 76).
template <int V> struct Vec;
template <> struct Vec<1> {
  float x;
  __device__ __forceinline__ Vec() {}
  __device__ __forceinline__ explicit Vec(float s) : x(s) {}
  __device__ __forceinline__ float get(int) const { return x; }
  __device__ __forceinline__ void set(int, float s) { x = s; }
};
template <> struct Vec<2> {
  unsigned long long x;                // one register pair from load to store: packing costs nothing
  __device__ __forceinline__ Vec() {}
  __device__ __forceinline__ explicit Vec(float s) : Vec(s, s) {}
  __device__ __forceinline__ Vec(float lo, float hi) { asm("mov.b64 %0, {%1, %2};" : "=l"(x) : "f"(lo), "f"(hi)); }
  __device__ __forceinline__ void halves(float& lo, float& hi) const { asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(x)); }
  __device__ __forceinline__ float get(int v) const {
    float lo, hi;
    halves(lo, hi);
    return v == 0 ? lo : hi;
  }
  __device__ __forceinline__ void set(int v, float s) { *this = v == 0 ? Vec(s, get(1)) : Vec(get(0), s); }
};
__device__ __forceinline__ Vec<1> vfma(Vec<1> a, Vec<1> b, Vec<1> c) { return Vec<1>(fmaf(a.x, b.x, c.x)); }
__device__ __forceinline__ Vec<1> vmul(Vec<1> a, Vec<1> b) { return Vec<1>(a.x * b.x); }
__device__ __forceinline__ Vec<1> vadd(Vec<1> a, Vec<1> b) { return Vec<1>(a.x + b.x); }
__device__ __forceinline__ Vec<1> vsub(Vec<1> a, Vec<1> b) { return Vec<1>(a.x - b.x); }
__device__ __forceinline__ Vec<2> vfma(Vec<2> a, Vec<2> b, Vec<2> c) {
  Vec<2> r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.x) : "l"(a.x), "l"(b.x), "l"(c.x));
  return r;
}
__device__ __forceinline__ Vec<2> vmul(Vec<2> a, Vec<2> b) {
  Vec<2> r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.x) : "l"(a.x), "l"(b.x));
  return r;
}
__device__ __forceinline__ Vec<2> vadd(Vec<2> a, Vec<2> b) {
  Vec<2> r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.x) : "l"(a.x), "l"(b.x));
  return r;
}
__device__ __forceinline__ Vec<2> vsub(Vec<2> a, Vec<2> b) { return vfma(b, Vec<2>(-1.f), a); }   // exact product: one rounding

__device__ __forceinline__ float exp2_(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float rcp_(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
constexpr float LOG2E = 1.4426950408889634f;
// 1 / (1 + exp2(x)), or with MINUS the negative of that; e receives exp2(x)
template <int V, bool MINUS = false> __device__ __forceinline__ Vec<V> gate_of(Vec<V> x, Vec<V>& e) {
#pragma unroll
  for (int v = 0; v < V; ++v) e.set(v, exp2_(x.get(v)));
  const Vec<V> den = MINUS ? vfma(e, Vec<V>(-1.f), Vec<V>(-1.f)) : vadd(e, Vec<V>(1.f));
  Vec<V> r;
#pragma unroll
  for (int v = 0; v < V; ++v) r.set(v, rcp_(den.get(v)));
  return r;
}

template <typename T, int V> struct Lane;                    // V adjacent channels as they are in memory
template <> struct Lane<float, 1> {
  typedef float Raw;
  static __device__ __forceinline__ Vec<1> get(Raw r) { return Vec<1>(r); }
  static __device__ __forceinline__ Raw put(Vec<1> v) { return v.x; }
  static __device__ __forceinline__ Raw put_minus(Vec<1> v) { return -v.x; }
};
template <> struct Lane<bf16, 1> {
  typedef unsigned short Raw;
  static __device__ __forceinline__ Vec<1> get(Raw r) { return Vec<1>(__uint_as_float((uint32_t)r << 16)); }
  static __device__ __forceinline__ Raw put(Vec<1> v) { return __bfloat16_as_ushort(__float2bfloat16_rn(v.x)); }
  static __device__ __forceinline__ Raw put_minus(Vec<1> v) { return __bfloat16_as_ushort(__float2bfloat16_rn(-v.x)); }
};
template <> struct Lane<bf16, 2> {
  typedef uint32_t Raw;
  static __device__ __forceinline__ Vec<2> get(Raw r) {
    return Vec<2>(__uint_as_float(r << 16), __uint_as_float(r & 0xFFFF0000u));
  }
  static __device__ __forceinline__ Raw put(Vec<2> v) {
    float lo, hi;
    v.halves(lo, hi);
    const __nv_bfloat162 p = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const Raw*>(&p);
  }
  static __device__ __forceinline__ Raw put_minus(Vec<2> v) { return put(v) ^ 0x80008000u; }
};

__device__ __forceinline__ uint32_t word_of(float x) { return x != x ? 0x7FFFFFFFu : __float_as_uint(x); }
__device__ __forceinline__ void publish(float2* at, Pair a) {
  asm volatile("st.relaxed.gpu.global.v2.b32 [%0], {%1, %2};" ::"l"(at), "r"(word_of(a.K)), "r"(word_of(a.H)) : "memory");
}
__device__ __forceinline__ void publish(float* at, float x) {
  asm volatile("st.relaxed.gpu.global.b32 [%0], %1;" ::"l"(at), "r"(word_of(x)) : "memory");
}
template <int N> __device__ __forceinline__ bool look(const void* at, uint32_t (&w)[N]) {
  if constexpr (N == 4)
    asm volatile("ld.relaxed.gpu.global.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]) : "l"(at) : "memory");
  else if constexpr (N == 2)
    asm volatile("ld.relaxed.gpu.global.v2.b32 {%0, %1}, [%2];" : "=r"(w[0]), "=r"(w[1]) : "l"(at) : "memory");
  else
    asm volatile("ld.relaxed.gpu.global.b32 %0, [%1];" : "=r"(w[0]) : "l"(at) : "memory");
  bool there = true;
#pragma unroll
  for (int k = 0; k < N; ++k) there = there && w[k] != NOT_YET;
  return there;
}
__device__ __forceinline__ void look_if(bool wanted, const float2* at, uint32_t (&w)[2]) {
  asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %3, 0;\n\t@p ld.relaxed.gpu.global.v2.b32 {%0, %1}, [%2];\n\t}"
               : "+r"(w[0]), "+r"(w[1]) : "l"(at), "r"((uint32_t)wanted));
}
__device__ __forceinline__ void look_if(bool wanted, const float* at, uint32_t& w) {
  asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %2, 0;\n\t@p ld.relaxed.gpu.global.b32 %0, [%1];\n\t}"
               : "+r"(w) : "l"(at), "r"((uint32_t)wanted));
}

// Bounds a polling loop that a whole warp runs together.
struct Patience {
  long spins = 0;
  unsigned long long t0 = 0;
  __device__ __forceinline__ bool left(const GlChain& ch, int step) {
    ++spins;
    bool stop = spins > ch.spin_limit;
    if ((spins & 255) == 0) {
      uint32_t aborted[1];
      look<1>(ch.ctrl + 1, aborted);
      const unsigned long long now = ptx::globaltimer_ns();
      if (t0 == 0) t0 = now;
      stop = stop || aborted[0] == 0 || now - t0 > ptx::kWaitDeadlineNs;
    }
    if (!__any_sync(0xFFFFFFFFu, stop)) return true;
    if ((threadIdx.x & 31) == 0) {
      asm volatile("st.relaxed.gpu.global.b32 [%0], %1;" ::"l"(ch.ctrl + 1), "r"(0) : "memory");
      report_timeout(ch.status, KID_GATED_LINEAR, step);
    }
    return false;
  }
};
// The whole warp waits until every lane's N words are there; false: gave up.
template <int N> __device__ __forceinline__ bool await(const void* at, uint32_t (&w)[N], const GlChain& ch, int step) {
  Patience patience;
  while (!__all_sync(0xFFFFFFFFu, look<N>(at, w)))
    if (!patience.left(ch, step)) return false;
  return true;
}

// What the scanning warps of a block share.  Every member is read between barriers that lie after the
// write and before the next tile's write.
template <int V, int W> struct Shared {
  Pair own[W][32 * V];             // the warps' pairs, in the scan's direction
  Pair before[GROUP - 1][32 * V];  // pairs of the tiles before in the group
  float start[32 * V];             // state at the group's start
  float enters[W][32 * V];         // state that enters each warp
  int next;                        // the block's next tile
  int gave_up;
};
// Barrier of the block's first `warps` warps.
__device__ __forceinline__ void warps_sync(int warps) {
  asm volatile("bar.sync 1, %0;" ::"r"(32 * warps) : "memory");
}

// From the warps' pairs to the state that enters each: all threads call it; `n` counts tiles and `w` warps in
// the scan's direction; `initial` is the state at the scan's start.  False: a
// wait gave up.
template <int V, int W, bool RESET>
__device__ __forceinline__ bool enter(Shared<V, W>& sh, int w, int warps, Vec<V> K, Vec<V> H, int n, int tiles,
                                      long base, long cols, Vec<V> initial, const GlChain& ch, int ticket,
                                      uint32_t grabbed, Vec<V>& S) {
  const int lane = threadIdx.x & 31, x = threadIdx.x;
#pragma unroll
  for (int v = 0; v < V; ++v) sh.own[w][lane * V + v] = Pair{K.get(v), H.get(v)};
  const int first = n / GROUP * GROUP, in_group = n - first;
  const bool ends_group = in_group == GROUP - 1, more = n + 1 < tiles && ticket != ch.stall;
  if (w == 0 && first == 0) {
#pragma unroll
    for (int v = 0; v < V; ++v) sh.start[lane * V + v] = initial.get(v);
  }
  warps_sync(warps);
  // `base` is the tile's first of `cols` channels; one thread per channel folds from here to the last barrier
  const long mine = base + x, col = base + lane * V, seen = col < cols ? col : cols - V;
  const bool on = x < 32 * V && mine < cols;
  if (on && more && !ends_group) {
    Pair all = sh.own[0][x];
    for (int k = 1; k < warps; ++k) all = join<RESET>(all, sh.own[k][x]);
    publish(ch.pairs + (long)n * cols + mine, all);
  }
  if (in_group > 0 || first > 0) {
    bool ok = true;
    for (int k = w; k < in_group && ok; k += warps) {
      uint32_t g[2 * V];
      ok = await<2 * V>(ch.pairs + (long)(first + k) * cols + seen, g, ch, n);
#pragma unroll
      for (int v = 0; v < V; ++v)
        sh.before[k][lane * V + v] = Pair{__uint_as_float(g[2 * v]), __uint_as_float(g[2 * v + 1])};
    }
    if (w == warps - 1 && first > 0 && ok) {
      uint32_t g[V];
      ok = await<V>(ch.states + (long)(first / GROUP - 1) * cols + seen, g, ch, n);
#pragma unroll
      for (int v = 0; v < V; ++v) sh.start[lane * V + v] = __uint_as_float(g[v]);
    }
    if (!ok && lane == 0) sh.gave_up = 1;
  }
  if (x == 0) sh.next = (int)(grabbed + 1u);
  if (tiles > 1) warps_sync(warps);
  if (sh.gave_up) return false;
  if (x < 32 * V) {
    float s = sh.start[x];
    for (int k = 0; k < in_group; ++k) s = pass<RESET>(s, sh.before[k][x]);
    for (int k = 0; k < warps; ++k) {
      sh.enters[k][x] = s;
      s = pass<RESET>(s, sh.own[k][x]);
    }
    if (on && more && ends_group) publish(ch.states + (long)(first / GROUP) * cols + mine, s);
  }
  warps_sync(warps);
#pragma unroll
  for (int v = 0; v < V; ++v) S.set(v, sh.enters[w][lane * V + v]);
  return true;
}

// A warp's scan from a zero state, from gates `nu` = -u (a packed fma has no negation): P, P - 1 and the state a step on.
template <int V> struct Scan {
  Vec<V> H, P, P_1;
  __device__ __forceinline__ Scan() : H(0.f), P(1.f), P_1(0.f) {}
  __device__ __forceinline__ void step(Vec<V> nu, Vec<V> c) {
    H = vfma(nu, vsub(H, c), H);
    P_1 = vfma(nu, P, P_1);
    P = vfma(nu, P, P);
  }
  __device__ __forceinline__ Vec<V> K() const {
    Vec<V> k;
#pragma unroll
    for (int v = 0; v < V; ++v) k.set(v, kept(P.get(v), P_1.get(v)));
    return k;
  }
};

// exp2's argument held at 115 (u = 2^-115), so that u (1 - u) = e u^2 stays a number; NaN passes.
template <int V> __device__ __forceinline__ Vec<V> held(Vec<V> x) {
#pragma unroll
  for (int v = 0; v < V; ++v) {
    float m;
    asm("min.NaN.f32 %0, %1, %2;" : "=f"(m) : "f"(x.get(v)), "f"(115.f));
    x.set(v, m);
  }
  return x;
}

// Steps of a warp whose document starts anew, as bits (lanes of one batch row agree).
template <int L> __device__ __forceinline__ uint32_t reset_bits(const GlParams& p, int t0, int b) {
  uint32_t bits = 0;
#pragma unroll
  for (int l = 0; l < L; ++l)
    if (t0 + l < p.T && p.reset[(long)(t0 + l) * p.B + b] != 0) bits |= 1u << l;
  return bits;
}
template <int V> __device__ __forceinline__ Vec<V> unless(bool cut, Vec<V> x) {
#pragma unroll
  for (int v = 0; v < V; ++v) x.set(v, cut ? 0.f : x.get(v));
  return x;
}

// L rows of a tensor, this lane's channels; rows past the end repeat the last one.
template <typename T, int V, int L>
__device__ __forceinline__ void load_rows(typename Lane<T, V>::Raw (&r)[L], const void* base, Strides s, int t0, int T_, int b, int i) {
  typedef typename Lane<T, V>::Raw Raw;
  const char* at = (const char*)base + (b * s.b + i) * (long)sizeof(T);
  const long step = s.t * (long)sizeof(T);
  if (t0 + L <= T_) {
    at += t0 * step;
#pragma unroll
    for (int l = 0; l < L; ++l) r[l] = __ldcs(reinterpret_cast<const Raw*>(at + l * step));
  } else {
#pragma unroll
    for (int l = 0; l < L; ++l) r[l] = __ldcs(reinterpret_cast<const Raw*>(at + (t0 + l < T_ ? t0 + l : T_ - 1) * step));
  }
}

constexpr int FW = 8, FL = 16;      // forward tile: 128 steps
constexpr int BW = 8, BL = 8;       // backward tile: GL_CHUNK steps, so that it starts at a saved state
static_assert(BW * BL == GL_CHUNK && GL_CHUNK % FL == 0, "saved states lie on tile and warp edges");

// A warp's last steps once more, from memory: for a state that the steps past the sequence's end, whose gates are zero, have
// turned from infinite into NaN (0 inf).
template <typename T, int V, bool RESET>
__device__ __forceinline__ Vec<V> walk(const GlParams& p, Vec<V> h, int t0, int b, int i) {
#pragma unroll
  for (int v = 0; v < V; ++v) {
    if (i + v >= p.d) continue;
    const T* f = (const T*)p.f + b * p.sf.b + i + v;
    const T* c = (const T*)p.c + b * p.sc.b + i + v;
    Vec<1> x(h.get(v)), e;
#pragma unroll 1
    for (int t = t0; t < p.T; ++t) {
      if (RESET && p.reset[(long)t * p.B + b] != 0) x = Vec<1>(0.f);
      x = vfma(gate_of<1, true>(vmul(Vec<1>(to_f(f[t * p.sf.t])), Vec<1>(LOG2E)), e), vsub(x, Vec<1>(to_f(c[t * p.sc.t]))), x);
    }
    h.set(v, x.x);
  }
  return h;
}
template <int V> __device__ __forceinline__ bool any_nan(Vec<V> h) {
  bool nan = false;
#pragma unroll
  for (int v = 0; v < V; ++v) nan = nan || h.get(v) != h.get(v);
  return nan;
}

// What both kernels know of the tile they are at.
template <int V> struct Tile {
  int n, b, i;
  long col, base;
  bool on;
  __device__ __forceinline__ Tile(int ticket, int col_groups, const GlParams& p) {
    const int lane = threadIdx.x & 31;
    const long cols = (long)p.B * p.d;
    n = ticket / col_groups;
    base = (long)(ticket - n * col_groups) * (32 * V);
    col = base + lane * V;
    on = col < cols;
    const long at = on ? col : cols - V;      // lanes past the last channel read it and write nothing
    b = (int)(at / p.d);
    i = (int)(at - (long)b * p.d);
  }
};

template <typename T, int V, bool RESET>
__global__ void __launch_bounds__(32 * FW, 2) gl_forward_tile_kernel(GlParams p, GlChain ch, int tiles, int col_groups) {
  typedef Lane<T, V> Ln;
  typedef Vec<V> F;
  __shared__ Shared<V, FW> sh;
  const int w = threadIdx.x >> 5, warps = blockDim.x >> 5;
  const long cols = (long)p.B * p.d;
  const int total = tiles * col_groups;
  ptx::wait_for_previous();
  if (threadIdx.x == 0) {
    sh.gave_up = 0;
    sh.next = tiles > 1 ? (int)(atomicAdd(ch.ctrl, 1u) + 1u) : (int)blockIdx.x;
  }
  __syncthreads();
  for (int ticket = sh.next; ticket < total;) {
    uint32_t grabbed = 0;
    if (tiles > 1 && threadIdx.x == 0) grabbed = atomicAdd(ch.ctrl, 1u);
    const Tile<V> at(ticket, col_groups, p);
    const int t0 = at.n * (FW * FL) + w * FL, steps = p.T - t0;
    typename Ln::Raw rf[FL], rc[FL], rz[FL];
    load_rows<T, V, FL>(rf, p.f, p.sf, t0, p.T, at.b, at.i);
    load_rows<T, V, FL>(rc, p.c, p.sc, t0, p.T, at.b, at.i);
    load_rows<T, V, FL>(rz, p.z, p.sz, t0, p.T, at.b, at.i);
    const uint32_t cut = RESET ? reset_bits<FL>(p, t0, at.b) : 0;
    F nu[FL], e, initial(0.f);
    if (w == 0 && at.n < GROUP && p.h0 != nullptr && at.on) {
#pragma unroll
      for (int v = 0; v < V; ++v) initial.set(v, p.h0[at.col + v]);
    }
#pragma unroll
    for (int l = 0; l < FL; ++l) nu[l] = gate_of<V, true>(vmul(Ln::get(rf[l]), F(LOG2E)), e);
    if (steps < FL) {
#pragma unroll
      for (int l = 0; l < FL; ++l)
        if (l >= steps) nu[l] = F(0.f);       // beyond the end: the state stays
    }
    Scan<V> scan;
#pragma unroll
    for (int l = 0; l < FL; ++l) {
      if (RESET) scan.H = unless(cut >> l & 1, scan.H);
      scan.step(nu[l], Ln::get(rc[l]));
    }
    F h;
    if (!enter<V, FW, RESET>(sh, w, warps, RESET && cut ? F(-1.f) : scan.K(), scan.H, at.n, tiles, at.base, cols, initial, ch, ticket, grabbed, h)) return;
    ticket = tiles > 1 ? sh.next : total;
    if (at.on && p.saved != nullptr && t0 % GL_CHUNK == 0 && steps > 0) {
#pragma unroll
      for (int v = 0; v < V; ++v) p.saved[(long)(t0 / GL_CHUNK) * cols + at.col + v] = h.get(v);
    }
    char* y = (char*)p.y + ((long)t0 * p.sy.t + at.b * p.sy.b + at.i) * (long)sizeof(T);
    const long step = p.sy.t * (long)sizeof(T);
#pragma unroll
    for (int l = 0; l < FL; ++l) {
      if (RESET) h = unless(cut >> l & 1, h);
      h = vfma(nu[l], vsub(h, Ln::get(rc[l])), h);
      const F z = Ln::get(rz[l]);
      const F out = vmul(h, vmul(z, gate_of(vmul(z, F(-LOG2E)), e)));
      if (at.on && l < steps) __stcs(reinterpret_cast<typename Ln::Raw*>(y + l * step), Ln::put(out));
    }
    if (at.on && steps > 0 && steps <= FL) {
      if (steps < FL && any_nan(h)) {
#pragma unroll
        for (int v = 0; v < V; ++v) h.set(v, sh.enters[w][(threadIdx.x & 31) * V + v]);
        h = walk<T, V, RESET>(p, h, t0, at.b, at.i);
      }
#pragma unroll
      for (int v = 0; v < V; ++v) p.h_last[at.col + v] = h.get(v);
    }
  }
}

template <typename T, int V, bool RESET>
__global__ void __launch_bounds__(32 * BW, 2) gl_backward_tile_kernel(GlParams p, GlChain ch, int tiles, int col_groups) {
  typedef Lane<T, V> Ln;
  typedef Vec<V> F;
  __shared__ Shared<V, BW> sh;
  __shared__ Pair ahead[BW][32 * V];      // the warps' pairs of the forward scan
  const int w = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = blockDim.x >> 5;
  const long cols = (long)p.B * p.d;
  const int total = tiles * col_groups;
  ptx::wait_for_previous();
  if (threadIdx.x == 0) {
    sh.gave_up = 0;
    sh.next = tiles > 1 ? (int)(atomicAdd(ch.ctrl, 1u) + 1u) : (int)blockIdx.x;
  }
  __syncthreads();
  for (int ticket = sh.next; ticket < total;) {
    uint32_t grabbed = 0;
    if (tiles > 1 && threadIdx.x == 0) grabbed = atomicAdd(ch.ctrl, 1u);
    const Tile<V> at(ticket, col_groups, p);
    const int chunk = tiles - 1 - at.n, t0 = chunk * GL_CHUNK + w * BL, steps = p.T - t0;
    typename Ln::Raw rf[BL], rc[BL], rz[BL], rdy[BL];
    load_rows<T, V, BL>(rf, p.f, p.sf, t0, p.T, at.b, at.i);
    load_rows<T, V, BL>(rc, p.c, p.sc, t0, p.T, at.b, at.i);
    load_rows<T, V, BL>(rz, p.z, p.sz, t0, p.T, at.b, at.i);
    load_rows<T, V, BL>(rdy, p.dy, p.sy, t0, p.T, at.b, at.i);
    F h(0.f), last(0.f);
    if (at.on) {
#pragma unroll
      for (int v = 0; v < V; ++v) h.set(v, p.saved[(long)chunk * cols + at.col + v]);
      if (steps > 0 && steps <= BL && p.dh_last != nullptr) {
#pragma unroll
        for (int v = 0; v < V; ++v) last.set(v, p.dh_last[at.col + v]);
      }
    }
    const uint32_t cut = RESET ? reset_bits<BL>(p, t0, at.b) : 0;
    // the states before the warp's steps
    F nu[BL], a[BL];
#pragma unroll
    for (int l = 0; l < BL; ++l) {
      F e;
      nu[l] = gate_of<V, true>(held(vmul(Ln::get(rf[l]), F(LOG2E))), e);
      a[l] = vmul(vmul(e, nu[l]), nu[l]);
    }
    if (steps < BL) {
#pragma unroll
      for (int l = 0; l < BL; ++l)
        if (l >= steps) nu[l] = F(0.f);
    }
    Scan<V> scan;
#pragma unroll
    for (int l = 0; l < BL; ++l) {
      if (RESET) scan.H = unless(cut >> l & 1, scan.H);
      scan.step(nu[l], Ln::get(rc[l]));
    }
    const F K = RESET && cut ? F(-1.f) : scan.K();
#pragma unroll
    for (int v = 0; v < V; ++v) ahead[w][lane * V + v] = Pair{K.get(v), scan.H.get(v)};
    __syncthreads();
#pragma unroll
    for (int v = 0; v < V; ++v) {
      float s = h.get(v);
      for (int k = 0; k < w; ++k) s = pass<RESET>(s, ahead[k][lane * V + v]);
      h.set(v, s);
    }
    // forward through the warp's steps: dz, and what the scan back needs
    char* dz = (char*)p.dz + ((long)t0 * p.sdz.t + at.b * p.sdz.b + at.i) * (long)sizeof(T);
    const long step_z = p.sdz.t * (long)sizeof(T);
    F q[BL], prev[BL];
#pragma unroll
    for (int l = 0; l < BL; ++l) {
      if (RESET) h = unless(cut >> l & 1, h);
      prev[l] = vsub(h, Ln::get(rc[l]));
      h = vfma(nu[l], prev[l], h);
      const F z = Ln::get(rz[l]), dy = Ln::get(rdy[l]);
      F e;
      const F s = gate_of(vmul(z, F(-LOG2E)), e), zs = vmul(z, s);
      q[l] = vmul(dy, zs);
      const F out = vmul(vmul(dy, h), vfma(zs, vsub(F(1.f), s), s));
      if (at.on && l < steps) __stcs(reinterpret_cast<typename Ln::Raw*>(dz + l * step_z), Ln::put(out));
    }
    if (steps <= BL) {
#pragma unroll
      for (int l = 0; l < BL; ++l) q[l] = l >= steps ? F(0.f) : l == steps - 1 ? vadd(q[l], last) : q[l];
    }
    F E(0.f), D;
#pragma unroll
    for (int l = BL - 1; l >= 0; --l) {
      const F g = vadd(q[l], E);
      E = vfma(nu[l], g, g);
      if (RESET) E = unless(cut >> l & 1, E);
    }
    if (!enter<V, BW, RESET>(sh, warps - 1 - w, warps, K, E, at.n, tiles, at.base, cols, F(0.f), ch, ticket, grabbed, D)) return;
    ticket = tiles > 1 ? sh.next : total;
    char* df = (char*)p.df + ((long)t0 * p.sdf.t + at.b * p.sdf.b + at.i) * (long)sizeof(T);
    char* dc = (char*)p.dc + ((long)t0 * p.sdc.t + at.b * p.sdc.b + at.i) * (long)sizeof(T);
    const long step_f = p.sdf.t * (long)sizeof(T), step_c = p.sdc.t * (long)sizeof(T);
#pragma unroll
    for (int l = BL - 1; l >= 0; --l) {
      const F g = vadd(q[l], D), minus_gu = vmul(g, nu[l]);
      const F of = vmul(vmul(g, prev[l]), a[l]);
      D = vfma(nu[l], g, g);
      if (RESET) D = unless(cut >> l & 1, D);
      if (at.on && l < steps) {
        __stcs(reinterpret_cast<typename Ln::Raw*>(dc + l * step_c), Ln::put_minus(minus_gu));
        __stcs(reinterpret_cast<typename Ln::Raw*>(df + l * step_f), Ln::put(of));
      }
    }
    if (at.on && t0 == 0) {
#pragma unroll
      for (int v = 0; v < V; ++v) p.dh0[at.col + v] = D.get(v);
    }
  }
}

// ---------------------------------------------------------------------------
// The same tiles fed by asynchronous copies: the next tile's rows arrive in one shared-memory stage while
// this tile is scanned from the other, so the loads never pause for the arithmetic.  A producer takes
// tiles from the counter and loads them; the other warps scan and link.  A tile lies within one batch row.  (Tiles loaded
// into registers by the scanning warps: T512 B32 d1280 forward and backward 165 us, fed 123.)
//
// FEED_TMA, for tensors whose base and row strides are multiples of 16 bytes: a box a tensor, rows past T and
// channels past d zero-filled; a lane owns the same 4-byte word of every row (two bf16 channels or one
// fp32 channel), results overwrite the inputs that made them and leave as bulk stores.
// FEED_ROWS4 and FEED_ROWS2, for all others, by what their rows' starts are multiples of: a copy a row, of the
// 16-byte blocks it touches, read at the row's own offset in them; results go out by plain stores.
// ---------------------------------------------------------------------------
constexpr int ROW_BYTES = 128;
enum FeedKind { FEED_TMA, FEED_ROWS4, FEED_ROWS2 };
constexpr int pitch_of(int feed) { return feed == FEED_TMA ? ROW_BYTES : ROW_BYTES + 16; }
template <int IN, int ROWS, int FEED> struct Stages {
  static constexpr int TENSOR = ROWS * pitch_of(FEED), STAGE = IN * TENSOR, BYTES = 2 * STAGE + 128;   // + alignment
};
// Scanning warps of the forward tile (16 steps each; two stages of longer rows leave room for seven).
constexpr int forward_warps(int feed) { return feed == FEED_TMA ? FW : 7; }
// Producer warps for rows copied in blocks: two channels a lane are short of registers (T4096 B16 d1001 bf16 forward 163 us
// with one, 197 with two, 227 with four), one is not (fp32 288, 245, 215).
constexpr int row_producers(int V) { return V == 2 ? 1 : 4; }
constexpr int producer_threads(int feed, int V) { return feed == FEED_TMA ? 32 : 32 * row_producers(V); }
struct GlTma {
  int tiles, groups_per_row, total;   // tiles in time; channel groups of a batch row; all tiles
  long cols;                          // channels as the chain counts them: whole groups
};
// Where a tile lies: its ticket (-1: no more tiles), its place in the scan's order, its batch row and channel group.
// The producer takes tickets apart; the divisions were a tenth of the backward tile's instructions.
struct alignas(16) TileAt { int ticket, n, b, group; };
struct Feed {                          // shared: producer <-> scanning and linking warps
  uint64_t full[2], done[2];
  TileAt tile[2];
  int gave_up;
};

template <int IN, int OUT, int ROWS>
__device__ __forceinline__ void produce(Feed& fd, uint8_t* smem, const CUtensorMap* const (&in)[IN],
                                        const CUtensorMap* const (&out)[OUT], int channels, bool backward,
                                        const GlTma& g, const GlChain& ch) {
  constexpr int TENSOR = Stages<IN, ROWS, FEED_TMA>::TENSOR, STAGE = Stages<IN, ROWS, FEED_TMA>::STAGE;
  volatile int* gave_up = &fd.gave_up;
  TileAt tile[2] = {{-1, 0, 0, 0}, {-1, 0, 0, 0}};
  const int per_time = g.total / g.tiles;
  auto row_of = [&](const TileAt& t) { return (backward ? g.tiles - 1 - t.n : t.n) * ROWS; };
  auto store = [&](int s) {
#pragma unroll
    for (int k = 0; k < OUT; ++k)
      tch::tma_store_3d(out[k], smem + s * STAGE + k * TENSOR, tile[s].group * channels, tile[s].b, row_of(tile[s]));
    tch::bulk_commit();
  };
  for (int it = 0;; ++it) {
    const int s = it & 1;
    if (it >= 2) {                                  // the tile that was here: its results leave
      if (!ptx::mbar_wait(&fd.done[s], (uint32_t)((it >> 1) - 1) & 1u, ch.spin_limit * 8, gave_up)) break;
      store(s);
    }
    const uint32_t next = g.tiles > 1 ? atomicAdd(ch.ctrl, 1u) + 1u
                                      : (uint32_t)(it == 0 ? blockIdx.x : g.total);
    TileAt t{-1, 0, 0, 0};
    if (next < (uint32_t)g.total) {
      t.ticket = (int)next;
      t.n = t.ticket / per_time;
      const int column = t.ticket - t.n * per_time;
      t.b = column / g.groups_per_row;
      t.group = column - t.b * g.groups_per_row;
    }
    tile[s] = t;
    fd.tile[s] = t;
    if (t.ticket < 0) {
      ptx::mbar_arrive(&fd.full[s]);                // nothing more: the scanning warps end here
      // the last tile's results
      if (it >= 1 && tile[s ^ 1].ticket >= 0 &&
          ptx::mbar_wait(&fd.done[s ^ 1], (uint32_t)((it - 1) >> 1) & 1u, ch.spin_limit * 8, gave_up))
        store(s ^ 1);
      break;
    }
    tch::bulk_wait_read_all();                      // the stage has been read out
    ptx::mbar_arrive_expect_tx(&fd.full[s], STAGE);
#pragma unroll
    for (int k = 0; k < IN; ++k)
      tch::tma_load_3d(smem + s * STAGE + k * TENSOR, in[k], t.group * channels, t.b, row_of(t), &fd.full[s]);
  }
  if (*gave_up != 0)
    for (int i = 0; i < 2000; ++i) __nanosleep(100);   // loads in flight land before the shared memory goes
  tch::bulk_wait_read_all();
}

// The producer warps for rows of any alignment: 16-byte copies of the blocks a row touches (eight, or nine), four rows
// an instruction.  (A bulk copy a row was measured too: T777 B5 d1001 fp32 forward 53 us instead of 21.)
template <typename T, int V, int IN, int ROWS, int FEED>
__device__ __forceinline__ void produce_rows(Feed& fd, uint8_t* smem, const void* const (&in)[IN], const Strides (&st)[IN], int which,
                                             const GlParams& p, bool backward, const GlTma& g, const GlChain& ch) {
  constexpr int PITCH = pitch_of(FEED), TENSOR = Stages<IN, ROWS, FEED>::TENSOR, STAGE = Stages<IN, ROWS, FEED>::STAGE;
  volatile int* gave_up = &fd.gave_up;
  const int lane = threadIdx.x & 31, per_time = g.total / g.tiles;
  for (int it = 0;; ++it) {
    const int s = it & 1;
    if (which == 0 && lane == 0) {
      TileAt t{-1, 0, 0, 0};
      if (it >= 2 && !ptx::mbar_wait(&fd.done[s], (uint32_t)((it >> 1) - 1) & 1u, ch.spin_limit * 8, gave_up)) {
        t.ticket = -2;                              // given up: nobody waits for the stage any more
      } else {
        const uint32_t next = g.tiles > 1 ? atomicAdd(ch.ctrl, 1u) + 1u : (uint32_t)(it == 0 ? blockIdx.x : g.total);
        if (next < (uint32_t)g.total) {
          t.ticket = (int)next;
          t.n = t.ticket / per_time;
          const int column = t.ticket - t.n * per_time;
          t.b = column / g.groups_per_row;
          t.group = column - t.b * g.groups_per_row;
        }
      }
      fd.tile[s] = t;
    }
    asm volatile("bar.sync 4, %0;" ::"n"(32 * row_producers(V)) : "memory");
    const TileAt t = fd.tile[s];
    if (t.ticket >= 0) {
      const int row0 = (backward ? g.tiles - 1 - t.n : t.n) * ROWS, i0 = t.group * (32 * V);
      const int rows = p.T - row0 < ROWS ? p.T - row0 : ROWS;
      const uintptr_t width = (uintptr_t)((p.d - i0 < 32 * V ? p.d - i0 : 32 * V) * (int)sizeof(T));
#pragma unroll
      for (int k = 0; k < IN; ++k) {
        const long step = st[k].t * (long)sizeof(T);
        const uintptr_t first = (uintptr_t)in[k] + (uintptr_t)((long)row0 * step + (t.b * st[k].b + i0) * (long)sizeof(T));
        const uint32_t to = ptx::smem_u32(smem + s * STAGE + k * TENSOR);
        auto copy = [&](int r, int block) {         // one 16-byte block of row r, if the row reaches into it
          const uintptr_t start = first + (uintptr_t)((long)r * step), from = (start & ~(uintptr_t)15) + 16u * block;
          if (r < rows && from < start + width)
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to + r * PITCH + 16 * block), "l"(from) : "memory");
        };
#pragma unroll 4
        for (int r = 4 * which + (lane >> 3); r < ROWS; r += 4 * row_producers(V)) copy(r, lane & 7);
        for (int r = 32 * which + lane; r < ROWS; r += 32 * row_producers(V)) copy(r, 8);
      }
      asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(ptx::smem_u32(&fd.full[s])) : "memory");
      if (which == 0 && lane == 0) ptx::mbar_arrive(&fd.full[s]);       // what it wrote of the tile is visible
    } else {
      if (t.ticket == -1) {
        ptx::mbar_arrive(&fd.full[s]);
        if (which == 0 && lane == 0) ptx::mbar_arrive(&fd.full[s]);
      }
      break;
    }
  }
  asm volatile("cp.async.wait_all;" ::: "memory");
}
constexpr int full_arrivals(int feed, int V) { return feed == FEED_TMA ? 1 : 32 * row_producers(V) + 1; }

// V channels of a state [B, d] from channel i on.
template <int V> __device__ __forceinline__ Vec<V> read_state(const float* from, int b, int i, int d) {
  Vec<V> x(0.f);
  if (from == nullptr) return x;
  from += (long)b * d + i;
#pragma unroll
  for (int v = 0; v < V; ++v)
    if (i + v < d) x.set(v, from[v]);
  return x;
}
template <int V> __device__ __forceinline__ void write_state(float* to, int b, int i, int d, Vec<V> x) {
  to += (long)b * d + i;
#pragma unroll
  for (int v = 0; v < V; ++v)
    if (i + v < d) to[v] = x.get(v);
}
__device__ __forceinline__ uint32_t lds_word(uint32_t addr) {
  uint32_t w;
  asm volatile("ld.shared.b32 %0, [%1];" : "=r"(w) : "r"(addr));
  return w;
}
__device__ __forceinline__ void sts_word(uint32_t addr, uint32_t w) {
  asm volatile("st.shared.b32 [%0], %1;" ::"r"(addr), "r"(w) : "memory");
}
template <typename T, int V> __device__ __forceinline__ Vec<V> from_word(uint32_t w) {
  typename Lane<T, V>::Raw r;
  memcpy(&r, &w, 4);
  return Lane<T, V>::get(r);
}
template <typename T, int V> __device__ __forceinline__ uint32_t to_word(Vec<V> x, bool minus) {
  const typename Lane<T, V>::Raw r = minus ? Lane<T, V>::put_minus(x) : Lane<T, V>::put(x);
  uint32_t w;
  memcpy(&w, &r, 4);
  return w;
}
// A lane's words of a warp's rows of one tensor in a stage.
template <typename T, int V, int FEED> struct RowsIn {
  uint32_t at, low, step;            // low, step: where the rows start (their low bits count)
  __device__ __forceinline__ RowsIn(uint32_t rows, const void* base, Strides s, int t0, int b, int i0) : at(rows + (threadIdx.x & 31) * 4) {
    low = (uint32_t)(uintptr_t)base + (uint32_t)(((long)t0 * s.t + b * s.b + i0) * (long)sizeof(T));
    step = (uint32_t)(s.t * (long)sizeof(T));
  }
  __device__ __forceinline__ uint32_t addr(int l) const {
    return FEED == FEED_TMA ? at + l * ROW_BYTES : at + l * pitch_of(FEED) + ((low + l * step) & 15u);
  }
  __device__ __forceinline__ Vec<V> get(int l) const {
    if constexpr (FEED == FEED_ROWS2)
      return from_word<T, V>((uint32_t)tch::lds_u16(addr(l)) | (uint32_t)tch::lds_u16(addr(l) + 2) << 16);
    else
      return from_word<T, V>(lds_word(addr(l)));
  }
  // rows from `steps` on were not copied: zeros (a zero gate alone would not keep what is not a number out)
  template <int L> __device__ __forceinline__ void clear_after(int steps) const {
    if (FEED == FEED_TMA || steps >= L) return;
#pragma unroll 1
    for (int l = steps > 0 ? steps : 0; l < L; ++l) {
      if constexpr (FEED == FEED_ROWS2) {
        tch::sts_u16(addr(l), 0);
        tch::sts_u16(addr(l) + 2, 0);
      } else {
        sts_word(addr(l), 0);
      }
    }
  }
};
// Where a lane's results go: into the stage, or out.
template <typename T, int V, int FEED> struct RowsOut {
  uint32_t stage;
  char* at;
  long step;
  int channels, steps;
  __device__ __forceinline__ RowsOut(uint32_t rows, void* base, Strides s, int t0, int b, int i, int d, int steps_)
      : stage(rows + (threadIdx.x & 31) * 4), steps(steps_) {
    at = (char*)base + ((long)t0 * s.t + b * s.b + i) * (long)sizeof(T);
    step = s.t * (long)sizeof(T);
    channels = d - i;
  }
  __device__ __forceinline__ void put(int l, Vec<V> x, bool minus = false) const {
    const uint32_t w = to_word<T, V>(x, minus);
    if constexpr (FEED == FEED_TMA) {
      sts_word(stage + l * ROW_BYTES, w);
    } else if (l < steps && channels > 0) {
      if constexpr (FEED == FEED_ROWS4) {
        __stcs(reinterpret_cast<uint32_t*>(at + l * step), w);
      } else {
        __stcs(reinterpret_cast<unsigned short*>(at + l * step), (unsigned short)w);
        if (channels > 1) __stcs(reinterpret_cast<unsigned short*>(at + l * step) + 1, (unsigned short)(w >> 16));
      }
    }
  }
};

// What the warps of such a block share.  The scanning warps leave their pairs (barrier 1, where they only
// arrive), warps of their own link the tile into the chain, one thread per channel, and hand back the
// state that enters each scanning warp (barrier 2).  Meanwhile the scanning warps work on what needs no
// state.  (Where the scanning warps folded the pairs themselves, that was a third of the backward tile's
// instructions.)
template <int V, int W> struct Links {
  Vec<V> P[W][32], P_1[W][32], H[W][32];   // the warps' stretches, in the scan's direction
  float enters[W][32 * V];         // state that enters each warp
  int gave_up[2];                  // somebody did, at this tile (even and odd ones apart: a slow warp may still look at the last)
};
// Each warp waits for a stage by itself, so one may give up (or leave early for another that did) where the rest still
// see it land.  The barriers have no limit: whoever leaves passes those of the tile first, whoever sees the end as
// well, and all the others leave behind the last of them.
template <int V, int W> __device__ __forceinline__ void leave_scan(Links<V, W>& sh, int s, bool given_up, bool backward) {
  if (given_up) sh.gave_up[s] = 1;
  if (backward) asm volatile("bar.sync 3, %0;" ::"n"(32 * W) : "memory");
  asm volatile("bar.arrive 1, %0;" ::"n"(32 * (W + V)) : "memory");
  asm volatile("bar.sync 2, %0;" ::"n"(32 * (W + V)) : "memory");
}
template <int V, int W> __device__ __forceinline__ void leave_link(Links<V, W>& sh, int s, bool given_up) {
  if (given_up) sh.gave_up[s] = 1;
  asm volatile("bar.sync 1, %0;" ::"n"(32 * (W + V)) : "memory");
  asm volatile("bar.sync 2, %0;" ::"n"(32 * (W + V)) : "memory");
}
template <int V, int W, bool RESET> __device__ __forceinline__ void leave_stretch(Links<V, W>& sh, int w, const Scan<V>& scan, Vec<V> H, uint32_t cut) {
  const int lane = threadIdx.x & 31;
  sh.P[w][lane] = scan.P;
  sh.P_1[w][lane] = RESET && cut ? Vec<V>(-2.f) : scan.P_1;
  sh.H[w][lane] = H;
  asm volatile("bar.arrive 1, %0;" ::"n"(32 * (W + V)) : "memory");
}
template <int V, int W> __device__ __forceinline__ bool take_state(Links<V, W>& sh, int s, int w, Vec<V>& S) {
  const int lane = threadIdx.x & 31;
  asm volatile("bar.sync 2, %0;" ::"n"(32 * (W + V)) : "memory");
#pragma unroll
  for (int v = 0; v < V; ++v) S.set(v, sh.enters[w][lane * V + v]);
  return sh.gave_up[s] == 0;
}
// One linking warp, one tile; x is the thread's channel in the tile.  False: a wait gave up.
// (`initial` is the caller's and may be any NaN: NOT_YET would send its lane to a state before the first.)
template <int V, int W, bool RESET>
__device__ __forceinline__ bool link(Links<V, W>& sh, int stage, int x, int n, int tiles, long base, long cols, float initial,
                                     const GlChain& ch, int ticket) {
  const int first = n / GROUP * GROUP, in_group = n - first;
  const bool ends_group = in_group == GROUP - 1, more = n + 1 < tiles && ticket != ch.stall;
  const float2* pairs = ch.pairs + (long)first * cols + base + x;
  const float* state = ch.states + (long)(first / GROUP - 1) * cols + base + x;
  uint32_t g[GROUP - 1][2], at_start = first > 0 ? NOT_YET : word_of(initial);
#pragma unroll
  for (int k = 0; k < GROUP - 1; ++k) g[k][0] = g[k][1] = k < in_group ? NOT_YET : 0u;
  auto fetch = [&]() {                             // what is missing: every load in flight before any is looked at
    look_if(at_start == NOT_YET, state, at_start);
#pragma unroll
    for (int k = 0; k < GROUP - 1; ++k) look_if(g[k][0] == NOT_YET || g[k][1] == NOT_YET, pairs + (long)k * cols, g[k]);
  };
  auto complete = [&]() {
    bool there = at_start != NOT_YET;
#pragma unroll
    for (int k = 0; k < GROUP - 1; ++k) there = there && g[k][0] != NOT_YET && g[k][1] != NOT_YET;
    return there;
  };
  fetch();                                         // while the scanning warps scan
  asm volatile("bar.sync 1, %0;" ::"n"(32 * (W + V)) : "memory");
  Stretch own[W];
#pragma unroll
  for (int k = 0; k < W; ++k)
    own[k] = Stretch{reinterpret_cast<const float*>(sh.P[k])[x], reinterpret_cast<const float*>(sh.P_1[k])[x],
                     reinterpret_cast<const float*>(sh.H[k])[x]};
  if (more && !ends_group) {
    Stretch all = own[0];
#pragma unroll
    for (int k = 1; k < W; ++k) all = join<RESET>(all, own[k]);
    publish(ch.pairs + (long)n * cols + base + x, pair_of<RESET>(all));
  }
  Patience patience;
  bool ok = true;
  while (ok && !__all_sync(0xFFFFFFFFu, complete())) {
    fetch();
    ok = patience.left(ch, n);
  }
  float s = __uint_as_float(at_start);
#pragma unroll
  for (int k = 0; k < GROUP - 1; ++k)
    if (k < in_group) s = pass<RESET>(s, Pair{__uint_as_float(g[k][0]), __uint_as_float(g[k][1])});
#pragma unroll
  for (int k = 0; k < W; ++k) {
    sh.enters[k][x] = s;
    s = pass<RESET>(s, own[k]);
  }
  if (more && ends_group) publish(ch.states + (long)(first / GROUP) * cols + base + x, s);
  if (!ok) sh.gave_up[stage] = 1;
  asm volatile("bar.sync 2, %0;" ::"n"(32 * (W + V)) : "memory");
  return sh.gave_up[stage] == 0;
}
// The linking warps' loop over the block's tiles.
template <int V, int W, bool RESET>
__device__ __forceinline__ void link_tiles(Links<V, W>& sh, Feed& fd, const GlParams& p, const GlChain& ch, const GlTma& g,
                                           const float* initial) {
  const int x = threadIdx.x - 32 * W;
  for (int it = 0;; ++it) {
    const int s = it & 1;
    const bool here = ptx::mbar_wait(&fd.full[s], (uint32_t)(it >> 1) & 1u, ch.spin_limit * 8, &fd.gave_up);
    if (!__all_sync(0xFFFFFFFFu, here && 32 * it + (int)(threadIdx.x >> 5) != ch.leave)) {
      fd.gave_up = 1;
      report_timeout(ch.status, KID_GATED_LINEAR, 0xFFFF);
      leave_link(sh, s, true);
      return;
    }
    const TileAt t = fd.tile[s];
    if (t.ticket < 0) {
      leave_link(sh, s, false);
      return;
    }
    const int i = t.group * (32 * V) + x;
    const long base = ((long)t.b * g.groups_per_row + t.group) * (32 * V);
    const float start = t.n < GROUP && initial != nullptr && i < p.d ? initial[(long)t.b * p.d + i] : 0.f;
    const bool ok = link<V, W, RESET>(sh, s, x, t.n, g.tiles, base, g.cols, start, ch, t.ticket);
    if (threadIdx.x % 32 == 0) ptx::mbar_arrive(&fd.done[s]);
    if (!ok) return;
  }
}

template <typename T, int V, bool RESET, int FEED>
__global__ void __launch_bounds__(32 * (forward_warps(FEED) + V) + producer_threads(FEED, V), 2)
gl_forward_fed_kernel(const __grid_constant__ CUtensorMap tf, const __grid_constant__ CUtensorMap tc,
                      const __grid_constant__ CUtensorMap tz, const __grid_constant__ CUtensorMap ty, GlParams p,
                      GlChain ch, GlTma g) {
  typedef Vec<V> F;
  static_assert(32 * V * sizeof(T) == ROW_BYTES, "a lane owns 4 bytes of a row");
  constexpr int W = forward_warps(FEED), ROWS = W * FL, TENSOR = Stages<3, ROWS, FEED>::TENSOR, STAGE = Stages<3, ROWS, FEED>::STAGE;
  extern __shared__ uint8_t raw[];
  __shared__ Links<V, W> sh;
  __shared__ Feed fd;
  uint8_t* smem = (uint8_t*)(((uintptr_t)raw + 127) & ~(uintptr_t)127);
  const int w = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    sh.gave_up[0] = sh.gave_up[1] = 0;
    fd.gave_up = 0;
    for (int s = 0; s < 2; ++s) {
      ptx::mbar_init(&fd.full[s], full_arrivals(FEED, V));
      ptx::mbar_init(&fd.done[s], W + V);
    }
    ptx::mbar_fence_init();
  }
  __syncthreads();
  ptx::wait_for_previous();
  if (w >= W + V) {
    if constexpr (FEED != FEED_TMA) {
      const void* const in[3] = {p.f, p.c, p.z};
      const Strides st[3] = {p.sf, p.sc, p.sz};
      produce_rows<T, V, 3, ROWS, FEED>(fd, smem, in, st, w - (W + V), p, false, g, ch);
    } else if (lane == 0) {
      const CUtensorMap* const in[3] = {&tf, &tc, &tz};
      const CUtensorMap* const out[1] = {&ty};
      produce<3, 1, ROWS>(fd, smem, in, out, 32 * V, false, g, ch);
    }
    return;
  }
  if (w >= W) {
    link_tiles<V, W, RESET>(sh, fd, p, ch, g, p.h0);
    return;
  }
  for (int it = 0;; ++it) {
    const int s = it & 1;
    const bool here = ptx::mbar_wait(&fd.full[s], (uint32_t)(it >> 1) & 1u, ch.spin_limit * 8, &fd.gave_up);
    if (!__all_sync(0xFFFFFFFFu, here && 32 * it + w != ch.leave)) {
      fd.gave_up = 1;
      report_timeout(ch.status, KID_GATED_LINEAR, 0xFFFF);
      leave_scan(sh, s, true, false);
      return;
    }
    const TileAt at = fd.tile[s];
    if (at.ticket < 0) {
      leave_scan(sh, s, false, false);
      return;
    }
    const int i = at.group * (32 * V) + lane * V;
    const int t0 = at.n * ROWS + w * FL, steps = p.T - t0;
    const uint32_t rows = ptx::smem_u32(smem + s * STAGE) + (uint32_t)(w * FL * pitch_of(FEED));
    const RowsIn<T, V, FEED> f(rows, p.f, p.sf, t0, at.b, i - lane * V), c(rows + TENSOR, p.c, p.sc, t0, at.b, i - lane * V),
        z(rows + 2 * TENSOR, p.z, p.sz, t0, at.b, i - lane * V);
    f.template clear_after<FL>(steps);
    c.template clear_after<FL>(steps);
    z.template clear_after<FL>(steps);
    const uint32_t cut = RESET ? reset_bits<FL>(p, t0, at.b) : 0;
    F nu[FL], zs[FL], e, h;
#pragma unroll
    for (int l = 0; l < FL; ++l) nu[l] = gate_of<V, true>(vmul(f.get(l), F(LOG2E)), e);
    if (steps < FL) {
#pragma unroll
      for (int l = 0; l < FL; ++l)
        if (l >= steps) nu[l] = F(0.f);
    }
    Scan<V> scan;
#pragma unroll
    for (int l = 0; l < FL; ++l) {
      if (RESET) scan.H = unless(cut >> l & 1, scan.H);
      scan.step(nu[l], c.get(l));
    }
    leave_stretch<V, W, RESET>(sh, w, scan, scan.H, cut);
#pragma unroll
    for (int l = 0; l < FL; ++l) {
      const F x = z.get(l);
      zs[l] = vmul(x, gate_of(vmul(x, F(-LOG2E)), e));
    }
    if (!take_state<V, W>(sh, s, w, h)) {
      fd.gave_up = 1;
      return;
    }
    const RowsOut<T, V, FEED> y(rows, p.y, p.sy, t0, at.b, i, p.d, steps);
    if (p.saved != nullptr && t0 % GL_CHUNK == 0 && steps > 0)
      write_state<V>(p.saved + (long)(t0 / GL_CHUNK) * p.B * p.d, at.b, i, p.d, h);
#pragma unroll
    for (int l = 0; l < FL; ++l) {
      if (RESET) h = unless(cut >> l & 1, h);
      h = vfma(nu[l], vsub(h, c.get(l)), h);
      y.put(l, vmul(h, zs[l]));
    }
    if (steps > 0 && steps <= FL) {
      if (steps < FL && any_nan(h)) {
#pragma unroll
        for (int v = 0; v < V; ++v) h.set(v, sh.enters[w][lane * V + v]);
        h = walk<T, V, RESET>(p, h, t0, at.b, i);
      }
      write_state<V>(p.h_last, at.b, i, p.d, h);
    }
    ptx::fence_proxy_async_smem();
    __syncwarp();
    if (lane == 0) ptx::mbar_arrive(&fd.done[s]);
  }
}

template <typename T, int V, bool RESET, int FEED>
__global__ void __launch_bounds__(32 * (BW + V) + producer_threads(FEED, V), 2)
gl_backward_fed_kernel(const __grid_constant__ CUtensorMap tf, const __grid_constant__ CUtensorMap tc,
                       const __grid_constant__ CUtensorMap tz, const __grid_constant__ CUtensorMap tdy,
                       const __grid_constant__ CUtensorMap tdf, const __grid_constant__ CUtensorMap tdc,
                       const __grid_constant__ CUtensorMap tdz, GlParams p, GlChain ch, GlTma g) {
  typedef Vec<V> F;
  constexpr int ROWS = BW * BL, TENSOR = Stages<4, ROWS, FEED>::TENSOR, STAGE = Stages<4, ROWS, FEED>::STAGE;
  extern __shared__ uint8_t raw[];
  __shared__ Links<V, BW> sh;
  __shared__ Vec<V> ahead_K[BW][32], ahead_H[BW][32], ahead_rest[BW][32];
  __shared__ Feed fd;
  uint8_t* smem = (uint8_t*)(((uintptr_t)raw + 127) & ~(uintptr_t)127);
  const int w = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    sh.gave_up[0] = sh.gave_up[1] = 0;
    fd.gave_up = 0;
    for (int s = 0; s < 2; ++s) {
      ptx::mbar_init(&fd.full[s], full_arrivals(FEED, V));
      ptx::mbar_init(&fd.done[s], BW + V);
    }
    ptx::mbar_fence_init();
  }
  __syncthreads();
  ptx::wait_for_previous();
  if (w >= BW + V) {
    if constexpr (FEED != FEED_TMA) {
      const void* const in[4] = {p.f, p.c, p.z, p.dy};
      const Strides st[4] = {p.sf, p.sc, p.sz, p.sy};
      produce_rows<T, V, 4, ROWS, FEED>(fd, smem, in, st, w - (BW + V), p, true, g, ch);
    } else if (lane == 0) {
      const CUtensorMap* const in[4] = {&tf, &tc, &tz, &tdy};
      const CUtensorMap* const out[3] = {&tdf, &tdc, &tdz};
      produce<4, 3, ROWS>(fd, smem, in, out, 32 * V, true, g, ch);
    }
    return;
  }
  if (w >= BW) {
    link_tiles<V, BW, RESET>(sh, fd, p, ch, g, nullptr);
    return;
  }
  for (int it = 0;; ++it) {
    const int s = it & 1;
    const bool here = ptx::mbar_wait(&fd.full[s], (uint32_t)(it >> 1) & 1u, ch.spin_limit * 8, &fd.gave_up);
    if (!__all_sync(0xFFFFFFFFu, here && 32 * it + w != ch.leave)) {
      fd.gave_up = 1;
      report_timeout(ch.status, KID_GATED_LINEAR, 0xFFFF);
      leave_scan(sh, s, true, true);
      return;
    }
    const TileAt at = fd.tile[s];
    if (at.ticket < 0) {
      leave_scan(sh, s, false, true);
      return;
    }
    const int i = at.group * (32 * V) + lane * V;
    const int chunk = g.tiles - 1 - at.n, t0 = chunk * ROWS + w * BL, steps = p.T - t0;
    const uint32_t rows = ptx::smem_u32(smem + s * STAGE) + (uint32_t)(w * BL * pitch_of(FEED));
    const RowsIn<T, V, FEED> f(rows, p.f, p.sf, t0, at.b, i - lane * V), c(rows + TENSOR, p.c, p.sc, t0, at.b, i - lane * V),
        z(rows + 2 * TENSOR, p.z, p.sz, t0, at.b, i - lane * V), dy(rows + 3 * TENSOR, p.dy, p.sy, t0, at.b, i - lane * V);
    f.template clear_after<BL>(steps);
    c.template clear_after<BL>(steps);
    z.template clear_after<BL>(steps);
    dy.template clear_after<BL>(steps);
    const uint32_t cut = RESET ? reset_bits<BL>(p, t0, at.b) : 0;
    F h = read_state<V>(p.saved + (long)chunk * p.B * p.d, at.b, i, p.d);
    F nu[BL], a[BL];
#pragma unroll
    for (int l = 0; l < BL; ++l) {
      F e;
      nu[l] = gate_of<V, true>(held(vmul(f.get(l), F(LOG2E))), e);
      a[l] = vmul(vmul(e, nu[l]), nu[l]);
    }
    if (steps < BL) {
#pragma unroll
      for (int l = 0; l < BL; ++l)
        if (l >= steps) nu[l] = F(0.f);
    }
    Scan<V> scan;
#pragma unroll
    for (int l = 0; l < BL; ++l) {
      if (RESET) scan.H = unless(cut >> l & 1, scan.H);
      scan.step(nu[l], c.get(l));
    }
    F K, rest;                            // pass() of both channels at once: h <- rest h + (K h + H)
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const bool near = scan.P_1.get(v) >= -0.5f;
      K.set(v, near ? scan.P_1.get(v) : scan.P.get(v));
      rest.set(v, RESET && cut ? -1.f : near ? 1.f : 0.f);
    }
    ahead_K[w][lane] = K;
    ahead_H[w][lane] = scan.H;
    ahead_rest[w][lane] = rest;
    asm volatile("bar.sync 3, %0;" ::"n"(32 * BW) : "memory");
#pragma unroll 1
    for (int k = 0; k < w; ++k) {
      const F H = ahead_H[k][lane], r = ahead_rest[k][lane];
      const F to = vfma(r, h, vfma(ahead_K[k][lane], h, H));
      h = RESET && r.get(0) < 0.f ? H : to;         // (a reset cuts all of a batch row's channels)
    }
    const RowsOut<T, V, FEED> dz(rows + 2 * TENSOR, p.dz, p.sdz, t0, at.b, i, p.d, steps);
    F q[BL];                              // a becomes (p - c) u (1 - u): df = g a
#pragma unroll
    for (int l = 0; l < BL; ++l) {
      if (RESET) h = unless(cut >> l & 1, h);
      const F prev = vsub(h, c.get(l));
      a[l] = vmul(a[l], prev);
      h = vfma(nu[l], prev, h);
      const F x = z.get(l), gy = dy.get(l);
      F e;
      const F sg = gate_of(vmul(x, F(-LOG2E)), e), zs = vmul(x, sg);
      q[l] = vmul(gy, zs);
      dz.put(l, vmul(vmul(gy, h), vfma(zs, vsub(F(1.f), sg), sg)));
    }
    if (steps <= BL) {                    // dh_last goes in with the last step (passed on to it, an infinite one would meet 0 inf)
      const F last = steps > 0 ? read_state<V>(p.dh_last, at.b, i, p.d) : F(0.f);
#pragma unroll
      for (int l = 0; l < BL; ++l) q[l] = l >= steps ? F(0.f) : l == steps - 1 ? vadd(q[l], last) : q[l];
    }
    F E(0.f), D;
#pragma unroll
    for (int l = BL - 1; l >= 0; --l) {
      const F gt = vadd(q[l], E);
      E = vfma(nu[l], gt, gt);
      if (RESET) E = unless(cut >> l & 1, E);
    }
    leave_stretch<V, BW, RESET>(sh, BW - 1 - w, scan, E, cut);
    if (!take_state<V, BW>(sh, s, BW - 1 - w, D)) {
      fd.gave_up = 1;
      return;
    }
    const RowsOut<T, V, FEED> df(rows, p.df, p.sdf, t0, at.b, i, p.d, steps), dc(rows + TENSOR, p.dc, p.sdc, t0, at.b, i, p.d, steps);
#pragma unroll
    for (int l = BL - 1; l >= 0; --l) {
      const F gt = vadd(q[l], D);
      df.put(l, vmul(gt, a[l]));
      dc.put(l, vmul(gt, nu[l]), true);
      D = vfma(nu[l], gt, gt);
      if (RESET) D = unless(cut >> l & 1, D);
    }
    if (t0 == 0) write_state<V>(p.dh0, at.b, i, p.d, D);
    ptx::fence_proxy_async_smem();
    __syncwarp();
    if (lane == 0) ptx::mbar_arrive(&fd.done[s]);
  }
}

GlParams params_of(const GatedLinearArgs& a) {
  GlParams p;
  p.T = a.T; p.B = a.B; p.d = a.d;
  p.f = a.f; p.c = a.c; p.z = a.z; p.dy = a.dy;
  auto s = [](const long* v) { return Strides{v[0], v[1]}; };
  p.sf = s(a.f_strides); p.sc = s(a.c_strides); p.sz = s(a.z_strides); p.sy = s(a.y_strides);
  p.sdf = s(a.df_strides); p.sdc = s(a.dc_strides); p.sdz = s(a.dz_strides);
  p.h0 = a.h0; p.reset = a.reset; p.saved = a.saved; p.y = a.y; p.h_last = a.h_last;
  p.dh_last = a.dh_last; p.df = a.df; p.dc = a.dc; p.dz = a.dz; p.dh0 = a.dh0;
  return p;
}

int tiles_of(int T, int steps) { return (int)(((long)T + steps - 1) / steps); }

size_t chain_bytes(int tiles, long cols) {
  if (tiles <= 1) return 0;
  return (256 + (size_t)tiles * cols * sizeof(float2) + (size_t)((tiles + GROUP - 1) / GROUP) * cols * sizeof(float) + 15) / 16 * 16;
}

// Two channels a lane where every row of every tensor allows 4-byte accesses.
bool pairs_of_channels(const GatedLinearArgs& a, bool bwd) {
  if (a.d % 2 != 0) return false;
  bool ok = true;
  auto see = [&](const void* base, const long* s) {
    ok = ok && ((uintptr_t)base & 3) == 0 && (a.T <= 1 || s[0] % 2 == 0) && (a.B <= 1 || s[1] % 2 == 0);
  };
  see(a.f, a.f_strides); see(a.c, a.c_strides); see(a.z, a.z_strides);
  see(bwd ? a.dy : a.y, a.y_strides);
  if (bwd) { see(a.df, a.df_strides); see(a.dc, a.dc_strides); see(a.dz, a.dz_strides); }
  return ok;
}

// Channels as a chain of whole TMA groups counts them: 128 bytes of a row each, within a batch row.
long whole_groups(int dtype, int d) {
  const int width = dtype == ELMAN_F32 ? 32 : 64;
  return ((long)d + width - 1) / width * width;
}
// A batch row's last group should not be mostly empty: narrower rows go to the kernels that count channels through, which
// reach about two thirds of the speed.
bool whole_width(int dtype, int d) { return whole_groups(dtype, d) <= (long)d + d / 2; }
FeedKind feed_of(int dtype, const GatedLinearArgs& a, bool bwd) {
  const long per16 = dtype == ELMAN_F32 ? 4 : 8, most = (1L << 39) / 4;
  bool ok = a.T <= (1 << 30) && a.B <= (1 << 30);
  auto see = [&](const void* base, const long* s) {
    ok = ok && ((uintptr_t)base & 15) == 0 && s[0] % per16 == 0 && s[0] < most &&
         (a.B <= 1 || (s[1] % per16 == 0 && s[1] > 0 && s[1] < most)) && s[0] > 0;
  };
  see(a.f, a.f_strides); see(a.c, a.c_strides); see(a.z, a.z_strides);
  see(bwd ? a.dy : a.y, a.y_strides);
  if (bwd) { see(a.df, a.df_strides); see(a.dc, a.dc_strides); see(a.dz, a.dz_strides); }
  return ok ? FEED_TMA : dtype == ELMAN_F32 || pairs_of_channels(a, bwd) ? FEED_ROWS4 : FEED_ROWS2;
}

// The workspace's start; the scan's launch overlaps it (T512 B32 d1280: a call takes 2 us less than behind a memset).
__global__ void __launch_bounds__(256) gl_fill_kernel(uint4* ws, long n) {
  ptx::let_next_start();
  const uint4 x = make_uint4(NOT_YET, NOT_YET, NOT_YET, NOT_YET);
  for (long i = (long)blockIdx.x * 256 + threadIdx.x; i < n; i += (long)gridDim.x * 256) ws[i] = x;
}

// The scan's launch, behind the workspace's where there is a chain.
template <typename... P, typename... A>
int launch_scan(void (*kernel)(P...), int tiles, long cols, void* workspace, unsigned grid, int threads, int smem, cudaStream_t st, A... args) {
  cudaLaunchAttribute attr = after_its_start();
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3((unsigned)threads);
  cfg.dynamicSmemBytes = (size_t)smem;
  cfg.stream = st;
  cfg.attrs = &attr;
  cfg.numAttrs = 0;
  if (tiles > 1) {
    const long pieces = (long)(chain_bytes(tiles, cols) / 16), blocks = (pieces + 255) / 256;
    gl_fill_kernel<<<(unsigned)(blocks < 148 * 8 ? blocks : 148 * 8), 256, 0, st>>>((uint4*)workspace, pieces);
    count_launch(false);
    cfg.numAttrs = 1;
  }
  ELMAN_CUDA_CHECK(cudaLaunchKernelEx(&cfg, kernel, args...));
  count_launch(false);
  ELMAN_CUDA_CHECK(cudaGetLastError());
  return ELMAN_OK;
}

void prepare_chain(GlChain& ch, const GatedLinearArgs& a, int tiles, long cols) {
  char* ws = (char*)a.workspace;
  ch.status = device_status_ptr();
  ch.spin_limit = options().spin_limit;
  ch.stall = (int)options().test_stall_step;
  ch.leave = (int)options().test_leave_warp;
  if (tiles <= 1) return;
  ch.ctrl = (uint32_t*)ws;
  ch.pairs = (float2*)(ws + 256);
  ch.states = (float*)(ws + 256 + (size_t)tiles * cols * sizeof(float2));
}

template <typename T, int V, bool RESET, int FEED>
int launch_fed(int dtype, const GatedLinearArgs& a, bool bwd, cudaStream_t st) {
  static std::mutex mutex;
  static bool sized[2][64];      // the kernel's shared-memory limit is set, per direction and device
  const int rows = bwd ? BW * BL : forward_warps(FEED) * FL;
  GlTma g{};
  g.tiles = tiles_of(a.T, rows);
  g.groups_per_row = (int)(whole_groups(dtype, a.d) / (32 * V));
  const long total = (long)g.groups_per_row * a.B * g.tiles;
  ELMAN_ARG_CHECK(total + 148 * 8 < (1L << 31), "too many channels for one call");
  g.total = (int)total;
  g.cols = (long)g.groups_per_row * a.B * 32 * V;
  const int smem = bwd ? Stages<4, BW * BL, FEED>::BYTES : Stages<3, forward_warps(FEED) * FL, FEED>::BYTES;
  const void* kernel = bwd ? (const void*)&gl_backward_fed_kernel<T, V, RESET, FEED> : (const void*)&gl_forward_fed_kernel<T, V, RESET, FEED>;
  int dev = 0;
  ELMAN_CUDA_CHECK(cudaGetDevice(&dev));
  {
    std::lock_guard<std::mutex> lock(mutex);
    if (dev >= 64 || !sized[bwd][dev]) {
      ELMAN_CUDA_CHECK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
      if (dev < 64) sized[bwd][dev] = true;
    }
  }
  CUtensorMap m[7];
  memset(m, 0, sizeof(m));
  if (FEED == FEED_TMA) {
    auto map = [&](int k, const void* base, const long* s) {
      const uint64_t one = a.B > 1 ? s[1] : s[0];     // (a single batch row: any valid stride)
      return make_tmap_3d(&m[k], dtype, base, a.d, a.B, a.T, one, s[0], 32 * V, 1, rows);
    };
    ELMAN_RETURN_IF(map(0, a.f, a.f_strides));
    ELMAN_RETURN_IF(map(1, a.c, a.c_strides));
    ELMAN_RETURN_IF(map(2, a.z, a.z_strides));
    ELMAN_RETURN_IF(map(3, bwd ? a.dy : a.y, a.y_strides));
    if (bwd) {
      ELMAN_RETURN_IF(map(4, a.df, a.df_strides));
      ELMAN_RETURN_IF(map(5, a.dc, a.dc_strides));
      ELMAN_RETURN_IF(map(6, a.dz, a.dz_strides));
    }
  }
  GlChain ch{};
  prepare_chain(ch, a, g.tiles, g.cols);
  const GlParams p = params_of(a);
  const unsigned grid = (unsigned)(g.tiles > 1 && total > 148 * 2 ? 148 * 2 : total);
  if (bwd)
    return launch_scan(&gl_backward_fed_kernel<T, V, RESET, FEED>, g.tiles, g.cols, a.workspace, grid,
                       32 * (BW + V) + producer_threads(FEED, V), smem, st, m[0], m[1], m[2], m[3], m[4], m[5], m[6], p, ch, g);
  return launch_scan(&gl_forward_fed_kernel<T, V, RESET, FEED>, g.tiles, g.cols, a.workspace, grid,
                     32 * (forward_warps(FEED) + V) + producer_threads(FEED, V), smem, st, m[0], m[1], m[2], m[3], p, ch, g);
}

template <typename T, int V, bool RESET>
int launch_tiles(const GatedLinearArgs& a, bool bwd, cudaStream_t st) {
  auto* kernel = bwd ? &gl_backward_tile_kernel<T, V, RESET> : &gl_forward_tile_kernel<T, V, RESET>;
  const long cols = (long)a.B * a.d;
  const int per_warp = bwd ? BL : FL, tile = bwd ? BW * BL : FW * FL;
  const int tiles = tiles_of(a.T, tile);
  // (a thread for each of the tile's channels at least)
  const int needed = tiles_of(a.T, per_warp), warps = tiles > 1 ? tile / per_warp : needed < V ? V : needed;
  const long col_groups = (cols + 32 * V - 1) / (32 * V);
  const long total = col_groups * tiles;
  ELMAN_ARG_CHECK(total + 148 * 8 < (1L << 31), "too many channels for one call");
  GlChain ch{};
  prepare_chain(ch, a, tiles, cols);
  long grid = total;
  if (tiles > 1) {
    const long resident = 148 * 2;       // the counter hands out the tiles
    if (grid > resident) grid = resident;
  }
  GlParams p = params_of(a);
  return launch_scan(kernel, tiles, cols, a.workspace, (unsigned)grid, 32 * warps, 0, st, p, ch, tiles, (int)col_groups);
}

template <bool RESET>
int launch_tiles(int dtype, const GatedLinearArgs& a, bool bwd, cudaStream_t st) {
  if (whole_width(dtype, a.d)) {
    const FeedKind feed = feed_of(dtype, a, bwd);
    if (dtype == ELMAN_F32)
      return feed == FEED_TMA ? launch_fed<float, 1, RESET, FEED_TMA>(dtype, a, bwd, st)
                              : launch_fed<float, 1, RESET, FEED_ROWS4>(dtype, a, bwd, st);
    return feed == FEED_TMA     ? launch_fed<bf16, 2, RESET, FEED_TMA>(dtype, a, bwd, st)
           : feed == FEED_ROWS4 ? launch_fed<bf16, 2, RESET, FEED_ROWS4>(dtype, a, bwd, st)
                                : launch_fed<bf16, 2, RESET, FEED_ROWS2>(dtype, a, bwd, st);
  }
  if (dtype == ELMAN_F32) return launch_tiles<float, 1, RESET>(a, bwd, st);
  if (pairs_of_channels(a, bwd)) return launch_tiles<bf16, 2, RESET>(a, bwd, st);
  return launch_tiles<bf16, 1, RESET>(a, bwd, st);
}

}  // namespace

int gated_linear_fwd(int dtype, const GatedLinearArgs& a, cudaStream_t st) {
  if (a.T > SEQ_STEPS)
    return a.reset != nullptr ? launch_tiles<true>(dtype, a, false, st) : launch_tiles<false>(dtype, a, false, st);
  const GlParams p = params_of(a);
  const long grid = ((long)a.B * a.d + 127) / 128;
  ELMAN_ARG_CHECK(grid < (1L << 31), "too many channels for one call");
  if (dtype == ELMAN_F32) gl_forward_seq_kernel<float><<<(unsigned)grid, 128, 0, st>>>(p);
  else gl_forward_seq_kernel<bf16><<<(unsigned)grid, 128, 0, st>>>(p);
  count_launch(false);
  ELMAN_CUDA_CHECK(cudaGetLastError());
  return ELMAN_OK;
}

int gated_linear_bwd(int dtype, const GatedLinearArgs& a, cudaStream_t st) {
  if (a.T > SEQ_STEPS)
    return a.reset != nullptr ? launch_tiles<true>(dtype, a, true, st) : launch_tiles<false>(dtype, a, true, st);
  const GlParams p = params_of(a);
  const long grid = ((long)a.B * a.d + 127) / 128;
  ELMAN_ARG_CHECK(grid < (1L << 31), "too many channels for one call");
  if (dtype == ELMAN_F32) gl_backward_seq_kernel<float><<<(unsigned)grid, 128, 0, st>>>(p);
  else gl_backward_seq_kernel<bf16><<<(unsigned)grid, 128, 0, st>>>(p);
  count_launch(false);
  ELMAN_CUDA_CHECK(cudaGetLastError());
  return ELMAN_OK;
}

size_t gated_linear_workspace(int dtype, int T, int B, int d) {
  // the backward pass has the shorter tiles
  return T > SEQ_STEPS ? chain_bytes(tiles_of(T, BW * BL), B * (whole_width(dtype, d) ? whole_groups(dtype, d) : (long)d)) : 0;
}

}  // namespace elman
