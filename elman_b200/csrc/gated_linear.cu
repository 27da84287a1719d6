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
#include "common.cuh"

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
// Sequences of more than a few steps: tiles of (W warps x L steps) x (32 V channels), each read once.
//
// A warp holds L steps of 32 lanes x V channels in registers and scans them from a zero state: the pair (R, H)
// with  h_out = h_in + (H - R h_in),  R = 1 - prod(1 - u) kept as the scan of the constant 1, so that
// it too keeps what 1 - u would lose.  R = -1 says that a reset lies inside: h_out = H, and h_in (which
// may be anything) is not read.  The tile's own pair goes to the tiles that follow in time through L2;
// they fold the pairs of their group of GROUP tiles onto the state at the group's start, which the last
// tile of the group before has published.  The association is fixed, so results do not depend on
// timing; the chain of dependent exchanges is one per GROUP tiles.  Backwards the same with time
// reversed, D in place of h, and the states recomputed from `saved`.
//
// Pairs and states are their own flags: the workspace starts as all ones, which no published value is
// (NaN goes out as 0x7fffffff), so an exchange is one store and one load.  Tiles are handed out in time
// order by a counter: whoever a tile waits for has started before it and waits for nobody behind it.
// ---------------------------------------------------------------------------
constexpr int GROUP = 16;
constexpr uint32_t NOT_YET = 0xFFFFFFFFu;

struct GlChain {             // workspace; all of it starts as NOT_YET
  uint32_t* ctrl;            // [0]: tiles handed out - 1; [1]: 0 once a wait has given up
  float2* pairs;             // [tiles in time][columns]
  float* states;             // [groups][columns]
  int* status;
  long spin_limit;
  int stall;                 // test hook: this tile publishes nothing
};

struct Pair { float R, H; };
__device__ __forceinline__ float pass(float S, Pair a) { return a.R < 0.f ? a.H : S + fmaf(-a.R, S, a.H); }
__device__ __forceinline__ Pair join(Pair a, Pair b) {       // a, then b
  if (b.R < 0.f) return b;
  return Pair{a.R < 0.f ? -1.f : a.R + fmaf(-b.R, a.R, b.R), a.H + fmaf(-b.R, a.H, b.H)};
}

template <typename T, int V> struct Lane;                    // V adjacent channels as they are in memory
template <> struct Lane<float, 1> {
  typedef float Raw;
  static __device__ __forceinline__ void get(Raw r, float (&x)[1]) { x[0] = r; }
  static __device__ __forceinline__ Raw put(const float (&x)[1]) { return x[0]; }
};
template <> struct Lane<bf16, 1> {
  typedef unsigned short Raw;
  static __device__ __forceinline__ void get(Raw r, float (&x)[1]) { x[0] = __uint_as_float((uint32_t)r << 16); }
  static __device__ __forceinline__ Raw put(const float (&x)[1]) { return __bfloat16_as_ushort(__float2bfloat16_rn(x[0])); }
};
template <> struct Lane<bf16, 2> {
  typedef uint32_t Raw;
  static __device__ __forceinline__ void get(Raw r, float (&x)[2]) {
    x[0] = __uint_as_float(r << 16);
    x[1] = __uint_as_float(r & 0xFFFF0000u);
  }
  static __device__ __forceinline__ Raw put(const float (&x)[2]) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(x[0], x[1]);
    return *reinterpret_cast<const Raw*>(&v);
  }
};

__device__ __forceinline__ uint32_t word_of(float x) { return x != x ? 0x7FFFFFFFu : __float_as_uint(x); }
template <int V> __device__ __forceinline__ void publish(float2* at, const Pair (&a)[V]) {
  if constexpr (V == 2)
    asm volatile("st.relaxed.gpu.global.v4.b32 [%0], {%1, %2, %3, %4};" ::"l"(at), "r"(word_of(a[0].R)), "r"(word_of(a[0].H)),
                 "r"(word_of(a[1].R)), "r"(word_of(a[1].H)) : "memory");
  else
    asm volatile("st.relaxed.gpu.global.v2.b32 [%0], {%1, %2};" ::"l"(at), "r"(word_of(a[0].R)), "r"(word_of(a[0].H)) : "memory");
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
// The whole warp waits until every lane's N words are there; false: gave up.
template <int N> __device__ __forceinline__ bool await(const void* at, uint32_t (&w)[N], const GlChain& ch, int step) {
  long spins = 0;
  unsigned long long t0 = 0;
  while (!__all_sync(0xFFFFFFFFu, look<N>(at, w))) {
    ++spins;
    bool stop = spins > ch.spin_limit;
    if ((spins & 255) == 0) {
      uint32_t aborted[1];
      look<1>(ch.ctrl + 1, aborted);
      stop = stop || aborted[0] == 0;
      unsigned long long now;
      asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(now));
      if (t0 == 0) t0 = now;
      else if (now - t0 > 2000000000ull) stop = true;
    }
    if (__any_sync(0xFFFFFFFFu, stop)) {
      if ((threadIdx.x & 31) == 0) {
        asm volatile("st.relaxed.gpu.global.b32 [%0], %1;" ::"l"(ch.ctrl + 1), "r"(0) : "memory");
        report_timeout(ch.status, KID_GATED_LINEAR, step);
      }
      return false;
    }
  }
  return true;
}

// Where a tile stands in the chain: `n` counts tiles from the end of time the scan starts at.
template <int V, int W> struct Chain {
  struct Shared {
    Pair own[2][W][32 * V];             // the warps' pairs (two tiles' worth: a slow warp may still read the last one's)
    Pair before[2][GROUP - 1][32 * V];  // pairs of the tiles before in the group
    float start[2][32 * V];             // state at the group's start
    int next;
    int gave_up;
  };
  // From the warp's own pair to the state that enters it.  All W warps (w = order in the scan's
  // direction) call it; `initial` is the state at the scan's start.  False: a wait gave up.
  static __device__ __forceinline__ bool enter(Shared& sh, int buf, int w, int warps, const Pair (&mine)[V], int n,
                                               int tiles, long col, long cols, bool lane_on, const float (&initial)[V],
                                               const GlChain& ch, int ticket, uint32_t* grabbed, float (&S)[V]) {
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int v = 0; v < V; ++v) sh.own[buf][w][lane * V + v] = mine[v];
    __syncthreads();
    const int first = n / GROUP * GROUP, in_group = n - first;
    const bool last_of_group = in_group == GROUP - 1;
    if (tiles > 1) {
      bool ok = true;
      if (w == 0 && n + 1 < tiles && !last_of_group && ticket != ch.stall) {
        Pair all[V];
#pragma unroll
        for (int v = 0; v < V; ++v) {
          all[v] = sh.own[buf][0][lane * V + v];
          for (int k = 1; k < warps; ++k) all[v] = join(all[v], sh.own[buf][k][lane * V + v]);
        }
        if (lane_on) publish<V>(ch.pairs + (long)n * cols + col, all);
      }
      for (int k = w; k < in_group && ok; k += warps) {
        uint32_t x[2 * V];
        ok = await<2 * V>(ch.pairs + (long)(first + k) * cols + col, x, ch, n);
#pragma unroll
        for (int v = 0; v < V; ++v)
          sh.before[buf][k][lane * V + v] = Pair{__uint_as_float(x[2 * v]), __uint_as_float(x[2 * v + 1])};
      }
      if (w == warps - 1) {
        uint32_t x[V];
        if (first > 0 && ok) ok = await<V>(ch.states + (long)(first / GROUP - 1) * cols + col, x, ch, n);
#pragma unroll
        for (int v = 0; v < V; ++v) sh.start[buf][lane * V + v] = first > 0 ? __uint_as_float(x[v]) : initial[v];
      }
      if (!ok && lane == 0) sh.gave_up = 1;
      if (threadIdx.x == 0) sh.next = (int)(*grabbed + 1u);
      __syncthreads();
      if (sh.gave_up) return false;
#pragma unroll
      for (int v = 0; v < V; ++v) {
        S[v] = sh.start[buf][lane * V + v];
        for (int k = 0; k < in_group; ++k) S[v] = pass(S[v], sh.before[buf][k][lane * V + v]);
      }
    } else {
#pragma unroll
      for (int v = 0; v < V; ++v) S[v] = initial[v];
    }
    if (w == 0 && last_of_group && n + 1 < tiles && ticket != ch.stall) {
      float end[V];
#pragma unroll
      for (int v = 0; v < V; ++v) {
        end[v] = S[v];
        for (int k = 0; k < warps; ++k) end[v] = pass(end[v], sh.own[buf][k][lane * V + v]);
        if (lane_on)
          asm volatile("st.relaxed.gpu.global.b32 [%0], %1;" ::"l"(ch.states + (long)(first / GROUP) * cols + col + v),
                       "r"(word_of(end[v])) : "memory");
      }
    }
#pragma unroll
    for (int v = 0; v < V; ++v)
      for (int k = 0; k < w; ++k) S[v] = pass(S[v], sh.own[buf][k][lane * V + v]);
    return true;
  }
};

// Steps of a warp whose document starts anew, as bits (lanes of one batch row agree).
template <int L> __device__ __forceinline__ uint32_t reset_bits(const GlParams& p, int t0, int b) {
  uint32_t bits = 0;
#pragma unroll
  for (int l = 0; l < L; ++l)
    if (t0 + l < p.T && p.reset[(long)(t0 + l) * p.B + b] != 0) bits |= 1u << l;
  return bits;
}

constexpr int FW = 8, FL = 16;      // forward tile: 128 steps
constexpr int BW = 8, BL = 8;       // backward tile: GL_CHUNK steps, so that it starts at a saved state
static_assert(BW * BL == GL_CHUNK && GL_CHUNK % FL == 0, "saved states lie on tile and warp edges");

template <typename T, int V, bool RESET>
__global__ void __launch_bounds__(32 * FW, 2) gl_forward_tile_kernel(GlParams p, GlChain ch, int tiles, int col_groups) {
  typedef typename Lane<T, V>::Raw Raw;
  __shared__ typename Chain<V, FW>::Shared sh;
  const int w = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = blockDim.x >> 5;
  const long cols = (long)p.B * p.d;
  const int total = tiles * col_groups;
  if (threadIdx.x == 0) {
    sh.gave_up = 0;
    sh.next = tiles > 1 ? (int)(atomicAdd(ch.ctrl, 1u) + 1u) : (int)blockIdx.x;
  }
  __syncthreads();
  for (int ticket = sh.next, buf = 0; ticket < total; buf ^= 1) {
    uint32_t grabbed = 0;
    if (tiles > 1 && threadIdx.x == 0) grabbed = atomicAdd(ch.ctrl, 1u);
    const int n = ticket / col_groups;
    const long mine = (long)(ticket - n * col_groups) * (32 * V) + lane * V;
    const bool lane_on = mine < cols;
    const long col = lane_on ? mine : cols - V;
    const int b = (int)(col / p.d), i = (int)(col - (long)b * p.d);
    const int t0 = n * (FW * FL) + w * FL;
    const Raw* f = reinterpret_cast<const Raw*>((const T*)p.f + (long)t0 * p.sf.t + b * p.sf.b + i);
    const Raw* c = reinterpret_cast<const Raw*>((const T*)p.c + (long)t0 * p.sc.t + b * p.sc.b + i);
    const Raw* z = reinterpret_cast<const Raw*>((const T*)p.z + (long)t0 * p.sz.t + b * p.sz.b + i);
    const int steps = p.T - t0;            // of this warp, L at most
    Raw rf[FL], rc[FL], rz[FL];
#pragma unroll
    for (int l = 0; l < FL; ++l) {
      rf[l] = Raw(0); rc[l] = Raw(0); rz[l] = Raw(0);
      if (l < steps) {
        rf[l] = __ldcs(f + l * (p.sf.t / V));
        rc[l] = __ldcs(c + l * (p.sc.t / V));
        rz[l] = __ldcs(z + l * (p.sz.t / V));
      }
    }
    const uint32_t cut = RESET ? reset_bits<FL>(p, t0, b) : 0;
    float u[FL][V], H[V], R[V];
#pragma unroll
    for (int v = 0; v < V; ++v) H[v] = R[v] = 0.f;
#pragma unroll
    for (int l = 0; l < FL; ++l) {
      float fx[V], cx[V], e;
      Lane<T, V>::get(rf[l], fx);
      Lane<T, V>::get(rc[l], cx);
#pragma unroll
      for (int v = 0; v < V; ++v) {
        u[l][v] = l < steps ? keep_gate(fx[v], e) : 0.f;     // beyond the end: the state stays
        if (RESET && (cut >> l & 1)) H[v] = 0.f;
        H[v] = fmaf(u[l][v], cx[v] - H[v], H[v]);
        R[v] = fmaf(u[l][v], 1.f - R[v], R[v]);
      }
    }
    Pair own[V];
    float h[V], initial[V];
#pragma unroll
    for (int v = 0; v < V; ++v) {
      own[v] = Pair{RESET && cut ? -1.f : R[v], H[v]};
      initial[v] = n < GROUP && p.h0 != nullptr ? p.h0[col + v] : 0.f;
    }
    if (!Chain<V, FW>::enter(sh, buf, w, warps, own, n, tiles, col, cols, lane_on, initial, ch, ticket, &grabbed, h)) return;
    ticket = tiles > 1 ? sh.next : total;
    if (lane_on && steps > 0) {
      if (p.saved != nullptr && t0 % GL_CHUNK == 0) {
#pragma unroll
        for (int v = 0; v < V; ++v) p.saved[(long)(t0 / GL_CHUNK) * cols + col + v] = h[v];
      }
      Raw* y = reinterpret_cast<Raw*>((T*)p.y + (long)t0 * p.sy.t + b * p.sy.b + i);
#pragma unroll
      for (int l = 0; l < FL; ++l) {
        float cx[V], zx[V], out[V];
        Lane<T, V>::get(rc[l], cx);
        Lane<T, V>::get(rz[l], zx);
#pragma unroll
        for (int v = 0; v < V; ++v) {
          if (RESET && (cut >> l & 1)) h[v] = 0.f;
          h[v] = fmaf(u[l][v], cx[v] - h[v], h[v]);
          out[v] = h[v] * siluf_(zx[v]);
        }
        if (l < steps) __stcs(y + l * (p.sy.t / V), Lane<T, V>::put(out));
      }
      if (steps <= FL) {
#pragma unroll
        for (int v = 0; v < V; ++v) p.h_last[col + v] = h[v];
      }
    }
  }
}

template <typename T, int V, bool RESET>
__global__ void __launch_bounds__(32 * BW, 2) gl_backward_tile_kernel(GlParams p, GlChain ch, int tiles, int col_groups) {
  typedef typename Lane<T, V>::Raw Raw;
  __shared__ typename Chain<V, BW>::Shared sh;
  __shared__ Pair ahead[2][BW][32 * V];      // the warps' pairs of the forward scan
  const int w = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = blockDim.x >> 5;
  const long cols = (long)p.B * p.d;
  const int total = tiles * col_groups;
  if (threadIdx.x == 0) {
    sh.gave_up = 0;
    sh.next = tiles > 1 ? (int)(atomicAdd(ch.ctrl, 1u) + 1u) : (int)blockIdx.x;
  }
  __syncthreads();
  for (int ticket = sh.next, buf = 0; ticket < total; buf ^= 1) {
    uint32_t grabbed = 0;
    if (tiles > 1 && threadIdx.x == 0) grabbed = atomicAdd(ch.ctrl, 1u);
    const int n = ticket / col_groups, chunk = tiles - 1 - n;
    const long mine = (long)(ticket - n * col_groups) * (32 * V) + lane * V;
    const bool lane_on = mine < cols;
    const long col = lane_on ? mine : cols - V;
    const int b = (int)(col / p.d), i = (int)(col - (long)b * p.d);
    const int t0 = chunk * GL_CHUNK + w * BL;
    const Raw* f = reinterpret_cast<const Raw*>((const T*)p.f + (long)t0 * p.sf.t + b * p.sf.b + i);
    const Raw* c = reinterpret_cast<const Raw*>((const T*)p.c + (long)t0 * p.sc.t + b * p.sc.b + i);
    const Raw* z = reinterpret_cast<const Raw*>((const T*)p.z + (long)t0 * p.sz.t + b * p.sz.b + i);
    const Raw* dy = reinterpret_cast<const Raw*>((const T*)p.dy + (long)t0 * p.sy.t + b * p.sy.b + i);
    const int steps = p.T - t0;
    Raw rf[BL], rc[BL], rz[BL], rdy[BL];
#pragma unroll
    for (int l = 0; l < BL; ++l) {
      rf[l] = Raw(0); rc[l] = Raw(0); rz[l] = Raw(0); rdy[l] = Raw(0);
      if (l < steps) {
        rf[l] = __ldcs(f + l * (p.sf.t / V));
        rc[l] = __ldcs(c + l * (p.sc.t / V));
        rz[l] = __ldcs(z + l * (p.sz.t / V));
        rdy[l] = __ldcs(dy + l * (p.sy.t / V));
      }
    }
    float h[V], D[V];
#pragma unroll
    for (int v = 0; v < V; ++v) {
      h[v] = p.saved[(long)chunk * cols + col + v];
      D[v] = n < GROUP && p.dh_last != nullptr ? p.dh_last[col + v] : 0.f;
    }
    const uint32_t cut = RESET ? reset_bits<BL>(p, t0, b) : 0;
    // the states before the warp's steps
    float u[BL][V], a[BL][V], H[V], R[V];
#pragma unroll
    for (int v = 0; v < V; ++v) H[v] = R[v] = 0.f;
#pragma unroll
    for (int l = 0; l < BL; ++l) {
      float fx[V], cx[V];
      Lane<T, V>::get(rf[l], fx);
      Lane<T, V>::get(rc[l], cx);
#pragma unroll
      for (int v = 0; v < V; ++v) {
        float e;
        u[l][v] = keep_gate(fx[v], e);
        a[l][v] = e * u[l][v] * u[l][v];                      // u (1 - u)
        if (l >= steps) u[l][v] = 0.f;
        if (RESET && (cut >> l & 1)) H[v] = 0.f;
        H[v] = fmaf(u[l][v], cx[v] - H[v], H[v]);
        R[v] = fmaf(u[l][v], 1.f - R[v], R[v]);
      }
    }
#pragma unroll
    for (int v = 0; v < V; ++v) {
      R[v] = RESET && cut ? -1.f : R[v];
      ahead[buf][w][lane * V + v] = Pair{R[v], H[v]};
    }
    __syncthreads();
#pragma unroll
    for (int v = 0; v < V; ++v)
      for (int k = 0; k < w; ++k) h[v] = pass(h[v], ahead[buf][k][lane * V + v]);
    // forward through the warp's steps: dz, and what the scan back needs
    Raw* dz = reinterpret_cast<Raw*>((T*)p.dz + (long)t0 * p.sdz.t + b * p.sdz.b + i);
    float q[BL][V], prev[BL][V];
#pragma unroll
    for (int l = 0; l < BL; ++l) {
      float cx[V], zx[V], gx[V], out[V];
      Lane<T, V>::get(rc[l], cx);
      Lane<T, V>::get(rz[l], zx);
      Lane<T, V>::get(rdy[l], gx);
#pragma unroll
      for (int v = 0; v < V; ++v) {
        if (RESET && (cut >> l & 1)) h[v] = 0.f;
        prev[l][v] = h[v] - cx[v];
        h[v] = fmaf(u[l][v], cx[v] - h[v], h[v]);
        const float sg = sigmoidf_(zx[v]);
        q[l][v] = gx[v] * zx[v] * sg;
        out[v] = gx[v] * h[v] * sg * (1.f + zx[v] * (1.f - sg));
      }
      if (lane_on && l < steps) __stcs(dz + l * (p.sdz.t / V), Lane<T, V>::put(out));
    }
    Pair own[V];
#pragma unroll
    for (int v = 0; v < V; ++v) {
      float E = 0.f;
#pragma unroll
      for (int l = BL - 1; l >= 0; --l) {
        const float g = q[l][v] + E;
        E = RESET && (cut >> l & 1) ? 0.f : fmaf(-u[l][v], g, g);
      }
      own[v] = Pair{R[v], E};
    }
    float start[V];
#pragma unroll
    for (int v = 0; v < V; ++v) start[v] = D[v];
    if (!Chain<V, BW>::enter(sh, buf, warps - 1 - w, warps, own, n, tiles, col, cols, lane_on, start, ch, ticket, &grabbed, D)) return;
    ticket = tiles > 1 ? sh.next : total;
    Raw* df = reinterpret_cast<Raw*>((T*)p.df + (long)t0 * p.sdf.t + b * p.sdf.b + i);
    Raw* dc = reinterpret_cast<Raw*>((T*)p.dc + (long)t0 * p.sdc.t + b * p.sdc.b + i);
#pragma unroll
    for (int l = BL - 1; l >= 0; --l) {
      float of[V], oc[V];
#pragma unroll
      for (int v = 0; v < V; ++v) {
        const float g = q[l][v] + D[v];
        oc[v] = g * u[l][v];
        of[v] = g * prev[l][v] * a[l][v];
        D[v] = RESET && (cut >> l & 1) ? 0.f : fmaf(-u[l][v], g, g);
      }
      if (lane_on && l < steps) {
        __stcs(dc + l * (p.sdc.t / V), Lane<T, V>::put(oc));
        __stcs(df + l * (p.sdf.t / V), Lane<T, V>::put(of));
      }
    }
    if (lane_on && t0 == 0) {
#pragma unroll
      for (int v = 0; v < V; ++v) p.dh0[col + v] = D[v];
    }
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
  return 256 + (size_t)tiles * cols * sizeof(float2) + (size_t)((tiles + GROUP - 1) / GROUP) * cols * sizeof(float);
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

template <typename T, int V, bool RESET>
int launch_tiles(const GatedLinearArgs& a, bool bwd, cudaStream_t st) {
  auto* kernel = bwd ? &gl_backward_tile_kernel<T, V, RESET> : &gl_forward_tile_kernel<T, V, RESET>;
  const long cols = (long)a.B * a.d;
  const int per_warp = bwd ? BL : FL, tile = bwd ? BW * BL : FW * FL;
  const int tiles = tiles_of(a.T, tile);
  const int warps = tiles > 1 ? tile / per_warp : tiles_of(a.T, per_warp);
  const long col_groups = (cols + 32 * V - 1) / (32 * V);
  const long total = col_groups * tiles;
  ELMAN_ARG_CHECK(total + 148 * 8 < (1L << 31), "too many channels for one call");
  GlChain ch{};
  long grid = total;
  if (tiles > 1) {
    char* ws = (char*)a.workspace;
    ch.ctrl = (uint32_t*)ws;
    ch.pairs = (float2*)(ws + 256);
    ch.states = (float*)(ws + 256 + (size_t)tiles * cols * sizeof(float2));
    ch.status = device_status_ptr();
    ch.spin_limit = options().spin_limit;
    ch.stall = (int)options().test_stall_step;
    ELMAN_CUDA_CHECK(cudaMemsetAsync(ws, 0xFF, chain_bytes(tiles, cols), st));
    const long resident = 148 * 4;       // more than stay resident: the counter hands out the tiles
    if (grid > resident) grid = resident;
  }
  GlParams p = params_of(a);
  kernel<<<(unsigned)grid, 32 * warps, 0, st>>>(p, ch, tiles, (int)col_groups);
  count_launch(false);
  ELMAN_CUDA_CHECK(cudaGetLastError());
  return ELMAN_OK;
}

template <bool RESET>
int launch_tiles(int dtype, const GatedLinearArgs& a, bool bwd, cudaStream_t st) {
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
  (void)dtype;
  // the backward pass has the shorter tiles
  return T > SEQ_STEPS ? chain_bytes(tiles_of(T, BW * BL), (long)B * d) : 0;
}

}  // namespace elman
