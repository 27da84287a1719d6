// Orthogonalising matrices by Newton-Schulz products, and the Muon update built on it:
//   X = G / (|G|_F + eps);  steps times:  A = X X^T,  B = b A + c A A,  X <- a X + B X
// (tall matrices: A = X^T X and X <- a X + X B, so that A has the smaller of the two extents, r).
// A and B are symmetric: only the tiles on and above the diagonal are computed and stored.  Per step 3 r^2 q + r^3
// flops with q the larger extent, three products for each of them (Numbers, below): bound by the tensor cores.
// Measured, five steps on bf16, the same inputs again and again: 18 x 1280 x 1280 1.79 ms (1260 TFLOP/s of such products, the
// tensor pipe 90 % busy; 2.11 ms with inputs that change, at the power limit), 1 x 4096 x 4096 2.98 ms (1380).  Small matrices
// are bound by the latency of 15 products one after another: 1 x 256 x 256 109 us, 7 us each.
//
// Numbers.  X, A and B are each kept as the sum of two fp16 numbers (22 significant bits), scaled by powers of two into
// their range: X by 2^12, A by 2^12, B by 2^10.  A product is three: high x high, high x low, low x high; every sum is
// fp32.  So a bf16 result is the exact one rounded (one fp16 number an operand leaves 1.3e-3 before that rounding,
// as much as the rounding itself), and an fp32 result is 5e-6 off.  The tensor cores cut their fp32 sums off rather than
// rounding them, which over a long contraction adds up (2.5e-5 at 33 x 2000 with one sum): for fp32 matrices the large
// products take turns in three sums and the small ones have a fourth (3.4e-6 at 200 x 2000, 1.2e-5 at 200 x 9000, 2.9e-5 at
// 1000 x 20000).  A step along K brings the high parts of both operands in one stage and the low parts in the next, for all
// three products: 4 x 1000 x 257 fp32 250 us with a stage a product, now 176.
// A start below 1e-4 (a norm far below eps) would lose its low parts under fp16's range: X is held as 2^e X, with an e for each
// matrix and step that follows from the norm and what the polynomial can make of it.
#include <math.h>

#include <mutex>
#include <type_traits>

#include "common.cuh"
#include "sm100_ptx.cuh"
#include "tc_helpers.cuh"

#include <cuda_fp16.h>

namespace elman {

namespace {

// One block's share of a tile is 128 rows of the product; a pair of blocks (cta_group::2) makes a tile of 256 x 256,
// a block by itself one of 128 x 128 or of 128 x 64.
constexpr int BK = 64, STAGES = 6, TICKETS = 4;
constexpr int EPI_WARPS = 8, THREADS = 128 + 32 * EPI_WARPS;
constexpr int BLOCK_BYTES = 64 * BK * 2;              // one TMA box: 64 x 64 fp16
constexpr int OPERAND_BYTES = 128 * BK * 2;
// Rows are finished in boxes of 32 x 32 through shared memory, a box's high and low parts a warp, with plain 16-byte
// accesses to global memory: the copy engine takes about two cycles a row of a box, and the operands' rows (512 a step
// along K of 1536 cycles) take most of its time already.
constexpr int BOX_BYTES = 32 * 64, BUFFER_BYTES = 2 * BOX_BYTES;
constexpr int NS_SMEM = STAGES * 2 * OPERAND_BYTES + EPI_WARPS * BUFFER_BYTES + 1024;
constexpr float SX = 4096.f, SA = 4096.f, SB = 1024.f;
constexpr int NORM_PARTS = 64;                        // partial sums of squares a matrix
constexpr int SHIFTS = 128;                           // exponents kept a matrix: one in front of each of 100 steps at most, and behind

enum Product { GRAM, SQUARE, UPDATE, LAST };
// An operand block of rows x K: stored [rows, K]; stored [K, rows] and read MN-major in place; or part of a
// symmetric matrix of which only the tiles on and above the diagonal are stored: below it the block is the
// mirrored one, read MN-major.
enum Form { ROWS_K, K_ROWS, UPPER };
__device__ __forceinline__ bool mn_major(int form, int row0, int k0, int edge) {
  return form == K_ROWS || (form == UPPER && row0 / edge > k0 / edge);
}

struct Split { __half* hi; __half* lo; };

// The matrix a step starts from: G, or Muon's momentum-weighted gradient.
struct NsSource {
  const void* in;            // [count, m, n], or the flat gradients
  const long long* offsets;  // Muon: where each matrix starts in the flat buffers (device); null: dense
  float* momentum;           // Muon: [count, m, n]
  float mu;
  int nesterov;
  const float* grad_scale;   // device, or null
};

// [high, low part] of a matrix: boxes of 128 rows x 64 (read along the rows) and of 64 x 64 (read MN-major).
struct NsMap { CUtensorMap rows[2], block[2]; };
struct NsMaps { NsMap x[2], a, b; };

// The whole iteration as one list of tiles: step by step, in a step all Gram tiles of all matrices, then the squares',
// then the updates'.  (Groups of matrices that stay in L2 from product to product were slower, with one product where
// there are three now: 18 x 1280 x 1280 as three groups 0.98 ms, as one 0.87: waiting for the matrix one reads costs more
// than reading it from HBM.)
struct NsPlan {
  int count, m, n, r, tall, steps;
  int edge, n_sym, n_upd;    // rows of a tile; columns of a symmetric product's tiles and of an update's
  int triangle, all;         // tiles of a symmetric product and of an update
  int per_step, total;       // items of the list
  float a, b, c;
  Split X[2], A, B;
  long ldx, ldr;
  void* result;              // [count, m, n], or the flat parameters
  const long long* offsets;
  int muon;
  float lr, decay, scale;    // Muon: p = p decay - lr scale X
  int* ticket;               // items handed out
  int* done;                 // [count]: warps' shares of tiles finished
  const unsigned char* shift;   // [count][SHIFTS]: step k starts from 2^shift X
  int* status;
  long spin_limit;
  int stall, leave;          // test hooks: a stage that is not loaded; 32 q + w: warp w gives up the wait for its block's item q
};

// One item of the list.  Taking it apart costs divisions, a thousand cycles of latency: the warp that takes items does
// it ahead of time and hands on the four numbers that the rest follows from.
struct alignas(16) NsSlot { int kind, mat, tile, step; };     // kind -1: no more; step with the exponents before and after it
__device__ __forceinline__ NsSlot slot_of(const NsPlan& p, int index) {
  NsSlot k;
  k.step = index / p.per_step;
  int w = index - k.step * p.per_step, ti, tj;
  const int gram = p.count * p.triangle;
  if (w < 2 * gram) {
    k.kind = w >= gram ? SQUARE : GRAM;
    if (w >= gram) w -= gram;
    k.mat = w / p.triangle;
    // column by column of blocks the blocks (i, j >= i), `per` tiles each
    const int t = w - k.mat * p.triangle, per = p.edge / p.n_sym, s = t / per;
    int j = (int)((sqrtf(8.f * (float)s + 1.f) - 1.f) * 0.5f);
    while ((j + 1) * (j + 2) / 2 <= s) ++j;
    while (j * (j + 1) / 2 > s) --j;
    const int rest = t - per * (j * (j + 1) / 2);
    tj = per * j + rest / (j + 1);
    ti = rest % (j + 1);
  } else {
    w -= 2 * gram;
    k.kind = k.step == p.steps - 1 ? LAST : UPDATE;
    k.mat = w / p.all;
    const int t = w - k.mat * p.all, tiles_n = (p.n + p.n_upd - 1) / p.n_upd;
    ti = t / tiles_n;
    tj = t - ti * tiles_n;
  }
  k.tile = ti << 16 | tj;
  const unsigned char* e = p.shift + (long)k.mat * SHIFTS + k.step;
  k.step |= e[0] << 8 | e[1] << 16;
  return k;
}
__device__ __forceinline__ int step_of(NsSlot k) { return k.step & 0xFF; }
struct NsItem {
  int kind, mat, ti, tj, step;
  int columns;                                 // of the tile
  int e, e_next;                               // X is held at 2^e of itself, and the step's result at 2^e_next
  int m, n, K, a_form, b_form;
};
__device__ __forceinline__ NsItem item_of(const NsPlan& p, NsSlot k) {
  NsItem it;
  it.kind = k.kind; it.mat = k.mat; it.ti = k.tile >> 16; it.tj = k.tile & 0xFFFF; it.step = step_of(k);
  it.e = k.step >> 8 & 0xFF; it.e_next = k.step >> 16;
  const bool symmetric = k.kind == GRAM || k.kind == SQUARE;
  it.columns = symmetric ? p.n_sym : p.n_upd;
  it.m = symmetric ? p.r : p.m;
  it.n = symmetric ? p.r : p.n;
  it.K = k.kind != GRAM ? p.r : p.tall ? p.m : p.n;
  if (k.kind == GRAM) it.a_form = it.b_form = p.tall ? K_ROWS : ROWS_K;
  else if (k.kind == SQUARE) it.a_form = it.b_form = UPPER;
  else {                                       // X B, or B X
    it.a_form = p.tall ? ROWS_K : UPPER;
    it.b_form = p.tall ? UPPER : K_ROWS;
  }
  return it;
}
// Tiles of its matrix that have to be finished before an item may start.
__device__ __forceinline__ int needed(const NsPlan& p, NsSlot k) {
  return step_of(k) * (2 * p.triangle + p.all) + (k.kind == GRAM ? 0 : k.kind == SQUARE ? p.triangle : 2 * p.triangle);
}

__device__ __forceinline__ void add_halves(float (&f)[8], uint4 x, float k) {
  const __half2* h = reinterpret_cast<const __half2*>(&x);
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    const float2 v = __half22float2(h[q]);
    f[2 * q] = fmaf(k, v.x, f[2 * q]);
    f[2 * q + 1] = fmaf(k, v.y, f[2 * q + 1]);
  }
}
__device__ __forceinline__ uint4 to_halves(const float (&f)[8]) {
  uint4 x;
  __half2* h = reinterpret_cast<__half2*>(&x);
#pragma unroll
  for (int q = 0; q < 4; ++q) h[q] = __floats2half2_rn(f[2 * q], f[2 * q + 1]);
  return x;
}

// ------------------------------------------------------------------ start: norm and scaling

// Muon's momentum moves by (1 - mu)(g - momentum); the update is it, or Nesterov's look ahead.
__device__ __forceinline__ float advance(const NsSource& s, float g, float gs, float& momentum) {
  g *= gs;
  momentum += (1.f - s.mu) * (g - momentum);
  return s.nesterov ? g + s.mu * (momentum - g) : momentum;
}
__device__ __forceinline__ float look_ahead(const NsSource& s, float g, float gs, float momentum) {
  g *= gs;
  return s.nesterov ? g + s.mu * (momentum - g) : momentum;
}
// Eight adjacent elements as one or two 16-byte accesses.
template <typename T> __device__ __forceinline__ void load8(const T* at, float (&f)[8]) {
  uint4 x[sizeof(T) / 2];
#pragma unroll
  for (int q = 0; q < (int)sizeof(T) / 2; ++q) x[q] = reinterpret_cast<const uint4*>(at)[q];
  const T* v = reinterpret_cast<const T*>(x);
#pragma unroll
  for (int j = 0; j < 8; ++j) f[j] = to_f(v[j]);
}
__device__ __forceinline__ void store8(float* at, const float (&f)[8]) {
#pragma unroll
  for (int q = 0; q < 2; ++q) reinterpret_cast<float4*>(at)[q] = make_float4(f[4 * q], f[4 * q + 1], f[4 * q + 2], f[4 * q + 3]);
}

// Sums of squares in fp64: a sum over millions of elements, of numbers whose squares leave fp32's range.  Also starts
// the counters of the products.
template <typename T>
__global__ void __launch_bounds__(256) ns_norm_kernel(NsSource s, long size, double* partial, int* ticket, int* done) {
  ptx::let_next_start();
  if (blockIdx.x == 0 && threadIdx.x == 0) {
    done[blockIdx.y] = 0;
    if (blockIdx.y == 0) *ticket = 0;
  }
  const T* in = (const T*)s.in + (s.offsets != nullptr ? s.offsets[blockIdx.y] : (long)blockIdx.y * size);
  float* momentum = s.momentum != nullptr ? s.momentum + (long)blockIdx.y * size : nullptr;
  const float gs = s.grad_scale != nullptr ? *s.grad_scale : 1.f;
  double sum = 0.;
  const bool vec = (((uintptr_t)in | (uintptr_t)momentum) & 15) == 0;
  const long whole = vec ? size / 8 : 0;
  for (long g = (long)blockIdx.x * 256 + threadIdx.x; g < whole; g += NORM_PARTS * 256) {
    float f[8];
    load8(in + 8 * g, f);
    if (momentum != nullptr) {
      float mom[8];
      load8(momentum + 8 * g, mom);
#pragma unroll
      for (int j = 0; j < 8; ++j) f[j] = advance(s, f[j], gs, mom[j]);
      store8(momentum + 8 * g, mom);
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) sum = fma((double)f[j], (double)f[j], sum);
  }
  for (long e = 8 * whole + (long)blockIdx.x * 256 + threadIdx.x; e < size; e += NORM_PARTS * 256) {
    float v = to_f(in[e]);
    if (momentum != nullptr) {
      float mom = momentum[e];
      v = advance(s, v, gs, mom);
      momentum[e] = mom;
    }
    sum = fma((double)v, (double)v, sum);
  }
  __shared__ double warp_sum[8];
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_down_sync(0xFFFFFFFFu, sum, o);
  if ((threadIdx.x & 31) == 0) warp_sum[threadIdx.x >> 5] = sum;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int k = 1; k < 8; ++k) sum += warp_sum[k];
    partial[(long)blockIdx.y * NORM_PARTS + blockIdx.x] = sum;
  }
}

struct Quintic { double a, b, c; };
// The largest |s (a + b s^2 + c s^4)| of s in [0, top].
__host__ __device__ inline double largest(Quintic q, double top) {
  auto poly = [&](double s2) { return fabs(sqrt(s2) * (q.a + s2 * (q.b + q.c * s2))); };
  double most = poly(top * top);
  auto see = [&](double s2) {
    if (s2 > 0. && s2 < top * top) most = fmax(most, poly(s2));
  };
  if (q.c != 0.) {
    const double disc = 9. * q.b * q.b - 20. * q.a * q.c;
    if (disc >= 0.) {
      see((-3. * q.b + sqrt(disc)) / (10. * q.c));
      see((-3. * q.b - sqrt(disc)) / (10. * q.c));
    }
  } else if (q.b != 0.) {
    see(-q.a / (3. * q.b));
  }
  return most;
}
// The exponent that brings values of up to `top` to between 1/2 and 1; those above stay, and NaN.
__host__ __device__ inline int lift(double top) { return !(top < 0.5) ? 0 : top < 0x1p-126 ? 126 : -ilogb(top) - 1; }

// A warp a row: X_0, scaled, as the sum of two fp16 numbers; and the exponents of the steps.  `shrinks`: the polynomial
// brings singular values of up to one below one half on its way.
template <typename T>
__global__ void __launch_bounds__(256) ns_scale_kernel(NsSource s, int m, int n, long ld, float eps, const double* partial, Split x,
                                                       unsigned char* shift, int steps, Quintic q, int shrinks) {
  ptx::let_next_start();
  ptx::wait_for_previous();
  const int lane = threadIdx.x & 31;
  static_assert(NORM_PARTS == 64, "two partial sums a lane");
  double total = partial[(long)blockIdx.y * NORM_PARTS + lane] + partial[(long)blockIdx.y * NORM_PARTS + 32 + lane];
  for (int o = 16; o > 0; o >>= 1) total += __shfl_xor_sync(0xFFFFFFFFu, total, o);
  // (a zero matrix stays zero without eps too; beyond fp32's range, or where it gets thin, the scale is two factors)
  const double norm = sqrt(total), start = norm / (norm + (double)eps);
  const bool plain = !(start < 0.5) && !shrinks;      // (NaN as well)
  const double whole = (total == 0. ? 0. : SX / (norm + (double)eps)) * (plain ? 1. : ldexp(1., lift(start)));
  const float first = whole > 0x1p90 ? 0x1p100f : whole < 0x1p-90 ? 0x1p-60f : 1.f, scale = (float)(whole / (double)first);
  if (blockIdx.x == 0 && threadIdx.x < 32) {
    shift += (long)blockIdx.y * SHIFTS;
    if (plain) {
      reinterpret_cast<uint32_t*>(shift)[lane] = 0;
    } else if (lane == 0) {
      double top = start;
      for (int k = 0; k <= steps; ++k) {
        shift[k] = (unsigned char)lift(top);
        top = largest(q, top);
      }
    }
  }
  const long size = (long)m * n;
  const T* in = (const T*)s.in + (s.offsets != nullptr ? s.offsets[blockIdx.y] : (long)blockIdx.y * size);
  const float* momentum = s.momentum != nullptr ? s.momentum + (long)blockIdx.y * size : nullptr;
  const float gs = s.grad_scale != nullptr ? *s.grad_scale : 1.f;
  const bool vec = n % 8 == 0 && (((uintptr_t)in | (uintptr_t)momentum) & 15) == 0;
  for (long row = (long)blockIdx.x * 8 + (threadIdx.x >> 5); row < m; row += (long)gridDim.x * 8) {
    const long from = row * n, to = ((long)blockIdx.y * m + row) * ld;
    if (vec) {
      for (int col = 8 * lane; col < n; col += 256) {
        float f[8];
        load8(in + from + col, f);
        if (momentum != nullptr) {
          float mom[8];
          load8(momentum + from + col, mom);
#pragma unroll
          for (int j = 0; j < 8; ++j) f[j] = look_ahead(s, f[j], gs, mom[j]);
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) f[j] = f[j] * first * scale;
        const uint4 h = to_halves(f);
        *reinterpret_cast<uint4*>(x.hi + to + col) = h;
        add_halves(f, h, -1.f);
        *reinterpret_cast<uint4*>(x.lo + to + col) = to_halves(f);
      }
    } else {
      for (int col = lane; col < n; col += 32) {
        float v = to_f(in[from + col]);
        if (momentum != nullptr) v = look_ahead(s, v, gs, momentum[from + col]);
        v = v * first * scale;
        const __half hi = __float2half_rn(v);
        x.hi[to + col] = hi;
        x.lo[to + col] = __float2half_rn(v - __half2float(hi));
      }
    }
  }
}

// ------------------------------------------------------------------ products

__device__ __forceinline__ void sts_u4(uint32_t addr, uint4 v) {
  asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}

__device__ __forceinline__ float power_of_two(int e) { return e < -126 ? 0.f : __int_as_float((e + 127) << 23); }
// What becomes of a product: k_acc * product + k_same * same; the last step's result times k_last.
struct Finish {
  float k_acc, k_same, k_last;
  Split same, out;                 // at the item's matrix
  long ld;
};
__device__ __forceinline__ Finish finish_of(const NsPlan& p, const NsItem& it) {
  Finish f;
  const int at = it.step & 1;
  if (it.kind == GRAM || it.kind == SQUARE) {
    f.ld = p.ldr;
    f.same = p.A;
    f.out = it.kind == GRAM ? p.A : p.B;
    // (A is that of 2^e X, B is X's)
    f.k_acc = it.kind == GRAM ? SA / (SX * SX) : p.c * (SB / (SA * SA)) * power_of_two(-4 * it.e);
    f.k_same = p.b * (SB / SA) * power_of_two(-2 * it.e);
  } else {
    f.ld = p.ldx;
    f.same = p.X[at];
    f.out = p.X[at ^ 1];
    const float to = it.kind == LAST ? 1.f / SX : power_of_two(it.e_next - it.e);
    f.k_acc = to / SB;
    f.k_same = p.a * to;
    f.k_last = power_of_two(-it.e);
  }
  const long off = (long)it.mat * it.m * f.ld;
  f.same.hi += off;
  f.same.lo += off;
  f.out.hi += off;
  f.out.lo += off;
  return f;
}
// A box's 16-byte pieces as a warp moves them: piece (lane & 3) of row 8 k + lane / 4.  Rows are whole groups of eight in
// memory: what lies past the last column is moved with it and used by nobody.
__device__ __forceinline__ uint32_t piece_at(uint32_t box, int r, int g) { return box + (uint32_t)(r * 64 + ((g ^ (r >> 1 & 3)) << 4)); }
struct Box { uint4 hi[4], lo[4]; };
__device__ __forceinline__ void fetch_box(Box& x, const Finish& f, const NsItem& it, int row0, int col0) {
  const int lane = threadIdx.x & 31, col = col0 + 8 * (lane & 3);
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const int row = row0 + 8 * k + (lane >> 2);
    if (it.kind == GRAM || row >= it.m || col >= it.n) continue;
    // (written by other blocks of this launch: from L2)
    x.hi[k] = __ldcg(reinterpret_cast<const uint4*>(f.same.hi + (long)row * f.ld + col));
    x.lo[k] = __ldcg(reinterpret_cast<const uint4*>(f.same.lo + (long)row * f.ld + col));
  }
}

// A box of the last step's result: from shared memory (row r of sizeof(T) * 32 bytes, 16-byte pieces xor-ed with the row)
// to the rows of X or of the parameters, a lane a column: any alignment, whole rows of the box an instruction.
template <typename T> __device__ __forceinline__ uint32_t result_at(uint32_t box, int r, int col) {
  constexpr int PER = 16 / sizeof(T), PIECES = 32 / PER;
  return box + (uint32_t)(r * 32 * (int)sizeof(T) + (((col / PER) ^ (PIECES == 4 ? r >> 1 & 3 : r & 7)) * 16) + col % PER * (int)sizeof(T));
}
template <typename T> __device__ __forceinline__ T lds_as(uint32_t addr);
template <> __device__ __forceinline__ float lds_as<float>(uint32_t addr) {
  float v;
  asm volatile("ld.shared.f32 %0, [%1];" : "=f"(v) : "r"(addr));
  return v;
}
template <> __device__ __forceinline__ bf16 lds_as<bf16>(uint32_t addr) { return __ushort_as_bfloat16(tch::lds_u16(addr)); }
// A parameter that Muon moves is rounded once: its share of X comes in fp32 (S).
template <typename T, typename S>
__device__ __forceinline__ void write_result(const NsPlan& p, const NsItem& it, uint32_t box, int row0, int col0) {
  const int lane = threadIdx.x & 31, rows = it.m - row0 < 32 ? it.m - row0 : 32;
  if (col0 + lane >= it.n) return;
  T* dst = (T*)p.result + (p.offsets != nullptr ? p.offsets[it.mat] : (long)it.mat * p.m * p.n) + (long)row0 * p.n + col0 + lane;
#pragma unroll 8
  for (int r = 0; r < 32; ++r) {
    if (r >= rows) break;
    const S x = lds_as<S>(result_at<S>(box, r, lane));
    if (p.muon) dst[(long)r * p.n] = from_f<T>(to_f(dst[(long)r * p.n]) * p.decay - p.lr * p.scale * to_f(x));
    else dst[(long)r * p.n] = from_f<T>(to_f(x));
  }
}

// All steps in one launch.  Blocks (or pairs) take items from a counter in the list's order; an item starts once the
// products it reads are finished (`done` of its matrix), which were handed out before it, so whoever waits, waits
// for someone who runs: no block has to be resident for another's sake, and launches may overlap.  With more than a
// few matrices the wait is over before it begins.
// Warp 3 of the even block takes items ahead of the others and waits until they may start, warps 0 and 2 load the
// two operands (one thread issues a stage's copies in about 1000 cycles, and a step's 1536 have two stages), warp 1
// issues the products (for both blocks), the others finish the rows: two accumulators, so a tile is finished under
// the next one's products.
template <typename T, bool PAIR>
__global__ void __launch_bounds__(THREADS, 1) ns_kernel(const __grid_constant__ NsMaps maps, const NsPlan p) {
  constexpr int EDGE = PAIR ? 256 : 128, BLOCKS = PAIR ? 2 : 1;
  constexpr bool SUMS = sizeof(T) == 4;              // fp32: four partial sums; else two accumulators in turn
  static_assert((SUMS ? 4 : 2) * EDGE <= 512, "tensor memory");
  static_assert(STAGES % 2 == 0, "high and low parts lie side by side");
  constexpr int sums = SUMS ? 1 : 2;
  extern __shared__ uint8_t raw[];
  __shared__ __align__(8) uint64_t full_bar[STAGES], empty_bar[STAGES], acc_full[2], acc_empty[2], tk_full[TICKETS], tk_empty[TICKETS], go[TICKETS];
  __shared__ NsSlot tk[TICKETS];
  __shared__ uint32_t tmem_slot;
  __shared__ int abort_flag;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const uint32_t rank = PAIR ? tch::cluster_ctarank() : 0;
  uint8_t* smem = (uint8_t*)(((uintptr_t)raw + 1023) & ~(uintptr_t)1023);
  uint8_t* sA = smem;
  uint8_t* sB = smem + STAGES * OPERAND_BYTES;
  if (tid == 0) {
    abort_flag = 0;
    for (int s = 0; s < STAGES; ++s) {
      ptx::mbar_init(&full_bar[s], 1);
      ptx::mbar_init(&empty_bar[s], 1);
    }
    for (int b = 0; b < 2; ++b) {
      ptx::mbar_init(&acc_full[b], 1);
      ptx::mbar_init(&acc_empty[b], BLOCKS * EPI_WARPS);
    }
    for (int k = 0; k < TICKETS; ++k) {
      ptx::mbar_init(&tk_full[k], 1);
      ptx::mbar_init(&go[k], 1);
      ptx::mbar_init(&tk_empty[k], 1 + BLOCKS * (EPI_WARPS + 2));   // products; rows and loads of both blocks
    }
    ptx::mbar_fence_init();
  }
  if (warp == 2 && lane < (int)(sizeof(NsMaps) / sizeof(CUtensorMap))) ptx::prefetch_tmap(reinterpret_cast<const CUtensorMap*>(&maps) + lane);
  if (warp == 1) {
    if constexpr (PAIR) {
      ptx::tmem_alloc_pair(&tmem_slot, 512);
      ptx::tmem_relinquish_pair();
    } else {
      ptx::tmem_alloc(&tmem_slot, 512);
      ptx::tmem_relinquish();
    }
  }
  ptx::tc_fence_before();
  __syncthreads();
  if constexpr (PAIR) tch::cluster_sync_all();
  ptx::tc_fence_after();
  const uint32_t tmem_base = tmem_slot;
  volatile int* abortp = &abort_flag;
  ptx::wait_for_previous();
  auto give_up = [&](int where) {
    abort_flag = 1;
    if constexpr (PAIR)
      asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(tch::mapa(ptx::smem_u32(&abort_flag), rank ^ 1u)), "r"(1) : "memory");
    report_timeout(p.status, KID_NEWTON_SCHULZ, where);
  };
  auto wait_for = [&](uint64_t* bar, int q) {         // item q's ticket or start (cluster-wide acquire: a pair's come from the even block)
    long spins = 0;
    unsigned long long t0 = 0;
    while (!(PAIR ? tch::mbar_try_wait_cluster(bar, (uint32_t)(q / TICKETS) & 1u) : ptx::mbar_try_wait(bar, (uint32_t)(q / TICKETS) & 1u))) {
      if (++spins > p.spin_limit * 8 || *abortp != 0) return false;
      if ((spins & 1023) == 0) {
        const unsigned long long now = ptx::globaltimer_ns();
        if (t0 == 0) t0 = now;
        else if (now - t0 > ptx::kWaitDeadlineNs) return false;
      }
    }
    return true;
  };
  auto free_ticket = [&](int q) {
    if constexpr (PAIR) ptx::mbar_arrive_cluster(tch::mapa(ptx::smem_u32(&tk_empty[q % TICKETS]), 0));
    else ptx::mbar_arrive(&tk_empty[q % TICKETS]);
  };

  auto finished = [&](NsSlot item) {                   // waits for the products an item reads
    const int want = needed(p, item) * BLOCKS * EPI_WARPS;
    long spins = 0;
    unsigned long long t0 = 0;
    while (ld_acquire_gpu(p.done + item.mat) < want) {
      __nanosleep(20);
      if (++spins > p.spin_limit || *abortp != 0) return false;
      if ((spins & 255) == 0) {
        const unsigned long long now = ptx::globaltimer_ns();
        if (t0 == 0) t0 = now;
        else if (now - t0 > ptx::kWaitDeadlineNs) return false;
      }
    }
    return true;
  };

  if (warp == 0 || warp == 2) {
    if (lane == 0) {
      const bool first = warp == 0;                   // operand A, or B
      uint8_t* const to = first ? sA : sB;
      const uint32_t bars = PAIR ? tch::mapa(ptx::smem_u32(full_bar), 0) : ptx::smem_u32(full_bar);
      uint32_t s = 0, ph = 0;
      long iteration = 0;
      for (int q = 0; abort_flag == 0; ++q) {
        const int k = q % TICKETS;
        if (!wait_for(&tk_full[k], q)) { give_up(0xFFFC); break; }
        const NsSlot slot = tk[k];
        if (slot.kind < 0) { free_ticket(q); break; }
        const NsItem it = item_of(p, slot);
        const int at = it.step & 1, form = first ? it.a_form : it.b_form;
        const int row0 = (first ? it.ti * EDGE : it.tj * it.columns) + 128 * (int)rank;
        const NsMap& map = it.kind == GRAM ? maps.x[at] : it.kind == SQUARE ? maps.a : first == (p.tall != 0) ? maps.x[at] : maps.b;
        auto claim = [&]() {                          // a stage to fill
          if (!ptx::mbar_wait(&empty_bar[s], ph ^ 1u, p.spin_limit, abortp)) return false;
          if (first && rank == 0) ptx::mbar_arrive_expect_tx(&full_bar[s], BLOCKS * OPERAND_BYTES + (uint32_t)it.columns * (BK * 2));
          return true;
        };
        bool claimed = claim(), ok = true;            // the first one before the item may start
        if (!claimed) { give_up(0xFFF9); break; }
        if (!wait_for(&go[k], q)) { give_up(0xFFF8); break; }
        free_ticket(q);                               // (not before: the start of the slot's next item would hide this one's)
        ptx::fence_proxy_async_global();              // written by other blocks, read here by TMA
        const int stages = 2 * ((it.K + BK - 1) / BK);   // high parts, low parts
        for (int i = 0; i < stages; ++i, ++iteration) {
          const int k0 = (i >> 1) * BK, low = i & 1;
          if (!claimed && !claim()) { give_up(k0); ok = false; break; }
          claimed = false;
          const bool mn = mn_major(form, row0, k0, EDGE);
          const uint32_t bar = bars + 8 * s;
          if (!(iteration == p.stall && blockIdx.x == 0)) {
            uint8_t* dst = to + s * OPERAND_BYTES;
            auto copy = [&](uint8_t* d, const CUtensorMap* m, int x, int y) {
              if constexpr (PAIR) ptx::tma_load_3d_pair(d, m, x, y, it.mat, bar);
              else tch::tma_load_3d(d, m, x, y, it.mat, &full_bar[s]);
            };
            if (!PAIR && !first && it.columns == 64) {
              copy(dst, &map.block[low], mn ? row0 : k0, mn ? k0 : row0);
            } else if (mn) {
              copy(dst, &map.block[low], row0, k0);
              copy(dst + BLOCK_BYTES, &map.block[low], row0 + 64, k0);
            } else {
              copy(dst, &map.rows[low], k0, row0);
            }
          }
          if (++s == STAGES) { s = 0; ph ^= 1u; }
        }
        if (!ok) break;
      }
    }
    __syncwarp();
  } else if (warp == 3) {
    if (lane == 0 && rank == 0) {
      for (int q = 0; abort_flag == 0; ++q) {
        const int k = q % TICKETS;
        if (!ptx::mbar_wait(&tk_empty[k], ((uint32_t)(q / TICKETS) & 1u) ^ 1u, p.spin_limit * 8, abortp)) { give_up(0xFFFB); break; }
        const int index = atomicAdd(p.ticket, 1);
        NsSlot slot{-1, 0, 0, 0};
        if (index < p.total) slot = slot_of(p, index);
        tk[k] = slot;
        ptx::mbar_arrive(&tk_full[k]);
        if constexpr (PAIR) {
          asm volatile("st.shared::cluster.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(tch::mapa(ptx::smem_u32(&tk[k]), 1)), "r"(slot.kind),
                       "r"(slot.mat), "r"(slot.tile), "r"(slot.step) : "memory");
          ptx::mbar_arrive_cluster(tch::mapa(ptx::smem_u32(&tk_full[k]), 1));
        }
        if (slot.kind < 0) break;
        if (!finished(slot)) { give_up(0xFFFA); break; }
        ptx::mbar_arrive(&go[k]);
        if constexpr (PAIR) ptx::mbar_arrive_cluster(tch::mapa(ptx::smem_u32(&go[k]), 1));
      }
    }
    __syncwarp();
  } else if (warp == 1) {
    if (lane == 0 && rank == 0) {
      uint32_t s = 0, ph = 0;
      bool ready = false, ok = true;
      for (int q = 0; ok; ++q) {
        if (!wait_for(&tk_full[q % TICKETS], q)) { give_up(0xFFFD); break; }
        const NsSlot slot = tk[q % TICKETS];
        free_ticket(q);
        if (slot.kind < 0) break;
        const NsItem it = item_of(p, slot);
        const int m0 = it.ti * EDGE, n0 = it.tj * it.columns / EDGE * EDGE;
        const int b = q % sums;
        if (!ptx::mbar_wait(&acc_empty[b], ((uint32_t)(q / sums) & 1u) ^ 1u, p.spin_limit * 8, abortp)) { give_up(0xFFFE); break; }
        ptx::tc_fence_after();
        // high x high, high x low, low x high, from two stages
        for (int k0 = 0, i = 0; k0 < it.K && ok;) {
          // the stretch of K in which both operands keep their form: an upper matrix changes at the diagonal
          int end = it.K;
          if (it.a_form == UPPER && k0 < m0) end = m0;
          if (it.b_form == UPPER && k0 < n0 && n0 < end) end = n0;
          const bool a_mn = mn_major(it.a_form, m0, k0, EDGE), b_mn = mn_major(it.b_form, n0, k0, EDGE);
          const uint32_t idesc = ptx::umma_idesc_f16(EDGE, PAIR ? EDGE : it.columns) | (a_mn ? 1u << 15 : 0u) | (b_mn ? 1u << 16 : 0u);
          const uint64_t a_step = a_mn ? 128 : 2, b_step = b_mn ? 128 : 2;
          const uint64_t da0 = a_mn ? ptx::umma_desc_mn_sw128(ptx::smem_u32(sA), BLOCK_BYTES) : ptx::umma_desc_k_sw128(ptx::smem_u32(sA));
          const uint64_t db0 = b_mn ? ptx::umma_desc_mn_sw128(ptx::smem_u32(sB), BLOCK_BYTES) : ptx::umma_desc_k_sw128(ptx::smem_u32(sB));
          for (; k0 < end; k0 += BK, ++i) {
            if (!ready && !ptx::mbar_wait(&full_bar[s], ph, p.spin_limit, abortp)) { give_up(i); ok = false; break; }
            const uint32_t low = s + 1;                 // (stages are even in number)
            const uint32_t next = low + 1 == STAGES ? 0 : low + 1, next_ph = ph ^ (next == 0 ? 1u : 0u);
            const uint64_t da = da0 + (uint64_t)(s * (OPERAND_BYTES / 16)), db = db0 + (uint64_t)(s * (OPERAND_BYTES / 16));
            const uint64_t da_low = da + OPERAND_BYTES / 16, db_low = db + OPERAND_BYTES / 16;
            const uint32_t large = tmem_base + (uint32_t)((SUMS ? i % 3 : b) * EDGE), small = tmem_base + (uint32_t)((SUMS ? 3 : b) * EDGE);
            const uint32_t large_on = i < (SUMS ? 3 : 1) ? 0u : 1u, small_on = SUMS && i == 0 ? 0u : 1u;
            auto products = [&](auto free, uint32_t sum, uint64_t x, uint64_t y, uint32_t on, uint32_t test, uint32_t test_ph) {
              constexpr bool FREE = decltype(free)::value;
              if constexpr (PAIR) return ptx::umma_stage_pair<FREE>(sum, x, y, a_step, b_step, idesc, on, &empty_bar[s], &full_bar[test], test_ph);
              else return ptx::umma_stage<FREE>(sum, x, y, a_step, b_step, idesc, on, &empty_bar[s], &full_bar[test], test_ph);
            };
            if (!products(std::false_type(), large, da, db, large_on, low, ph) &&
                !ptx::mbar_wait(&full_bar[low], ph, p.spin_limit, abortp)) { give_up(i); ok = false; break; }
            products(std::false_type(), small, da, db_low, small_on, next, next_ph);
            ready = products(std::true_type(), small, da_low, db, 1u, next, next_ph);
            if constexpr (PAIR) ptx::umma_commit_pair(&empty_bar[low], 3);
            else ptx::umma_commit(&empty_bar[low]);
            s = next;
            ph = next_ph;
          }
        }
        if (ok) {
          if constexpr (PAIR) ptx::umma_commit_pair(&acc_full[b], 3);
          else ptx::umma_commit(&acc_full[b]);
        }
      }
    }
    __syncwarp();
  } else {
    // warp w may read TMEM lanes [32 (w % 4), +32); the two warps of a quarter split the tile's columns
    const int quarter = warp & 3, mine = warp - 4, half = mine >> 2;
    const uint32_t buffer = ptx::smem_u32(smem) + STAGES * 2 * OPERAND_BYTES + (uint32_t)(mine * BUFFER_BYTES);
    for (int q = 0;; ++q) {
      bool ok = __all_sync(0xFFFFFFFFu, wait_for(&tk_full[q % TICKETS], q) && 32 * q + warp != p.leave), end = false;
      NsItem it;
      Finish fin;
      Box same;
      int b = 0, row0 = 0, col0 = 0;
      if (ok) {
        const NsSlot slot = tk[q % TICKETS];
        __syncwarp();
        end = slot.kind < 0;
        if (!end) {
          it = item_of(p, slot);
          b = q % sums;
          row0 = it.ti * EDGE + 128 * (int)rank + quarter * 32;
          col0 = it.tj * it.columns + half * (it.columns / 2);
          fin = finish_of(p, it);
          ok = __all_sync(0xFFFFFFFFu, it.kind == GRAM || wait_for(&go[q % TICKETS], q));
        }
        if (lane == 0) free_ticket(q);
        if (ok && !end) {
          fetch_box(same, fin, it, row0, col0);        // under the products
          ok = ptx::mbar_wait(&acc_full[b], (uint32_t)(q / sums) & 1u, p.spin_limit * 8, abortp);
        }
      }
      if (!ok && abort_flag == 0) give_up(0xFFFF);
      // One verdict for all of them, at the end too: a warp that gave up there would wait for those that have left.
      uint32_t stop;
      asm volatile(
          "{\n\t.reg .pred pp, qq;\n\t"
          "setp.ne.b32 pp, %1, 0;\n\t"
          "bar.red.or.pred qq, 1, %2, pp;\n\t"
          "selp.b32 %0, 1, 0, qq;\n\t}"
          : "=r"(stop)
          : "r"((uint32_t)(!ok || end || abort_flag != 0)), "n"(32 * EPI_WARPS)
          : "memory");
      if (stop) break;
      ptx::tc_fence_after();
      const uint32_t tsrc = tmem_base + ((uint32_t)(quarter * 32) << 16) + (uint32_t)(b * EDGE + half * (it.columns / 2));
      const int nk = (it.K + BK - 1) / BK, boxes = it.columns / 64;
#pragma unroll 1
      for (int c = 0; c < boxes; ++c) {
        uint32_t r[32];
        ptx::tmem_ld32(tsrc + (uint32_t)(c * 32), r);
        const int col = col0 + c * 32;
        if (it.kind != GRAM) {                        // `same`, from the lanes that fetched it to the rows' lanes
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const uint32_t at = piece_at(buffer, 8 * k + (lane >> 2), lane & 3);
            sts_u4(at, same.hi[k]);
            sts_u4(at + BOX_BYTES, same.lo[k]);
          }
          __syncwarp();
          if (c + 1 < boxes) fetch_box(same, fin, it, row0, col + 32);
        }
        ptx::tmem_ld_wait();
        for (int sum = 1; sum < (SUMS ? 4 : 1); ++sum) {
          if (sum < 3 && sum >= nk) continue;
          uint32_t more[32];
          ptx::tmem_ld32(tsrc + (uint32_t)(sum * EDGE + c * 32), more);
          ptx::tmem_ld_wait();
#pragma unroll
          for (int j = 0; j < 32; ++j) r[j] = __float_as_uint(__uint_as_float(r[j]) + __uint_as_float(more[j]));
        }
        if (c == boxes - 1) {                            // the accumulator is free again
          ptx::tc_fence_before();
          __syncwarp();
          if (lane == 0) {
            if constexpr (PAIR) ptx::mbar_arrive_cluster(tch::mapa(ptx::smem_u32(&acc_empty[b]), 0));
            else ptx::mbar_arrive(&acc_empty[b]);
          }
        }
        if (row0 >= it.m || col >= it.n) continue;
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          float f[8];
#pragma unroll
          for (int j = 0; j < 8; ++j) f[j] = fin.k_acc * __uint_as_float(r[8 * g + j]);
          const uint32_t piece = piece_at(buffer, lane, g);
          if (it.kind != GRAM) {
            add_halves(f, tch::lds_u4(piece), fin.k_same);
            add_halves(f, tch::lds_u4(piece + BOX_BYTES), fin.k_same);
          }
          if (it.kind == LAST) {
#pragma unroll
            for (int j = 0; j < 8; ++j) r[8 * g + j] = __float_as_uint(f[j] * fin.k_last);
            continue;
          }
          const uint4 h = to_halves(f);
          sts_u4(piece, h);
          add_halves(f, h, -1.f);
          sts_u4(piece + BOX_BYTES, to_halves(f));
        }
        __syncwarp();
        if (it.kind == LAST) {
          auto leave = [&](auto as) {
            typedef decltype(as) S;
#pragma unroll
            for (int j = 0; j < 32; j += 16 / (int)sizeof(S)) {
              alignas(16) S x[16 / sizeof(S)];
#pragma unroll
              for (int k = 0; k < (int)(16 / sizeof(S)); ++k) x[k] = from_f<S>(__uint_as_float(r[j + k]));
              sts_u4(result_at<S>(buffer, lane, j), *reinterpret_cast<const uint4*>(x));
            }
            __syncwarp();
            write_result<T, S>(p, it, buffer, row0, col);
          };
          if (p.muon) leave(0.f);
          else leave(T());
        } else {
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const int row = row0 + 8 * k + (lane >> 2), to = col + 8 * (lane & 3);
            if (row >= it.m || to >= it.n) continue;
            const uint32_t at = piece_at(buffer, 8 * k + (lane >> 2), lane & 3);
            *reinterpret_cast<uint4*>(fin.out.hi + (long)row * fin.ld + to) = tch::lds_u4(at);
            *reinterpret_cast<uint4*>(fin.out.lo + (long)row * fin.ld + to) = tch::lds_u4(at + BOX_BYTES);
          }
        }
        __syncwarp();
      }
      if (it.kind != LAST && lane == 0) red_release_gpu_add(p.done + it.mat, 1);
    }
  }
  if (abort_flag != 0)
    for (int i = 0; i < 2000; ++i) __nanosleep(100);   // copies in flight land before the shared memory goes
  ptx::tc_fence_before();
  __syncthreads();
  if constexpr (PAIR) {
    tch::cluster_sync_all();                           // the pair's MMAs read both blocks' operands
    if (warp == 1) ptx::tmem_dealloc_pair(tmem_base, 512);
  } else {
    if (warp == 1) ptx::tmem_dealloc(tmem_base, 512);
  }
}

// ------------------------------------------------------------------ host

long padded(long x) { return (x + 7) / 8 * 8; }       // rows start on 16 bytes

struct NsBuffers {
  Split X[2], A, B;
  double* partial;
  int* ticket;
  int* done;
  unsigned char* shift;
  long ldx, ldr;
  size_t bytes;
};
NsBuffers carve(void* ws, int count, int m, int n) {
  NsBuffers b{};
  char* base = (char*)ws;
  size_t off = 0;
  auto take = [&](size_t bytes) {
    void* p = base + off;
    off += (bytes + 255) / 256 * 256;
    return p;
  };
  const int r = m < n ? m : n;
  b.ldx = padded(n);
  b.ldr = padded(r);
  const size_t x = (size_t)count * m * b.ldx * 2, a = (size_t)count * r * b.ldr * 2;
  for (int k = 0; k < 2; ++k) {
    b.X[k].hi = (__half*)take(x);
    b.X[k].lo = (__half*)take(x);
  }
  b.A.hi = (__half*)take(a);
  b.A.lo = (__half*)take(a);
  b.B.hi = (__half*)take(a);
  b.B.lo = (__half*)take(a);
  b.partial = (double*)take((size_t)count * NORM_PARTS * sizeof(double));
  b.ticket = (int*)take(sizeof(int));
  b.done = (int*)take((size_t)count * sizeof(int));
  b.shift = (unsigned char*)take((size_t)count * SHIFTS);
  b.bytes = off;
  return b;
}

// The largest singular value that `steps` applications make of values in [0, 1], and the largest |B|: both
// have to stay inside fp16's range at their scales.
bool stays_in_range(int steps, Quintic q) {
  double top = 1.;
  for (int k = 0; k < steps; ++k) {
    auto inner = [&](double s2) { return fabs(s2 * (q.b + q.c * s2)); };
    const double most = largest(q, top), turn = q.c != 0. ? -q.b / (2. * q.c) : 0.;
    const double most_b = turn > 0. && turn < top * top ? fmax(inner(top * top), inner(turn)) : inner(top * top);
    if (!(most_b <= 60.) || !(most <= 3.5)) return false;
    top = most;
  }
  return true;
}
bool shrinks(int steps, Quintic q) {
  double top = 1.;
  for (int k = 0; k < steps; ++k)
    if ((top = largest(q, top)) < 0.5) return true;
  return false;
}

// Pairs make four times the tile of a single block with half as many units.  Measured, us: a step along K (three products)
// 1.32 in pairs and 0.95 in single blocks where tiles follow one another, 0.5 and 1.5 a tile on top; where a matrix's products
// wait for one another a step 0.9 and 0.7 and a product 9.8 and 5.9 more.  The smaller of the two times is covered by the
// other but for a fifth.  Single blocks also waste fewer rows of ragged matrices.
// 18 x 1280 x 1280 takes 1.79 ms in pairs and 2.31 in single blocks, 4 x 1280 x 1280 484 us and 572, 3 x 1280 x 1280 459 and 461,
// 6 x 640 x 1280 363 and 273, 18 x 512 x 512 282 and 217, 2 x 200 x 9000 869 and 617, 1 x 2048 x 2048 690 and 610.
bool pays_as_pairs(const NsPlan& p) {
  auto cost = [&](int edge, int units, double stage, double tile, double alone, double latency) {     // of a step
    const double side = (p.r + edge - 1) / edge, q = p.tall ? p.m : p.n, k_gram = ceil(q / BK), k = ceil((double)p.r / BK);
    const double tri = p.count * side * (side + 1) / 2 / units, all = p.count * side * ceil(q / edge) / units;
    const double busy = tri * (k_gram * stage + tile) + (tri + all) * (k * stage + tile), chain = (k_gram + 2 * k) * alone + 3 * latency;
    return fmax(busy, chain) + 0.2 * fmin(busy, chain);
  };
  return cost(256, 74, 1.32, 0.5, 0.9, 9.8) < cost(128, 148, 0.95, 1.5, 0.7, 5.9);
}
bool as_pairs(int dtype, const NsPlan& p) { return dtype == ELMAN_BF16 && pays_as_pairs(p); }
// Tiles of the blocks (i, j >= i) of a symmetric product.
int triangle_of(int r, int edge, int columns) {
  const int per = edge / columns, strips = (r + columns - 1) / columns, whole = strips / per;
  return per * (whole * (whole + 1) / 2) + strips % per * (whole + 1);
}
// Single blocks: tiles of 64 columns where they spread a product over more of the device.  From start to end they take
// 8700 cycles and 1270 a step along K, tiles of 128 columns 11300 and 1330 (measured): 1 x 256 x 256 109 us against 131,
// 4 x 512 x 512 156 and 176; but 18 x 512 x 512 309 and 217.
int columns_of(const NsPlan& p, int wide, int narrow, int stages) {
  auto cost = [&](int tiles, double stage, double tile) { return ceil((double)tiles * p.count / 148) * (stage * stages + tile); };
  return cost(narrow, 1270, 8700) < cost(wide, 1330, 11300) ? 64 : 128;
}

template <typename T, bool PAIR>
int launch(const NsMaps& maps, const NsPlan& p, cudaStream_t st) {
  static std::mutex mutex;
  static bool sized[64];
  int dev = 0;
  ELMAN_CUDA_CHECK(cudaGetDevice(&dev));
  {
    std::lock_guard<std::mutex> lock(mutex);
    if (dev >= 64 || !sized[dev]) {
      ELMAN_CUDA_CHECK(cudaFuncSetAttribute(ns_kernel<T, PAIR>, cudaFuncAttributeMaxDynamicSharedMemorySize, NS_SMEM));
      if (dev < 64) sized[dev] = true;
    }
  }
  // no more than a product's tiles: the next products run where code and tensor maps are warm
  const int blocks = PAIR ? 2 : 1, most = p.count * (p.triangle > p.all ? p.triangle : p.all);
  const int units = most < 148 / blocks ? most : 148 / blocks;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)(blocks * units));
  cfg.blockDim = dim3(THREADS);
  cfg.dynamicSmemBytes = NS_SMEM;
  cfg.stream = st;
  cudaLaunchAttribute attrs[2];
  attrs[0] = after_its_start();
  attrs[1].id = cudaLaunchAttributeClusterDimension;
  attrs[1].val.clusterDim.x = blocks;
  attrs[1].val.clusterDim.y = attrs[1].val.clusterDim.z = 1;
  cfg.attrs = attrs;
  cfg.numAttrs = PAIR ? 2 : 1;
  ELMAN_CUDA_CHECK(cudaLaunchKernelEx(&cfg, ns_kernel<T, PAIR>, maps, p));
  count_launch(true);
  return ELMAN_OK;
}

template <typename T>
int run(const NewtonSchulzArgs& g, const NsSource& src, NsPlan p, cudaStream_t st) {
  const NsBuffers buf = carve(g.workspace, g.count, g.m, g.n);
  p.count = g.count; p.m = g.m; p.n = g.n; p.tall = g.m > g.n;
  p.r = p.tall ? g.n : g.m;
  p.steps = g.steps;
  p.a = g.a; p.b = g.b; p.c = g.c;
  const Quintic quintic{g.a, g.b, g.c};
  p.X[0] = buf.X[0]; p.X[1] = buf.X[1]; p.A = buf.A; p.B = buf.B;
  p.ldx = buf.ldx; p.ldr = buf.ldr;
  p.ticket = buf.ticket; p.done = buf.done; p.shift = buf.shift;
  p.status = device_status_ptr();
  p.spin_limit = options().spin_limit;
  p.stall = (int)options().test_stall_step;
  p.leave = (int)options().test_leave_warp;
  const bool pair = as_pairs(g.dtype, p);
  const int edge = pair ? 256 : 128;
  p.edge = p.n_sym = p.n_upd = edge;
  const int upd_rows = (p.m + edge - 1) / edge;
  if (!pair) {
    const int gram = ((p.tall ? p.m : p.n) + BK - 1) / BK, inner = (p.r + BK - 1) / BK;
    p.n_sym = columns_of(p, triangle_of(p.r, 128, 128), triangle_of(p.r, 128, 64), (gram + inner) / 2);
    p.n_upd = columns_of(p, upd_rows * ((p.n + 127) / 128), upd_rows * ((p.n + 63) / 64), inner);
  }
  p.triangle = triangle_of(p.r, edge, p.n_sym);
  p.all = upd_rows * ((p.n + p.n_upd - 1) / p.n_upd);
  const double total = (double)p.steps * p.count * (2. * p.triangle + p.all);
  ELMAN_ARG_CHECK(total + 1024 < (double)(1L << 31), "matrices too large");
  p.per_step = p.count * (2 * p.triangle + p.all);
  p.total = p.steps * p.per_step;
  NsMaps maps;
  auto map = [&](NsMap& out, const Split& x, int rows, int cols, long ld) {
    for (int low = 0; low < 2; ++low) {
      const __half* base = low ? x.lo : x.hi;
      const uint64_t all = (uint64_t)rows * ld;
      ELMAN_RETURN_IF(make_tmap_f16(&out.rows[low], base, cols, rows, p.count, ld, all, 128));
      ELMAN_RETURN_IF(make_tmap_f16(&out.block[low], base, cols, rows, p.count, ld, all, 64));
    }
    return (int)ELMAN_OK;
  };
  ELMAN_RETURN_IF(map(maps.x[0], buf.X[0], p.m, p.n, buf.ldx));
  ELMAN_RETURN_IF(map(maps.x[1], buf.X[1], p.m, p.n, buf.ldx));
  ELMAN_RETURN_IF(map(maps.a, buf.A, p.r, p.r, buf.ldr));
  ELMAN_RETURN_IF(map(maps.b, buf.B, p.r, p.r, buf.ldr));
  const long size = (long)p.m * p.n, blocks = (p.m + 7) / 8;
  ns_norm_kernel<T><<<dim3(NORM_PARTS, p.count), 256, 0, st>>>(src, size, buf.partial, buf.ticket, buf.done);
  count_launch(false);
  cudaLaunchAttribute attr = after_its_start();
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)(blocks < 1024 ? blocks : 1024), p.count);
  cfg.blockDim = dim3(256);
  cfg.stream = st;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  ELMAN_CUDA_CHECK(cudaLaunchKernelEx(&cfg, ns_scale_kernel<T>, src, p.m, p.n, buf.ldx, g.eps, (const double*)buf.partial, buf.X[0],
                                     buf.shift, p.steps, quintic, (int)shrinks(p.steps, quintic)));
  count_launch(false);
  ELMAN_CUDA_CHECK(cudaGetLastError());
  if constexpr (sizeof(T) == 2)
    if (pair) return launch<T, true>(maps, p, st);
  return launch<T, false>(maps, p, st);
}

}  // namespace

size_t newton_schulz_workspace(int, int count, int m, int n) { return carve(nullptr, count, m, n).bytes; }
int newton_schulz_tile(int dtype, int count, int m, int n) {
  NsPlan p{};
  p.count = count; p.m = m; p.n = n; p.tall = m > n; p.r = p.tall ? n : m;
  return as_pairs(dtype, p) ? 256 : 128;
}
bool newton_schulz_in_range(int steps, float a, float b, float c) { return stays_in_range(steps, Quintic{a, b, c}); }

int newton_schulz(const NewtonSchulzArgs& a, cudaStream_t st) {
  NsSource src{};
  src.in = a.in;
  NsPlan p{};
  p.result = a.out;
  return a.dtype == ELMAN_F32 ? run<float>(a, src, p, st) : run<bf16>(a, src, p, st);
}

int muon_step(const NewtonSchulzArgs& a, const MuonArgs& u, cudaStream_t st) {
  NsSource src{};
  src.in = u.grads;
  src.offsets = u.offsets;
  src.momentum = u.momentum;
  src.mu = u.mu;
  src.nesterov = u.nesterov;
  src.grad_scale = u.grad_scale;
  NsPlan p{};
  p.result = u.params;
  p.offsets = u.offsets;
  p.muon = 1;
  p.lr = u.lr;
  p.decay = 1.f - u.lr * u.weight_decay;
  p.scale = u.scale;
  return a.dtype == ELMAN_F32 ? run<float>(a, src, p, st) : run<bf16>(a, src, p, st);
}

}  // namespace elman
