// Orthogonalising matrices by Newton-Schulz products, and the Muon update built on it:
//   X = G / (|G|_F + eps);  steps times:  A = X X^T,  B = b A + c A A,  X <- a X + B X
// (tall matrices: A = X^T X and X <- a X + X B, so that A has the smaller of the two extents, r).
// A and B are symmetric: only the tiles on and above the diagonal are computed and stored.  Per step 3 r^2 q + r^3 flops with q the larger extent: bound by the tensor cores.
//
// Numbers.  The operands are fp16 (11 significant bits; bf16 has 8), scaled by powers of two into its
// range: X by 2^12, A by 2^12, B by 2^10; every sum is fp32.  The polynomial multiplies small singular
// values by a (3.44) a step, and with them what rounding X puts into their directions: a gradient with a
// few strong directions above noise comes out 1.1e-2 off with X in fp16 alone (8e-2 in bf16).  So X is kept
// as the sum of two fp16 numbers, and the term a X takes both, in all but the last two steps: 7e-4.  Near the end
// the polynomial's slope is small and rounding a X and B X alike is what keeps the error small.
// fp32 matrices take both parts of X, A and B into the products as well (three products for one): 5e-6.  The tensor
// cores cut their fp32 sums off rather than rounding them, which over a long contraction adds up (2.5e-5 at
// 33 x 2000 with one sum): there the large products take turns in three sums and the small ones have a fourth.
#include <math.h>

#include <mutex>

#include "common.cuh"
#include "sm100_ptx.cuh"
#include "tc_helpers.cuh"

#include <cuda_fp16.h>

namespace elman {

namespace {

constexpr int TILE = 128, BK = 64, STAGES = 3;
constexpr int BLOCK_BYTES = 64 * BK * 2;              // one TMA box: 64 x 64 fp16
constexpr int OPERAND_BYTES = TILE * BK * 2;
constexpr int NS_SMEM = STAGES * 2 * OPERAND_BYTES + 1024;
constexpr float SX = 4096.f, SA = 4096.f, SB = 1024.f;
constexpr int NORM_PARTS = 64;                        // partial sums of squares a matrix

enum Product { GRAM, SQUARE, UPDATE, LAST };
// An operand block of rows x K: stored [rows, K]; stored [K, rows] and read MN-major in place; or part of a
// symmetric matrix of which only the tiles on and above the diagonal are stored: below it the block is the
// mirrored one, read MN-major.
enum Form { ROWS_K, K_ROWS, UPPER };
__device__ __forceinline__ bool mn_major(int form, int row0, int k0) {
  return form == K_ROWS || (form == UPPER && row0 / TILE > k0 / TILE);
}

struct Split { __half* hi; __half* lo; };             // lo may be null

// The matrix a step starts from: G, or Muon's momentum-weighted gradient.
struct NsSource {
  const void* in;            // [count, m, n], or the flat gradients
  const long long* offsets;  // Muon: where each matrix starts in the flat buffers (device); null: dense
  float* momentum;           // Muon: [count, m, n]
  float mu;
  int nesterov;
  const float* grad_scale;   // device, or null
};

struct NsParams {
  int kind, m, n;            // extents of the output
  int K, parts;              // contraction extent; 1, or 3 products of high and low parts
  int a_form, b_form;        // how an operand lies in memory: Form
  int symmetric;
  long ld;                   // row stride of the fp16 output (and of `same`)
  long stride;               // elements between matrices of the output (and of `same`)
  float k_acc, k_same;       // output = k_acc * product + k_same * same
  Split same, out;
  void* result;              // LAST: [count, m, n], or the flat parameters
  const long long* offsets;
  int muon;
  float lr, decay, scale;    // Muon: p = p decay - lr scale X
  int* status;
  long spin_limit;
  int stall;
};

__device__ __forceinline__ void split_half(float v, __half& hi, __half& lo) {
  hi = __float2half_rn(v);
  lo = __float2half_rn(v - __half2float(hi));
}

// ------------------------------------------------------------------ start: norm and scaling

template <typename T> __device__ __forceinline__ float source_at(const NsSource& s, long at, long dense, float gs, bool advance) {
  float g = to_f(((const T*)s.in)[at]);
  if (s.momentum == nullptr) return g;
  g *= gs;
  float mom = s.momentum[dense];
  if (advance) {
    mom += (1.f - s.mu) * (g - mom);
    s.momentum[dense] = mom;
  }
  return s.nesterov ? g + s.mu * (mom - g) : mom;
}

// Sums of squares in fp64: a sum over millions of elements, of numbers whose squares leave fp32's range.
template <typename T>
__global__ void __launch_bounds__(256) ns_norm_kernel(NsSource s, long size, double* partial) {
  const long base = s.offsets != nullptr ? s.offsets[blockIdx.y] : (long)blockIdx.y * size;
  const float gs = s.grad_scale != nullptr ? *s.grad_scale : 1.f;
  double sum = 0.;
  for (long e = (long)blockIdx.x * 256 + threadIdx.x; e < size; e += NORM_PARTS * 256) {
    const double v = source_at<T>(s, base + e, (long)blockIdx.y * size + e, gs, true);
    sum += v * v;
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

template <typename T>
__global__ void __launch_bounds__(256) ns_scale_kernel(NsSource s, int m, int n, long ld, float eps, const double* partial, Split x) {
  __shared__ double total;
  if (threadIdx.x == 0) {
    double t = 0.;
    for (int k = 0; k < NORM_PARTS; ++k) t += partial[(long)blockIdx.y * NORM_PARTS + k];
    total = t;
  }
  __syncthreads();
  const float scale = (float)(SX / (sqrt(total) + (double)eps));
  const float gs = s.grad_scale != nullptr ? *s.grad_scale : 1.f;
  const long size = (long)m * n, base = s.offsets != nullptr ? s.offsets[blockIdx.y] : (long)blockIdx.y * size;
  const long to = (long)blockIdx.y * m * ld;
  for (long e = (long)blockIdx.x * 256 + threadIdx.x; e < size; e += (long)gridDim.x * 256) {
    const long row = e / n, col = e - row * n;
    __half hi, lo;
    split_half(source_at<T>(s, base + e, (long)blockIdx.y * size + e, gs, false) * scale, hi, lo);
    x.hi[to + row * ld + col] = hi;
    if (x.lo != nullptr) x.lo[to + row * ld + col] = lo;
  }
}

// ------------------------------------------------------------------ products

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
// Eight adjacent values of the result: X, or the parameters moved by it.
template <typename T> __device__ __forceinline__ void store8(const NsParams& p, T* dst, const float (&f)[8], int cols) {
  if (cols >= 8 && ((uintptr_t)dst & 15) == 0) {
    uint4 x[sizeof(T) / 2];
    T* v = reinterpret_cast<T*>(x);
    if (p.muon) {
#pragma unroll
      for (int q = 0; q < (int)sizeof(T) / 2; ++q) x[q] = reinterpret_cast<const uint4*>(dst)[q];
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = from_f<T>(p.muon ? to_f(v[j]) * p.decay - p.lr * p.scale * f[j] : f[j]);
#pragma unroll
    for (int q = 0; q < (int)sizeof(T) / 2; ++q) reinterpret_cast<uint4*>(dst)[q] = x[q];
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (j < cols) dst[j] = from_f<T>(p.muon ? to_f(dst[j]) * p.decay - p.lr * p.scale * f[j] : f[j]);
  }
}

// 32 columns of one output row as they come out of tensor memory.  Rows of the fp16 matrices are whole groups of
// eight: what lies past the last column is written with it and read by nobody.
template <typename T>
__device__ __forceinline__ void finish_row(const NsParams& p, int mat, int row, int col0, const uint32_t (&r)[32]) {
  if (row >= p.m) return;
  const long at = (long)mat * p.stride + (long)row * p.ld + col0;
  uint4 hi[4], lo[4];
#pragma unroll
  for (int g = 0; g < 4; ++g) {
    hi[g] = lo[g] = make_uint4(0, 0, 0, 0);
    if (p.kind != GRAM && col0 + 8 * g < p.n) {
      hi[g] = *reinterpret_cast<const uint4*>(p.same.hi + at + 8 * g);
      if (p.same.lo != nullptr) lo[g] = *reinterpret_cast<const uint4*>(p.same.lo + at + 8 * g);
    }
  }
#pragma unroll
  for (int g = 0; g < 4; ++g) {
    const int cols = p.n - col0 - 8 * g;
    if (cols <= 0) break;
    float f[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) f[j] = p.k_acc * __uint_as_float(r[8 * g + j]);
    add_halves(f, hi[g], p.k_same);
    add_halves(f, lo[g], p.k_same);
    if (p.kind == LAST) {
      store8(p, (T*)p.result + (p.offsets != nullptr ? p.offsets[mat] : (long)mat * p.m * p.n) + (long)row * p.n + col0 + 8 * g,
             f, cols);
      continue;
    }
    const uint4 h = to_halves(f);
    *reinterpret_cast<uint4*>(p.out.hi + at + 8 * g) = h;
    if (p.out.lo != nullptr) {
      add_halves(f, h, -1.f);
      *reinterpret_cast<uint4*>(p.out.lo + at + 8 * g) = to_halves(f);
    }
  }
}

// One block: one 128 x 128 tile.  Thread 0 of warp 0 loads, thread 0 of warp 1 issues the products, all
// four warps finish the rows.
template <typename T>
__global__ void __launch_bounds__(128, 2)
ns_product_kernel(const __grid_constant__ CUtensorMap tAh, const __grid_constant__ CUtensorMap tAl,
                  const __grid_constant__ CUtensorMap tBh, const __grid_constant__ CUtensorMap tBl, NsParams p) {
  extern __shared__ uint8_t raw[];
  __shared__ __align__(8) uint64_t full_bar[STAGES], empty_bar[STAGES], acc_bar;
  __shared__ uint32_t tmem_slot;
  __shared__ int abort_flag;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, mat = blockIdx.y;
  uint8_t* smem = (uint8_t*)(((uintptr_t)raw + 1023) & ~(uintptr_t)1023);
  uint8_t* sA = smem;
  uint8_t* sB = smem + STAGES * OPERAND_BYTES;
  int ti, tj;
  const int tiles_n = (p.n + TILE - 1) / TILE;
  if (p.symmetric) {             // blocks count the tiles (i, j >= i) column by column
    tj = (int)((sqrtf(8.f * blockIdx.x + 1.f) - 1.f) * 0.5f);
    while ((tj + 1) * (tj + 2) / 2 <= (int)blockIdx.x) ++tj;
    while (tj * (tj + 1) / 2 > (int)blockIdx.x) --tj;
    ti = blockIdx.x - tj * (tj + 1) / 2;
  } else {
    ti = blockIdx.x / tiles_n;
    tj = blockIdx.x - ti * tiles_n;
  }
  const int m0 = ti * TILE, n0 = tj * TILE;
  const int nk = (p.K + BK - 1) / BK, iters = nk * p.parts;
  if (tid == 0) {
    abort_flag = 0;
    for (int s = 0; s < STAGES; ++s) {
      ptx::mbar_init(&full_bar[s], 1);
      ptx::mbar_init(&empty_bar[s], 1);
    }
    ptx::mbar_init(&acc_bar, 1);
    ptx::mbar_fence_init();
  }
  const uint32_t tmem_cols = p.parts > 1 ? 4 * TILE : TILE;
  if (warp == 0) {
    ptx::tmem_alloc(&tmem_slot, tmem_cols);
    ptx::tmem_relinquish();
  }
  ptx::tc_fence_before();
  __syncthreads();
  ptx::tc_fence_after();
  const uint32_t tmem_base = tmem_slot;
  volatile int* abortp = &abort_flag;
  if (warp == 0) {
    if (lane == 0) {
      for (int i = 0; i < iters; ++i) {
        const int s = i % STAGES, part = i / nk, k0 = (i - part * nk) * BK;
        if (!ptx::mbar_wait(&empty_bar[s], ((uint32_t)(i / STAGES) & 1u) ^ 1u, p.spin_limit, abortp)) {
          abort_flag = 1;
          report_timeout(p.status, KID_NEWTON_SCHULZ, i);
          break;
        }
        ptx::mbar_arrive_expect_tx(&full_bar[s], 2 * OPERAND_BYTES);
        if (i == p.stall && blockIdx.x == 0 && mat == 0) continue;
        const bool a_mn = mn_major(p.a_form, m0, k0), b_mn = mn_major(p.b_form, n0, k0);
        const CUtensorMap* A = part == 2 ? &tAl : &tAh;      // high x high, high x low, low x high
        const CUtensorMap* B = part == 1 ? &tBl : &tBh;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          tch::tma_load_3d(sA + s * OPERAND_BYTES + h * BLOCK_BYTES, A, a_mn ? m0 + 64 * h : k0, a_mn ? k0 : m0 + 64 * h, mat,
                           &full_bar[s]);
          tch::tma_load_3d(sB + s * OPERAND_BYTES + h * BLOCK_BYTES, B, b_mn ? n0 + 64 * h : k0, b_mn ? k0 : n0 + 64 * h, mat,
                           &full_bar[s]);
        }
      }
    }
    __syncwarp();
  } else if (warp == 1) {
    if (lane == 0) {
      bool ok = true;
      for (int i = 0; i < iters && ok; ++i) {
        const int s = i % STAGES;
        if (!ptx::mbar_wait(&full_bar[s], (uint32_t)(i / STAGES) & 1u, p.spin_limit, abortp)) {
          abort_flag = 1;
          report_timeout(p.status, KID_NEWTON_SCHULZ, i);
          ok = false;
          break;
        }
        ptx::tc_fence_after();
        const uint32_t a_addr = ptx::smem_u32(sA + s * OPERAND_BYTES), b_addr = ptx::smem_u32(sB + s * OPERAND_BYTES);
        const int k0 = (i % nk) * BK;
        const bool a_mn = mn_major(p.a_form, m0, k0), b_mn = mn_major(p.b_form, n0, k0);
        const uint32_t idesc = ptx::umma_idesc_f16(TILE, TILE) | (a_mn ? 1u << 15 : 0u) | (b_mn ? 1u << 16 : 0u);
        const uint64_t a_step = a_mn ? 128 : 2, b_step = b_mn ? 128 : 2;
        const uint64_t da = a_mn ? ptx::umma_desc_mn_sw128(a_addr, BLOCK_BYTES) : ptx::umma_desc_k_sw128(a_addr);
        const uint64_t db = b_mn ? ptx::umma_desc_mn_sw128(b_addr, BLOCK_BYTES) : ptx::umma_desc_k_sw128(b_addr);
        const int sum = p.parts == 1 ? 0 : i < nk ? i % 3 : 3;
        const bool opens = p.parts == 1 ? i == 0 : i < 3 ? i < nk || i == nk : i == nk;
#pragma unroll
        for (int k = 0; k < BK / 16; ++k)
          ptx::umma_bf16(tmem_base + (uint32_t)(sum * TILE), da + a_step * k, db + b_step * k, idesc, opens && k == 0 ? 0u : 1u);
        ptx::umma_commit(&empty_bar[s]);
      }
      if (ok) ptx::umma_commit(&acc_bar);
    }
    __syncwarp();
  }
  bool ok = ptx::mbar_wait(&acc_bar, 0, p.spin_limit * 8, abortp);
  if (!ok && abort_flag == 0) {
    abort_flag = 1;
    report_timeout(p.status, KID_NEWTON_SCHULZ, 0xFFFF);
  }
  ok = __all_sync(0xffffffffu, ok);
  ptx::tc_fence_after();
  if (ok) {
    for (int c = 0; c < TILE / 32; ++c) {
      uint32_t r[32];
      ptx::tmem_ld32(tmem_base + ((uint32_t)(warp * 32) << 16) + (uint32_t)(c * 32), r);
      ptx::tmem_ld_wait();
      for (int sum = 1; sum < 4 && p.parts > 1; ++sum) {
        if (sum < 3 && sum >= nk) continue;
        uint32_t more[32];
        ptx::tmem_ld32(tmem_base + ((uint32_t)(warp * 32) << 16) + (uint32_t)(sum * TILE + c * 32), more);
        ptx::tmem_ld_wait();
#pragma unroll
        for (int j = 0; j < 32; ++j) r[j] = __float_as_uint(__uint_as_float(r[j]) + __uint_as_float(more[j]));
      }
      if (n0 + c * 32 < p.n) finish_row<T>(p, mat, m0 + warp * 32 + lane, n0 + c * 32, r);
    }
  }
  if (abort_flag != 0)
    for (int i = 0; i < 2000; ++i) __nanosleep(100);   // copies in flight land before the shared memory goes
  ptx::tc_fence_before();
  __syncthreads();
  if (warp == 0) ptx::tmem_dealloc(tmem_base, tmem_cols);
}

// ------------------------------------------------------------------ host

long padded(long x) { return (x + 7) / 8 * 8; }       // rows start on 16 bytes

struct NsBuffers {
  Split X[2], A, B;
  double* partial;
  long ldx, ldr;
  size_t bytes;
};
NsBuffers carve(void* ws, int dtype, int count, int m, int n) {
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
  b.B.hi = (__half*)take(a);
  if (dtype == ELMAN_F32) {
    b.A.lo = (__half*)take(a);
    b.B.lo = (__half*)take(a);
  }
  b.partial = (double*)take((size_t)count * NORM_PARTS * sizeof(double));
  b.bytes = off;
  return b;
}

// The largest singular value that `steps` applications make of values in [0, 1], and the largest |B|: both
// have to stay inside fp16's range at their scales.
bool stays_in_range(int steps, double a, double b, double c) {
  double top = 1.;
  for (int k = 0; k < steps; ++k) {
    auto poly = [&](double s) { return fabs(s * (a + s * s * (b + c * s * s))); };
    auto inner = [&](double s) { return fabs(s * s * (b + c * s * s)); };
    double most = poly(top), most_b = inner(top);
    auto see = [&](double s2) {
      if (s2 > 0. && s2 < top * top) {
        most = fmax(most, poly(sqrt(s2)));
        most_b = fmax(most_b, inner(sqrt(s2)));
      }
    };
    if (c != 0.) {
      const double disc = 9. * b * b - 20. * a * c;
      if (disc >= 0.) {
        see((-3. * b + sqrt(disc)) / (10. * c));
        see((-3. * b - sqrt(disc)) / (10. * c));
      }
      see(-b / (2. * c));
    } else if (b != 0.) {
      see(-a / (3. * b));
    }
    if (!(most_b <= 60.) || !(most <= 3.5)) return false;
    top = most;
  }
  return true;
}

template <typename T>
int run(int dtype, int count, int m, int n, const NsSource& src, int steps, float a, float b, float c, float eps, NsParams last,
        void* ws, cudaStream_t st) {
  const NsBuffers buf = carve(ws, dtype, count, m, n);
  const bool split = dtype == ELMAN_F32, tall = m > n;
  const int r = tall ? n : m;
  static std::mutex mutex;
  static bool sized[64];
  int dev = 0;
  ELMAN_CUDA_CHECK(cudaGetDevice(&dev));
  {
    std::lock_guard<std::mutex> lock(mutex);
    if (dev >= 64 || !sized[dev]) {
      ELMAN_CUDA_CHECK(cudaFuncSetAttribute(ns_product_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, NS_SMEM));
      if (dev < 64) sized[dev] = true;
    }
  }
  auto takes_low = [&](int step) { return split || step < steps - 2; };
  ns_norm_kernel<T><<<dim3(NORM_PARTS, count), 256, 0, st>>>(src, (long)m * n, buf.partial);
  count_launch(false);
  const long blocks = ((long)m * n + 256 * 8 - 1) / (256 * 8);
  Split x0 = buf.X[0];
  if (!takes_low(0)) x0.lo = nullptr;
  ns_scale_kernel<T><<<dim3((unsigned)(blocks < 1024 ? blocks : 1024), count), 256, 0, st>>>(src, m, n, buf.ldx, eps, buf.partial, x0);
  count_launch(false);
  CUtensorMap mx[2][2], ma[2], mb[2];
  auto map = [&](CUtensorMap* out, const __half* base, int rows, int cols, long ld) {
    return make_tmap_f16_sw128(out, base, cols, rows, count, ld, (long)rows * ld);
  };
  for (int k = 0; k < 2; ++k) {
    ELMAN_RETURN_IF(map(&mx[k][0], buf.X[k].hi, m, n, buf.ldx));
    ELMAN_RETURN_IF(map(&mx[k][1], split ? buf.X[k].lo : buf.X[k].hi, m, n, buf.ldx));
  }
  ELMAN_RETURN_IF(map(&ma[0], buf.A.hi, r, r, buf.ldr));
  ELMAN_RETURN_IF(map(&ma[1], split ? buf.A.lo : buf.A.hi, r, r, buf.ldr));
  ELMAN_RETURN_IF(map(&mb[0], buf.B.hi, r, r, buf.ldr));
  ELMAN_RETURN_IF(map(&mb[1], split ? buf.B.lo : buf.B.hi, r, r, buf.ldr));
  const int side = (r + TILE - 1) / TILE, triangle = side * (side + 1) / 2;
  const int all = ((m + TILE - 1) / TILE) * ((n + TILE - 1) / TILE);
  NsParams p = last;
  p.parts = split ? 3 : 1;
  p.status = device_status_ptr();
  p.spin_limit = options().spin_limit;
  p.stall = (int)options().test_stall_step;
  for (int step = 0; step < steps; ++step) {
    const int at = step & 1;
    // A = X X^T, or X^T X
    p.kind = GRAM; p.m = p.n = r; p.K = tall ? m : n; p.a_form = p.b_form = tall ? K_ROWS : ROWS_K; p.symmetric = 1;
    p.ld = buf.ldr; p.stride = (long)r * buf.ldr; p.k_acc = SA / (SX * SX); p.k_same = 0.f; p.out = buf.A;
    ns_product_kernel<T><<<dim3(triangle, count), 128, NS_SMEM, st>>>(mx[at][0], mx[at][1], mx[at][0], mx[at][1], p);
    count_launch(true);
    // B = b A + c A A
    p.kind = SQUARE; p.K = r; p.a_form = p.b_form = UPPER; p.k_acc = c * SB / (SA * SA); p.k_same = b * SB / SA;
    p.same = buf.A; p.out = buf.B;
    ns_product_kernel<T><<<dim3(triangle, count), 128, NS_SMEM, st>>>(ma[0], ma[1], ma[0], ma[1], p);
    count_launch(true);
    // X <- a X + B X, or a X + X B
    const bool ends = step == steps - 1;
    p.kind = ends ? LAST : UPDATE; p.m = m; p.n = n; p.symmetric = 0; p.ld = buf.ldx; p.stride = (long)m * buf.ldx;
    p.k_acc = 1.f / SB; p.k_same = a;
    if (ends) { p.k_acc /= SX; p.k_same /= SX; }
    p.same = buf.X[at]; p.out = buf.X[at ^ 1];
    if (!takes_low(step)) p.same.lo = nullptr;
    if (!ends && !takes_low(step + 1)) p.out.lo = nullptr;
    if (tall) {
      p.a_form = ROWS_K;
      ns_product_kernel<T><<<dim3(all, count), 128, NS_SMEM, st>>>(mx[at][0], mx[at][1], mb[0], mb[1], p);
    } else {
      p.b_form = K_ROWS;
      ns_product_kernel<T><<<dim3(all, count), 128, NS_SMEM, st>>>(mb[0], mb[1], mx[at][0], mx[at][1], p);
    }
    count_launch(true);
  }
  ELMAN_CUDA_CHECK(cudaGetLastError());
  return ELMAN_OK;
}

}  // namespace

size_t newton_schulz_workspace(int dtype, int count, int m, int n) { return carve(nullptr, dtype, count, m, n).bytes; }
bool newton_schulz_in_range(int steps, float a, float b, float c) { return stays_in_range(steps, a, b, c); }

int newton_schulz(const NewtonSchulzArgs& a, cudaStream_t st) {
  NsSource src{};
  src.in = a.in;
  NsParams last{};
  last.result = a.out;
  return a.dtype == ELMAN_F32 ? run<float>(a.dtype, a.count, a.m, a.n, src, a.steps, a.a, a.b, a.c, a.eps, last, a.workspace, st)
                              : run<bf16>(a.dtype, a.count, a.m, a.n, src, a.steps, a.a, a.b, a.c, a.eps, last, a.workspace, st);
}

int muon_step(const NewtonSchulzArgs& a, const MuonArgs& u, cudaStream_t st) {
  NsSource src{};
  src.in = u.grads;
  src.offsets = u.offsets;
  src.momentum = u.momentum;
  src.mu = u.mu;
  src.nesterov = u.nesterov;
  src.grad_scale = u.grad_scale;
  NsParams last{};
  last.result = u.params;
  last.offsets = u.offsets;
  last.muon = 1;
  last.lr = u.lr;
  last.decay = 1.f - u.lr * u.weight_decay;
  last.scale = u.scale;
  return a.dtype == ELMAN_F32 ? run<float>(a.dtype, a.count, a.m, a.n, src, a.steps, a.a, a.b, a.c, a.eps, last, a.workspace, st)
                              : run<bf16>(a.dtype, a.count, a.m, a.n, src, a.steps, a.a, a.b, a.c, a.eps, last, a.workspace, st);
}

}  // namespace elman
