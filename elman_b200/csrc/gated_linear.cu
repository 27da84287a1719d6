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

// One thread per channel walks the sequence.
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
  float before[GL_CHUNK];
  for (int k = (p.T - 1) / GL_CHUNK; k >= 0 && p.T > 0; --k) {
    const int t0 = k * GL_CHUNK, n = p.T - t0 < GL_CHUNK ? p.T - t0 : GL_CHUNK;
    float h = p.saved[(long)k * cols + col];
    for (int j = 0; j < n; ++j) {
      const int t = t0 + j;
      if (p.reset != nullptr && p.reset[(long)t * p.B + b] != 0) h = 0.f;
      before[j] = h;
      float e;
      const float u = keep_gate(to_f(f[t * p.sf.t]), e);
      h = fmaf(u, to_f(c[t * p.sc.t]) - h, h);
    }
    for (int j = n - 1; j >= 0; --j) {
      const int t = t0 + j;
      float e;
      const float u = keep_gate(to_f(f[t * p.sf.t]), e), cv = to_f(c[t * p.sc.t]), zv = to_f(z[t * p.sz.t]);
      const float g0 = to_f(dy[t * p.sy.t]), prev = before[j];
      const float now = fmaf(u, cv - prev, prev);
      const float g = fmaf(g0, siluf_(zv), D);
      dz[t * p.sdz.t] = from_f<T>(g0 * now * dsiluf_(zv));
      dc[t * p.sdc.t] = from_f<T>(g * u);
      df[t * p.sdf.t] = from_f<T>(g * (prev - cv) * u * (e * u));
      D = p.reset != nullptr && p.reset[(long)t * p.B + b] != 0 ? 0.f : fmaf(-u, g, g);
    }
  }
  p.dh0[col] = D;
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

}  // namespace

int gated_linear_fwd(int dtype, const GatedLinearArgs& a, cudaStream_t st) {
  const long cols = (long)a.B * a.d;
  if (cols == 0) return ELMAN_OK;
  const GlParams p = params_of(a);
  const int grid = (int)((cols + 127) / 128);
  if (dtype == ELMAN_F32) gl_forward_seq_kernel<float><<<grid, 128, 0, st>>>(p);
  else gl_forward_seq_kernel<bf16><<<grid, 128, 0, st>>>(p);
  count_launch(false);
  ELMAN_CUDA_CHECK(cudaGetLastError());
  return ELMAN_OK;
}

int gated_linear_bwd(int dtype, const GatedLinearArgs& a, cudaStream_t st) {
  const long cols = (long)a.B * a.d;
  if (cols == 0) return ELMAN_OK;
  const GlParams p = params_of(a);
  const int grid = (int)((cols + 127) / 128);
  if (dtype == ELMAN_F32) gl_backward_seq_kernel<float><<<grid, 128, 0, st>>>(p);
  else gl_backward_seq_kernel<bf16><<<grid, 128, 0, st>>>(p);
  count_launch(false);
  ELMAN_CUDA_CHECK(cudaGetLastError());
  return ELMAN_OK;
}

size_t gated_linear_workspace(int dtype, int T, int B, int d) {
  (void)dtype; (void)T; (void)B; (void)d;
  return 0;
}

}  // namespace elman
