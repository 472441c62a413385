// Layer norm over rows of D, forward and backward, with an optional residual:
//     s = x (+ residual),  y = (s - mean) rstd w + b
//     ds += rstd (dy w - mean(dy w) - hat mean(dy w hat)),  hat = (s - mean) rstd
//     dw = sum_rows dy hat,  db = sum_rows dy
// Bandwidth bound.  A row is held in registers by G threads (a power of two:
// part of a warp, a warp, or a CTA of up to 512), read once; the
// statistics are taken in two passes over the registers, so a large mean costs
// no precision.  The backward's CTAs walk rows in a fixed stride and keep the
// dw, db terms of their own columns in registers; a second kernel adds the
// CTAs' sums, so the result does not depend on timing.
#include <type_traits>

#include "linear_attn.cuh"
#include "profile.cuh"

namespace gdn2 {
namespace {

enum Residual { kNone = 0, kSame = 1, kF32 = 2 };  // no residual, of x's type, fp32 beside bf16 x

template <typename T, int N>
GDN2_DEV void ldv(const T* p, float (&x)[N]) {
  if constexpr (N == 8) ld8(p, x);
  else if constexpr (N == 4) {
    const float4 a = *reinterpret_cast<const float4*>(p);
    x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w;
  } else x[0] = to_f(p[0]);
}
template <typename T, int N>
GDN2_DEV void stv(T* p, const float (&x)[N]) {
  if constexpr (N == 8) st8(p, x);
  else if constexpr (N == 4) *reinterpret_cast<float4*>(p) = make_float4(x[0], x[1], x[2], x[3]);
  else p[0] = from_f<T>(x[0]);
}
template <int N>
GDN2_DEV void ldw(const void* p, int64_t i, int dtype, float (&x)[N]) {
  if (dtype == GDN2_BF16) {
#pragma unroll
    for (int e = 0; e < N; ++e) x[e] = to_f(static_cast<const __nv_bfloat16*>(p)[i + e]);
  } else {
#pragma unroll
    for (int e = 0; e < N; ++e) x[e] = static_cast<const float*>(p)[i + e];
  }
}

// sums over the G threads of a row; every one of them gets the result
template <int M>
GDN2_DEV void group_sum(float (&x)[M], int G, float (*sh)[M]) {
  for (int o = min(G, 32) >> 1; o > 0; o >>= 1)
#pragma unroll
    for (int m = 0; m < M; ++m) x[m] += __shfl_xor_sync(0xffffffffu, x[m], o);
  if (G <= 32) return;
  const int warp = threadIdx.x >> 5, nw = G >> 5, w0 = warp / nw * nw;
  __syncthreads();
  if ((threadIdx.x & 31) == 0)
#pragma unroll
    for (int m = 0; m < M; ++m) sh[warp][m] = x[m];
  __syncthreads();
#pragma unroll
  for (int m = 0; m < M; ++m) x[m] = 0.f;
  for (int w = 0; w < nw; ++w)
#pragma unroll
    for (int m = 0; m < M; ++m) x[m] += sh[w0 + w][m];
}

template <typename T, int RES>
struct ResType {
  using type = typename std::conditional<RES == kF32, float, T>::type;
};

// CTAs of 512 threads only for the longest rows
template <int VEC, int NV>
constexpr int kMaxThreads = VEC * NV * 256 >= 32768 / 2 ? 512 : 256;

template <typename T, int RES, int VEC, int NV>
__global__ void __launch_bounds__((kMaxThreads<VEC, NV>)) layer_norm_fwd_kernel(const gdn2_layer_norm_args a, int G) {
  using R = typename ResType<T, RES>::type;
  __shared__ float sh[32][1];
  const int lane = threadIdx.x % G;
  const int64_t row = (int64_t)blockIdx.x * (blockDim.x / G) + threadIdx.x / G;
  const int64_t D = a.D;
  const bool in = row < a.rows;
  const T* x = static_cast<const T*>(a.x) + row * D;
  const R* r = static_cast<const R*>(a.residual) + row * D;
  float s[NV][VEC];
  float sum[1] = {0.f};
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int64_t c = (int64_t)(lane + i * G) * VEC;
#pragma unroll
    for (int e = 0; e < VEC; ++e) s[i][e] = 0.f;
    if (in && c < D) {
      ldv(x + c, s[i]);
      if (RES != kNone) {
        float y[VEC];
        ldv(r + c, y);
#pragma unroll
        for (int e = 0; e < VEC; ++e) s[i][e] = to_f(from_f<R>(s[i][e] + y[e]));
        stv(static_cast<R*>(a.s) + row * D + c, s[i]);
      }
    }
#pragma unroll
    for (int e = 0; e < VEC; ++e) sum[0] += s[i][e];
  }
  group_sum(sum, G, sh);
  const float mean = sum[0] / (float)D;
  float sq[1] = {0.f};
#pragma unroll
  for (int i = 0; i < NV; ++i)
    if ((int64_t)(lane + i * G) * VEC < D)
#pragma unroll
      for (int e = 0; e < VEC; ++e) sq[0] += (s[i][e] - mean) * (s[i][e] - mean);
  group_sum(sq, G, sh);
  const float rstd = rsqrtf(sq[0] / (float)D + a.eps);
  if (!in) return;
  if (a.mean && lane == 0) {
    a.mean[row] = mean;
    a.rstd[row] = rstd;
  }
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int64_t c = (int64_t)(lane + i * G) * VEC;
    if (c < D) {
      float w[VEC], b[VEC], y[VEC];
#pragma unroll
      for (int e = 0; e < VEC; ++e) w[e] = 1.f, b[e] = 0.f;
      if (a.weight) ldw(a.weight, c, a.dtype_weight, w);
      if (a.bias) ldw(a.bias, c, a.dtype_weight, b);
#pragma unroll
      for (int e = 0; e < VEC; ++e) y[e] = fmaf((s[i][e] - mean) * rstd, w[e], b[e]);
      stv(static_cast<T*>(a.y) + row * D + c, y);
    }
  }
}

template <typename T, int RES, int VEC, int NV>
__global__ void __launch_bounds__((kMaxThreads<VEC, NV>)) layer_norm_bwd_kernel(const gdn2_layer_norm_args a, const gdn2_layer_norm_grads g, int G, float* part) {
  using R = typename ResType<T, RES>::type;
  extern __shared__ float cols[];  // [2][D] when several rows share the CTA
  __shared__ float sh[32][2];
  const int lane = threadIdx.x % G, set = threadIdx.x / G, sets = blockDim.x / G;
  const int64_t D = a.D;
  float dw[NV][VEC], db[NV][VEC], w[NV][VEC];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int64_t c = (int64_t)(lane + i * G) * VEC;
#pragma unroll
    for (int e = 0; e < VEC; ++e) dw[i][e] = db[i][e] = 0.f, w[i][e] = 1.f;
    if (a.weight && c < D) ldw(a.weight, c, a.dtype_weight, w[i]);
  }
  for (int64_t r0 = (int64_t)blockIdx.x * sets; r0 < a.rows; r0 += (int64_t)gridDim.x * sets) {
    const int64_t row = r0 + set;
    const bool in = row < a.rows;
    const float mean = in ? a.mean[row] : 0.f, rstd = in ? a.rstd[row] : 0.f;
    float hat[NV][VEC], d[NV][VEC], sum[2] = {0.f, 0.f};
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int64_t c = (int64_t)(lane + i * G) * VEC;
#pragma unroll
      for (int e = 0; e < VEC; ++e) hat[i][e] = d[i][e] = 0.f;
      if (in && c < D) {
        ldv(static_cast<const R*>(g.s) + row * D + c, hat[i]);
        ldv(static_cast<const T*>(g.dy) + row * D + c, d[i]);
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
          hat[i][e] = (hat[i][e] - mean) * rstd;
          dw[i][e] = fmaf(d[i][e], hat[i][e], dw[i][e]);
          db[i][e] += d[i][e];
          d[i][e] *= w[i][e];
          sum[0] += d[i][e];
          sum[1] = fmaf(d[i][e], hat[i][e], sum[1]);
        }
      }
    }
    group_sum(sum, G, sh);
    const float m0 = sum[0] / (float)D, m1 = sum[1] / (float)D;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int64_t c = (int64_t)(lane + i * G) * VEC;
      if (in && c < D) {
        float x[VEC];
#pragma unroll
        for (int e = 0; e < VEC; ++e) x[e] = rstd * (d[i][e] - m0 - hat[i][e] * m1);
        if (RES != kNone && g.ds) {
          float y[VEC];
          ldv(static_cast<const R*>(g.ds) + row * D + c, y);
#pragma unroll
          for (int e = 0; e < VEC; ++e) x[e] += y[e];
        }
        if (g.dx) stv(static_cast<T*>(g.dx) + row * D + c, x);
        if (RES != kNone && g.dresidual) stv(static_cast<R*>(g.dresidual) + row * D + c, x);
      }
    }
  }
  if (!part) return;
  float* out = part + (int64_t)blockIdx.x * 2 * D;
  for (int k = 0; k < sets; ++k) {  // the row sets of a CTA, one after the other
    if (sets > 1) __syncthreads();
    if (set == k)
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int64_t c = (int64_t)(lane + i * G) * VEC;
        if (c < D)
#pragma unroll
          for (int e = 0; e < VEC; ++e) {
            float x = dw[i][e], y = db[i][e];
            if (k > 0) x += cols[c + e], y += cols[D + c + e];
            if (k + 1 < sets) cols[c + e] = x, cols[D + c + e] = y;
            else out[c + e] = x, out[D + c + e] = y;
          }
      }
  }
}

// dw, db: the CTAs' sums in order; a warp per 32 columns and 8 strided shares of the CTAs
__global__ void __launch_bounds__(256) layer_norm_sum_kernel(const float* part, int n, int64_t D, void* dw, void* db,
                                                             int dtype) {
  __shared__ float sh[8][32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t c = (int64_t)blockIdx.x * 32 + lane;  // over [dw | db]
  float x = 0.f;
  if (c < 2 * D)
    for (int i = warp; i < n; i += 8) x += part[(int64_t)i * 2 * D + c];
  sh[warp][lane] = x;
  __syncthreads();
  if (warp == 0 && c < 2 * D) {
    x = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) x += sh[i][lane];
    void* out = c < D ? dw : db;
    if (out) {
      if (dtype == GDN2_BF16) static_cast<__nv_bfloat16*>(out)[c < D ? c : c - D] = __float2bfloat16_rn(x);
      else static_cast<float*>(out)[c < D ? c : c - D] = x;
    }
  }
}

struct Plan {
  bool vec;
  int NV, G, threads;  // vectors per thread, threads per row, threads per CTA
};

// One vector per thread up to 256 threads a row, then more vectors, then 512 threads.
Plan plan(const gdn2_layer_norm_args& a, bool vec) {
  const int per = vec ? (a.dtype == GDN2_BF16 ? 8 : 4) : 1;
  const int64_t units = (a.D + per - 1) / per;
  const int least = vec ? 1 : 4;
  Plan p{vec, least, 8, 256};
  while ((int64_t)p.G * least < units && p.G < 256) p.G *= 2;
  if (vec) {
    while ((int64_t)p.G * p.NV < units && p.NV < 4) p.NV *= 2;
  } else if ((int64_t)p.G * p.NV < units) {
    p.NV = 32;
  }
  if ((int64_t)p.G * p.NV < units) {
    p.G = p.threads = 512;
    p.NV = 32768 / (512 * per);
  }
  return p;
}

bool aligned(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

int bwd_ctas(const gdn2_layer_norm_args& a, const Plan& p) {
  const int64_t sets = p.threads / p.G, need = (a.rows + sets - 1) / sets;
  const int64_t most = 148 * (p.threads > 256 ? 1 : 3);
  return need < 1 ? 1 : (int)(need < most ? need : most);
}

template <typename T, int RES>
int fwd(const gdn2_layer_norm_args& a, const Plan& p, cudaStream_t s) {
  const int64_t rows_per = p.threads / p.G;
  const unsigned grid = (unsigned)((a.rows + rows_per - 1) / rows_per);
  constexpr int VEC = sizeof(T) == 2 ? 8 : 4;
  ProfScope ps(kKLayerNormFwd, s);
#define LN_FWD(V, N) layer_norm_fwd_kernel<T, RES, V, N><<<grid, p.threads, 0, s>>>(a, p.G)
  if (p.vec) {
    if (p.NV == 1) LN_FWD(VEC, 1);
    else if (p.NV == 2) LN_FWD(VEC, 2);
    else if (p.NV == 4) LN_FWD(VEC, 4);
    else LN_FWD(VEC, 64 / VEC);
  } else {
    if (p.NV == 4) LN_FWD(1, 4);
    else if (p.NV == 32) LN_FWD(1, 32);
    else LN_FWD(1, 64);
  }
#undef LN_FWD
  GDN2_LAUNCH_CHECK();
  return 0;
}

template <typename T, int RES>
int bwd(const gdn2_layer_norm_args& a, const gdn2_layer_norm_grads& g, const Plan& p, float* part, cudaStream_t s) {
  const int ctas = bwd_ctas(a, p);
  const size_t sm = p.threads / p.G > 1 ? 2 * a.D * 4 : 0;
  constexpr int VEC = sizeof(T) == 2 ? 8 : 4;
  {
    ProfScope ps(kKLayerNormBwd, s);
#define LN_BWD(V, N) layer_norm_bwd_kernel<T, RES, V, N><<<ctas, p.threads, sm, s>>>(a, g, p.G, part)
    if (p.vec) {
      if (p.NV == 1) LN_BWD(VEC, 1);
      else if (p.NV == 2) LN_BWD(VEC, 2);
      else if (p.NV == 4) LN_BWD(VEC, 4);
      else LN_BWD(VEC, 64 / VEC);
    } else {
      if (p.NV == 4) LN_BWD(1, 4);
      else if (p.NV == 32) LN_BWD(1, 32);
      else LN_BWD(1, 64);
    }
#undef LN_BWD
    GDN2_LAUNCH_CHECK();
  }
  if (part) {
    layer_norm_sum_kernel<<<(unsigned)((2 * a.D + 31) / 32), 256, 0, s>>>(part, ctas, a.D, g.dweight, g.dbias,
                                                                          a.dtype_weight);
    GDN2_LAUNCH_CHECK();
  }
  return 0;
}

}  // namespace

int layer_norm_fwd_launch(const gdn2_layer_norm_args& a, cudaStream_t s) {
  const bool vec = a.D % (a.dtype == GDN2_BF16 ? 8 : 4) == 0 && aligned(a.x) && aligned(a.y) && aligned(a.residual) &&
                   aligned(a.s);
  const Plan p = plan(a, vec);
  if (a.dtype == GDN2_F32) return a.residual ? fwd<float, kSame>(a, p, s) : fwd<float, kNone>(a, p, s);
  if (!a.residual) return fwd<__nv_bfloat16, kNone>(a, p, s);
  return a.dtype_residual == GDN2_F32 ? fwd<__nv_bfloat16, kF32>(a, p, s) : fwd<__nv_bfloat16, kSame>(a, p, s);
}

size_t layer_norm_bwd_ws(const gdn2_layer_norm_args& a) {
  const int v = bwd_ctas(a, plan(a, true)), n = bwd_ctas(a, plan(a, false));
  return (size_t)(v > n ? v : n) * 2 * (size_t)a.D * 4;
}

int layer_norm_bwd_launch(const gdn2_layer_norm_args& a, const gdn2_layer_norm_grads& g, void* ws, cudaStream_t s) {
  const bool vec = a.D % (a.dtype == GDN2_BF16 ? 8 : 4) == 0 && aligned(g.s) && aligned(g.dy) && aligned(g.ds) &&
                   aligned(g.dx) && aligned(g.dresidual);
  const Plan p = plan(a, vec);
  float* part = (g.dweight || g.dbias) ? static_cast<float*>(ws) : nullptr;
  if (a.dtype == GDN2_F32) return a.residual ? bwd<float, kSame>(a, g, p, part, s) : bwd<float, kNone>(a, g, p, part, s);
  if (!a.residual) return bwd<__nv_bfloat16, kNone>(a, g, p, part, s);
  return a.dtype_residual == GDN2_F32 ? bwd<__nv_bfloat16, kF32>(a, g, p, part, s)
                                      : bwd<__nv_bfloat16, kSame>(a, g, p, part, s);
}

}  // namespace gdn2
