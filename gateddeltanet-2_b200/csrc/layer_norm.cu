// Layer norm over rows of D, forward and backward, with an optional residual:
//     s = x (+ residual),  y = (s - mean) rstd w + b
//     ds += rstd (dy w - mean(dy w) - hat mean(dy w hat)),  hat = (s - mean) rstd
//     dw = sum_rows dy hat,  db = sum_rows dy
// Bandwidth bound: what counts is how many bytes are on the way.  A row is held
// in registers by G threads, read once; the statistics are taken in two passes
// over the registers, so a large mean costs no precision.  Rows of up to 256
// vectors (16 bytes) belong to a warp or part of one, several short rows side by side in each
// thread, and need no barrier; longer rows belong to a CTA of 256 or 512.
// The backward keeps the dw, db terms of a thread's columns in registers while
// its CTA walks rows in a fixed stride (short rows several at a time, CTA-wide rows with the
// next one already loading); a second kernel adds the CTAs' sums in order, so the
// result does not depend on timing.
// Measured, bf16 rows: 16384 x 2048 onto an fp32 residual, forward 62 us (402 MB,
// 6.5 TB/s) and backward 98 us (537 MB, 5.5 TB/s); 262144 x 128, forward 31 us
// (134 MB, 4.3 TB/s) and backward 53 us (201 MB, 3.8 TB/s), then 9 us for the sum.
// Those short rows wait: 126 registers a thread leave two CTAs an SM (a quarter of the
// warps), the backward loads a turn's rows only when it comes to them, and SM and DRAM
// are both near half busy or below (forward 52 and 36%, backward 39 and 43%); the
// sum runs on 8 CTAs.  Rows off the 16-byte grid (D no multiple of 4 in fp32, of 8 in
// bf16, or unaligned views) go element by element: 50000 x 1001 bf16 164 us forward
// and 158 us backward, 25000 x 1001 fp32 81 and 83 us, some 1.2 to 3.6 TB/s.
#include <type_traits>

#include "linear_attn.cuh"
#include "profile.cuh"
#include "tc.cuh"

namespace gdn2 {
namespace {

enum Residual { kNone = 0, kSame = 1, kF32 = 2 };  // no residual, of x's type, fp32 beside bf16 x

// N elements as they lie in memory (16-byte pieces, or one element)
template <typename T, int N>
struct Raw {
  static constexpr int kWords = (int)sizeof(T) * N >= 16 ? (int)sizeof(T) * N / 4 : 1;
  uint32_t w[kWords];
  GDN2_DEV void zero() {
#pragma unroll
    for (int i = 0; i < kWords; ++i) w[i] = 0;
  }
  GDN2_DEV void load(const T* p) {
    if constexpr (kWords >= 4) {
#pragma unroll
      for (int i = 0; i < kWords; i += 4) {
        const uint4 u = reinterpret_cast<const uint4*>(p)[i / 4];
        w[i] = u.x; w[i + 1] = u.y; w[i + 2] = u.z; w[i + 3] = u.w;
      }
    } else if constexpr (sizeof(T) == 2) {
      w[0] = *reinterpret_cast<const uint16_t*>(p);
    } else {
      w[0] = *reinterpret_cast<const uint32_t*>(p);
    }
  }
  GDN2_DEV float operator[](int e) const {
    if constexpr (sizeof(T) == 4) return __uint_as_float(w[e]);
    else return __uint_as_float(e & 1 ? w[e / 2] & 0xffff0000u : w[e / 2] << 16);
  }
};
template <typename T, int N>
GDN2_DEV void stv(T* p, const float (&x)[N]) {
  if constexpr (N == 8) st8(p, x);
  else if constexpr (N == 4) *reinterpret_cast<float4*>(p) = make_float4(x[0], x[1], x[2], x[3]);
  else p[0] = from_f<T>(x[0]);
}
// N elements of a weight from column i on, 1 where there is none; wide loads where `vec` says that they are aligned
template <int N>
GDN2_DEV void ldw(const void* p, int64_t i, int dtype, bool vec, float none, float (&x)[N]) {
  if (!p) {
#pragma unroll
    for (int e = 0; e < N; ++e) x[e] = none;
  } else if (dtype == GDN2_BF16) {
    const __nv_bfloat16* q = static_cast<const __nv_bfloat16*>(p) + i;
    if (N == 8 && vec) {
      Raw<__nv_bfloat16, 8> r;
      r.load(q);
#pragma unroll
      for (int e = 0; e < N; ++e) x[e] = r[e];
    } else {
#pragma unroll
      for (int e = 0; e < N; ++e) x[e] = to_f(q[e]);
    }
  } else {
    const float* q = static_cast<const float*>(p) + i;
    if (N >= 4 && vec) {
      Raw<float, N < 4 ? 4 : N> r;
      r.load(q);
#pragma unroll
      for (int e = 0; e < N; ++e) x[e] = r[e];
    } else {
#pragma unroll
      for (int e = 0; e < N; ++e) x[e] = q[e];
    }
  }
}

// Arithmetic on N elements, two per instruction where N is even: on short rows
// a vector's conversions and multiply-adds count beside its loads.
template <int N, typename F1, typename F2>
GDN2_DEV void each(F1 one, F2 two) {
  if constexpr (N % 2 == 0) {
#pragma unroll
    for (int e = 0; e < N; e += 2) two(e);
  } else {
#pragma unroll
    for (int e = 0; e < N; ++e) one(e);
  }
}
template <int N>
GDN2_DEV void add_to(float (&x)[N], float c) {  // x += c
  const uint64_t c2 = tc::pack2(c, c);
  each<N>([&](int e) { x[e] += c; },
          [&](int e) { tc::unpack2(tc::add2(tc::pack2(x[e], x[e + 1]), c2), x[e], x[e + 1]); });
}
template <int N>
GDN2_DEV void scale_by(float (&x)[N], float c) {  // x *= c
  const uint64_t c2 = tc::pack2(c, c);
  each<N>([&](int e) { x[e] *= c; },
          [&](int e) { tc::unpack2(tc::mul2(tc::pack2(x[e], x[e + 1]), c2), x[e], x[e + 1]); });
}
template <int N>
GDN2_DEV void mul_by(float (&x)[N], const float (&y)[N]) {  // x *= y
  each<N>([&](int e) { x[e] *= y[e]; }, [&](int e) {
    tc::unpack2(tc::mul2(tc::pack2(x[e], x[e + 1]), tc::pack2(y[e], y[e + 1])), x[e], x[e + 1]);
  });
}
template <int N>
GDN2_DEV void add_up(float (&s)[N], const float (&x)[N]) {  // s += x
  each<N>([&](int e) { s[e] += x[e]; }, [&](int e) {
    tc::unpack2(tc::add2(tc::pack2(s[e], s[e + 1]), tc::pack2(x[e], x[e + 1])), s[e], s[e + 1]);
  });
}
template <int N>
GDN2_DEV void fma_up(float (&s)[N], const float (&x)[N], const float (&y)[N]) {  // s += x y
  each<N>([&](int e) { s[e] = fmaf(x[e], y[e], s[e]); }, [&](int e) {
    tc::unpack2(tc::fma2(tc::pack2(x[e], x[e + 1]), tc::pack2(y[e], y[e + 1]), tc::pack2(s[e], s[e + 1])), s[e], s[e + 1]);
  });
}
template <int N>
GDN2_DEV void fma_by(float (&x)[N], const float (&w)[N], const float (&b)[N]) {  // x = x w + b
  each<N>([&](int e) { x[e] = fmaf(x[e], w[e], b[e]); }, [&](int e) {
    tc::unpack2(tc::fma2(tc::pack2(x[e], x[e + 1]), tc::pack2(w[e], w[e + 1]), tc::pack2(b[e], b[e + 1])), x[e], x[e + 1]);
  });
}
template <int N>
GDN2_DEV void fma_to(float (&x)[N], const float (&y)[N], float c) {  // x += c y
  const uint64_t c2 = tc::pack2(c, c);
  each<N>([&](int e) { x[e] = fmaf(y[e], c, x[e]); }, [&](int e) {
    tc::unpack2(tc::fma2(tc::pack2(y[e], y[e + 1]), c2, tc::pack2(x[e], x[e + 1])), x[e], x[e + 1]);
  });
}
template <int N>
GDN2_DEV float total(const float (&x)[N]) {
  float s = x[0];
#pragma unroll
  for (int e = 1; e < N; ++e) s += x[e];
  return s;
}

// sums over the G threads of a row (M of them at once); every one of them gets the results
template <int M>
GDN2_DEV void group_sum(float (&x)[M], int G, float (*sh)[M]) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1)
    if (o < G)
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

// CTAs of 512 threads for the longest rows, and for single elements beyond 4 a thread
template <int VEC, int NV>
constexpr int kMaxThreads = VEC * NV == 64 || (VEC == 1 && NV > 4) ? 512 : 256;

// What one turn of the forward reads: R rows of a group of G threads, NV vectors of VEC elements of each per thread
template <typename T, typename S, int RES, int VEC, int NV, int R>
struct FwdTurn {
  Raw<T, VEC> x[R][NV];
  Raw<S, VEC> res[RES == kNone ? 1 : R][RES == kNone ? 1 : NV];
  GDN2_DEV void load(const gdn2_layer_norm_args& a, int64_t row0, int sets, int lane, int G) {
#pragma unroll
    for (int k = 0; k < R; ++k) {
      const int64_t row = row0 + k * sets;
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int64_t c = (int64_t)(lane + i * G) * VEC, at = row * a.D + c;
        const bool in = row < a.rows && c < a.D;
        if (in) x[k][i].load(static_cast<const T*>(a.x) + at);
        else x[k][i].zero();
        if constexpr (RES != kNone) {
          if (in) res[k][i].load(static_cast<const S*>(a.residual) + at);
          else res[k][i].zero();
        }
      }
    }
  }
  // the row that is normalised: with a residual, as it is stored
  GDN2_DEV float at(int k, int i, int e) const {
    if constexpr (RES != kNone) return to_f(from_f<S>(x[k][i][e] + res[k][i][e]));
    else return x[k][i][e];
  }
};

template <typename T, int RES, int VEC, int NV, int R, bool kAhead>
__global__ void __launch_bounds__((kMaxThreads<VEC, NV>))
layer_norm_fwd_kernel(const gdn2_layer_norm_args a, int G, bool vecw) {
  using S = typename ResType<T, RES>::type;
  __shared__ float sh[32][R];
  const int lane = threadIdx.x % G, set = threadIdx.x / G, sets = blockDim.x / G;
  const int64_t D = a.D, stride = (int64_t)gridDim.x * sets * R, first = (int64_t)blockIdx.x * sets * R;
  FwdTurn<T, S, RES, VEC, NV, R> t;
  if (kAhead) t.load(a, first + set, sets, lane, G);
  float w[NV][VEC], b[NV][VEC];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int64_t c = (int64_t)(lane + i * G) * VEC;
    ldw(c < D ? a.weight : nullptr, c, a.dtype_weight, vecw, 1.f, w[i]);
    ldw(c < D ? a.bias : nullptr, c, a.dtype_weight, vecw, 0.f, b[i]);
  }
  const float inv = 1.f / (float)D;
  for (int64_t r0 = first; r0 < a.rows; r0 += stride) {  // (the CTA's bounds: there are barriers inside)
    [[maybe_unused]] FwdTurn<T, S, RES, VEC, NV, R> next;
    if constexpr (kAhead) next.load(a, r0 + stride + set, sets, lane, G);
    else t.load(a, r0 + set, sets, lane, G);
    float c[R][NV][VEC], sum[R], sq[R];
#pragma unroll
    for (int k = 0; k < R; ++k) {
      float acc[VEC];
#pragma unroll
      for (int i = 0; i < NV; ++i) {
#pragma unroll
        for (int e = 0; e < VEC; ++e) c[k][i][e] = t.at(k, i, e);
        const int64_t row = r0 + set + k * sets, col = (int64_t)(lane + i * G) * VEC;
        if (RES != kNone && row < a.rows && col < D) stv(static_cast<S*>(a.s) + row * D + col, c[k][i]);
        if (i == 0) {
#pragma unroll
          for (int e = 0; e < VEC; ++e) acc[e] = c[k][0][e];
        } else {
          add_up(acc, c[k][i]);
        }
      }
      sum[k] = total(acc);
    }
    group_sum(sum, G, sh);
#pragma unroll
    for (int k = 0; k < R; ++k) {
      sum[k] *= inv;
      float acc[VEC];
#pragma unroll
      for (int e = 0; e < VEC; ++e) acc[e] = 0.f;
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        add_to(c[k][i], -sum[k]);
        if ((int64_t)(lane + i * G) * VEC < D) fma_up(acc, c[k][i], c[k][i]);
      }
      sq[k] = total(acc);
    }
    group_sum(sq, G, sh);
#pragma unroll
    for (int k = 0; k < R; ++k) {
      const int64_t row = r0 + set + k * sets;
      if (row >= a.rows) continue;
      const float rstd = rsqrtf(fmaf(sq[k], inv, a.eps));
      if (a.mean && lane == 0) {
        a.mean[row] = sum[k];
        a.rstd[row] = rstd;
      }
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int64_t col = (int64_t)(lane + i * G) * VEC;
        if (col >= D) continue;
        scale_by(c[k][i], rstd);
        fma_by(c[k][i], w[i], b[i]);
        stv(static_cast<T*>(a.y) + row * D + col, c[k][i]);
      }
    }
    if constexpr (kAhead) t = next;
  }
}

// What one turn of the backward reads: R rows of a group
template <typename T, typename S, int RES, int VEC, int NV, int R>
struct Turn {
  Raw<S, VEC> s[R][NV];
  Raw<T, VEC> dy[R][NV];
  Raw<S, VEC> ds[RES == kNone ? 1 : R][RES == kNone ? 1 : NV];
  float mean[R], rstd[R];
  GDN2_DEV void load(const gdn2_layer_norm_args& a, const gdn2_layer_norm_grads& g, int64_t row0, int sets, int lane,
                     int G) {
#pragma unroll
    for (int k = 0; k < R; ++k) {
      const int64_t row = row0 + k * sets;
      const bool row_in = row < a.rows;
      mean[k] = row_in ? a.mean[row] : 0.f;
      rstd[k] = row_in ? a.rstd[row] : 0.f;
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int64_t c = (int64_t)(lane + i * G) * VEC, at = row * a.D + c;
        const bool in = row_in && c < a.D;
        if (in) s[k][i].load(static_cast<const S*>(g.s) + at);
        else s[k][i].zero();
        if (in) dy[k][i].load(static_cast<const T*>(g.dy) + at);
        else dy[k][i].zero();
        if constexpr (RES != kNone) {
          if (in && g.ds) ds[k][i].load(static_cast<const S*>(g.ds) + at);
          else ds[k][i].zero();
        }
      }
    }
  }
};

template <typename T, int RES, int VEC, int NV, int R, bool kAhead>
__global__ void __launch_bounds__((kMaxThreads<VEC, NV>))
layer_norm_bwd_kernel(const gdn2_layer_norm_args a, const gdn2_layer_norm_grads g, int G, bool vecw, float* part) {
  using S = typename ResType<T, RES>::type;
  extern __shared__ float cols[];  // [2][D] when several rows share the CTA
  __shared__ float sh[32][2 * R];
  const int lane = threadIdx.x % G, set = threadIdx.x / G, sets = blockDim.x / G;
  const int64_t D = a.D, stride = (int64_t)gridDim.x * sets * R;
  const float inv = 1.f / (float)D;
  float dw[NV][VEC], db[NV][VEC], w[NV][VEC];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int64_t c = (int64_t)(lane + i * G) * VEC;
#pragma unroll
    for (int e = 0; e < VEC; ++e) dw[i][e] = db[i][e] = 0.f;
    ldw(c < D ? a.weight : nullptr, c, a.dtype_weight, vecw, 1.f, w[i]);
  }
  const int64_t first = (int64_t)blockIdx.x * sets * R;  // (the loop's bounds are the CTA's: it has barriers)
  Turn<T, S, RES, VEC, NV, R> t;
  if (kAhead && first < a.rows) t.load(a, g, first + set, sets, lane, G);
  for (int64_t r0 = first; r0 < a.rows; r0 += stride) {
    [[maybe_unused]] Turn<T, S, RES, VEC, NV, R> next;
    if constexpr (kAhead) {
      if (r0 + stride < a.rows) next.load(a, g, r0 + stride + set, sets, lane, G);
    } else {
      t.load(a, g, r0 + set, sets, lane, G);
    }
    float hat[R][NV][VEC], d[R][NV][VEC], sum[2 * R];
#pragma unroll
    for (int k = 0; k < R; ++k) {
      float s0[VEC], s1[VEC];
#pragma unroll
      for (int e = 0; e < VEC; ++e) s0[e] = s1[e] = 0.f;
#pragma unroll
      for (int i = 0; i < NV; ++i) {  // (zeros past the row's end and the last row add nothing)
#pragma unroll
        for (int e = 0; e < VEC; ++e) hat[k][i][e] = t.s[k][i][e], d[k][i][e] = t.dy[k][i][e];
        add_to(hat[k][i], -t.mean[k]);
        scale_by(hat[k][i], t.rstd[k]);
        fma_up(dw[i], d[k][i], hat[k][i]);
        add_up(db[i], d[k][i]);
        mul_by(d[k][i], w[i]);
        add_up(s0, d[k][i]);
        fma_up(s1, d[k][i], hat[k][i]);
      }
      sum[2 * k] = total(s0);
      sum[2 * k + 1] = total(s1);
    }
    group_sum(sum, G, sh);
#pragma unroll
    for (int k = 0; k < R; ++k) {
      const int64_t row = r0 + set + k * sets;
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int64_t c = (int64_t)(lane + i * G) * VEC;
        if (row >= a.rows || c >= D) continue;
        add_to(d[k][i], -sum[2 * k] * inv);
        fma_to(d[k][i], hat[k][i], -sum[2 * k + 1] * inv);
        scale_by(d[k][i], t.rstd[k]);
        if constexpr (RES != kNone) {
          float y[VEC];
#pragma unroll
          for (int e = 0; e < VEC; ++e) y[e] = t.ds[k][i][e];
          add_up(d[k][i], y);
        }
        if (g.dx) stv(static_cast<T*>(g.dx) + row * D + c, d[k][i]);
        if (RES != kNone && g.dresidual) stv(static_cast<S*>(g.dresidual) + row * D + c, d[k][i]);
      }
    }
    if constexpr (kAhead) t = next;
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

// dw, db: the CTAs' sums in order; a CTA per 32 columns, its 16 warps a strided share of the CTAs each
__global__ void __launch_bounds__(512) layer_norm_sum_kernel(const float* part, int n, int64_t D, void* dw, void* db,
                                                             int dtype) {
  __shared__ float sh[16][32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t c = (int64_t)blockIdx.x * 32 + lane;  // over [dw | db]
  float x = 0.f;
  if (c < 2 * D)
#pragma unroll 8
    for (int i = warp; i < n; i += 16) x += part[(int64_t)i * 2 * D + c];
  sh[warp][lane] = x;
  __syncthreads();
  if (warp == 0 && c < 2 * D) {
    x = 0.f;
#pragma unroll
    for (int i = 0; i < 16; ++i) x += sh[i][lane];
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

// One vector per thread up to 256 threads a row, then two or four, then 512
// threads.  A row of more than a warp takes whole warps, not a power of two.
Plan plan(const gdn2_layer_norm_args& a, bool vec) {
  const int per = vec ? (a.dtype == GDN2_BF16 ? 8 : 4) : 1;
  const int64_t units = (a.D + per - 1) / per;
  Plan p{vec, vec ? 1 : 4, 8, 0};
  if (units > 1024) {
    p.G = p.threads = 512;
    p.NV = vec ? 64 / per : units <= 4096 ? 8 : units <= 8192 ? 16 : 64;
    return p;
  }
  if (vec) p.NV = units <= 256 ? 1 : units <= 512 ? 2 : 4;
  const int threads = (int)((units + p.NV - 1) / p.NV);
  while (p.G < threads && p.G < 32) p.G *= 2;
  if (threads > 32) p.G = (threads + 31) / 32 * 32;
  p.threads = 256 / p.G * p.G;
  return p;
}

bool aligned(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// Rows side by side in a thread: four where a row is a warp's or less; `wide`
// (fewer barriers per row) where it is a CTA's, one vector per thread, and
// there are rows enough for every CTA to walk several turns.
int rows_per_group(const gdn2_layer_norm_args& a, const Plan& p, int wide) {
  if (!p.vec) return 1;
  if (p.G <= 32) return 4;
  return p.NV == 1 && a.rows >= (int64_t)kLaSms * 16 * (p.threads / p.G) ? wide : 1;
}

int ctas(const gdn2_layer_norm_args& a, const Plan& p, int rows, int per_sm) {
  const int64_t per = (int64_t)(p.threads / p.G) * rows, need = (a.rows + per - 1) / per;
  const int64_t most = kLaSms * (p.threads > 256 ? 2 : per_sm);
  return need < 1 ? 1 : (int)(need < most ? need : most);
}
// CTAs per SM: forward 6, backward 4 (16384 x 2048 with a residual, with 3 / 4 / 6
// of them: forward 62 / 70 / 61 us, backward 109 / 94 / 100 us).  Chosen on that shape
// and used for all: where registers hold fewer, as for short rows, a part of the CTAs starts later.
constexpr int kFwdCtas = 6, kBwdCtas = 4;
int bwd_rows(const gdn2_layer_norm_args& a, const Plan& p) { return rows_per_group(a, p, a.residual ? 1 : 2); }
int bwd_ctas(const gdn2_layer_norm_args& a, const Plan& p) { return ctas(a, p, bwd_rows(a, p), kBwdCtas); }

template <typename T, int RES>
int fwd(const gdn2_layer_norm_args& a, const Plan& p, bool vecw, cudaStream_t s) {
  constexpr int kWide = RES == kNone ? 4 : 2;
  const int rows = rows_per_group(a, p, kWide), n = ctas(a, p, rows, kFwdCtas);
  constexpr int VEC = sizeof(T) == 2 ? 8 : 4;
  ProfScope ps(kKLayerNormFwd, s);
#define LN_FWD(V, N, R, A) layer_norm_fwd_kernel<T, RES, V, N, R, A><<<n, p.threads, 0, s>>>(a, p.G, vecw)
  if (p.vec) {
    if (p.threads == 512) LN_FWD(VEC, 64 / VEC, 1, false);
    else if (p.G <= 32) LN_FWD(VEC, 1, 4, true);
    else if (p.NV == 1 && rows == kWide) LN_FWD(VEC, 1, kWide, true);
    else if (p.NV == 1) LN_FWD(VEC, 1, 1, true);
    else if (p.NV == 2) LN_FWD(VEC, 2, 1, true);
    else LN_FWD(VEC, 4, 1, true);
  } else {
    if (p.NV == 4) LN_FWD(1, 4, 1, true);
    else if (p.NV == 8) LN_FWD(1, 8, 1, true);
    else if (p.NV == 16) LN_FWD(1, 16, 1, true);
    else LN_FWD(1, 64, 1, false);
  }
#undef LN_FWD
  GDN2_LAUNCH_CHECK();
  return 0;
}

template <typename T, int RES>
int bwd(const gdn2_layer_norm_args& a, const gdn2_layer_norm_grads& g, const Plan& p, bool vecw, float* part,
        cudaStream_t s) {
  constexpr int kWide = RES == kNone ? 2 : 1;
  const int rows = bwd_rows(a, p), n = bwd_ctas(a, p);
  const size_t sm = p.threads / p.G > 1 ? 2 * a.D * 4 : 0;
  constexpr int VEC = sizeof(T) == 2 ? 8 : 4;
  {
    ProfScope ps(kKLayerNormBwd, s);
#define LN_BWD(V, N, R, A) layer_norm_bwd_kernel<T, RES, V, N, R, A><<<n, p.threads, sm, s>>>(a, g, p.G, vecw, part)
    if (p.vec) {
      if (p.threads == 512) LN_BWD(VEC, 64 / VEC, 1, false);
      else if (p.G <= 32) LN_BWD(VEC, 1, 4, false);
      else if (p.NV == 1 && rows == kWide) LN_BWD(VEC, 1, kWide, true);
      else if (p.NV == 1) LN_BWD(VEC, 1, 1, true);
      else if (p.NV == 2) LN_BWD(VEC, 2, 1, true);
      else LN_BWD(VEC, 4, 1, false);
    } else {
      if (p.NV == 4) LN_BWD(1, 4, 1, true);
      else if (p.NV == 8) LN_BWD(1, 8, 1, false);
      else if (p.NV == 16) LN_BWD(1, 16, 1, false);
      else LN_BWD(1, 64, 1, false);
    }
#undef LN_BWD
    GDN2_LAUNCH_CHECK();
  }
  if (part) {
    layer_norm_sum_kernel<<<(unsigned)((2 * a.D + 31) / 32), 512, 0, s>>>(part, n, a.D, g.dweight, g.dbias,
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
  const bool vw = vec && aligned(a.weight) && aligned(a.bias);
  if (a.dtype == GDN2_F32) return a.residual ? fwd<float, kSame>(a, p, vw, s) : fwd<float, kNone>(a, p, vw, s);
  if (!a.residual) return fwd<__nv_bfloat16, kNone>(a, p, vw, s);
  return a.dtype_residual == GDN2_F32 ? fwd<__nv_bfloat16, kF32>(a, p, vw, s) : fwd<__nv_bfloat16, kSame>(a, p, vw, s);
}

size_t layer_norm_bwd_ws(const gdn2_layer_norm_args& a) {
  const int v = bwd_ctas(a, plan(a, true)), n = bwd_ctas(a, plan(a, false));
  return (size_t)(v > n ? v : n) * 2 * (size_t)a.D * 4;
}

int layer_norm_bwd_launch(const gdn2_layer_norm_args& a, const gdn2_layer_norm_grads& g, void* ws, cudaStream_t s) {
  const bool vec = a.D % (a.dtype == GDN2_BF16 ? 8 : 4) == 0 && aligned(g.s) && aligned(g.dy) && aligned(g.ds) &&
                   aligned(g.dx) && aligned(g.dresidual);
  const Plan p = plan(a, vec);
  const bool vw = vec && aligned(a.weight);
  float* part = (g.dweight || g.dbias) ? static_cast<float*>(ws) : nullptr;
  if (a.dtype == GDN2_F32) return a.residual ? bwd<float, kSame>(a, g, p, vw, part, s) : bwd<float, kNone>(a, g, p, vw, part, s);
  if (!a.residual) return bwd<__nv_bfloat16, kNone>(a, g, p, vw, part, s);
  return a.dtype_residual == GDN2_F32 ? bwd<__nv_bfloat16, kF32>(a, g, p, vw, part, s)
                                      : bwd<__nv_bfloat16, kSame>(a, g, p, vw, part, s);
}

}  // namespace gdn2
