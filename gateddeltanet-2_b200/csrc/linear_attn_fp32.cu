// Linear attention with a decay for each head, fp32 arithmetic throughout
// (the fp32 path).  With G the running sum of g inside a chunk of C = 64
// tokens and S, dS' the state entering and the state cotangent leaving it:
//     P_ij = e^{G_i - G_j} (q_i . k_j),  E_ij = e^{G_i - G_j} (do_i . v_j)   (i >= j)
//     o  = scale (P v + e^G q S)          S' = e^{G_C} S + sum_j e^{G_C - G_j} k_j v_j^T
//     dq = scale (E k + e^G do S^T)       dk = scale E^T q + e^{G_C - G} v dS'^T
//     dv = scale P^T do + e^{G_C - G} k dS'
//     dS = e^{G_C} dS' + scale sum_i e^{G_i} q_i do_i^T
//     dg_t = sum_{i>=t} (sum_{j<i} M_ij + q_i . dq_i^inter) - sum_{j>=t} sum_{i>j} M_ij
//            + sum_{j<t} k_j . dk_j^inter + e^{G_C} <S, dS'>,   M = scale P E / e^{G_i - G_j}
// (the diagonal of M cancels and is left out, so a token that no decay acts
// on gets an exact zero).  Three steps each way: every chunk's own state term,
// a running sum of those over the chunks of a sequence, and every chunk's
// outputs.  Running sums of g and their differences are held in fp64: their
// exponentials then carry only their own rounding, however long or strong the decay.
// Measured, both directions: 2 x 1000 tokens, 4 heads of 64 (128 CTAs of one wave) 75 us
// in six launches, 4 x 4096 tokens, 16 heads of 128, 3.3 ms; with operands loaded word by
// word 107 us and 5.0 ms.  That is 12 and 25 TFLOP/s of these kernels' own 0.9 and 82 GFLOP,
// a sixth and a third of the CUDA cores' fp32 rate: a product of 64 x 64 x 64 takes 16 FMAs
// a step of k in each of 256 threads, for 3 to 5 wavefronts of operands, every phase ends
// at a barrier, and one CTA an SM (205 KB of tiles at K = V = 128) has nothing to run
// while it loads the next half of a state.
#include "linear_attn.cuh"
#include "profile.cuh"

namespace gdn2 {
namespace {

constexpr int kC = kLaChunkF32;
constexpr int kThreads = 256;
constexpr int kPad = 4;  // rows of tiles stay on 16 bytes, and 8 of them start in 8 groups of banks
constexpr int kLdP = kC + kPad;

// acc[r][c] += sum_k A(4 ty + r, k) B(k, tx + 16 c), four k at a time.  kAt: A is
// stored k by rows (row k holds all i), else i by rows; kBt: B is stored column by
// column (row j holds all k), else k by rows.  What lies along a row is loaded 16 bytes at a
// time: 3 or 5 shared-memory wavefronts a step of k instead of 8 of single words.
template <bool kAt, bool kBt, int NJ>
GDN2_DEV void tile_mm(float (&acc)[4][NJ], const float* A, int lda, const float* B, int ldb, int kdim) {
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  A += kAt ? 4 * ty : 4 * ty * lda;
  B += kBt ? tx * ldb : tx;
#pragma unroll 2
  for (int k = 0; k < kdim; k += 4) {
    float x[4][4], y[NJ][4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const float4 v = *reinterpret_cast<const float4*>(kAt ? A + (k + u) * lda : A + u * lda + k);
      const float w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
      for (int e = 0; e < 4; ++e) (kAt ? x[e][u] : x[u][e]) = w[e];
    }
#pragma unroll
    for (int c = 0; c < NJ; ++c) {
      if constexpr (kBt) {
        const float4 v = *reinterpret_cast<const float4*>(B + 16 * c * ldb + k);
        y[c][0] = v.x; y[c][1] = v.y; y[c][2] = v.z; y[c][3] = v.w;
      } else {
#pragma unroll
        for (int u = 0; u < 4; ++u) y[c][u] = B[(k + u) * ldb + 16 * c];
      }
    }
#pragma unroll
    for (int u = 0; u < 4; ++u)
#pragma unroll
      for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int c = 0; c < NJ; ++c) acc[r][c] = fmaf(x[r][u], y[c][u], acc[r][c]);
  }
}

template <int NJ>
GDN2_DEV void zero(float (&acc)[4][NJ]) {
#pragma unroll
  for (int r = 0; r < 4; ++r)
#pragma unroll
    for (int c = 0; c < NJ; ++c) acc[r][c] = 0.f;
}

// L rows of D elements (row stride st, 16-byte steps) into a padded tile, zero rows after them; all loads at once
template <int D>
GDN2_DEV void load_rows(float* dst, const float* src, int64_t st, int L) {
  constexpr int kEach = kC * D / 4 / kThreads;
  float4 x[kEach];
#pragma unroll
  for (int e = 0; e < kEach; ++e) {
    const int i = threadIdx.x + e * kThreads, r = i / (D / 4), c = i % (D / 4) * 4;
    x[e] = r < L ? *reinterpret_cast<const float4*>(src + r * st + c) : make_float4(0.f, 0.f, 0.f, 0.f);
  }
#pragma unroll
  for (int e = 0; e < kEach; ++e) {
    const int i = threadIdx.x + e * kThreads, r = i / (D / 4), c = i % (D / 4) * 4;
    *reinterpret_cast<float4*>(dst + r * (D + kPad) + c) = x[e];
  }
}
// ROWS rows of 64 or more columns of a state with V columns
template <int ROWS, int COLS>
GDN2_DEV void load_state(float* dst, const float* src, int V) {
  constexpr int kEach = ROWS * COLS / 4 / kThreads;
  float4 x[kEach];
#pragma unroll
  for (int e = 0; e < kEach; ++e) {
    const int i = threadIdx.x + e * kThreads, r = i / (COLS / 4), c = i % (COLS / 4) * 4;
    x[e] = *reinterpret_cast<const float4*>(src + (int64_t)r * V + c);
  }
#pragma unroll
  for (int e = 0; e < kEach; ++e) {
    const int i = threadIdx.x + e * kThreads, r = i / (COLS / 4), c = i % (COLS / 4) * 4;
    *reinterpret_cast<float4*>(dst + r * (COLS + kPad) + c) = x[e];
  }
}

// running sums of the chunk's log-decays (warp 0; two tokens per lane)
GDN2_DEV void chunk_sums(double* G, const LaDecay& d, int64_t b, int64_t t0, int64_t hv, int L) {
  if (threadIdx.x < 32) {
    const int lane = threadIdx.x;
    const double x0 = 2 * lane < L ? d.at(b, t0 + 2 * lane, hv) : 0.0;
    const double x1 = 2 * lane + 1 < L ? d.at(b, t0 + 2 * lane + 1, hv) : 0.0;
    double s = x0 + x1;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const double y = __shfl_up_sync(0xffffffffu, s, o);
      if (lane >= o) s += y;
    }
    const double before = __shfl_up_sync(0xffffffffu, s, 1);
    G[2 * lane] = (lane ? before : 0.0) + x0;
    G[2 * lane + 1] = s;
  }
}

struct Where {
  int64_t n, c, b, t0, tok0;  // sequence, chunk in it, batch row, first token in that row, and over all rows
  int L;
};
GDN2_DEV bool locate(const LaGeom& geo, int64_t id, Where& w) {
  if (!geo.chunk(id, w.n, w.c)) return false;
  int64_t bos, len;
  geo.seq(w.n, bos, len);
  const int64_t left = len - w.c * kC;
  w.L = (int)min(left, (int64_t)kC);
  w.tok0 = bos + w.c * kC;
  w.b = geo.cu ? 0 : w.n;
  w.t0 = geo.cu ? w.tok0 : w.c * kC;
  return w.L > 0;
}

// One chunk's own term of the state recurrence, sum_t w_t x_t y_t^T: forward
// x = k, y = v, w_t = e^{G_C - G_t}; backward x = q, y = do, w_t = scale e^{G_t}.
// 8 x 8 (or smaller) outputs per thread.
template <int K, int V, bool kBack>
__global__ void __launch_bounds__(kThreads) la_state_kernel(const float* x, int64_t xb, int64_t xt, int64_t xh, const float* y,
                                                            int64_t yb, int64_t yt, int64_t yh, LaDecay dec,
                                                            LaGeom geo, int HV, int group, float scale, float* states,
                                                            float* total) {
  extern __shared__ __align__(16) float sm[];
  float* X = sm;
  float* Y = X + kC * (K + kPad);
  __shared__ double G[kC];
  __shared__ float weight[kC];
  Where w;
  const int hv = blockIdx.y;
  if (!locate(geo, blockIdx.x, w)) return;
  load_rows<K>(X, x + w.b * xb + w.t0 * xt + (hv / group) * xh, xt, w.L);
  load_rows<V>(Y, y + w.b * yb + w.t0 * yt + hv * yh, yt, w.L);
  chunk_sums(G, dec, w.b, w.t0, hv, w.L);
  __syncthreads();
  if (threadIdx.x == 0 && total) total[(int64_t)blockIdx.x * HV + hv] = expf((float)G[kC - 1]);
  if (threadIdx.x < kC)
    weight[threadIdx.x] =
        kBack ? scale * expf((float)G[threadIdx.x]) : expf((float)(G[kC - 1] - G[threadIdx.x]));
  __syncthreads();
  constexpr int R = K / 16, NJ = V / 16;
  float acc[R][NJ];
#pragma unroll
  for (int r = 0; r < R; ++r)
#pragma unroll
    for (int c = 0; c < NJ; ++c) acc[r][c] = 0.f;
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
#pragma unroll 4
  for (int t = 0; t < w.L; ++t) {
    float a[R], bb[NJ];
#pragma unroll
    for (int r = 0; r < R; r += 4) {
      const float4 x = *reinterpret_cast<const float4*>(X + t * (K + kPad) + R * ty + r);
      a[r] = x.x; a[r + 1] = x.y; a[r + 2] = x.z; a[r + 3] = x.w;
    }
    const float f = weight[t];
#pragma unroll
    for (int c = 0; c < NJ; ++c) bb[c] = f * Y[t * (V + kPad) + tx + 16 * c];
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
      for (int c = 0; c < NJ; ++c) acc[r][c] = fmaf(a[r], bb[c], acc[r][c]);
  }
  float* dst = states + ((int64_t)blockIdx.x * HV + hv) * K * V;
#pragma unroll
  for (int r = 0; r < R; ++r)
#pragma unroll
    for (int c = 0; c < NJ; ++c) dst[(R * ty + r) * V + tx + 16 * c] = acc[r][c];
}

// The running sum over a sequence's chunks, in place: states[c] becomes the
// state entering chunk c (forward), or the cotangent leaving it (backward, from
// the last chunk).  Four elements per thread; the loads of kAhead chunks are in flight.
template <bool kBack>
__global__ void __launch_bounds__(128) la_prefix_kernel(float* states, const float* total, const float* init, float* fin,
                                                        LaGeom geo, int HV, int64_t KV) {
  constexpr int kAhead = 8;
  const int64_t nh = blockIdx.x, n = nh / HV, hv = nh % HV;
  const int64_t e = ((int64_t)blockIdx.y * 128 + threadIdx.x) * 4;
  if (e >= KV) return;
  int64_t bos, len;
  geo.seq(n, bos, len);
  const int64_t nch = geo.chunks(n, len), c0 = geo.chunk0(n);
  float4 s = init ? *reinterpret_cast<const float4*>(init + nh * KV + e) : make_float4(0.f, 0.f, 0.f, 0.f);
  for (int64_t i0 = 0; i0 < nch; i0 += kAhead) {
    float4 add[kAhead];
    float f[kAhead];
#pragma unroll
    for (int i = 0; i < kAhead; ++i)
      if (i0 + i < nch) {
        const int64_t c = c0 + (kBack ? nch - 1 - (i0 + i) : i0 + i);
        add[i] = *reinterpret_cast<const float4*>(states + (c * HV + hv) * KV + e);
        f[i] = total[c * HV + hv];
      }
#pragma unroll
    for (int i = 0; i < kAhead; ++i)
      if (i0 + i < nch) {
        const int64_t c = c0 + (kBack ? nch - 1 - (i0 + i) : i0 + i);
        *reinterpret_cast<float4*>(states + (c * HV + hv) * KV + e) = s;
        s.x = fmaf(s.x, f[i], add[i].x);
        s.y = fmaf(s.y, f[i], add[i].y);
        s.z = fmaf(s.z, f[i], add[i].z);
        s.w = fmaf(s.w, f[i], add[i].w);
      }
  }
  if (fin) *reinterpret_cast<float4*>(fin + nh * KV + e) = s;
}

template <int K, int V>
__global__ void __launch_bounds__(kThreads) la_out_kernel(gdn2_linear_attn_args a, LaDecay dec, LaGeom geo,
                                                          const float* states) {
  extern __shared__ __align__(16) float sm[];
  float* Q = sm;
  float* Kt = Q + kC * (K + kPad);
  float* Vt = Kt + kC * (K + kPad);
  float* P = Vt + kC * (V + kPad);
  float* S = P + kC * kLdP;  // 64 rows of the state at a time
  __shared__ double G[kC];
  Where w;
  const int64_t HV = a.HV, hv = blockIdx.y, h = hv / (HV / a.H);
  if (!locate(geo, blockIdx.x, w)) return;
  load_rows<K>(Q, static_cast<const float*>(a.q) + w.b * a.q_stride[0] + w.t0 * a.q_stride[1] + h * a.q_stride[2],
                  a.q_stride[1], w.L);
  load_rows<K>(Kt, static_cast<const float*>(a.k) + w.b * a.k_stride[0] + w.t0 * a.k_stride[1] + h * a.k_stride[2],
                  a.k_stride[1], w.L);
  load_rows<V>(Vt, static_cast<const float*>(a.v) + w.b * a.v_stride[0] + w.t0 * a.v_stride[1] + hv * a.v_stride[2],
                  a.v_stride[1], w.L);
  chunk_sums(G, dec, w.b, w.t0, hv, w.L);
  __syncthreads();
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  {
    float p[4][4];
    zero(p);
    tile_mm<false, true>(p, Q, K + kPad, Kt, K + kPad, K);
#pragma unroll
    for (int r = 0; r < 4; ++r)
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const int i = 4 * ty + r, j = tx + 16 * c;
        P[i * kLdP + j] = i >= j ? p[r][c] * expf((float)(G[i] - G[j])) : 0.f;
      }
  }
  constexpr int NJ = V / 16;
  float o[4][NJ];
  zero(o);
  const float* st = states + ((int64_t)blockIdx.x * HV + hv) * K * V;
  for (int k0 = 0; k0 < K; k0 += 64) {
    __syncthreads();
    load_state<64, V>(S, st + k0 * V, V);
    __syncthreads();
    tile_mm<false, false>(o, Q + k0, K + kPad, S, V + kPad, 64);
  }
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    const float f = expf((float)G[4 * ty + r]);
#pragma unroll
    for (int c = 0; c < NJ; ++c) o[r][c] *= f;
  }
  tile_mm<false, false>(o, P, kLdP, Vt, V + kPad, kC);
  float* out = static_cast<float*>(a.o);
#pragma unroll
  for (int r = 0; r < 4; ++r)
#pragma unroll
    for (int c = 0; c < NJ; ++c)
      if (4 * ty + r < w.L)
        out[((w.tok0 + 4 * ty + r) * HV + hv) * V + tx + 16 * c] = a.scale * o[r][c];
}

// sum over the 16 threads tx of a row group; every one of them gets it
GDN2_DEV float row_sum(float x) {
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
  return x;
}

// One CTA per (chunk, key head): the value heads of the group one after the
// other, their shares of dq and dk added up in registers.
template <int K, int V>
__global__ void __launch_bounds__(kThreads) la_bwd_kernel(gdn2_linear_attn_args a, gdn2_linear_attn_grads gr,
                                                          LaDecay dec, LaGeom geo, const float* states,
                                                          const float* dstates, float* dgf) {
  extern __shared__ __align__(16) float sm[];
  float* Q = sm;
  float* Kt = Q + kC * (K + kPad);
  float* Vt = Kt + kC * (K + kPad);
  float* D = Vt + kC * (V + kPad);
  float* P = D + kC * (V + kPad);
  float* E = P + kC * kLdP;
  float* S = E + kC * kLdP;  // half of a state, 64 rows, or 64 columns
  __shared__ double G[kC];
  __shared__ float colw[8][kC], rows[kC], qint[kC], kint[kC], wsum[8];
  Where w;
  const int64_t H = a.H, HV = a.HV, h = blockIdx.y;
  const int group = (int)(HV / H);
  if (!locate(geo, blockIdx.x, w)) return;
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  constexpr int NK = K / 16, NV = V / 16;
  const bool want_dg = gr.dg != nullptr;
  float dq[4][NK], dk[4][NK];
  zero(dq);
  zero(dk);
  load_rows<K>(Q, static_cast<const float*>(a.q) + w.b * a.q_stride[0] + w.t0 * a.q_stride[1] + h * a.q_stride[2],
                  a.q_stride[1], w.L);
  load_rows<K>(Kt, static_cast<const float*>(a.k) + w.b * a.k_stride[0] + w.t0 * a.k_stride[1] + h * a.k_stride[2],
                  a.k_stride[1], w.L);
  for (int j = 0; j < group; ++j) {
    const int64_t hv = h * group + j;
    __syncthreads();
    load_rows<V>(Vt, static_cast<const float*>(a.v) + w.b * a.v_stride[0] + w.t0 * a.v_stride[1] + hv * a.v_stride[2],
                    a.v_stride[1], w.L);
    load_rows<V>(D, static_cast<const float*>(gr.dout) + (w.tok0 * HV + hv) * V, HV * V, w.L);
    chunk_sums(G, dec, w.b, w.t0, hv, w.L);
    __syncthreads();
    const float* st = states + ((int64_t)blockIdx.x * HV + hv) * K * V;
    const float* dst = dstates + ((int64_t)blockIdx.x * HV + hv) * K * V;
    const double GC = G[kC - 1];
    {
      float p[4][4], e[4][4], col[4] = {0.f, 0.f, 0.f, 0.f};
      zero(p);
      zero(e);
      tile_mm<false, true>(p, Q, K + kPad, Kt, K + kPad, K);
      tile_mm<false, true>(e, D, V + kPad, Vt, V + kPad, V);
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        float row = 0.f;
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          const int i = 4 * ty + r, jj = tx + 16 * c;
          const float f = i >= jj ? a.scale * expf((float)(G[i] - G[jj])) : 0.f;
          P[i * kLdP + jj] = i >= jj ? p[r][c] * f : 0.f;
          E[i * kLdP + jj] = i >= jj ? e[r][c] * f : 0.f;
          if (i > jj) {
            const float m = p[r][c] * e[r][c] * f;
            row += m;
            col[c] += m;
          }
        }
        if (want_dg) {
          row = row_sum(row);
          if (tx == 0) rows[4 * ty + r] = row;
        }
      }
      if (want_dg) {
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          const float x = col[c] + __shfl_xor_sync(0xffffffffu, col[c], 16);
          if (lane < 16) colw[warp][tx + 16 * c] = x;
        }
      }
    }
    {  // dv = e^{G_C - G} k dS' + P^T do
      float acc[4][NV];
      zero(acc);
      for (int k0 = 0; k0 < K; k0 += 64) {
        __syncthreads();
        load_state<64, V>(S, dst + k0 * V, V);
        __syncthreads();
        tile_mm<false, false>(acc, Kt + k0, K + kPad, S, V + kPad, 64);
      }
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const float f = expf((float)(GC - G[4 * ty + r]));
#pragma unroll
        for (int c = 0; c < NV; ++c) acc[r][c] *= f;
      }
      tile_mm<true, false>(acc, P, kLdP, D, V + kPad, kC);
      float* out = static_cast<float*>(gr.dv);
#pragma unroll
      for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int c = 0; c < NV; ++c)
          if (4 * ty + r < w.L) out[((w.tok0 + 4 * ty + r) * HV + hv) * V + tx + 16 * c] = acc[r][c];
    }
    {  // dq += scale e^G do S^T + E k
      float acc[4][NK];
      zero(acc);
      for (int v0 = 0; v0 < V; v0 += 64) {
        __syncthreads();
        load_state<K, 64>(S, st + v0, V);
        __syncthreads();
        tile_mm<false, true>(acc, D + v0, V + kPad, S, 64 + kPad, 64);
      }
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const float f = a.scale * expf((float)G[4 * ty + r]);
        float x = 0.f;
#pragma unroll
        for (int c = 0; c < NK; ++c) {
          acc[r][c] *= f;
          x = fmaf(acc[r][c], Q[(4 * ty + r) * (K + kPad) + tx + 16 * c], x);
        }
        if (want_dg) {
          x = row_sum(x);
          if (tx == 0) qint[4 * ty + r] = x;
        }
      }
      tile_mm<false, false>(acc, E, kLdP, Kt, K + kPad, kC);
#pragma unroll
      for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int c = 0; c < NK; ++c) dq[r][c] += acc[r][c];
    }
    {  // dk += e^{G_C - G} v dS'^T + E^T q
      float acc[4][NK];
      zero(acc);
      for (int v0 = 0; v0 < V; v0 += 64) {
        __syncthreads();
        load_state<K, 64>(S, dst + v0, V);
        __syncthreads();
        tile_mm<false, true>(acc, Vt + v0, V + kPad, S, 64 + kPad, 64);
      }
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const float f = expf((float)(GC - G[4 * ty + r]));
        float x = 0.f;
#pragma unroll
        for (int c = 0; c < NK; ++c) {
          acc[r][c] *= f;
          x = fmaf(acc[r][c], Kt[(4 * ty + r) * (K + kPad) + tx + 16 * c], x);
        }
        if (want_dg) {
          x = row_sum(x);
          if (tx == 0) kint[4 * ty + r] = x;
        }
      }
      tile_mm<true, false>(acc, E, kLdP, Q, K + kPad, kC);
#pragma unroll
      for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int c = 0; c < NK; ++c) dk[r][c] += acc[r][c];
    }
    if (want_dg) {
      float x = 0.f;
#pragma unroll 4
      for (int i = threadIdx.x; i < K * V / 4; i += kThreads) {
        const float4 y = reinterpret_cast<const float4*>(st)[i], z = reinterpret_cast<const float4*>(dst)[i];
        x = fmaf(y.x, z.x, x);
        x = fmaf(y.y, z.y, x);
        x = fmaf(y.z, z.z, x);
        x = fmaf(y.w, z.w, x);
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
      if (lane == 0) wsum[warp] = x;
      __syncthreads();
      if (warp == 0) {  // two tokens per lane: sums to the chunk's end, and of kint from its start
        float x0 = 0.f, e[2], k[2];
#pragma unroll
        for (int i = 0; i < 8; ++i) x0 += wsum[i];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const int t = 2 * lane + u;
          float cs = 0.f;
#pragma unroll
          for (int ww = 0; ww < 8; ++ww) cs += colw[ww][t];
          e[u] = rows[t] + qint[t] - cs;
          k[u] = kint[t];
        }
        float after = e[0] + e[1], before = k[0] + k[1];
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const float y = __shfl_down_sync(0xffffffffu, after, o), z = __shfl_up_sync(0xffffffffu, before, o);
          if (lane + o < 32) after += y;
          if (lane >= o) before += z;
        }
        after = __shfl_down_sync(0xffffffffu, after, 1);
        before = __shfl_up_sync(0xffffffffu, before, 1);
        const float base = expf((float)GC) * x0 + (lane < 31 ? after : 0.f) + (lane ? before : 0.f) + e[1];
        const float d[2] = {base + e[0], base + k[0]};
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const int t = 2 * lane + u;
          if (t < w.L) {
            const int64_t at = (w.tok0 + t) * HV + hv;
            if (dgf) dgf[at] = d[u];
            else if (a.dtype_g == GDN2_BF16) static_cast<__nv_bfloat16*>(gr.dg)[at] = __float2bfloat16_rn(d[u]);
            else static_cast<float*>(gr.dg)[at] = d[u];
          }
        }
      }
    }
  }
  float* oq = static_cast<float*>(gr.dq);
  float* ok = static_cast<float*>(gr.dk);
#pragma unroll
  for (int r = 0; r < 4; ++r)
#pragma unroll
    for (int c = 0; c < NK; ++c)
      if (4 * ty + r < w.L) {
        const int64_t at = ((w.tok0 + 4 * ty + r) * H + h) * K + tx + 16 * c;
        oq[at] = dq[r][c];
        ok[at] = dk[r][c];
      }
}

// Gradient of one decay per head: the sum of its tokens' (fixed order).  A CTA a head, in
// steps of HV floats: 14 of a training step's 270 us at 4 x 4096 tokens, 16 heads of 128.
__global__ void __launch_bounds__(256) la_head_sum_kernel(const float* dg, int64_t tokens, int HV, void* out, int dtype,
                                                          LaGeom geo) {
  __shared__ double part[8];
  const int hv = blockIdx.x;
  double s = 0.0;
  for (int64_t n = 0; n < geo.N; ++n) {
    int64_t bos, len;
    geo.seq(n, bos, len);
    for (int64_t t = threadIdx.x; t < len; t += 256) s += dg[(bos + t) * HV + hv];
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = s;
  __syncthreads();
  if (threadIdx.x == 0) {
    s = 0.0;
    for (int i = 0; i < 8; ++i) s += part[i];
    if (dtype == GDN2_BF16) static_cast<__nv_bfloat16*>(out)[hv] = __float2bfloat16_rn((float)s);
    else static_cast<float*>(out)[hv] = (float)s;
  }
}

// (sequence, chunk) of every chunk id of a packed batch, and each sequence's
// first chunk; the same for segments, of which an empty sequence has one.  One
// CTA walks the lengths 1024 at a time with a block prefix sum.
GDN2_DEV void chunk_map(const LaGeom& geo, int64_t unit, int64_t least, LaChunk* map, int32_t* first, int64_t NT) {
  __shared__ int64_t warp_sum[32];
  __shared__ int64_t carry;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  if (tid == 0) carry = 0;
  __syncthreads();
  for (int64_t n0 = 0; n0 < geo.N; n0 += 1024) {
    const int64_t n = n0 + tid;
    int64_t bos = 0, len = 0;
    if (n < geo.N) geo.seq(n, bos, len);
    const int64_t nch = n < geo.N ? max((len + unit - 1) / unit, least) : 0;
    int64_t s = nch;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t y = __shfl_up_sync(0xffffffffu, s, o);
      if (lane >= o) s += y;
    }
    if (lane == 31) warp_sum[warp] = s;
    __syncthreads();
    int64_t base = carry;
    for (int i = 0; i < warp; ++i) base += warp_sum[i];
    if (n < geo.N) first[n] = (int32_t)min(base + s - nch, NT);
    __syncthreads();
    if (tid == 1023) carry = base + s;
    __syncthreads();
  }
  const int64_t all = min(carry, NT);
  if (tid == 0) first[geo.N] = (int32_t)all;
  __syncthreads();
  for (int64_t id = tid; id < NT; id += 1024) {
    LaChunk m{-1, 0};
    if (id < all) {  // the last sequence whose first chunk is <= id
      int64_t lo = 0, hi = geo.N;
      while (hi - lo > 1) {
        const int64_t mid = (lo + hi) / 2;
        if (first[mid] <= id) lo = mid;
        else hi = mid;
      }
      m.n = (int32_t)lo;
      m.c = (int32_t)(id - first[lo]);
    }
    map[id] = m;
  }
  __syncthreads();
}

// The entries of a scan, long ones first (a counting sort over 1024 classes of
// lengths; the order within one is of no consequence), so that the CTAs' turns
// through them add up to nearly the same; after them, how many are full.
GDN2_DEV void order_entries(const LaGeom& geo, const LaSegs& seg, int32_t* order) {
  __shared__ int32_t count[1024];
  __shared__ int32_t warp_sum[32];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  auto cls = [&](int64_t e) -> int {
    int64_t n, s, bos, len, chunks = 0;
    if (seg.get(e, geo, n, s)) {
      geo.seq(n, bos, len);
      chunks = max((len + geo.C - 1) / geo.C - s * seg.len, (int64_t)0);
    }
    return chunks >= seg.len ? 0 : 1 + (int)((seg.len - 1 - chunks) * 1022 / max(seg.len - 1, 1));
  };
  count[tid] = 0;
  __syncthreads();
  for (int64_t e = tid; e < seg.entries; e += 1024) atomicAdd(&count[cls(e)], 1);
  __syncthreads();
  const int32_t mine = count[tid];
  int32_t s = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int32_t y = __shfl_up_sync(0xffffffffu, s, o);
    if (lane >= o) s += y;
  }
  if (lane == 31) warp_sum[warp] = s;
  __syncthreads();
  for (int i = 0; i < warp; ++i) s += warp_sum[i];
  count[tid] = s - mine;
  if (tid == 0) order[seg.entries] = mine;
  __syncthreads();
  for (int64_t e = tid; e < seg.entries; e += 1024) order[atomicAdd(&count[cls(e)], 1)] = (int32_t)e;
}

// What a packed batch needs before its forward pass: CTA 0 lays out chunks and
// segments, the others clear rows.  (One launch: they are a few microseconds each.)
struct LaPacked {
  LaGeom geo;
  LaSegs seg;
  LaRows rows;
  LaChunk *map, *seg_map;  // or NULL
  int32_t *first, *seg_first, *order;
  int64_t NT;
};
__global__ void __launch_bounds__(1024) la_packed_kernel(LaPacked p) {
  if (blockIdx.x > 0) {
    zero_outside(p.rows, p.geo, blockIdx.x - 1, gridDim.x - 1);
    return;
  }
  if (p.map) chunk_map(p.geo, p.geo.C, 0, p.map, p.first, p.NT);
  if (p.seg_map) chunk_map(p.geo, (int64_t)p.geo.C * p.seg.len, 1, p.seg_map, p.seg_first, p.seg.entries);
  if (p.order) order_entries(p.geo, p.seg, p.order);
}
__global__ void __launch_bounds__(256) la_zero_outside_kernel(LaRows r, LaGeom geo) {
  zero_outside(r, geo, blockIdx.x, gridDim.x);
}

template <int K, int V>
int fwd(const gdn2_linear_attn_args& a, const LaWs& ws, cudaStream_t s) {
  const LaGeom geo = la_geom(a, ws);
  const LaDecay dec = la_decay(a);
  const int64_t NT = la_num_chunks(a);
  const int HV = (int)a.HV, group = (int)(a.HV / a.H);
  const float* h0 = (a.flags & GDN2_HAS_H0) ? a.h0 : nullptr;
  float* ht = (a.flags & GDN2_STORE_FINAL) ? a.ht : nullptr;
  ProfScope ps(kKLinAttnFp32, s);
  if (NT > 0) {
    const size_t sm = kC * (K + V + 2 * kPad) * 4;
    if (int st = (smem_opt_in<la_state_kernel<K, V, false>>(sm))) return st;
    la_state_kernel<K, V, false><<<dim3((unsigned)NT, HV), kThreads, sm, s>>>(
        static_cast<const float*>(a.k), a.k_stride[0], a.k_stride[1], a.k_stride[2], static_cast<const float*>(a.v),
        a.v_stride[0], a.v_stride[1], a.v_stride[2], dec, geo, HV, group, 1.f, ws.states, ws.total);
    GDN2_LAUNCH_CHECK();
  }
  la_prefix_kernel<false><<<dim3((unsigned)(a.N * HV), (K * V + 511) / 512), 128, 0, s>>>(ws.states, ws.total, h0, ht,
                                                                                          geo, HV, K * V);
  GDN2_LAUNCH_CHECK();
  if (NT > 0) {
    const size_t sm = (2 * kC * (K + kPad) + kC * (V + kPad) + kC * kLdP + 64 * (V + kPad)) * 4;
    if (int st = (smem_opt_in<la_out_kernel<K, V>>(sm))) return st;
    la_out_kernel<K, V><<<dim3((unsigned)NT, HV), kThreads, sm, s>>>(a, dec, geo, ws.states);
    GDN2_LAUNCH_CHECK();
  }
  return 0;
}

template <int K, int V>
int bwd(const gdn2_linear_attn_args& a, const gdn2_linear_attn_grads& gr, const LaWs& ws, const LaBwdWs& bw,
        cudaStream_t s) {
  const LaGeom geo = la_geom(a, ws);
  const LaDecay dec = la_decay(a);
  const int64_t NT = la_num_chunks(a);
  const int HV = (int)a.HV, group = (int)(a.HV / a.H);
  ProfScope ps(kKLinAttnFp32, s);
  if (NT > 0) {
    const size_t sm = kC * (K + V + 2 * kPad) * 4;
    if (int st = (smem_opt_in<la_state_kernel<K, V, true>>(sm))) return st;
    la_state_kernel<K, V, true><<<dim3((unsigned)NT, HV), kThreads, sm, s>>>(
        static_cast<const float*>(a.q), a.q_stride[0], a.q_stride[1], a.q_stride[2], static_cast<const float*>(gr.dout),
        a.T * HV * V, (int64_t)HV * V, V, dec, geo, HV, group, a.scale, bw.dstates, nullptr);
    GDN2_LAUNCH_CHECK();
  }
  la_prefix_kernel<true><<<dim3((unsigned)(a.N * HV), (K * V + 511) / 512), 128, 0, s>>>(
      bw.dstates, ws.total, gr.dht, gr.dh0, geo, HV, K * V);
  GDN2_LAUNCH_CHECK();
  if (NT > 0) {
    constexpr int half = 64 * (V + kPad) > K * (64 + kPad) ? 64 * (V + kPad) : K * (64 + kPad);
    const size_t sm = (2 * kC * (K + kPad) + 2 * kC * (V + kPad) + 2 * kC * kLdP + half) * 4;
    if (int st = (smem_opt_in<la_bwd_kernel<K, V>>(sm))) return st;
    la_bwd_kernel<K, V><<<dim3((unsigned)NT, (unsigned)a.H), kThreads, sm, s>>>(
        a, gr, dec, geo, ws.states, bw.dstates, a.decay == GDN2_DECAY_HEAD ? bw.dg : nullptr);
    GDN2_LAUNCH_CHECK();
  }
  return 0;
}

template <typename F>
int by_dims(const gdn2_linear_attn_args& a, F f) {
  if (a.K == 128) return a.V == 128 ? f.template operator()<128, 128>() : f.template operator()<128, 64>();
  return a.V == 128 ? f.template operator()<64, 128>() : f.template operator()<64, 64>();
}

struct FwdCall {
  const gdn2_linear_attn_args& a;
  const LaWs& ws;
  cudaStream_t s;
  template <int K, int V>
  int operator()() const { return fwd<K, V>(a, ws, s); }
};
struct BwdCall {
  const gdn2_linear_attn_args& a;
  const gdn2_linear_attn_grads& gr;
  const LaWs& ws;
  const LaBwdWs& bw;
  cudaStream_t s;
  template <int K, int V>
  int operator()() const { return bwd<K, V>(a, gr, ws, bw, s); }
};

}  // namespace

int la_fwd_launch(const gdn2_linear_attn_args& a, const LaWs& ws, cudaStream_t s) {
  const LaGeom geo = la_geom(a, ws);
  const bool any = a.B * a.T > 0;
  if (a.cu_seqlens) {
    const int64_t e = a.dtype == GDN2_BF16 ? 2 : 4;
    LaPacked p{geo, {}, {{any ? a.o : nullptr}, {a.HV * a.V * e}}, ws.map, nullptr, ws.first, nullptr, nullptr, la_num_chunks(a)};
    if (la_tc(a)) {
      p.seg = la_segs(a, ws.seg);
      p.seg_map = ws.seg.map;
      p.seg_first = ws.seg.first;
      p.order = ws.seg.order;
    }
    la_packed_kernel<<<33, 1024, 0, s>>>(p);
    GDN2_LAUNCH_CHECK();
  }
  if (!any) {  // no tokens: the final states are the initial ones
    if (!(a.flags & GDN2_STORE_FINAL)) return 0;
    const size_t bytes = (size_t)(a.N * a.HV * a.K * a.V) * 4;
    if (a.flags & GDN2_HAS_H0) GDN2_CUDA_TRY(cudaMemcpyAsync(a.ht, a.h0, bytes, cudaMemcpyDeviceToDevice, s));
    else GDN2_CUDA_TRY(cudaMemsetAsync(a.ht, 0, bytes, s));
    return 0;
  }
  if (la_tc(a)) return la_tc_fwd_launch(a, ws, s);
  return by_dims(a, FwdCall{a, ws, s});
}

int la_bwd_launch(const gdn2_linear_attn_args& a, const gdn2_linear_attn_grads& gr, const LaWs& ws,
                  const LaBwdWs& bw, cudaStream_t s) {
  if (a.B * a.T == 0) {
    const size_t bytes = (size_t)(a.N * a.HV * a.K * a.V) * 4;
    if (gr.dh0 && gr.dht) GDN2_CUDA_TRY(cudaMemcpyAsync(gr.dh0, gr.dht, bytes, cudaMemcpyDeviceToDevice, s));
    else if (gr.dh0) GDN2_CUDA_TRY(cudaMemsetAsync(gr.dh0, 0, bytes, s));
    if (gr.dg && a.decay == GDN2_DECAY_HEAD)
      GDN2_CUDA_TRY(cudaMemsetAsync(gr.dg, 0, (size_t)a.HV * (a.dtype_g == GDN2_BF16 ? 2 : 4), s));
    return 0;
  }
  if (a.cu_seqlens) {
    const int64_t e = a.dtype == GDN2_BF16 ? 2 : 4, eg = a.dtype_g == GDN2_BF16 ? 2 : 4;
    const bool token = a.decay == GDN2_DECAY_TOKEN;
    la_zero_outside_kernel<<<32, 256, 0, s>>>(LaRows{{gr.dq, gr.dk, gr.dv, token ? gr.dg : nullptr},
                                                     {a.H * a.K * e, a.H * a.K * e, a.HV * a.V * e, a.HV * eg}},
                                              la_geom(a, ws));
    GDN2_LAUNCH_CHECK();
  }
  if (la_tc(a)) {
    if (int st = la_tc_bwd_launch(a, gr, ws, bw, s)) return st;
  } else if (int st = by_dims(a, BwdCall{a, gr, ws, bw, s})) {
    return st;
  }
  if (gr.dg && a.decay == GDN2_DECAY_HEAD) {
    la_head_sum_kernel<<<(unsigned)a.HV, 256, 0, s>>>(bw.dg, a.B * a.T, (int)a.HV, gr.dg, a.dtype_g, la_geom(a, ws));
    GDN2_LAUNCH_CHECK();
  }
  return 0;
}

}  // namespace gdn2
