// Token-serial linear attention with a decay for each head (decoding):
//     S <- e^g S + k v^T,  o = scale S^T q
// One CTA holds a [K x VT] tile of one (sequence, value head) state in
// registers: read once, taken through the sequence's tokens, written once, so
// the bytes of the state are the whole cost.  A thread owns one float4 of
// columns in K / (threads / (VT / 4)) rows; all its loads are issued before
// anything waits on them.  o needs one reduction over the rows: each thread's
// own rows, the lanes of its warp that share its columns, then the warps
// through shared memory.  Tiles are 64 columns wide: 32 floats of state a thread
// at K = 128, four CTAs an SM.
// Bound by bandwidth: 256 sequences of 16 heads, K = V = 128 (541 MB) take 88 us,
// 6.15 TB/s; four sequences 8 us, which is the launch and one trip to memory and back.
// Several tokens: each one's q, k, v are loaded after the barrier that ends the token
// before, so a call of one sequence, 16 heads, takes 0.8 us a token (53 us for 64).
// The last CTAs of a packed batch clear the rows outside of every sequence.
#include "linear_attn.cuh"
#include "profile.cuh"

namespace gdn2 {
namespace {

constexpr int kThreads = 256;
constexpr int kClear = 32;  // CTAs that clear rows outside of packed sequences

template <typename T, int K, int VT>
__global__ void __launch_bounds__(kThreads)
la_recurrent_kernel(const gdn2_linear_attn_args a, const LaDecay dec, const LaGeom geo, unsigned tiles_in_all) {
  constexpr int kGroups = VT / 4;                 // float4 columns of the tile
  constexpr int kRowSets = kThreads / kGroups;    // threads that share a column
  constexpr int kRows = K / kRowSets;             // rows per thread
  __shared__ float s_q[K], s_k[K], s_v[VT];
  __shared__ float s_o[kThreads / 32][VT];
  __shared__ float s_decay;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int64_t V = a.V, HV = a.HV;
  if (blockIdx.x >= tiles_in_all) {  // packed batches: the last CTAs clear the rows that no sequence covers
    zero_outside(LaRows{{a.o}, {HV * V * (int64_t)sizeof(T)}}, geo, blockIdx.x - tiles_in_all, kClear);
    return;
  }
  const int tiles = (int)(V / VT);
  const int64_t nh = blockIdx.x / tiles, n = nh / HV, hv = nh % HV, h = hv / (HV / a.H);
  const int v0 = (int)(blockIdx.x % tiles) * VT;
  int64_t bos, len;
  geo.seq(n, bos, len);
  const int64_t b = geo.cu ? 0 : n, t0 = geo.cu ? bos : 0;
  const int cg = tid % kGroups, r0 = tid / kGroups;
  T* o = static_cast<T*>(a.o);

  int64_t slot = n;
  if (a.state_indices) {
    slot = a.state_indices[n];
    if (slot < 0 || slot >= a.num_slots) {  // a padding entry of the batch
      for (int64_t i = tid; i < len * VT; i += kThreads)
        o[((bos + i / VT) * HV + hv) * V + v0 + i % VT] = from_f<T>(0.f);
      return;
    }
  }
  float st[kRows][4];
  const bool load = a.flags & GDN2_HAS_H0;
  const float* src = a.h0 + slot * a.state_stride_in + hv * K * V + v0 + 4 * cg;
#pragma unroll
  for (int i = 0; i < kRows; ++i) {
    const float4 x = load ? *reinterpret_cast<const float4*>(src + (int64_t)(r0 + i * kRowSets) * V)
                          : make_float4(0.f, 0.f, 0.f, 0.f);
    st[i][0] = x.x; st[i][1] = x.y; st[i][2] = x.z; st[i][3] = x.w;
  }
  const T* q = static_cast<const T*>(a.q) + b * a.q_stride[0] + h * a.q_stride[2];
  const T* k = static_cast<const T*>(a.k) + b * a.k_stride[0] + h * a.k_stride[2];
  const T* v = static_cast<const T*>(a.v) + b * a.v_stride[0] + hv * a.v_stride[2] + v0;
  for (int64_t t = 0; t < len; ++t) {
    for (int i = tid; i < K; i += kThreads) {
      s_q[i] = a.scale * to_f(q[(t0 + t) * a.q_stride[1] + i]);
      s_k[i] = to_f(k[(t0 + t) * a.k_stride[1] + i]);
    }
    if (tid >= kThreads - VT) s_v[tid - (kThreads - VT)] = to_f(v[(t0 + t) * a.v_stride[1] + tid - (kThreads - VT)]);
    if (tid == 0) s_decay = expf((float)dec.at(b, t0 + t, hv));
    __syncthreads();
    const float d = s_decay;
    float vv[4], acc[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int e = 0; e < 4; ++e) vv[e] = s_v[4 * cg + e];
#pragma unroll
    for (int i = 0; i < kRows; ++i) {
      const float kr = s_k[r0 + i * kRowSets], qr = s_q[r0 + i * kRowSets];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        st[i][e] = fmaf(kr, vv[e], d * st[i][e]);
        acc[e] = fmaf(qr, st[i][e], acc[e]);
      }
    }
#pragma unroll
    for (int off = kGroups; off < 32; off <<= 1)
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[e] += __shfl_xor_sync(0xffffffffu, acc[e], off);
    if (lane < kGroups)
#pragma unroll
      for (int e = 0; e < 4; ++e) s_o[warp][4 * cg + e] = acc[e];
    __syncthreads();
    if (tid < VT) {
      float x = 0.f;
#pragma unroll
      for (int w = 0; w < kThreads / 32; ++w) x += s_o[w][tid];
      o[((bos + t) * HV + hv) * V + v0 + tid] = from_f<T>(x);
    }
    // the next token's vectors are written after this barrier's readers (s_q, s_k, s_v) are done
  }
  if (a.flags & GDN2_STORE_FINAL) {
    float* dst = a.ht + slot * a.state_stride_out + hv * K * V + v0 + 4 * cg;
#pragma unroll
    for (int i = 0; i < kRows; ++i)
      *reinterpret_cast<float4*>(dst + (int64_t)(r0 + i * kRowSets) * V) =
          make_float4(st[i][0], st[i][1], st[i][2], st[i][3]);
  }
}

template <typename T, int K, int VT>
int launch(const gdn2_linear_attn_args& a, cudaStream_t s) {
  const LaGeom geo{a.cu_seqlens, a.T, a.N, 1, a.T, nullptr, nullptr};
  ProfScope ps(kKLinAttnRec, s);
  const unsigned tiles = (unsigned)(a.N * a.HV * (a.V / VT));
  la_recurrent_kernel<T, K, VT><<<tiles + (a.cu_seqlens ? kClear : 0), kThreads, 0, s>>>(a, la_decay(a), geo, tiles);
  GDN2_LAUNCH_CHECK();
  return 0;
}

template <typename T>
int dispatch(const gdn2_linear_attn_args& a, cudaStream_t s) {
  if (a.K == 128) return launch<T, 128, 64>(a, s);
  return launch<T, 64, 64>(a, s);
}

}  // namespace

int la_recurrent_launch(const gdn2_linear_attn_args& a, cudaStream_t s) {
  return a.dtype == GDN2_F32 ? dispatch<float>(a, s) : dispatch<__nv_bfloat16>(a, s);
}

}  // namespace gdn2
