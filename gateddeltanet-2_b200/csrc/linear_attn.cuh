// Linear attention with a decay for each head: geometry, workspace layout and
// the launchers behind the gdn2_linear_attn_* entry points.
#pragma once

#include <algorithm>
#include <atomic>

#include "common.cuh"

namespace gdn2 {

constexpr int kLaChunkF32 = 64;   // tokens per chunk of the fp32 kernels
constexpr int kLaChunkTc = 128;   // and of the tensor-core kernels
// The shared-memory opt-in of a kernel, asked for once per device.
template <auto kKernel>
inline int smem_opt_in(size_t bytes) {
  static std::atomic<uint64_t> done{0};
  int dev = 0;
  GDN2_CUDA_TRY(cudaGetDevice(&dev));
  const uint64_t bit = dev < 64 ? uint64_t(1) << dev : 0;
  if (done.load(std::memory_order_relaxed) & bit) return 0;
  GDN2_CUDA_TRY(cudaFuncSetAttribute(kKernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes));
  done.fetch_or(bit, std::memory_order_relaxed);
  return 0;
}

constexpr int kLaSms = 148;       // CTAs of a persistent kernel: one per SM of a B200

// A chunk of a packed batch: its sequence (-1: past the last chunk) and its index there.
struct LaChunk {
  int32_t n, c;
};

struct LaGeom {
  const int64_t* cu;
  int64_t T, N;
  int C;              // tokens per chunk
  int64_t nts;        // chunks per sequence (dense)
  const LaChunk* map;   // [NT] (packed)
  const int32_t* first; // [N + 1] first chunk of each sequence (packed)

  // first row and length of sequence n, clipped to the tensor (packed rows: B == 1)
  GDN2_DEV void seq(int64_t n, int64_t& bos, int64_t& len) const {
    if (cu) {
      bos = min(max(cu[n], (int64_t)0), T);
      len = min(max(cu[n + 1], bos), T) - bos;
    } else {
      bos = n * T;
      len = T;
    }
  }
  GDN2_DEV int64_t chunk0(int64_t n) const { return cu ? (int64_t)first[n] : n * nts; }
  // chunks of sequence n (a packed batch needs `first`), as far as the buffers hold them: all of
  // them, unless offsets decrease and sequences overlap
  GDN2_DEV int64_t chunks(int64_t n, int64_t len) const {
    const int64_t all = (len + C - 1) / C;
    return cu ? min(all, (int64_t)(first[n + 1] - first[n])) : all;
  }
  // chunk id -> (sequence, chunk in it); false past the last chunk
  GDN2_DEV bool chunk(int64_t id, int64_t& n, int64_t& c) const {
    if (cu) {
      const LaChunk m = map[id];
      n = m.n;
      c = m.c;
      return n >= 0;
    }
    n = id / nts;
    c = id - n * nts;
    return true;
  }
};

// Sequences cut into segments of `len` chunks for the scans over time, so that
// few sequences and heads over a long axis still fill the GPU.
struct LaSegs {
  int len;              // chunks per segment
  bool multi;           // some sequence may have several
  bool cut;             // packed and cut: the entries are looked up in `map`
  int64_t per;          // segments per sequence (dense)
  int64_t entries;      // segments over all sequences (packed and cut: an upper bound)
  const LaChunk* map;   // [entries] (sequence, segment), packed and cut only
  const int32_t* first; // [N + 1] first entry of each sequence
  const int32_t* order; // [entries] long entries first, then how many hold `len` chunks; packed only
  float* X;             // [entries, HV, K, V] states, where cut
  float* D;             // [entries, HV] decay over the segment
  GDN2_DEV bool get(int64_t entry, const LaGeom&, int64_t& n, int64_t& s) const {
    if (map) {
      n = map[entry].n;
      s = map[entry].c;
      return n >= 0;
    }
    n = (uint32_t)entry / (uint32_t)per;
    s = entry - n * per;
    return true;
  }
  GDN2_DEV int64_t first_of(int64_t n) const { return map ? (int64_t)first[n] : n * per; }
  // segments of sequence n, as far as the buffers hold them
  GDN2_DEV int64_t count(int64_t n, int64_t chunks) const {
    const int64_t all = chunks > 0 ? (chunks + len - 1) / len : 1;
    return map ? min(all, (int64_t)(first[n + 1] - first[n])) : all;
  }
};

struct LaSegWs {
  LaChunk* map;
  int32_t* first;
  int32_t* order;
  float* X;
  float* D;
};

struct LaWs {
  LaChunk* map;     // [NT]   packed only
  int32_t* first;   // [N+1]  packed only
  float* total;     // [NT, HV] exp of each chunk's summed decay (fp32 kernels)
  float* states;    // [NT, HV, K, V] fp32 (fp32 kernels)
  __nv_bfloat16* states16;  // [NT, HV, K, V] bf16 (tensor-core kernels, for the backward)
  LaSegWs seg;
};
struct LaBwdWs {
  float* dstates;   // [NT, HV, K, V] fp32 (fp32 kernels)
  __nv_bfloat16* dstates16;  // [NT, HV, K, V] bf16 (tensor-core kernels)
  float* acc;       // [CTAs, 2, 128, K] running sums over a group of value heads (tensor-core kernels)
  LaSegWs seg;
  float* dg;        // [B, T, HV] fp32, the terms of a per-head decay's gradient
};

inline bool la_tc(const gdn2_linear_attn_args& a) { return a.dtype == GDN2_BF16; }
inline int la_chunk(const gdn2_linear_attn_args& a) { return la_tc(a) ? kLaChunkTc : kLaChunkF32; }

// chunks over all sequences: exact for dense batches, an upper bound for packed
// ones (the lengths stay on the device): sum ceil(len / C) <= T / C + N
inline int64_t la_num_chunks(const gdn2_linear_attn_args& a) {
  const int64_t C = la_chunk(a);
  return a.cu_seqlens ? a.T / C + a.N : a.B * ((a.T + C - 1) / C);
}

// The cut of the scans: as many segments as SMs for each 64-column slice of a
// head (rounded down: 16 heads of 128 get 4, 128 tasks for 148 SMs), none shorter than 4 chunks.  A cut costs a second pass over k and v and two
// launches, so it has to take two segments and 8 chunks off the walk.  One sequence,
// 16 heads, K = V = 128, uncut and cut: 1024 tokens 22 and 30 us (2 x 4 chunks: not
// cut), 2048 tokens 37 and 33 us (4 x 4; 2 x 8: 41 us), 16384 tokens 261 and 121 us;
// one head, 16384 tokens: 243 us, and 44 or 39 us with at least 8 or 4 chunks.
inline LaSegs la_segs(const gdn2_linear_attn_args& a, const LaSegWs& ws) {
  const int64_t C = kLaChunkTc, NT = la_num_chunks(a), slices = a.HV * (a.V / 64);
  const int64_t most = (a.T + C - 1) / C;                      // chunks of the longest sequence
  const int64_t want = std::max<int64_t>(1, kLaSms / slices);  // segments over all sequences
  LaSegs g{};
  int64_t len = most;
  if (a.cu_seqlens) len = (NT + want - 1) / want;
  else if (a.N < want) len = (most + want / std::max<int64_t>(a.N, 1) - 1) / (want / std::max<int64_t>(a.N, 1));
  len = std::max<int64_t>(len, 4);
  g.multi = most >= 2 * len + 8;
  g.len = (int)(g.multi ? len : std::max<int64_t>(most, 1));
  g.per = g.multi ? (most + len - 1) / len : 1;
  g.entries = a.cu_seqlens ? (g.multi ? a.T / (C * len) + a.N : a.N) : a.N * g.per;
  g.order = ws.order;
  if (g.multi) {
    g.map = a.cu_seqlens ? ws.map : nullptr;
    g.first = ws.first;
    g.cut = a.cu_seqlens != nullptr;
    g.X = ws.X;
    g.D = ws.D;
  }
  return g;
}

inline size_t la_align(size_t x) { return (x + 255) & ~size_t(255); }

inline size_t la_ws_layout(const gdn2_linear_attn_args& a, void* base, LaWs* out) {
  size_t off = 0;
  auto take = [&](size_t bytes) {
    const size_t o = off;
    off = la_align(off + bytes);
    return base ? (void*)((char*)base + o) : nullptr;
  };
  LaWs w{};
  const size_t NT = (size_t)la_num_chunks(a), HV = (size_t)a.HV, KV = (size_t)(a.K * a.V);
  const bool save = a.flags & GDN2_SAVE_FOR_BWD;
  if (a.cu_seqlens && (save || !la_tc(a))) {
    w.map = (LaChunk*)take(NT * sizeof(LaChunk));
    w.first = (int32_t*)take(((size_t)a.N + 1) * 4);
  }
  if (la_tc(a)) {
    const LaSegs g = la_segs(a, w.seg);
    if (a.cu_seqlens) w.seg.order = (int32_t*)take(((size_t)g.entries + 1) * 4);
    if (g.multi) {
      if (a.cu_seqlens) {
        w.seg.map = (LaChunk*)take((size_t)g.entries * sizeof(LaChunk));
        w.seg.first = (int32_t*)take(((size_t)a.N + 1) * 4);
      }
      w.seg.X = (float*)take((size_t)g.entries * HV * KV * 4);
      w.seg.D = (float*)take((size_t)g.entries * HV * 4);
    }
    if (save) w.states16 = (__nv_bfloat16*)take(NT * HV * KV * 2);
    if (out) *out = w;
    return off;
  }
  w.total = (float*)take(NT * HV * 4);
  w.states = (float*)take(NT * HV * KV * 4);
  if (out) *out = w;
  return off;
}

inline size_t la_bwd_ws_layout(const gdn2_linear_attn_args& a, void* base, LaBwdWs* out) {
  size_t off = 0;
  auto take = [&](size_t bytes) {
    const size_t o = off;
    off = la_align(off + bytes);
    return base ? (void*)((char*)base + o) : nullptr;
  };
  LaBwdWs w{};
  const size_t NT = (size_t)la_num_chunks(a), HV = (size_t)a.HV, KV = (size_t)(a.K * a.V);
  if (la_tc(a)) {
    const LaSegs g = la_segs(a, w.seg);
    if (g.multi) {
      w.seg.X = (float*)take((size_t)g.entries * HV * KV * 4);
      w.seg.D = (float*)take((size_t)g.entries * HV * 4);
    }
    w.dstates16 = (__nv_bfloat16*)take(NT * HV * KV * 2);
    if (a.HV > a.H) w.acc = (float*)take((size_t)kLaSms * 2 * kLaChunkTc * (size_t)a.K * 4);
  } else {
    w.dstates = (float*)take(NT * HV * KV * 4);
  }
  if (a.decay == GDN2_DECAY_HEAD) w.dg = (float*)take((size_t)(a.B * a.T) * HV * 4);
  if (out) *out = w;
  return off;
}

inline LaGeom la_geom(const gdn2_linear_attn_args& a, const LaWs& ws) {
  const int C = la_chunk(a);
  return LaGeom{a.cu_seqlens, a.T, a.N, C, (a.T + C - 1) / C, ws.map, ws.first};
}

// Rows of packed tensors that lie in no sequence (before the first offset,
// after the last) get zeros, a row by a CTA.  Offsets that cover the row, the usual case, leave nothing to do.
struct LaRows {
  void* p[4];
  int64_t bytes[4];  // of one row
};
GDN2_DEV void zero_outside(const LaRows& r, const LaGeom& geo, int block, int blocks) {
  int64_t b0, l0, b1, l1;
  geo.seq(0, b0, l0);
  geo.seq(geo.N - 1, b1, l1);
  const int64_t end = b1 + l1, rows = b0 + (geo.T - end);
  for (int64_t k = block; k < rows; k += blocks) {
    const int64_t row = k < b0 ? k : end + (k - b0);
#pragma unroll 1
    for (int i = 0; i < 4; ++i) {
      if (!r.p[i]) continue;
      uint16_t* p = static_cast<uint16_t*>(r.p[i]) + row * (r.bytes[i] / 2);  // every row is a whole number of 2-byte units
#pragma unroll 1
      for (int64_t x = threadIdx.x; x < r.bytes[i] / 2; x += blockDim.x) p[x] = 0;
    }
  }
}

// The log-decay of one token.  Values below -150 (and -inf) count as -150: exp
// of it is zero in fp32, and differences of running sums never become
// inf - inf.  NaN stays NaN.
struct LaDecay {
  const void* g;
  int64_t sb, st, sh;
  int kind, dtype;
  // the bits as they lie in memory (to be loaded ahead), and their value
  GDN2_DEV uint32_t raw(int64_t b, int64_t t, int64_t hv) const {
    if (kind == GDN2_DECAY_NONE) return 0;
    const int64_t i = kind == GDN2_DECAY_HEAD ? hv * sh : b * sb + t * st + hv * sh;
    return dtype == GDN2_BF16 ? static_cast<const uint16_t*>(g)[i] : static_cast<const uint32_t*>(g)[i];
  }
  GDN2_DEV double value(uint32_t bits) const {
    const float x = __uint_as_float(dtype == GDN2_BF16 ? bits << 16 : bits);
    return x < -150.f ? -150.0 : (double)x;
  }
  GDN2_DEV double at(int64_t b, int64_t t, int64_t hv) const { return value(raw(b, t, hv)); }
};
inline LaDecay la_decay(const gdn2_linear_attn_args& a) {
  return LaDecay{a.g, a.g_stride[0], a.g_stride[1], a.g_stride[2], a.decay, a.dtype_g};
}

int la_fwd_launch(const gdn2_linear_attn_args& a, const LaWs& ws, cudaStream_t s);
int la_bwd_launch(const gdn2_linear_attn_args& a, const gdn2_linear_attn_grads& gr, const LaWs& ws,
                         const LaBwdWs& bw, cudaStream_t s);
int la_tc_fwd_launch(const gdn2_linear_attn_args& a, const LaWs& ws, cudaStream_t s);
// fault word of the tensor-core kernels: bit 0 = a bounded wait gave up
int la_fault_read(int clear, unsigned int* out);
int la_tc_bwd_launch(const gdn2_linear_attn_args& a, const gdn2_linear_attn_grads& gr, const LaWs& ws,
                     const LaBwdWs& bw, cudaStream_t s);
int la_recurrent_launch(const gdn2_linear_attn_args& a, cudaStream_t s);

int layer_norm_fwd_launch(const gdn2_layer_norm_args& a, cudaStream_t s);
int layer_norm_bwd_launch(const gdn2_layer_norm_args& a, const gdn2_layer_norm_grads& g, void* ws, cudaStream_t s);
size_t layer_norm_bwd_ws(const gdn2_layer_norm_args& a);

}  // namespace gdn2
