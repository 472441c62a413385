// Linear attention with a decay for each head on 5th-generation tensor cores
// (tcgen05 + TMEM + TMA), bf16 operands, fp32 accumulation: the scan over time.
//
// Chunks of C = 128 tokens, G the running sum of g inside one, S the state entering it:
//     P_ij = e^{G_i - G_j} (q_i . k_j) for i >= j           o = scale (P v + e^G q S)
//     S'   = e^{G_C} S + sum_j k_j (e^{G_C - G_j} v_j)^T
// and, run backwards with x = q, y = do, the state cotangent (no outputs):
//     dS   = e^{G_C} dS' + sum_i q_i (scale e^{G_i} do_i)^T
// A CTA walks the chunks of one (sequence, value head, 64 columns of V); two
// CTAs side by side share q and k through L2.  CTAs are persistent: the roles
// below run through the chunks of all its tasks as one pipeline, so a task's
// loads overlap the end of the one before.
//   warp 0      TMA loads into two stages (q, k; v)
//   warp 1      allocates TMEM, issues the MMAs: Q K^T (the next chunk's), Q S,
//               K^T (w v), P V (P from TMEM)
//   warp 2      running sums of g in fp64 and the factors made from them
//   warp 3      TMA stores: o, the chunk's entering state
//   warps 4-7   scores: Q K^T out of TMEM, decayed, back as the bf16 operand P.
//               Off the diagonal e^{G_i - G_j} = e^{G_i - G_r} e^{G_r - G_j} with r
//               the first row of the 32-row block: both factors are at most 1 for
//               decays, one is per row, the other per block and column, so only the
//               32 diagonal columns take an exponential each.
//   warps 8-11  w v in bf16, and the state in registers (thread = row k of S):
//               S <- e^{G_C} S + what the MMA left in TMEM; bf16 copy for Q S
//   warps 12-15 o out of TMEM (thread = token), bf16, into the stage's own v slot
// Precision: P, S and w v are rounded to bf16 as MMA operands (2^-9 each, as the
// result itself).  Where the final state (or the initial state's gradient) is
// asked for, w v goes in as the sum of two bf16 values, so the state that leaves
// in fp32 carries 16 bits or more of every product.
// Every wait is bounded (tc::kWaitLimitNs); one that gives up sets g_la_fault.
#include <cuda.h>
#include <cudaTypedefs.h>

#include <algorithm>

#include "linear_attn.cuh"
#include "profile.cuh"
#include "tc.cuh"

namespace gdn2 {

__device__ unsigned int g_la_fault;

namespace {

constexpr int kC = kLaChunkTc;
constexpr float kLog2e = 1.44269504088896340736f;
constexpr uint32_t kTile = 128 * 64 * 2;  // one [128 x 64] bf16 swizzled tile

struct alignas(16) Factors {  // of one chunk; cf[w - 1][j] = e^{G_{32 w} - G_j}, j < 32 w
  float rowE[kC];     // e^{G_i}
  float r[kC];        // e^{G_i - G_{32 floor(i / 32)}}
  float g2[kC];       // (G_i - G_{32 floor(i / 32)}) log2 e
  float yw[kC];       // e^{G_C - G_j} (backwards: scale e^{G_i}); 0 past the last token
  float cf[3][kC];
  float total;        // e^{G_C}
};

template <int K, bool kOut>
struct alignas(1024) ScanSmem {
  __nv_bfloat16 X[2][K / 64][128 * 64];
  __nv_bfloat16 Q[kOut ? 2 : 1][kOut ? K / 64 : 1][kOut ? 128 * 64 : 512];
  __nv_bfloat16 Y[2][128 * 64];
  __nv_bfloat16 YW[2][128 * 64];  // two chunks' w v, or (exact) the two terms of one
  __nv_bfloat16 S[K * 64];        // bf16 state, rows k
  Factors f[2];
  uint64_t full_x[2], full_y[2], empty_x[2], empty_y[2], f_full[2], f_empty[2], qk_full[2], p_full[2], ds_full[2];
  uint64_t yw_full[2], o_staged[2], s_full, s_free, o_full, o_free;
  uint32_t tbase;
};

static_assert(sizeof(Factors) % 16 == 0 && offsetof(Factors, g2) % 16 == 0 && offsetof(Factors, cf) % 16 == 0,
              "16-byte reads of the factors");

struct ScanArgs {
  gdn2_linear_attn_args a;
  LaDecay dec;
  LaGeom geo;
  LaSegs seg;
  int64_t tasks;
  int pre;               // 1: the pass that only takes segments' own states to X and their decays to D
  const float* init;     // h0 / dht, or NULL
  float* fin;            // ht / dh0, or NULL
};

struct Task {
  int64_t n, hv, h, bos, len, entry, chunk0;
  int z, cb, ce;
  bool head, tail;  // holds the first / last segment in the direction of the walk
};

template <bool kBack>
GDN2_DEV bool get_task(const ScanArgs& p, int64_t id, Task& t) {
  const int vs = (int)(p.a.V >> 6);
  t.z = (int)(id % vs);
  const int64_t r = id / vs;
  t.hv = r % p.a.HV;
  t.entry = r / p.a.HV;
  t.h = t.hv / (p.a.HV / p.a.H);
  int64_t s;
  if (!p.seg.get(t.entry, p.geo, t.n, s)) return false;
  p.geo.seq(t.n, t.bos, t.len);
  const int nch = (int)((t.len + kC - 1) / kC);
  t.chunk0 = p.geo.cu && !p.geo.first ? 0 : p.geo.chunk0(t.n);  // (used where states are stored)
  t.cb = (int)s * p.seg.len;
  t.ce = min(t.cb + p.seg.len, nch);
  const bool first = s == 0, last = t.ce >= nch;
  t.head = kBack ? last : first;
  t.tail = kBack ? first : last;
  if (p.pre && t.tail) return false;  // nobody needs the state that leaves the last segment
  return true;
}

GDN2_DEV uint64_t kmaj(const void* p, int kk) {  // K-major tile, 16-column step kk
  return tc::sdesc_sw128(tc::smem_u32(p) + kk * 32, 16, 1024);
}
GDN2_DEV uint64_t nmaj(const void* p, int kk) {  // M- or N-major tile, 16-row step kk; 64-column blocks one tile apart
  return tc::sdesc_sw128(tc::smem_u32(p) + kk * 2048, kTile, 1024);
}
GDN2_DEV bool warp_wait(uint64_t* bar, uint32_t parity) {
  return __all_sync(0xffffffffu, tc::mbar_wait(bar, parity));
}

template <int K, bool kOut, bool kStore, bool kBack, bool kExact>
__global__ void __launch_bounds__(kOut ? 512 : 256, 1)
la_scan_kernel(const ScanArgs p, const __grid_constant__ CUtensorMap tmX, const __grid_constant__ CUtensorMap tmQ,
               const __grid_constant__ CUtensorMap tmY, const __grid_constant__ CUtensorMap tmO,
               const __grid_constant__ CUtensorMap tmS) {
  extern __shared__ unsigned char smem_raw[];
  using Sm = ScanSmem<K, kOut>;
  Sm& sm = *reinterpret_cast<Sm*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  constexpr bool kS16 = kOut || kStore;  // the bf16 state is used
  constexpr uint32_t kColQK = 0, kColO1 = 256, kColO2 = 320, kColDS = kOut ? 384 : 0;
  constexpr uint32_t kCols = kOut ? 512 : 128;
  constexpr int kNB = kExact ? 1 : 2;  // chunks of w v held
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  if (tid == 0) {
    for (int i = 0; i < 2; ++i) {
      tc::mbar_init(&sm.full_x[i], 1);
      tc::mbar_init(&sm.full_y[i], 1);
      tc::mbar_init(&sm.empty_x[i], 1);
      tc::mbar_init(&sm.empty_y[i], kOut ? 1 : 128);
      tc::mbar_init(&sm.f_full[i], 32);
      tc::mbar_init(&sm.f_empty[i], kOut ? 12 : 4);
      tc::mbar_init(&sm.qk_full[i], 1);
      tc::mbar_init(&sm.p_full[i], 128);
      tc::mbar_init(&sm.ds_full[i], 1);
      tc::mbar_init(&sm.yw_full[i], 128);
      tc::mbar_init(&sm.o_staged[i], 128);
    }
      tc::mbar_init(&sm.s_full, 128);
    tc::mbar_init(&sm.s_free, 1);
    tc::mbar_init(&sm.o_full, 1);
    tc::mbar_init(&sm.o_free, 128);
    tc::mbar_fence_init();
  }
  if (warp == 1) tc::tmem_alloc(&sm.tbase, kCols);
  tc::tc_fence_before();
  __syncthreads();
  tc::tc_fence_after();
  const uint32_t tb = sm.tbase;
  bool ok = true;
  uint32_t it = 0;  // chunks this role has been through, over all tasks
  Task t{};
  auto nth = [&](int i) { return kBack ? t.ce - 1 - i : t.cb + i; };  // i-th chunk of the task
  auto rows = [&](int c) { return (int)min(t.len - (int64_t)c * kC, (int64_t)kC); };
  // the token coordinate and batch of chunk c in the tensor maps
  auto tok = [&](int c) { return (int)((p.geo.cu ? t.bos : 0) + (int64_t)c * kC); };
  const int64_t step = gridDim.x;

  if (warp == 0) {
    // ---------------------------------------------------------------- loads
    if (lane == 0) {
      tc::prefetch_tensormap(&tmX);
      tc::prefetch_tensormap(&tmY);
      if (kOut) tc::prefetch_tensormap(&tmQ);
      for (int64_t id = blockIdx.x; id < p.tasks && ok; id += step) {
        if (!get_task<kBack>(p, id, t)) continue;
        const int b = p.geo.cu ? 0 : (int)t.n;
        for (int i = 0; i < t.ce - t.cb; ++i, ++it) {
          const int s = it & 1, tt = tok(nth(i));
          const uint32_t par = ((it >> 1) & 1) ^ 1;
          if (it >= 2 && !(ok = tc::mbar_wait(&sm.empty_x[s], par))) break;
          tc::mbar_arrive_expect_tx(&sm.full_x[s], (kOut ? 2 : 1) * (K / 64) * kTile);
#pragma unroll
          for (int c = 0; c < K / 64; ++c) {
            tc::tma_load_4d(sm.X[s][c], &tmX, &sm.full_x[s], 64 * c, (int)t.h, tt, b);
            if constexpr (kOut) tc::tma_load_4d(sm.Q[s][c], &tmQ, &sm.full_x[s], 64 * c, (int)t.h, tt, b);
          }
          if (it >= 2 && !(ok = tc::mbar_wait(&sm.empty_y[s], par))) break;
          tc::mbar_arrive_expect_tx(&sm.full_y[s], kTile);
          tc::tma_load_4d(sm.Y[s], &tmY, &sm.full_y[s], 64 * t.z, (int)t.hv, tt, b);
        }
      }
      // loads in flight land before the CTA exits, also after a wait that gave up
      for (uint32_t j = it > 2 ? it - 2 : 0; !ok && j < it; ++j) {
        tc::mbar_wait(&sm.full_x[j & 1], (j >> 1) & 1);
        tc::mbar_wait(&sm.full_y[j & 1], (j >> 1) & 1);
      }
    }
  } else if (warp == 1) {
    // ----------------------------------------------------------------- MMAs
    if (lane == 0) {
      constexpr uint32_t iQK = tc::idesc_bf16(128, 128, 0, 0), iNV = tc::idesc_bf16(128, 64, 0, 1);
      constexpr uint32_t iDS = tc::idesc_bf16(K, 64, 1, 1);
      auto qk = [&](uint32_t j) {
        const int s = j & 1;
        if (!tc::mbar_wait(&sm.full_x[s], (j >> 1) & 1)) return false;
        tc::tc_fence_after();
#pragma unroll
        for (int kk = 0; kk < K / 16; ++kk)
          tc::mma_bf16(tb + kColQK + 128 * s, kmaj(sm.Q[s][kk >> 2], kk & 3), kmaj(sm.X[s][kk >> 2], kk & 3), iQK,
                       kk > 0);
        tc::mma_commit(&sm.qk_full[s]);
        return true;
      };
      uint32_t total = 0;  // chunks over all tasks
      for (int64_t id = blockIdx.x; id < p.tasks; id += step)
        if (get_task<kBack>(p, id, t)) total += (uint32_t)max(t.ce - t.cb, 0);
      if (kOut && total > 0) ok = qk(0);
      for (; ok && it < total; ++it) {
        const int s = it & 1, y = kNB == 2 ? s : 0;
        if constexpr (kOut) {
          if (!(ok = tc::mbar_wait(&sm.s_full, it & 1))) break;
          if (it > 0 && !(ok = tc::mbar_wait(&sm.o_free, (it - 1) & 1))) break;
          tc::tc_fence_after();
#pragma unroll
          for (int kk = 0; kk < K / 16; ++kk)
            tc::mma_bf16(tb + kColO1, kmaj(sm.Q[s][kk >> 2], kk & 3), nmaj(sm.S, kk), iNV, kk > 0);
        } else if (!(ok = tc::mbar_wait(&sm.full_x[s], (it >> 1) & 1))) {
          break;
        }
        if (!(ok = tc::mbar_wait(&sm.yw_full[s], (it >> 1) & 1))) break;
        tc::tc_fence_after();
#pragma unroll
        for (int kk = 0; kk < 8; ++kk)
          tc::mma_bf16(tb + kColDS + 64 * s, nmaj(sm.X[s], kk), nmaj(sm.YW[y], kk), iDS, kk > 0);
        if constexpr (kExact) {
#pragma unroll
          for (int kk = 0; kk < 8; ++kk)
            tc::mma_bf16(tb + kColDS + 64 * s, nmaj(sm.X[s], kk), nmaj(sm.YW[1], kk), iDS, 1);
        }
        tc::mma_commit(&sm.ds_full[s]);
        tc::mma_commit(&sm.empty_x[s]);
        if constexpr (kOut) {
          if (it + 1 < total && !(ok = qk(it + 1))) break;
          if (!(ok = tc::mbar_wait(&sm.full_y[s], (it >> 1) & 1) && tc::mbar_wait(&sm.p_full[s], (it >> 1) & 1))) break;
          tc::tc_fence_after();
#pragma unroll
          for (int kk = 0; kk < 8; ++kk)
            tc::mma_bf16_ts(tb + kColO2, tb + kColQK + 128 * s + 8 * kk, nmaj(sm.Y[s], kk), iNV, kk > 0);
          tc::mma_commit(&sm.o_full);
        }
      }
      // what was issued has completed before TMEM is released (the last commits, when all went well)
      if (ok && total > 0) {
        const uint32_t j = total - 1;
        if (!(kOut ? tc::mbar_wait(&sm.o_full, j & 1) : tc::mbar_wait(&sm.ds_full[j & 1], (j >> 1) & 1))) ok = false;
      } else if (!ok) {  // a commit of its own covers them
        tc::mma_commit(&sm.o_full);
        tc::mbar_wait(&sm.o_full, it & 1);
      }
    }
  } else if (warp == 2) {
    // -------------------------------------------------------------- factors
    for (int64_t id = blockIdx.x; id < p.tasks && ok; id += step) {
      if (!get_task<kBack>(p, id, t)) continue;
      const int64_t b = p.geo.cu ? 0 : t.n;
      double x[4], sum = 0.0;
      auto load = [&](int c) {
        const int L = rows(c);
        const int64_t t0 = (p.geo.cu ? t.bos : 0) + (int64_t)c * kC;
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] = 4 * lane + e < L ? p.dec.at(b, t0 + 4 * lane + e, t.hv) : 0.0;
      };
      const int nloc = t.ce - t.cb;
      if (nloc > 0) load(nth(0));
      for (int i = 0; i < nloc; ++i, ++it) {
        const int s = it & 1, L = rows(nth(i));
        double G[4] = {x[0], x[0] + x[1], 0.0, 0.0};
        G[2] = G[1] + x[2];
        G[3] = G[2] + x[3];
        double inc = G[3];
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const double y = __shfl_up_sync(0xffffffffu, inc, o);
          if (lane >= o) inc += y;
        }
        const double before = __shfl_up_sync(0xffffffffu, inc, 1);
#pragma unroll
        for (int e = 0; e < 4; ++e) G[e] += lane ? before : 0.0;
        const double GC = __shfl_sync(0xffffffffu, inc, 31);
        double ref[4];
#pragma unroll
        for (int w = 0; w < 4; ++w) ref[w] = __shfl_sync(0xffffffffu, G[0], 8 * w);
        sum += GC;
        if (i + 1 < nloc) load(nth(i + 1));
        if (it >= 2 && !(ok = warp_wait(&sm.f_empty[s], ((it >> 1) & 1) ^ 1))) break;
        Factors& f = sm.f[s];
        const int own = lane >> 3;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int j = 4 * lane + e;
          f.yw[j] = j >= L ? 0.f : kBack ? p.a.scale * expf((float)G[e]) : expf((float)(GC - G[e]));
          if constexpr (kOut) {
            double rw = ref[0];
#pragma unroll
            for (int w = 1; w < 4; ++w) rw = own == w ? ref[w] : rw;
            f.rowE[j] = expf((float)G[e]);
            f.r[j] = expf((float)(G[e] - rw));
            f.g2[j] = (float)(G[e] - rw) * kLog2e;
#pragma unroll
            for (int w = 1; w < 4; ++w)
              if (own < w) f.cf[w - 1][j] = expf((float)(ref[w] - G[e]));
          }
        }
        if (lane == 0) f.total = expf((float)GC);
        tc::mbar_arrive(&sm.f_full[s]);
      }
      if (p.pre && lane == 0 && t.z == 0) p.seg.D[t.entry * p.a.HV + t.hv] = expf((float)sum);
    }
  } else if (warp == 3) {
    // --------------------------------------------------------------- stores
    if (lane == 0 && (kOut || kStore)) {
      for (int64_t id = blockIdx.x; id < p.tasks && ok; id += step) {
        if (!get_task<kBack>(p, id, t)) continue;
        const int b = p.geo.cu ? 0 : (int)t.n;
        for (int i = 0; i < t.ce - t.cb; ++i, ++it) {
          const int c = nth(i);
          if constexpr (kStore) {
            if (!(ok = tc::mbar_wait(&sm.s_full, it & 1))) break;
            tc::tma_store_2d(&tmS, sm.S, 64 * t.z, (int)(((t.chunk0 + c) * p.a.HV + t.hv) * K));
            tc::bulk_commit();
            tc::bulk_wait_read_all();
            tc::mbar_arrive(&sm.s_free);
          }
          if constexpr (kOut) {
            if (!(ok = tc::mbar_wait(&sm.o_staged[it & 1], (it >> 1) & 1))) break;
            if (!p.geo.cu || rows(c) == kC) {  // (the last rows of a packed sequence: stored by their threads)
              tc::tma_store_4d(&tmO, sm.Y[it & 1], 64 * t.z, (int)t.hv, tok(c), b);
              tc::bulk_commit();
              tc::bulk_wait_read_all();
            }
            tc::mbar_arrive(&sm.empty_y[it & 1]);
          }
        }
      }
      tc::bulk_wait_all();
    }
  } else if (kOut && warp < 8) {
    // --------------------------------------------------------------- scores
    const int w = warp - 4, i = 32 * w + lane;
    for (int64_t id = blockIdx.x; id < p.tasks && ok; id += step) {
      if (!get_task<kBack>(p, id, t)) continue;
      for (int j = 0; j < t.ce - t.cb; ++j, ++it) {
        const int s = it & 1;
        const uint32_t tp = tb + kColQK + 128 * s + ((uint32_t)(32 * w) << 16);
        if (!(ok = warp_wait(&sm.f_full[s], (it >> 1) & 1) && warp_wait(&sm.qk_full[s], (it >> 1) & 1))) break;
        tc::tc_fence_after();
        const Factors& f = sm.f[s];
        const float ri = f.r[i], gi = f.g2[i];
#pragma unroll 1
        for (int J = 0; J < 4; ++J) {
          uint32_t pk[16];
          if (J > w) {
#pragma unroll
            for (int e = 0; e < 16; ++e) pk[e] = 0;
          } else {
            float x[32];
            tc::tmem_ld32(tp + 32 * J, x);
            if (J < w) {
              const float4* cf = reinterpret_cast<const float4*>(f.cf[w - 1] + 32 * J);
              tc::tmem_wait_ld();
#pragma unroll
              for (int e = 0; e < 8; ++e) {
                const float4 cc = cf[e];
                pk[2 * e] = pack_bf16(x[4 * e] * cc.x * ri, x[4 * e + 1] * cc.y * ri);
                pk[2 * e + 1] = pack_bf16(x[4 * e + 2] * cc.z * ri, x[4 * e + 3] * cc.w * ri);
              }
            } else {
              const float4* gj = reinterpret_cast<const float4*>(f.g2 + 32 * J);
              tc::tmem_wait_ld();
#pragma unroll
              for (int e = 0; e < 8; ++e) {
                const float4 gg = gj[e];
                const float d[4] = {gg.x, gg.y, gg.z, gg.w};
                float y[4];
#pragma unroll
                for (int u = 0; u < 4; ++u) y[u] = 4 * e + u <= lane ? x[4 * e + u] * exp2_approx(gi - d[u]) : 0.f;
                pk[2 * e] = pack_bf16(y[0], y[1]);
                pk[2 * e + 1] = pack_bf16(y[2], y[3]);
              }
            }
          }
          tc::tmem_st16(tp + 16 * J, pk);
        }
        tc::tmem_wait_st();
        tc::tc_fence_before();
        tc::mbar_arrive(&sm.p_full[s]);
        if (lane == 0) tc::mbar_arrive(&sm.f_empty[s]);
      }
    }
  } else if (kOut ? warp < 12 : warp >= 4 && warp < 8) {
    // ---------------------------------------------------------------- state
    const int w = warp & 3, row = K == 128 ? 32 * w + lane : 16 * w + (lane & 15), j = 32 * w + lane;
    const bool own = K == 128 || lane < 16;  // M = 64: rows in the first 16 lanes of each quarter
    const uint32_t td = tb + kColDS + ((uint32_t)(32 * w) << 16);
    float st[64];
    uint32_t done = 0;   // chunks whose state term has been taken
    // w v of chunk `it`
    auto weigh = [&](int c) -> bool {
      const int s = it & 1, L = rows(c);
      if (!warp_wait(&sm.f_full[s], (it >> 1) & 1) || !warp_wait(&sm.full_y[s], (it >> 1) & 1)) return false;
      char* src = reinterpret_cast<char*>(sm.Y[s]) + j * 128;
      char* hi = reinterpret_cast<char*>(sm.YW[kNB == 2 ? s : 0]) + j * 128;
      char* lo = reinterpret_cast<char*>(sm.YW[1]) + j * 128;
      const float f = sm.f[s].yw[j];
      const bool inside = j < L;
#pragma unroll
      for (int q = 0; q < 8; ++q) {
        const int at = (q ^ (j & 7)) << 4;
        float x[8];
        ld8(reinterpret_cast<const __nv_bfloat16*>(src + at), x);
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = inside ? x[e] * f : 0.f;
        const uint4 h = pack8(x);
        *reinterpret_cast<uint4*>(hi + at) = h;
        if constexpr (kExact) {
          float y[8];
          ld8(reinterpret_cast<const __nv_bfloat16*>(&h), y);
#pragma unroll
          for (int e = 0; e < 8; ++e) x[e] -= y[e];
          *reinterpret_cast<uint4*>(lo + at) = pack8(x);
        }
      }
      if (p.geo.cu && L < kC) {  // the next sequence's rows in this tile: none of them may reach a sum
        if (!warp_wait(&sm.full_x[s], (it >> 1) & 1)) return false;
        if (!inside) {
#pragma unroll
          for (int q = 0; q < 8; ++q) {
            *reinterpret_cast<uint4*>(src + 16 * q) = make_uint4(0, 0, 0, 0);
#pragma unroll
            for (int b = 0; b < K / 64; ++b)
              *reinterpret_cast<uint4*>(reinterpret_cast<char*>(sm.X[s][b]) + j * 128 + 16 * q) = make_uint4(0, 0, 0, 0);
          }
        }
      }
      tc::fence_proxy_async();
      tc::mbar_arrive(&sm.yw_full[s]);
      if constexpr (!kOut) tc::mbar_arrive(&sm.empty_y[s]);
      return true;
    };
    // S <- total S + the term of chunk `done`
    auto take = [&]() -> bool {
      const int s = done & 1;
      const float f = sm.f[s].total;
      if (!warp_wait(&sm.ds_full[s], (done >> 1) & 1)) return false;
      tc::tc_fence_after();
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        float x[32];
        tc::tmem_ld32(td + 64 * s + 32 * h, x);
        tc::tmem_wait_ld();
#pragma unroll
        for (int e = 0; e < 32; ++e) st[32 * h + e] = fmaf(st[32 * h + e], f, x[e]);
      }
      tc::tc_fence_before();
      __syncwarp();
      if (lane == 0) tc::mbar_arrive(&sm.f_empty[s]);
      ++done;
      return true;
    };
    // the bf16 state of chunk `it`
    auto publish = [&]() -> bool {
      if constexpr (kS16) {
        if (kStore && it > 0 && !warp_wait(&sm.s_free, (it - 1) & 1)) return false;
        char* dst = reinterpret_cast<char*>(sm.S) + row * 128;
        if (own) {
#pragma unroll
          for (int q = 0; q < 8; ++q) *reinterpret_cast<uint4*>(dst + ((q ^ (row & 7)) << 4)) = pack8(st + 8 * q);
        }
        tc::fence_proxy_async();
        tc::mbar_arrive(&sm.s_full);
      }
      return true;
    };
    for (int64_t id = blockIdx.x; id < p.tasks && ok; id += step) {
      if (!get_task<kBack>(p, id, t)) continue;
      const int64_t KV = (int64_t)K * p.a.V, at = (int64_t)row * p.a.V + 64 * t.z;
      const float* src = t.head ? (p.init ? p.init + (t.n * p.a.HV + t.hv) * KV : nullptr)
                         : p.pre ? nullptr
                                 : p.seg.X + ((t.entry + (kBack ? 1 : -1)) * p.a.HV + t.hv) * KV;
#pragma unroll
      for (int q = 0; q < 16; ++q) {
        const float4 x = src ? *reinterpret_cast<const float4*>(src + at + 4 * q) : make_float4(0.f, 0.f, 0.f, 0.f);
        st[4 * q] = x.x; st[4 * q + 1] = x.y; st[4 * q + 2] = x.z; st[4 * q + 3] = x.w;
      }
      const int nloc = t.ce - t.cb;
      for (int i = 0; i < nloc; ++i, ++it) {
        // with two buffers the next w v is made while the MMA of the chunk before still runs
        if (kNB == 2 && !(ok = weigh(nth(i)))) break;
        if (i > 0 && !(ok = take())) break;
        if (!(ok = publish())) break;
        if (kNB == 1 && !(ok = weigh(nth(i)))) break;
      }
      if (ok && nloc > 0) ok = take();
      if (!ok) break;
      float* dst = p.pre ? p.seg.X + (t.entry * p.a.HV + t.hv) * KV
                   : t.tail && p.fin ? p.fin + (t.n * p.a.HV + t.hv) * KV : nullptr;
      if (dst && own) {
#pragma unroll
        for (int q = 0; q < 16; ++q)
          *reinterpret_cast<float4*>(dst + at + 4 * q) = make_float4(st[4 * q], st[4 * q + 1], st[4 * q + 2], st[4 * q + 3]);
      }
    }
  } else if (kOut && warp >= 12) {
    // --------------------------------------------------------------- output
    const int w = warp & 3, i = 32 * w + lane;
    const uint32_t to = tb + ((uint32_t)(32 * w) << 16);
    for (int64_t id = blockIdx.x; id < p.tasks && ok; id += step) {
      if (!get_task<kBack>(p, id, t)) continue;
      for (int j = 0; j < t.ce - t.cb; ++j, ++it) {
        const int s = it & 1, c = nth(j), L = rows(c);
        if (!(ok = warp_wait(&sm.f_full[s], (it >> 1) & 1))) break;
        const float f = sm.f[s].rowE[i];
        if (!(ok = warp_wait(&sm.o_full, it & 1))) break;
        tc::tc_fence_after();
        uint4 out[8];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          float x[32], y[32];
          tc::tmem_ld32(to + kColO1 + 32 * h, x);
          tc::tmem_ld32(to + kColO2 + 32 * h, y);
          tc::tmem_wait_ld();
#pragma unroll
          for (int e = 0; e < 32; ++e) x[e] = p.a.scale * fmaf(f, x[e], y[e]);
#pragma unroll
          for (int q = 0; q < 4; ++q) out[4 * h + q] = pack8(x + 8 * q);
        }
        tc::tc_fence_before();
        tc::mbar_arrive(&sm.o_free);
        __syncwarp();
        if (lane == 0) tc::mbar_arrive(&sm.f_empty[s]);
        if (!p.geo.cu || L == kC) {
          char* dst = reinterpret_cast<char*>(sm.Y[s]) + i * 128;
#pragma unroll
          for (int q = 0; q < 8; ++q) *reinterpret_cast<uint4*>(dst + ((q ^ (i & 7)) << 4)) = out[q];
          tc::fence_proxy_async();
        } else if (i < L) {
          __nv_bfloat16* dst = static_cast<__nv_bfloat16*>(p.a.o) +
                               ((t.bos + (int64_t)c * kC + i) * p.a.HV + t.hv) * p.a.V + 64 * t.z;
#pragma unroll
          for (int q = 0; q < 8; ++q) *reinterpret_cast<uint4*>(dst + 8 * q) = out[q];
        }
        tc::mbar_arrive(&sm.o_staged[s]);
      }
    }
  }
  if (!ok) atomicOr(&g_la_fault, 1u);
  tc::tc_fence_before();
  __syncthreads();
  tc::tc_fence_after();
  if (warp == 1) tc::tmem_dealloc(tb, kCols);
}

// Entering states of the segments from their own terms: X[s] <- D[s] X[s - 1] + X[s]
// (backwards from the other end), four elements of one state per thread.
template <bool kBack>
__global__ void __launch_bounds__(128) la_segment_kernel(LaSegs seg, LaGeom geo, int64_t HV, int64_t KV) {
  const int64_t n = blockIdx.x / HV, hv = blockIdx.x % HV;
  const int64_t e = ((int64_t)blockIdx.y * 128 + threadIdx.x) * 4;
  int64_t bos, len;
  geo.seq(n, bos, len);
  const int64_t nch = (len + kC - 1) / kC, ns = nch > 0 ? (nch + seg.len - 1) / seg.len : 1;
  const int64_t e0 = seg.first_of(n);
  if (e >= KV || ns < 3) return;  // the first segment's term is a whole state already, the last one's is not used
  auto at = [&](int64_t s) {
    return reinterpret_cast<float4*>(seg.X + ((e0 + (kBack ? ns - 1 - s : s)) * HV + hv) * KV + e);
  };
  float4 x = *at(0);
  for (int64_t s = 1; s < ns - 1; ++s) {
    const float f = seg.D[(e0 + (kBack ? ns - 1 - s : s)) * HV + hv];
    float4 y = *at(s);
    x = make_float4(fmaf(f, x.x, y.x), fmaf(f, x.y, y.y), fmaf(f, x.z, y.z), fmaf(f, x.w, y.w));
    *at(s) = x;
  }
}

// ---------------------------------------------------------------------------
// host
// ---------------------------------------------------------------------------
PFN_cuTensorMapEncodeTiled_v12000 encode_fn() {
  static PFN_cuTensorMapEncodeTiled_v12000 fn = nullptr;
  if (!fn) {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) == cudaSuccess &&
        q == cudaDriverEntryPointSuccess)
      fn = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(p);
  }
  return fn;
}

// [B, T, H, D] bf16 with the given element steps -> boxes of 128 tokens x 64
// elements of one head; rows past T read as zero and are not written
bool token_map(CUtensorMap* m, const void* base, int64_t D, int64_t H, int64_t T, int64_t B, const int64_t* step) {
  auto enc = encode_fn();
  if (!enc || !base) return false;
  // the step of a dimension with one element is never taken
  const cuuint64_t sh = H > 1 ? step[2] * 2 : D * 2, st = T > 1 ? step[1] * 2 : D * 2, sb = B > 1 ? step[0] * 2 : D * 2;
  cuuint64_t dims[4] = {(cuuint64_t)D, (cuuint64_t)H, (cuuint64_t)T, (cuuint64_t)B};
  cuuint64_t strides[3] = {sh, st, sb};
  cuuint32_t box[4] = {64, 1, 128, 1};
  cuuint32_t es[4] = {1, 1, 1, 1};
  return enc(m, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, const_cast<void*>(base), dims, strides, box, es,
             CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
             CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// [rows, V] bf16 states -> boxes of K rows x 64 columns
bool state_map(CUtensorMap* m, const void* base, int64_t V, int64_t rows, int64_t K) {
  auto enc = encode_fn();
  if (!enc || !base) return false;
  cuuint64_t dims[2] = {(cuuint64_t)V, (cuuint64_t)rows};
  cuuint64_t strides[1] = {(cuuint64_t)V * 2};
  cuuint32_t box[2] = {64, (cuuint32_t)K};
  cuuint32_t es[2] = {1, 1};
  return enc(m, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, const_cast<void*>(base), dims, strides, box, es,
             CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
             CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

struct ScanMaps {
  CUtensorMap x, q, y, o, s;
};

template <int K, bool kOut, bool kStore, bool kBack, bool kExact>
int run_scan(const ScanArgs& p, const ScanMaps& m, cudaStream_t s) {
  auto kern = la_scan_kernel<K, kOut, kStore, kBack, kExact>;
  constexpr size_t bytes = sizeof(ScanSmem<K, kOut>) + 1024;
  static_assert(bytes <= 227 * 1024, "shared memory of the scan");
  GDN2_CUDA_TRY(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes));
  ProfScope ps(kOut ? kKLinAttnScan : kKLinAttnStates, s);
  kern<<<(unsigned)std::min<int64_t>(p.tasks, kLaSms), kOut ? 512 : 256, bytes, s>>>(p, m.x, m.q, m.y, m.o, m.s);
  GDN2_LAUNCH_CHECK();
  return 0;
}

// one direction of the scan: the segments' own states and their sum first where the sequences are cut
template <int K, bool kBack>
int scan(ScanArgs& p, const ScanMaps& m, bool out, bool store, bool exact, cudaStream_t s) {
  if (p.seg.multi) {
    p.pre = 1;
    if (int st = run_scan<K, false, false, kBack, true>(p, m, s)) return st;
    const int64_t KV = p.a.K * p.a.V;
    la_segment_kernel<kBack><<<dim3((unsigned)(p.a.N * p.a.HV), (unsigned)((KV + 511) / 512)), 128, 0, s>>>(
        p.seg, p.geo, p.a.HV, KV);
    GDN2_LAUNCH_CHECK();
    p.pre = 0;
  }
  if constexpr (kBack) {
    return exact ? run_scan<K, false, true, true, true>(p, m, s) : run_scan<K, false, true, true, false>(p, m, s);
  } else {
    if (store)
      return exact ? run_scan<K, true, true, false, true>(p, m, s) : run_scan<K, true, true, false, false>(p, m, s);
    return exact ? run_scan<K, true, false, false, true>(p, m, s) : run_scan<K, true, false, false, false>(p, m, s);
  }
}

}  // namespace

int la_tc_fwd_launch(const gdn2_linear_attn_args& a, const LaWs& ws, cudaStream_t s) {
  ScanArgs p{a, la_decay(a), la_geom(a, ws), la_segs(a, ws.seg), 0, 0, (a.flags & GDN2_HAS_H0) ? a.h0 : nullptr,
             (a.flags & GDN2_STORE_FINAL) ? a.ht : nullptr};
  p.tasks = p.seg.entries * a.HV * (a.V / 64);
  const bool save = a.flags & GDN2_SAVE_FOR_BWD;
  ScanMaps m;
  const int64_t ostep[3] = {a.T * a.HV * a.V, a.HV * a.V, a.V};
  if (!token_map(&m.x, a.k, a.K, a.H, a.T, a.B, a.k_stride) || !token_map(&m.q, a.q, a.K, a.H, a.T, a.B, a.q_stride) ||
      !token_map(&m.y, a.v, a.V, a.HV, a.T, a.B, a.v_stride) || !token_map(&m.o, a.o, a.V, a.HV, a.T, a.B, ostep))
    return GDN2_ERR_TENSOR_MAP;
  m.s = m.o;
  if (save && !state_map(&m.s, ws.states16, a.V, la_num_chunks(a) * a.HV * a.K, a.K)) return GDN2_ERR_TENSOR_MAP;
  const bool exact = a.flags & GDN2_STORE_FINAL;
  return a.K == 128 ? scan<128, false>(p, m, true, save, exact, s) : scan<64, false>(p, m, true, save, exact, s);
}

int la_fault_read(int clear, unsigned int* out) {
  GDN2_CUDA_TRY(cudaMemcpyFromSymbol(out, g_la_fault, sizeof(unsigned)));
  if (clear) {
    const unsigned zero = 0;
    GDN2_CUDA_TRY(cudaMemcpyToSymbol(g_la_fault, &zero, sizeof(unsigned)));
  }
  return 0;
}

}  // namespace gdn2
