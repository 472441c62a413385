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
//   warp 0      TMA loads (q, k: two stages, three without outputs; v: three)
//   warp 1      MMAs: Q K^T of chunk i, P V of chunk i - 1 (P from TMEM)
//   warp 2      running sums of g in fp64, handed on as a float and what it misses;
//               TMA stores of the chunks' entering states (without outputs: warp 1)
//   warp 3      MMAs: K^T (w v) and Q S.  Two issuers: neither chain waits for the other's
//               barriers, and an issuer ahead of the tensor pipe holds up the memory
//               instructions of its own quarter of the SM only
//   warps 4-11  scores (64 columns per four warps): Q K^T out of TMEM, decayed,
//               back as the bf16 operand P.  Off the diagonal e^{G_i - G_j} =
//               e^{G_i - G_r} e^{G_r - G_j} with r the first row of the 32-row block:
//               both factors are at most 1 for decays, one is per row, the other per
//               block and column, so only the 32 diagonal columns take an exponential each.
//   warps 12-15 the state in registers (thread = row k of S): S <- e^{G_C} S + what
//               the MMA left in TMEM; bf16 copy for Q S (without outputs also w v)
//   warps 16-19 w v; o out of TMEM (thread = token), straight to memory, 32 bytes a store
// P V lags by a chunk, which gives the scores more than a chunk's time.
// Precision: P and S are rounded to bf16 as MMA operands (as the result itself
// is).  w v goes in as the sum of two bf16 values, so the fp32 state carries 16
// bits or more of every product: with one it would hold 8, and o as many again less.
// Why 64 columns of V a CTA: two score buffers (256 TMEM columns), Q S of two
// chunks (128), P V (64) and the state's term (64) then fill TMEM's 512 exactly, the
// stages fill shared memory, and a sequence has twice as many CTAs; the price is
// Q K^T once per 64 columns.
// What bounds it: a chunk's products keep the tensor pipe busy for some 2050 clocks
// and read their operands from shared memory for some 2950 (K = 128); the roles'
// hand-overs bring that to 3400 (batches in L2) to 4300.  Measured at 16 heads, K = V = 128:
// 4 sequences of 4096 tokens 76 us (268 MB, 3.5 TB/s; 83 us where the states are kept
// for the backward, 48 us for the reverse scan without outputs); 65536 tokens 267 us
// after 139 us for the segments' own states (4 segments: 128 CTAs of 148 have a task, 96
// in the first pass, where the last segments have none); 23 packed sequences of 9001
// tokens 74 us.  Without outputs the same four warps make w v and then update the state.
// Every wait is bounded (tc::kWaitLimitNs); one that gives up sets g_la_fault.
#include <cuda.h>
#include <cudaTypedefs.h>

#include <algorithm>
#include <type_traits>

#include "linear_attn.cuh"
#include "profile.cuh"
#include "tc.cuh"

namespace gdn2 {

__device__ unsigned int g_la_fault;

namespace {

constexpr int kC = kLaChunkTc;
constexpr float kLog2e = 1.44269504088896340736f;
constexpr uint32_t kTile = 128 * 64 * 2;  // one [128 x 64] bf16 swizzled tile

// Running sums of one chunk's log-decays: fp64 values as a float and what it
// misses (8 bits of that are plenty)
struct alignas(16) Sums {
  float hi[kC];
  __nv_bfloat16 lo[kC];
};
// e^x: the hardware's base-2 exponential (2^-22) of x log2 e (rounded: another 2^-24 |x|)
GDN2_DEV float exp_of(float x) { return exp2_approx(x * kLog2e); }
// G_i - G_j
GDN2_DEV float sum_diff(const Sums& g, int i, int j) {
  return (g.hi[i] - g.hi[j]) + (__bfloat162float(g.lo[i]) - __bfloat162float(g.lo[j]));
}

template <int K, bool kOut>
struct alignas(1024) ScanSmem {
  static constexpr int NX = kOut ? 2 : 3, NY = 3;  // stages
  static constexpr int NB = kOut ? 1 : 2;          // chunks of w v held
  __nv_bfloat16 X[NX][(kOut ? 2 : 1) * K / 64][128 * 64];  // k; with outputs then q
  __nv_bfloat16 Y[NY][128 * 64];
  __nv_bfloat16 YW[NB][2][128 * 64];  // w v as the sum of two bf16 values
  __nv_bfloat16 S[K * 64];  // bf16 state, rows k
  Sums f[2];
  float cw[kOut ? 320 : 4];  // column factors of the score warps, 32 (w + 1) for w = 0..3
  uint64_t full_x[NX], empty_x[NX], full_y[NY], empty_y[NY], f_full[2], f_empty[2], qk_full[2], p_full[2];
  uint64_t yw_full[NB], ds_full[NB], ds_free, s_full, s_free, y_ready[NY], o_full[2], o_free[2], drained;
  uint32_t tbase;
};

struct ScanArgs {
  gdn2_linear_attn_args a;
  LaDecay dec;
  LaGeom geo;
  LaSegs seg;
  int64_t tasks;
  int group;             // value heads per key head
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
GDN2_DEV bool find_task(const ScanArgs& p, int64_t id, Task& t) {
  // the CTAs' turns go back and forth through the tasks, whose lengths fall where they are ordered
  const uint32_t turn = (uint32_t)id / kLaSms;
  if (!p.pre && (turn & 1) && (int64_t)(turn + 1) * kLaSms <= p.tasks) id = (int64_t)(2 * turn + 1) * kLaSms - 1 - id;
  const uint32_t two = (uint32_t)(p.a.V >> 7), HV = (uint32_t)p.a.HV, r = (uint32_t)id >> two;  // 64-column slices: 1 or 2
  t.z = (int)((uint32_t)id & two);
  t.entry = r / HV;
  t.hv = r - (uint32_t)t.entry * HV;
  if (p.seg.order) t.entry = p.seg.order[t.entry];
  t.h = (uint32_t)t.hv / (uint32_t)p.group;
  int64_t s;
  if (!p.seg.get(t.entry, p.geo, t.n, s)) return false;
  p.geo.seq(t.n, t.bos, t.len);
  const bool stored = !p.geo.cu || p.geo.first;  // states are: their rows have an end
  const int nch = (int)(stored ? p.geo.chunks(t.n, t.len) : (t.len + kC - 1) / kC);
  t.chunk0 = stored ? p.geo.chunk0(t.n) : 0;
  t.cb = (int)s * p.seg.len;
  t.ce = min(t.cb + p.seg.len, nch);
  const bool first = s == 0, last = t.ce >= nch;
  t.head = kBack ? last || t.entry + 1 >= p.seg.entries : first;  // (entries end early where offsets decrease)
  t.tail = kBack ? first : last;
  if (p.pre && t.tail) return false;  // nobody needs the state that leaves the last segment
  return true;
}

// A value that all lanes share, in a form that the compiler knows to be shared:
// loops and branches on it are then known to keep the warp converged, and the
// shuffles inside them are single instructions instead of ten.
template <typename T>
GDN2_DEV T uniform(T x) { return __shfl_sync(0xffffffffu, x, 0); }

// find_task for a whole warp
template <bool kBack>
GDN2_DEV bool get_task(const ScanArgs& p, int64_t id, Task& t) {
  const bool any = __all_sync(0xffffffffu, find_task<kBack>(p, id, t));
  t.n = uniform(t.n);
  t.bos = uniform(t.bos);
  t.len = uniform(t.len);
  t.cb = uniform(t.cb);
  t.ce = uniform(t.ce);
  t.head = __all_sync(0xffffffffu, t.head);
  t.tail = __all_sync(0xffffffffu, t.tail);
  return any;
}

// Operand descriptors from a shared-memory address in 16-byte units: the low
// word is that address plus constants, the high word a constant (8-row groups
// 1024 bytes apart, version 1, 128-byte swizzle).
constexpr uint32_t kDescHi = (1024 >> 4) | (1u << 14) | (2u << 29);
GDN2_DEV uint64_t desc(uint32_t lo) { return (static_cast<uint64_t>(kDescHi) << 32) | lo; }
GDN2_DEV uint32_t addr16(const void* p) { return tc::smem_u32(p) >> 4; }
// K-major tiles of 64 columns, 16-column step kk over all of them
GDN2_DEV uint64_t kmaj(uint32_t a16, int kk) { return desc(a16 + (kk >> 2) * (kTile >> 4) + (kk & 3) * 2 + (1u << 16)); }
// M- or N-major tile, 16-row step kk; 64-column blocks one tile apart
GDN2_DEV uint64_t nmaj(uint32_t a16, int kk) { return desc(a16 + kk * 128 + ((kTile >> 4) << 16)); }
// a whole 32-byte sector per thread where the tensor allows it
GDN2_DEV void st_32bytes(void* p, const uint4& a, const uint4& b) {
  if ((reinterpret_cast<uintptr_t>(p) & 31) == 0) {
    asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(a.x), "r"(a.y), "r"(a.z),
                 "r"(a.w), "r"(b.x), "r"(b.y), "r"(b.z), "r"(b.w)
                 : "memory");
  } else {
    static_cast<uint4*>(p)[0] = a;
    static_cast<uint4*>(p)[1] = b;
  }
}
GDN2_DEV void ld_32bytes(const float* p, float* x) {
  uint32_t r[8];
  if ((reinterpret_cast<uintptr_t>(p) & 31) == 0) {
    asm volatile("ld.global.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
                 : "l"(p)
                 : "memory");
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) r[e] = __float_as_uint(p[e]);
  }
#pragma unroll
  for (int e = 0; e < 8; ++e) x[e] = __uint_as_float(r[e]);
}
// Bounded waits.  One lane: the retry loop is one copy of code.  A whole warp:
// votes keep it converged in a way that the compiler can see (a call would not).
__device__ __noinline__ bool wait_slow(uint64_t* bar, uint32_t parity) { return tc::mbar_wait(bar, parity); }
GDN2_DEV bool wait(uint64_t* bar, uint32_t parity) {
  return tc::mbar_try_wait(tc::smem_u32(bar), parity) || wait_slow(bar, parity);
}
GDN2_DEV bool warp_wait(uint64_t* bar, uint32_t parity) {
  const uint32_t addr = tc::smem_u32(bar);
  bool r = __all_sync(0xffffffffu, tc::mbar_try_wait(addr, parity));
  if (!r) {
    const uint64_t t0 = tc::globaltimer_ns();
    do {
      r = __all_sync(0xffffffffu, tc::mbar_try_wait(addr, parity));
    } while (!r && __all_sync(0xffffffffu, tc::globaltimer_ns() - t0 < tc::kWaitLimitNs));
  }
  return r;
}

template <int K, bool kOut, bool kStore, bool kBack>
__global__ void __launch_bounds__(kOut ? 640 : 256, 1)
la_scan_kernel(const __grid_constant__ ScanArgs p, const __grid_constant__ CUtensorMap tmX, const __grid_constant__ CUtensorMap tmQ,
               const __grid_constant__ CUtensorMap tmY, const __grid_constant__ CUtensorMap tmS) {
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  using Sm = ScanSmem<K, kOut>;
  Sm& sm = *reinterpret_cast<Sm*>(smem_raw);
  constexpr uint32_t NX = Sm::NX, NY = Sm::NY, NB = Sm::NB;
  // TMEM columns: two score buffers, Q S of two chunks, P V, the state term
  constexpr uint32_t kColQK = 0, kColO1 = 256, kColO2 = 384, kColDS = kOut ? 448 : 0;
  constexpr uint32_t kCols = kOut ? 512 : 128;
  const int tid = threadIdx.x, warp = uniform(tid >> 5), lane = tid & 31;
  if (tid == 0) {
    for (uint32_t i = 0; i < NX; ++i) {
      tc::mbar_init(&sm.full_x[i], 1);
      tc::mbar_init(&sm.empty_x[i], kOut ? 2 : 1);  // one per issuer
    }
    for (uint32_t i = 0; i < NY; ++i) {
      tc::mbar_init(&sm.full_y[i], 1);
      tc::mbar_init(&sm.empty_y[i], kOut ? 1 : 128);
      tc::mbar_init(&sm.y_ready[i], 128);
    }
    for (int i = 0; i < 2; ++i) {
      tc::mbar_init(&sm.f_full[i], 32);
      tc::mbar_init(&sm.f_empty[i], kOut ? 16 : 4);  // one per warp that reads them
      tc::mbar_init(&sm.qk_full[i], 1);
      tc::mbar_init(&sm.p_full[i], 256);
      tc::mbar_init(&sm.o_full[i], 2);  // Q S and P V
      tc::mbar_init(&sm.o_free[i], 128);
    }
    for (uint32_t i = 0; i < NB; ++i) {
      tc::mbar_init(&sm.yw_full[i], 128);
      tc::mbar_init(&sm.ds_full[i], 1);
    }
    tc::mbar_init(&sm.ds_free, 128);
    tc::mbar_init(&sm.s_full, 128);
    tc::mbar_init(&sm.s_free, 1);
    tc::mbar_init(&sm.drained, kOut ? 2 : 1);  // one per issuer
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
  int64_t tasks = p.tasks;
  if constexpr (!kOut && !kBack) {  // only segments that are full have one after them
    if (p.pre && p.seg.order) tasks = uniform(min(tasks, (int64_t)p.seg.order[p.seg.entries] * p.a.HV * (p.a.V >> 6)));
  }
  auto count_chunks = [&]() {  // over all tasks
    uint32_t n = 0;
    for (int64_t id = blockIdx.x; id < tasks; id += step)
      if (find_task<kBack>(p, id, t)) n += (uint32_t)max(t.ce - t.cb, 0);
    return n;
  };
  // w v of chunk `it`, row j of its tile (token j): made in registers, so that it can
  // be ready before the MMAs have read the chunk before's, then put in shared memory.
  // f_row: e^{G_j}, total: e^{G_C}.
  uint32_t wh[32], wl[32];
  auto prepare = [&](int c, int j, float& f_row, float& total) -> bool {
    const int s = it & 1;
    const uint32_t sy = it % NY;
    if (!warp_wait(&sm.f_full[s], (it >> 1) & 1)) return false;
    const Sums& g = sm.f[s];
    f_row = exp_of(g.hi[j]);
    total = exp_of(g.hi[kC - 1] + __bfloat162float(g.lo[kC - 1]));
    const float f = j >= rows(c) ? 0.f : kBack ? p.a.scale * f_row : exp_of(sum_diff(g, kC - 1, j));
    __syncwarp();
    if (lane == 0) tc::mbar_arrive(&sm.f_empty[s]);
    const uint32_t fh = pack_bf16(f, f);
    const float fr = f - bf16_round(f);
    const uint32_t fl = pack_bf16(fr, fr);
    const char* src = reinterpret_cast<const char*>(sm.Y[sy]) + j * 128;
    if (!warp_wait(&sm.full_y[sy], (it / NY) & 1)) return false;
#pragma unroll
    for (int q = 0; q < 8; ++q) {
      const uint4 v4 = *reinterpret_cast<const uint4*>(src + ((q ^ (j & 7)) << 4));
      const uint32_t v[4] = {v4.x, v4.y, v4.z, v4.w};
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        wh[4 * q + e] = tc::bmul2(v[e], fh);
        // what the product of the leading parts lost (exact), and the trailing part's product; of an
        // infinity, which the leading part carries, those of the largest finite value: not inf - inf
        const uint32_t u = tc::bmin_abs2(v[e], 0x7f7f7f7fu);
        wl[4 * q + e] = tc::bfma2(u, fl, tc::bfma2(u, fh, tc::bmul2(u, fh) ^ 0x80008000u));
      }
    }
    return true;
  };
  auto put = [&](int c, int j) -> bool {
    const uint32_t sy = it % NY, b = it % NB;
    const int L = rows(c);
    char* hi = reinterpret_cast<char*>(sm.YW[b][0]) + j * 128;
    char* lo = reinterpret_cast<char*>(sm.YW[b][1]) + j * 128;
    // rows of the next sequence in this tile: none of them may reach a sum
    const bool clear = p.geo.cu && L < kC;
    if (clear && !warp_wait(&sm.full_x[it % NX], (it / NX) & 1)) return false;
    if (it >= NB && !warp_wait(&sm.ds_full[b], (it / NB - 1) & 1)) return false;  // YW has been read
    if (clear && j >= L) {
#pragma unroll
      for (int q = 0; q < 32; ++q) wh[q] = wl[q] = 0;
      for (int q = 0; q < 8; ++q) {
        *reinterpret_cast<uint4*>(reinterpret_cast<char*>(sm.Y[sy]) + j * 128 + 16 * q) = make_uint4(0, 0, 0, 0);
#pragma unroll
        for (int e = 0; e < K / 64; ++e)
          *reinterpret_cast<uint4*>(reinterpret_cast<char*>(sm.X[it % NX][e]) + j * 128 + 16 * q) = make_uint4(0, 0, 0, 0);
      }
    }
#pragma unroll
    for (int q = 0; q < 8; ++q) {
      const int at = (q ^ (j & 7)) << 4;
      *reinterpret_cast<uint4*>(hi + at) = make_uint4(wh[4 * q], wh[4 * q + 1], wh[4 * q + 2], wh[4 * q + 3]);
      *reinterpret_cast<uint4*>(lo + at) = make_uint4(wl[4 * q], wl[4 * q + 1], wl[4 * q + 2], wl[4 * q + 3]);
    }
    tc::fence_proxy_async();
    tc::mbar_arrive(&sm.yw_full[b]);
    if constexpr (kOut) tc::mbar_arrive(&sm.y_ready[sy]);  // landed, and clear of other sequences' rows
    else tc::mbar_arrive(&sm.empty_y[sy]);
    return true;
  };

  if (warp == 0) {
    // ---------------------------------------------------------------- loads
    if (lane == 0) {
      tc::prefetch_tensormap(&tmX);
      tc::prefetch_tensormap(&tmY);
      if (kOut) tc::prefetch_tensormap(&tmQ);
      for (int64_t id = blockIdx.x; id < tasks && ok; id += step) {
        if (!find_task<kBack>(p, id, t)) continue;
        const int b = p.geo.cu ? 0 : (int)t.n;
        if (t.head && p.init && t.z == 0)  // both slices' state, ahead of the task's turn
          l2_prefetch(p.init + (t.n * p.a.HV + t.hv) * K * p.a.V, (int)(K * p.a.V * 4));
        for (int i = 0; i < t.ce - t.cb; ++i, ++it) {
          const uint32_t sx = it % NX, sy = it % NY;
          const int tt = tok(nth(i));
          if (it >= NY && !(ok = wait(&sm.empty_y[sy], (it / NY - 1) & 1))) break;
          tc::mbar_arrive_expect_tx(&sm.full_y[sy], kTile);
          tc::tma_load_4d(sm.Y[sy], &tmY, &sm.full_y[sy], 64 * t.z, (int)t.hv, tt, b);
          if (it >= NX && !(ok = wait(&sm.empty_x[sx], (it / NX - 1) & 1))) {
            wait(&sm.full_y[sy], (it / NY) & 1);
            break;
          }
          tc::mbar_arrive_expect_tx(&sm.full_x[sx], (kOut ? 2 : 1) * (K / 64) * kTile);
#pragma unroll
          for (int c = 0; c < K / 64; ++c) {
            tc::tma_load_4d(sm.X[sx][c], &tmX, &sm.full_x[sx], 64 * c, (int)t.h, tt, b);
            if constexpr (kOut) tc::tma_load_4d(sm.X[sx][K / 64 + c], &tmQ, &sm.full_x[sx], 64 * c, (int)t.h, tt, b);
          }
        }
      }
      // loads in flight land before the CTA exits, also after a wait that gave up
      for (uint32_t j = it > NY ? it - NY : 0; !ok && j < it; ++j) {
        wait(&sm.full_x[j % NX], (j / NX) & 1);
        wait(&sm.full_y[j % NY], (j / NY) & 1);
      }
    }
  } else if (warp == 1) {
    // ---------------------- MMAs: Q K^T, P V; without outputs: entering states out
    if constexpr (!kOut) {
      if (kStore && lane == 0) {
        for (int64_t id = blockIdx.x; id < tasks && ok; id += step) {
          if (!find_task<kBack>(p, id, t)) continue;
          for (int i = 0; i < t.ce - t.cb; ++i, ++it) {
            if (!(ok = wait(&sm.s_full, it & 1))) break;
            tc::tma_store_2d(&tmS, sm.S, 64 * t.z, (int)(((t.chunk0 + nth(i)) * p.a.HV + t.hv) * K));
            tc::bulk_commit();
            tc::bulk_wait_read_all();
            tc::mbar_arrive(&sm.s_free);
          }
        }
        tc::bulk_wait_all();
      }
    } else if (tc::elect_one()) {
      constexpr uint32_t iQK = tc::idesc_bf16(128, 128, 0, 0), iNV = tc::idesc_bf16(128, 64, 0, 1);
      const uint32_t aX = addr16(sm.X), aY = addr16(sm.Y), total = count_chunks();
      for (; it < total + (total > 0 ? 1 : 0); ++it) {
        const uint32_t s = it & 1, sx = it % NX;
        if (it < total) {
          const uint32_t ax = aX + sx * (uint32_t)(sizeof(sm.X[0]) >> 4), aq = ax + (K / 64) * (kTile >> 4);
          if (!(ok = wait(&sm.full_x[sx], (it / NX) & 1))) break;
          tc::tc_fence_after();
#pragma unroll
          for (int kk = 0; kk < K / 16; ++kk)
            tc::mma_bf16(tb + kColQK + 128 * s, kmaj(aq, kk), kmaj(ax, kk), iQK, kk > 0);
          tc::mma_commit(&sm.qk_full[s]);
          tc::mma_commit(&sm.empty_x[sx]);
        }
        if (it > 0) {
          const uint32_t j = it - 1, sj = j & 1, sy = j % NY;
          if (j > 0 && !(ok = wait(&sm.o_free[(j - 1) & 1], ((j - 1) >> 1) & 1))) break;  // P V of the chunk before has left TMEM
          if (!(ok = wait(&sm.y_ready[sy], (j / NY) & 1) && wait(&sm.p_full[sj], (j >> 1) & 1))) break;
          tc::tc_fence_after();
#pragma unroll
          for (int kk = 0; kk < 8; ++kk)  // P: columns 0-31 and 64-95 of the score buffer
            tc::mma_bf16_ts(tb + kColO2, tb + kColQK + 128 * sj + 8 * kk + (kk < 4 ? 0 : 32),
                            nmaj(aY + sy * (kTile >> 4), kk), iNV, kk > 0);
          tc::mma_commit(&sm.o_full[sj]);
          tc::mma_commit(&sm.empty_y[sy]);
        }
      }
      tc::mma_commit(&sm.drained);  // what was issued has completed before TMEM is released
      if (!wait(&sm.drained, 0)) ok = false;
    }
  } else if (warp == 3) {
    // --------------------------------------------- MMAs: K^T (w v), Q S
    if (tc::elect_one()) {
      constexpr uint32_t iNV = tc::idesc_bf16(128, 64, 0, 1), iDS = tc::idesc_bf16(K, 64, 1, 1);
      const uint32_t aX = addr16(sm.X), aW = addr16(sm.YW), aS = addr16(sm.S), total = count_chunks();
      for (; it < total; ++it) {
        const uint32_t s = it & 1, sx = it % NX, b = it % NB;
        const uint32_t ax = aX + sx * (uint32_t)(sizeof(sm.X[0]) >> 4), aq = ax + (K / 64) * (kTile >> 4);
        if (!(ok = wait(&sm.full_x[sx], (it / NX) & 1) && wait(&sm.yw_full[b], (it / NB) & 1))) break;
        if constexpr (kOut) {  // the state term of the chunk before has left TMEM
          if (it > 0 && !(ok = wait(&sm.ds_free, (it - 1) & 1))) break;
        }
        tc::tc_fence_after();
#pragma unroll
        for (int e = 0; e < 2; ++e)
#pragma unroll
          for (int kk = 0; kk < 8; ++kk)
            tc::mma_bf16(tb + kColDS + 64 * b, nmaj(ax, kk), nmaj(aW + (2 * b + e) * (kTile >> 4), kk), iDS, e + kk > 0);
        tc::mma_commit(&sm.ds_full[b]);
        if constexpr (kOut) {
          // Q S of two chunks before has left TMEM.  (A barrier per buffer: its next phase needs the
          // Q S below.  With one barrier for both, the output of the chunk between, which needs nothing
          // more from this warp, could end its phase first, and this wait would see the other parity.)
          if (it >= 2 && !(ok = wait(&sm.o_free[s], ((it >> 1) & 1) ^ 1))) break;
          if (!(ok = wait(&sm.s_full, it & 1))) break;
          tc::tc_fence_after();
#pragma unroll
          for (int kk = 0; kk < K / 16; ++kk)
            tc::mma_bf16(tb + kColO1 + 64 * s, kmaj(aq, kk), nmaj(aS, kk), iNV, kk > 0);
          tc::mma_commit(&sm.o_full[s]);
        }
        tc::mma_commit(&sm.empty_x[sx]);  // also: S has been read
      }
      tc::mma_commit(&sm.drained);
      if (!wait(&sm.drained, 0)) ok = false;
    }
  } else if (warp == 2) {
    // ---------------------------- sums; with outputs also the entering states out
    constexpr bool kStoreHere = kOut && kStore;
    // (the sums run ahead of the states, so each turn stores the one of two chunks before)
    int out_row[2] = {0, 0}, out_z[2] = {0, 0};
    auto store = [&](uint32_t d) -> bool {
      if (!warp_wait(&sm.s_full, d & 1)) return false;
      if (lane == 0) {
        tc::tma_store_2d(&tmS, sm.S, 64 * (d & 1 ? out_z[1] : out_z[0]), d & 1 ? out_row[1] : out_row[0]);
        tc::bulk_commit();
        tc::bulk_wait_read_all();
        tc::mbar_arrive(&sm.s_free);
      }
      __syncwarp();
      return true;
    };
    for (int64_t id = blockIdx.x; id < tasks && ok; id += step) {
      if (!get_task<kBack>(p, id, t)) continue;
      // this lane's four tokens of a chunk lie `gs` bytes apart (0: one decay for all)
      const int es = p.dec.dtype == GDN2_BF16 ? 2 : 4;
      const bool token = p.dec.kind == GDN2_DECAY_TOKEN;
      const int64_t gs = token ? p.dec.st * es : 0;
      const char* g0 = static_cast<const char*>(p.dec.g) +
                       (t.hv * p.dec.sh + (token ? (p.geo.cu ? t.bos * p.dec.st : t.n * p.dec.sb) : 0)) * es;
      uint32_t raw[4];
      double sum = 0.0;
      auto load = [&](int c) {
        const int left = p.dec.kind == GDN2_DECAY_NONE ? 0 : rows(c) - 4 * lane;
        const char* g = g0 + ((int64_t)c * kC + 4 * lane) * gs;
#pragma unroll
        for (int e = 0; e < 4; ++e)
          raw[e] = e >= left ? 0
                   : es == 2 ? *reinterpret_cast<const uint16_t*>(g + e * gs) : *reinterpret_cast<const uint32_t*>(g + e * gs);
      };
      const int nloc = t.ce - t.cb;
      if (nloc > 0) load(nth(0));
      for (int i = 0; i < nloc; ++i, ++it) {
        const int s = it & 1;
        double G[4];
        G[0] = p.dec.value(raw[0]);
#pragma unroll
        for (int e = 1; e < 4; ++e) G[e] = G[e - 1] + p.dec.value(raw[e]);
        if (i + 1 < nloc) load(nth(i + 1));  // in flight until the next turn
        double inc = G[3];
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const double y = __shfl_up_sync(0xffffffffu, inc, o);
          if (lane >= o) inc += y;
        }
        const double before = __shfl_up_sync(0xffffffffu, inc, 1);
        float hi[4], lo[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          G[e] += lane ? before : 0.0;
          hi[e] = (float)G[e];
          lo[e] = (float)(G[e] - (double)hi[e]);
        }
        if (p.pre) sum += __shfl_sync(0xffffffffu, inc, 31);
        if constexpr (kStoreHere) {
          if (it >= 2 && !(ok = store(it - 2))) break;
        }
        if (it >= 2 && !(ok = warp_wait(&sm.f_empty[s], ((it >> 1) & 1) ^ 1))) break;
        reinterpret_cast<float4*>(sm.f[s].hi)[lane] = make_float4(hi[0], hi[1], hi[2], hi[3]);
        reinterpret_cast<uint2*>(sm.f[s].lo)[lane] = make_uint2(pack_bf16(lo[0], lo[1]), pack_bf16(lo[2], lo[3]));
        tc::mbar_arrive(&sm.f_full[s]);
        if constexpr (kStoreHere) {
          const int r = (int)(((t.chunk0 + nth(i)) * p.a.HV + t.hv) * K);
          if (s) out_row[1] = r, out_z[1] = t.z;
          else out_row[0] = r, out_z[0] = t.z;
        }
      }
      if (p.pre && lane == 0 && t.z == 0) p.seg.D[t.entry * p.a.HV + t.hv] = expf((float)sum);
    }
    if constexpr (kStoreHere) {
      if (ok && it > 1) ok = store(it - 2);
      if (ok && it > 0) ok = store(it - 1);
      if (lane == 0) tc::bulk_wait_all();
    }
  } else if (kOut && warp < 12) {
    // --------------------------------------------------------------- scores
    const int w = warp & 3, i = 32 * w + lane, p2 = (warp - 4) >> 2;  // columns 64 p2 .. 64 p2 + 63
    for (int64_t id = blockIdx.x; id < tasks && ok; id += step) {
      if (!get_task<kBack>(p, id, t)) continue;
      for (int j = 0; j < t.ce - t.cb; ++j, ++it) {
        const int s = it & 1;
        const uint32_t tp = tb + kColQK + 128 * s + 64 * p2 + ((uint32_t)(32 * w) << 16);
        if (!(ok = warp_wait(&sm.f_full[s], (it >> 1) & 1))) break;
        const Sums& f = sm.f[s];
        const float gi = sum_diff(f, i, 32 * w) * kLog2e;
        float* cw = sm.cw + 16 * w * (w + 1);  // (both warps with this w: each its own columns)
        if (64 * p2 < 32 * w) cw[64 * p2 + lane] = exp2_approx(sum_diff(f, 32 * w, 64 * p2 + lane) * kLog2e);
        if (64 * p2 + 32 < 32 * w) cw[64 * p2 + 32 + lane] = exp2_approx(sum_diff(f, 32 * w, 64 * p2 + 32 + lane) * kLog2e);
        if (p2 == w >> 1) cw[i] = gi;
        __syncwarp();
        if (lane == 0) tc::mbar_arrive(&sm.f_empty[s]);
        const float ri = exp2_approx(gi);
        const uint64_t ri2 = tc::pack2(ri, ri);
        if (!(ok = warp_wait(&sm.qk_full[s], (it >> 1) & 1))) break;
        tc::tc_fence_after();
#pragma unroll 1
        for (int b = 0; b < 4; ++b) {  // 16 columns a turn: a short loop stays in the instruction cache
          const int c0 = 64 * p2 + 16 * b, d0 = c0 - 32 * w;  // first column, and its place in the diagonal block
          const float4* cc = reinterpret_cast<const float4*>(cw + c0);
          uint32_t pk[8];
          if (d0 >= 32) {
#pragma unroll
            for (int e = 0; e < 8; ++e) pk[e] = 0;
          } else {
            float x[16];
            tc::tmem_ld16(tp + 16 * b, x);
            tc::tmem_wait_ld();
            if (d0 < 0) {
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                const float4 c = cc[e];
                float y[4];
                tc::unpack2(tc::mul2(tc::mul2(tc::pack2(x[4 * e], x[4 * e + 1]), tc::pack2(c.x, c.y)), ri2), y[0], y[1]);
                tc::unpack2(tc::mul2(tc::mul2(tc::pack2(x[4 * e + 2], x[4 * e + 3]), tc::pack2(c.z, c.w)), ri2), y[2],
                            y[3]);
                pk[2 * e] = pack_bf16(y[0], y[1]);
                pk[2 * e + 1] = pack_bf16(y[2], y[3]);
              }
            } else {
              const int last = lane - d0;  // columns up to this one are not in the future
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                const float4 c = cc[e];
                const float d[4] = {c.x, c.y, c.z, c.w};
                float y[4];
#pragma unroll
                for (int u = 0; u < 4; ++u) y[u] = 4 * e + u <= last ? x[4 * e + u] * exp2_approx(gi - d[u]) : 0.f;
                pk[2 * e] = pack_bf16(y[0], y[1]);
                pk[2 * e + 1] = pack_bf16(y[2], y[3]);
              }
            }
          }
          tc::tmem_st8(tp + 8 * b, pk);
        }
        tc::tmem_wait_st();
        tc::tc_fence_before();
        tc::mbar_arrive(&sm.p_full[s]);
      }
    }
  } else if (kOut ? warp < 16 : warp >= 4) {
    // ---------------------------------------------------------------- state
    const int w = warp & 3, row = K == 128 ? 32 * w + lane : 16 * w + (lane & 15), j = 32 * w + lane;
    const bool own = K == 128 || lane < 16;  // M = 64: rows in the first 16 lanes of each quarter
    const uint32_t td = tb + kColDS + ((uint32_t)(32 * w) << 16);
    float st[64];
    float total = 0.f, total_next = 0.f;  // e^{G_C} of the chunk before, of this one
    // S <- total S + the term of chunk d
    auto take = [&](uint32_t d) -> bool {
      const uint32_t b = d % NB;
      const uint64_t f2 = tc::pack2(total, total);
      if (!warp_wait(&sm.ds_full[b], (d / NB) & 1)) return false;
      tc::tc_fence_after();
#pragma unroll
      for (int h = 0; h < 4; ++h) {
        float x[16];
        tc::tmem_ld16(td + 64 * b + 16 * h, x);
        tc::tmem_wait_ld();
#pragma unroll
        for (int e = 0; e < 16; e += 2) {
          float* y = st + 16 * h + e;
          tc::unpack2(tc::fma2(tc::pack2(y[0], y[1]), f2, tc::pack2(x[e], x[e + 1])), y[0], y[1]);
        }
      }
      tc::tc_fence_before();
      if constexpr (kOut) tc::mbar_arrive(&sm.ds_free);
      return true;
    };
    // the bf16 state of chunk `it`
    auto publish = [&]() -> bool {
      if (kStore && it > 0 && !warp_wait(&sm.s_free, (it - 1) & 1)) return false;
      if constexpr (kOut) {  // Q S of the chunk before is done
        if (it > 0 && !warp_wait(&sm.empty_x[(it - 1) % NX], ((it - 1) / NX) & 1)) return false;
      }
      char* dst = reinterpret_cast<char*>(sm.S) + row * 128;
      if (own) {
#pragma unroll
        for (int q = 0; q < 8; ++q) *reinterpret_cast<uint4*>(dst + ((q ^ (row & 7)) << 4)) = pack8(st + 8 * q);
      }
      tc::fence_proxy_async();
      tc::mbar_arrive(&sm.s_full);
      return true;
    };
    const int64_t KV = (int64_t)K * p.a.V;
    for (int64_t id = blockIdx.x; id < tasks && ok; id += step) {
      if (!get_task<kBack>(p, id, t)) continue;
      const int64_t at = (int64_t)row * p.a.V + 64 * t.z;
      const float* src = t.head ? (p.init ? p.init + (t.n * p.a.HV + t.hv) * KV : nullptr)
                         : p.pre ? nullptr
                                 : p.seg.X + ((t.entry + (kBack ? 1 : -1)) * p.a.HV + t.hv) * KV;
#pragma unroll
      for (int q = 0; q < 64; ++q) st[q] = 0.f;
      if (src) {
#pragma unroll
        for (int q = 0; q < 64; q += 8) ld_32bytes(src + at + q, st + q);
      }
      const int nloc = t.ce - t.cb;
      for (int i = 0; i <= nloc; ++i) {
        if constexpr (kOut) {
          if (i < nloc) {
            const int f = it & 1;
            if (!(ok = warp_wait(&sm.f_full[f], (it >> 1) & 1))) break;
            total_next = exp_of(sm.f[f].hi[kC - 1] + __bfloat162float(sm.f[f].lo[kC - 1]));
            __syncwarp();
            if (lane == 0) tc::mbar_arrive(&sm.f_empty[f]);
          }
        } else {  // (two buffers: the next w v goes in before the MMA of the chunk before has ended)
          float f_row;
          if (i < nloc && !(ok = prepare(nth(i), j, f_row, total_next) && put(nth(i), j))) break;
        }
        if (i > 0 && !(ok = take(it - 1))) break;
        total = total_next;
        if (i == nloc) break;
        if constexpr (kOut || kStore) {
          if (!(ok = publish())) break;
        }
        ++it;
      }
      if (!ok) break;
      float* dst = p.pre ? p.seg.X + (t.entry * p.a.HV + t.hv) * KV
                   : t.tail && p.fin ? p.fin + (t.n * p.a.HV + t.hv) * KV : nullptr;
      if (dst && own) {
#pragma unroll
        for (int q = 0; q < 16; ++q)
          *reinterpret_cast<float4*>(dst + at + 4 * q) = make_float4(st[4 * q], st[4 * q + 1], st[4 * q + 2], st[4 * q + 3]);
      }
    }
  } else if (kOut) {
    // ---------------------------------------------------------- w v, output
    // Chunk it's w v comes before chunk it - 2's output, across tasks too: the
    // MMAs of chunk it wait for the one and go before the other's end.
    const int w = warp & 3, i = 32 * w + lane;
    const uint32_t to = tb + ((uint32_t)(32 * w) << 16);
    const uint64_t sc2 = tc::pack2(p.a.scale, p.a.scale);
    const int64_t chunk_step = (int64_t)kC * p.a.HV * p.a.V;
    // of chunks it - 2 and it - 1: e^{G_i}, and this thread's row of o (NULL past the sequence's end)
    float f = 0.f, f1 = 0.f, f_next = 0.f, total;
    __nv_bfloat16 *dst = nullptr, *dst1 = nullptr;
    auto output = [&](uint32_t d) -> bool {
      if (!warp_wait(&sm.o_full[d & 1], (d >> 1) & 1)) return false;
      tc::tc_fence_after();
      const uint64_t f2 = tc::mul2(sc2, tc::pack2(f, f));
#pragma unroll 1
      for (int h = 0; h < 4; ++h) {
        float x[16], y[16];
        tc::tmem_ld16(to + kColO1 + 64 * (d & 1) + 16 * h, x);
        tc::tmem_ld16(to + kColO2 + 16 * h, y);
        tc::tmem_wait_ld();
#pragma unroll
        for (int e = 0; e < 16; e += 2)
          tc::unpack2(tc::fma2(f2, tc::pack2(x[e], x[e + 1]), tc::mul2(sc2, tc::pack2(y[e], y[e + 1]))), x[e], x[e + 1]);
        if (dst) st_32bytes(dst + 16 * h, pack8(x), pack8(x + 8));
      }
      tc::tc_fence_before();
      tc::mbar_arrive(&sm.o_free[d & 1]);
      return true;
    };
    for (int64_t id = blockIdx.x; id < tasks && ok; id += step) {
      if (!get_task<kBack>(p, id, t)) continue;
      __nv_bfloat16* const row0 =
          static_cast<__nv_bfloat16*>(p.a.o) + ((t.bos + i) * p.a.HV + t.hv) * p.a.V + 64 * t.z;
      for (int j = 0; j < t.ce - t.cb; ++j, ++it) {
        const int c = nth(j);
        if (!(ok = prepare(c, i, f_next, total) && put(c, i))) break;
        if (it > 1 && !(ok = output(it - 2))) break;
        f = f1;
        dst = dst1;
        f1 = f_next;
        dst1 = i < rows(c) ? row0 + c * chunk_step : nullptr;
      }
    }
    if (ok && it > 1) ok = output(it - 2);
    f = f1;
    dst = dst1;
    if (ok && it > 0) ok = output(it - 1);
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
  int64_t bos, len;
  geo.seq(n, bos, len);
  const int64_t ns = seg.count(n, (len + kC - 1) / kC);
  const int64_t e0 = seg.first_of(n);
  if (ns < 3) return;  // the first segment's term is a whole state already, the last one's is not used
  for (int64_t e = ((int64_t)blockIdx.y * 128 + threadIdx.x) * 4; e < KV; e += (int64_t)gridDim.y * 512) {
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
}

// sum of 8 products of bf16 pairs
GDN2_DEV float dot8(const uint4& a, const uint4& b) {
  const uint32_t x[4] = {a.x, a.y, a.z, a.w}, y[4] = {b.x, b.y, b.z, b.w};
  float s = 0.f, t = 0.f;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    s = fmaf(__uint_as_float(x[i] << 16), __uint_as_float(y[i] << 16), s);
    t = fmaf(__uint_as_float(x[i] & 0xffff0000u), __uint_as_float(y[i] & 0xffff0000u), t);
  }
  return s + t;
}
// 16 bf16 of a swizzled row (pieces p0, p0 + 1) times 16 floats
GDN2_DEV float dot16(const unsigned char* row_base, int p0, int row, const float (&y)[16]) {
  float s = 0.f, t = 0.f;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const uint4 v = *reinterpret_cast<const uint4*>(row_base + (((p0 + h) ^ (row & 7)) << 4));
    const uint32_t x[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      s = fmaf(__uint_as_float(x[i] << 16), y[8 * h + 2 * i], s);
      t = fmaf(__uint_as_float(x[i] & 0xffff0000u), y[8 * h + 2 * i + 1], t);
    }
  }
  return s + t;
}

// ---------------------------------------------------------------------------
// Backward, one chunk of 128 tokens and one value head at a time (all chunks in
// parallel), from the chunk's entering state S and leaving cotangent dS':
//     P^T_ji = scale e^{G_i - G_j} (k_j . q_i),  E^T_ji = scale e^{G_i - G_j} (v_j . do_i)   (i >= j)
//     dq = scale e^G do S^T + E k      dk = e^{G_C - G} v dS'^T + E^T q      dv = e^{G_C - G} k dS' + P^T do
// Nine products of M = 128 tokens.  The scores come out transposed (rows j), so
// that P^T and E^T are TMEM operands of dv and dk as they are; E^T also goes to
// shared memory, where it is the M-major operand of dq.  The products with the
// states land in the gradients' accumulators first; their rows are scaled
// there, then the products within the chunk add to them.
// dg: with X_i = q_i . dq_i and Y_j = k_j . dk_j (fp32, before rounding), whose parts from within the
// chunk use the same bf16 E and so cancel where they must,
//     dg_t = sum_{i>=t} (X_i - Y_i) + sum_j k_j . (e^{G_C - G_j} v_j dS'^T) + e^{G_C} <S, dS'>.
// A sequence's first token without an initial state decays nothing: exactly zero.
// Y's part from within the chunk is sum_i E_ij (k_j . q_i), taken from the scores as they are weighed, so that
// k is not read again.  Shared memory holds one chunk's six tiles and E^T; S, v and dS' make room for the next
// chunk's q, k and do while this one is being finished, then k, q and do for its v, S and dS'.
//   warp 0 loads, warp 1 dg, warp 2 running sums, warp 3 MMAs,
//   warps 4-19: thread = token (TMEM lane) and a quarter of the columns
// What bounds it: a chunk's six tiles fill shared memory at K = V = 128 (and have the same
// room at 64, where two chunks' would fit), so little of the next one's
// loads, and none of its products, runs beside this one's chain of products and row
// passes; the nine products are 4600 of some 16000 clocks.  Sixteen row warps instead
// of eight overlap the passes' TMEM latencies: 136 -> 127 us.  Measured at 4 sequences
// of 4096 tokens, 16 heads, K = V = 128: 125 us (604 MB, 4.8 TB/s), 112 us without dg
// (the next chunk's tiles fetched into L2 beforehand: no change, so it is the chain).
// ---------------------------------------------------------------------------
constexpr float kLoUnit = 1.f / 16777216.f / 127.f;

enum Tile { kTQ = 0, kTK, kTO, kTV, kTS, kTD };  // q, k, do, v, S, dS'

struct alignas(1024) BwdSmem {
  __nv_bfloat16 slot[6][128 * 128];
  __nv_bfloat16 E[2][128 * 64];  // E^T, rows j
  float hi[kC];                  // running sums of g, and
  int8_t lo[kC];                 // what they miss, in 127ths of |hi| 2^-24 (half a unit in hi's last place at most)
  float g2[kC];                  // (G_i - G_{32 floor(i / 32)}) log2 e
  float r[kC];                   // 2^g2
  float xy[2][kC];               // X - Y, per half of the columns (two terms on a zero: their order is nothing)
  float part[32];                // per warp: sum of k . dk (state part), e^{G_C} <S, dS'>
  uint64_t full[6], empty[6], f_full, f_empty, clean, g1, g2_, pe, rmw1, g3, rmw2, g4a, g4b, qk_free, dv_free, xy_full,
      xy_free, aborted;
  uint32_t tbase;
};

struct BwdArgs {
  gdn2_linear_attn_args a;
  gdn2_linear_attn_grads gr;
  LaDecay dec;
  LaGeom geo;
  int64_t items;  // chunks (bound) x key heads
  float* acc;     // [CTAs, 2, 128, K] running sums of dq, dk over a group of value heads
  float* dgf;     // [B, T, HV] fp32 terms of a per-head decay's gradient, or NULL
};

template <int K, int V, bool kDg>
__global__ void __launch_bounds__(640, 1)
la_bwd_tc_kernel(const __grid_constant__ BwdArgs p, const __grid_constant__ CUtensorMap tmQ,
                 const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV,
                 const __grid_constant__ CUtensorMap tmO, const __grid_constant__ CUtensorMap tmS,
                 const __grid_constant__ CUtensorMap tmD) {
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  BwdSmem& sm = *reinterpret_cast<BwdSmem*>(smem_raw);
  constexpr uint32_t kColA1 = 0, kColA2 = 128, kColDq = 256, kColDk = 384;  // dv: over A2
  const int tid = threadIdx.x, warp = uniform(tid >> 5), lane = tid & 31;
  if (tid == 0) {
    for (int i = 0; i < 6; ++i) {
      tc::mbar_init(&sm.full[i], 1);
      tc::mbar_init(&sm.empty[i], 17);  // the MMAs' commit and the row warps
    }
    tc::mbar_init(&sm.f_full, 32);
    tc::mbar_init(&sm.f_empty, 16);
    tc::mbar_init(&sm.clean, 512);
    tc::mbar_init(&sm.g1, 1);
    tc::mbar_init(&sm.g2_, 1);
    tc::mbar_init(&sm.pe, 512);
    tc::mbar_init(&sm.rmw1, 512);
    tc::mbar_init(&sm.g3, 1);
    tc::mbar_init(&sm.rmw2, 512);
    tc::mbar_init(&sm.g4a, 1);
    tc::mbar_init(&sm.g4b, 1);
    tc::mbar_init(&sm.qk_free, 512);
    tc::mbar_init(&sm.dv_free, 512);
    tc::mbar_init(&sm.xy_full, 512);
    tc::mbar_init(&sm.xy_free, 32);
    tc::mbar_init(&sm.aborted, 1);
    tc::mbar_fence_init();
  }
  if (tid < 2 * kC) sm.xy[0][tid] = 0.f;
  if (warp == 1) tc::tmem_alloc(&sm.tbase, 512);
  tc::tc_fence_before();
  __syncthreads();
  tc::tc_fence_after();
  const uint32_t tb = sm.tbase;
  const int group = (int)(p.a.HV / p.a.H);
  bool ok = true;
  uint32_t n = 0;  // (chunk, value head) pairs this role has been through
  struct {
    int64_t n, c, bos;
    int h, L;
  } w{};
  // item -> sequence, chunk, key head; false past the last chunk
  auto item = [&](int64_t id) -> bool {
    const uint32_t H = (uint32_t)p.a.H, ch = (uint32_t)id / H;
    w.h = (int)((uint32_t)id % H);
    if (!p.geo.chunk(ch, w.n, w.c)) return false;
    int64_t len;
    p.geo.seq(w.n, w.bos, len);
    w.L = (int)min(len - w.c * kC, (int64_t)kC);
    return w.L > 0;
  };
  auto witem = [&](int64_t id) -> bool {
    const bool any = __all_sync(0xffffffffu, item(id));
    w.n = uniform(w.n);
    w.c = uniform(w.c);
    w.bos = uniform(w.bos);
    w.L = uniform(w.L);
    return any;
  };
  // q <-> S, k <-> v, do <-> dS' from one pair to the next
  auto slot_of = [&](int x) -> int { return (n & 1) ? (int)((0x201534u >> (4 * x)) & 7) : x; };
  const int64_t step = gridDim.x;

  if (warp == 0) {
    // ---------------------------------------------------------------- loads
    if (tc::elect_one()) {
      for (int64_t id = blockIdx.x; id < p.items && ok; id += step) {
        if (!item(id)) continue;
        const int b = p.geo.cu ? 0 : (int)w.n, t = (int)((p.geo.cu ? w.bos : 0) + w.c * kC);
        for (int j = 0; j < group && ok; ++j, ++n) {
          const int hv = w.h * group + j;
          const int row = (int)(((p.geo.chunk0(w.n) + w.c) * p.a.HV + hv) * K);
#pragma unroll 1
          for (int x = 0; x < 6; ++x) {
            const int s = slot_of(x);
            if (n > 0 && !(ok = wait(&sm.empty[s], (n - 1) & 1))) break;
            unsigned char* dst = reinterpret_cast<unsigned char*>(sm.slot[s]);
            uint64_t* bar = &sm.full[s];
            const bool state = x >= kTS, key = x <= kTK;
            const int blocks = (key ? K : V) / 64;
            const uint32_t bytes = state ? (uint32_t)K * 128 : kTile;
            tc::mbar_arrive_expect_tx(bar, blocks * bytes);
            const CUtensorMap* m = x == kTQ ? &tmQ : x == kTK ? &tmK : x == kTO ? &tmO : x == kTV ? &tmV
                                                                             : x == kTS ? &tmS : &tmD;
            for (int c = 0; c < blocks; ++c) {
              if (state) tc::tma_load_2d(dst + c * bytes, m, bar, 64 * c, row);
              else tc::tma_load_4d(dst + c * bytes, m, bar, 64 * c, key ? w.h : hv, t, b);
            }
          }
          if (!ok) break;
        }
      }
      if (!ok)  // loads in flight land before the CTA exits, also after a wait that gave up
        for (int s = 0; s < 6; ++s) {
          wait(&sm.full[s], n & 1);
          wait(&sm.full[s], (n + 1) & 1);
        }
    }
  } else if (warp == 3) {
    // ----------------------------------------------------------------- MMAs
    if (tc::elect_one()) {
      constexpr int kRoll = 4;
      constexpr uint32_t iA = tc::idesc_bf16(128, 128, 0, 0), iK = tc::idesc_bf16(128, K, 0, 0);
      constexpr uint32_t iVn = tc::idesc_bf16(128, V, 0, 1), iKn = tc::idesc_bf16(128, K, 0, 1);
      constexpr uint32_t iKmn = tc::idesc_bf16(128, K, 1, 1);
      constexpr uint32_t kBlk = K * 128 / 16;  // a state's 64-column block, in 16-byte units
      const uint32_t a0 = addr16(sm.slot), aE = addr16(sm.E);
      for (int64_t id = blockIdx.x; id < p.items && ok; id += step) {
        if (!item(id)) continue;
        for (int j = 0; j < group; ++j, ++n) {
          const uint32_t par = n & 1, prev = par ^ 1;
          auto at = [&](int x) { return a0 + (uint32_t)slot_of(x) * (sizeof(sm.slot[0]) >> 4); };
          const uint32_t aq = at(kTQ), ak = at(kTK), ao = at(kTO), av = at(kTV), as = at(kTS), ad = at(kTD);
          auto full = [&](int x) { return wait(&sm.full[slot_of(x)], par); };
          if (!(ok = full(kTQ) && full(kTK) && wait(&sm.clean, par))) break;
          tc::tc_fence_after();
#pragma unroll kRoll
          for (int kk = 0; kk < K / 16; ++kk)
            tc::mma_bf16(tb + kColA1, kmaj(ak, kk), kmaj(aq, kk), iA, kk > 0);
          if (!(ok = full(kTO) && full(kTV) && (n == 0 || wait(&sm.dv_free, prev)))) break;
          tc::tc_fence_after();
#pragma unroll kRoll
          for (int kk = 0; kk < V / 16; ++kk)
            tc::mma_bf16(tb + kColA2, kmaj(av, kk), kmaj(ao, kk), iA, kk > 0);
          tc::mma_commit(&sm.g1);
          if (!(ok = full(kTS) && (n == 0 || wait(&sm.qk_free, prev)))) break;
          tc::tc_fence_after();
#pragma unroll kRoll
          for (int kk = 0; kk < V / 16; ++kk)
            tc::mma_bf16(tb + kColDq, kmaj(ao, kk), desc(as + (kk >> 2) * kBlk + (kk & 3) * 2 + (1u << 16)), iK, kk > 0);
          if (!(ok = full(kTD))) break;
          tc::tc_fence_after();
#pragma unroll kRoll
          for (int kk = 0; kk < V / 16; ++kk)
            tc::mma_bf16(tb + kColDk, kmaj(av, kk), desc(ad + (kk >> 2) * kBlk + (kk & 3) * 2 + (1u << 16)), iK, kk > 0);
          tc::mma_commit(&sm.g2_);
          tc::mma_commit(&sm.empty[slot_of(kTV)]);
          tc::mma_commit(&sm.empty[slot_of(kTS)]);
          if (!(ok = wait(&sm.pe, par))) break;
          tc::tc_fence_after();
#pragma unroll kRoll
          for (int kk = 0; kk < K / 16; ++kk)
            tc::mma_bf16(tb + kColA2, kmaj(ak, kk), desc(ad + kk * 128 + (kBlk << 16)), iVn, kk > 0);
          tc::mma_commit(&sm.g3);
          tc::mma_commit(&sm.empty[slot_of(kTD)]);
          if (!(ok = wait(&sm.rmw1, par))) break;
          tc::tc_fence_after();
#pragma unroll kRoll
          for (int kk = 0; kk < 128 / 16; ++kk)
            tc::mma_bf16(tb + kColDq, nmaj(aE, kk), nmaj(ak, kk), iKmn, 1);
#pragma unroll kRoll
          for (int kk = 0; kk < 128 / 16; ++kk)
            tc::mma_bf16_ts(tb + kColDk, tb + kColA1 + 32 * (kk >> 1) + 16 + 8 * (kk & 1), nmaj(aq, kk), iKn, 1);
          tc::mma_commit(&sm.g4a);
          tc::mma_commit(&sm.empty[slot_of(kTQ)]);
          tc::mma_commit(&sm.empty[slot_of(kTK)]);
          if (!(ok = wait(&sm.rmw2, par))) break;
          tc::tc_fence_after();
#pragma unroll kRoll
          for (int kk = 0; kk < 128 / 16; ++kk)
            tc::mma_bf16_ts(tb + kColA2, tb + kColA1 + 32 * (kk >> 1) + 8 * (kk & 1), nmaj(ao, kk), iVn, 1);
          tc::mma_commit(&sm.g4b);
          tc::mma_commit(&sm.empty[slot_of(kTO)]);
        }
      }
      tc::mma_commit(&sm.aborted);  // what was issued has completed before TMEM is released
      if (!wait(&sm.aborted, 0)) ok = false;
    }
  } else if (warp == 2) {
    // ----------------------------------------------------------------- sums
    for (int64_t id = blockIdx.x; id < p.items && ok; id += step) {
      if (!witem(id)) continue;
      const int64_t b = p.geo.cu ? 0 : w.n, t0 = (p.geo.cu ? w.bos : 0) + w.c * kC;
      for (int j = 0; j < group; ++j, ++n) {
        double G[4], x[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] = 4 * lane + e < w.L ? p.dec.at(b, t0 + 4 * lane + e, w.h * group + j) : 0.0;
        G[0] = x[0];
#pragma unroll
        for (int e = 1; e < 4; ++e) G[e] = G[e - 1] + x[e];
        double inc = G[3];
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const double y = __shfl_up_sync(0xffffffffu, inc, o);
          if (lane >= o) inc += y;
        }
        const double before = __shfl_up_sync(0xffffffffu, inc, 1);
#pragma unroll
        for (int e = 0; e < 4; ++e) G[e] += lane ? before : 0.0;
        const double ref = __shfl_sync(0xffffffffu, G[0], lane & 24);  // of this lane's block of 32 tokens
        float hi[4], g2[4], r[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          hi[e] = (float)G[e];
          g2[e] = (float)(G[e] - ref) * kLog2e;
          r[e] = exp2_approx(g2[e]);
        }
        char4 lo;
        auto rest = [&](int e) {  // (hi = 0: 0 times infinity is NaN, which converts to 0)
          return (signed char)__float2int_rn((float)(G[e] - (double)hi[e]) * __frcp_rn(fabsf(hi[e]) * kLoUnit));
        };
        lo.x = rest(0), lo.y = rest(1), lo.z = rest(2), lo.w = rest(3);
        if (n > 0 && !(ok = warp_wait(&sm.f_empty, (n - 1) & 1))) break;
        reinterpret_cast<float4*>(sm.hi)[lane] = make_float4(hi[0], hi[1], hi[2], hi[3]);
        reinterpret_cast<char4*>(sm.lo)[lane] = lo;
        reinterpret_cast<float4*>(sm.g2)[lane] = make_float4(g2[0], g2[1], g2[2], g2[3]);
        reinterpret_cast<float4*>(sm.r)[lane] = make_float4(r[0], r[1], r[2], r[3]);
        tc::mbar_arrive(&sm.f_full);
      }
    }
  } else if (warp == 1) {
    // ------------------------------------------------------------------- dg
    if constexpr (kDg) {
      for (int64_t id = blockIdx.x; id < p.items && ok; id += step) {
        if (!witem(id)) continue;
        for (int j = 0; j < group; ++j, ++n) {
          if (!(ok = warp_wait(&sm.xy_full, n & 1))) break;
          const float4 x0 = reinterpret_cast<const float4*>(sm.xy[0])[lane];
          const float4 x1 = reinterpret_cast<const float4*>(sm.xy[1])[lane];
          float base = sm.part[lane];
          reinterpret_cast<float4*>(sm.xy[0])[lane] = make_float4(0.f, 0.f, 0.f, 0.f);
          reinterpret_cast<float4*>(sm.xy[1])[lane] = make_float4(0.f, 0.f, 0.f, 0.f);
          __syncwarp();
          tc::mbar_arrive(&sm.xy_free);
          float d[4] = {x0.x + x1.x, x0.y + x1.y, x0.z + x1.z, x0.w + x1.w};
#pragma unroll
          for (int o = 16; o > 0; o >>= 1) base += __shfl_xor_sync(0xffffffffu, base, o);
          // sums from each token to the chunk's end
#pragma unroll
          for (int e = 2; e >= 0; --e) d[e] += d[e + 1];
          float s = d[0];
#pragma unroll
          for (int o = 1; o < 32; o <<= 1) {
            const float y = __shfl_down_sync(0xffffffffu, s, o);
            if (lane + o < 32) s += y;
          }
          const float after = s - d[0] + base;
          const int64_t hv = w.h * group + j;
          const bool fresh = w.c == 0 && !(p.a.flags & GDN2_HAS_H0);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int t = 4 * lane + e;
            if (t < w.L) {
              const float v = fresh && t == 0 ? 0.f : d[e] + after;
              const int64_t at = (w.bos + w.c * kC + t) * p.a.HV + hv;
              if (p.dgf) p.dgf[at] = v;
              else if (p.a.dtype_g == GDN2_BF16) static_cast<__nv_bfloat16*>(p.gr.dg)[at] = __float2bfloat16_rn(v);
              else static_cast<float*>(p.gr.dg)[at] = v;
            }
          }
        }
      }
    }
  } else {
    // ----------------------------------------------------------------- rows
    const int q4 = warp & 3, row = 32 * q4 + lane, quarter = (warp - 4) >> 2;
    const uint32_t tl = tb + ((uint32_t)(32 * q4) << 16);
    const int64_t H = p.a.H, HV = p.a.HV;
    float* acc = p.acc + ((int64_t)blockIdx.x * 2 * kC + row) * K + quarter * (K / 4);
    for (int64_t id = blockIdx.x; id < p.items && ok; id += step) {
      if (!witem(id)) continue;
      const int64_t tok = w.bos + w.c * kC + row;
      const bool inside = row < w.L;
      for (int j = 0; j < group; ++j, ++n) {
        const uint32_t par = n & 1;
        const int hv = w.h * group + j;
        auto tile = [&](int x) { return reinterpret_cast<unsigned char*>(sm.slot[slot_of(x)]); };
        auto release = [&](int x) {
          __syncwarp();
          if (lane == 0) tc::mbar_arrive(&sm.empty[slot_of(x)]);
        };
        // rows of the next sequence in these tiles: none of them may reach a sum
        if (p.geo.cu && w.L < kC) {
          for (int x = kTQ; x <= kTV; ++x)
            if (!(ok = warp_wait(&sm.full[slot_of(x)], par))) break;
          if (!ok) break;
          if (!inside) {
#pragma unroll 1
            for (int x = kTQ; x <= kTV; ++x) {
              if ((x <= kTK ? K : V) == 64 && quarter > 1) continue;  // a block of 64 columns: two quarters
              uint4* dst = reinterpret_cast<uint4*>(tile(x) + (quarter >> 1) * kTile + row * 128) + 4 * (quarter & 1);
              for (int e = 0; e < 4; ++e) dst[e] = make_uint4(0, 0, 0, 0);
            }
          }
          tc::fence_proxy_async();
        }
        tc::mbar_arrive(&sm.clean);
        if (!(ok = warp_wait(&sm.f_full, par))) break;
        const float hj = sm.hi[row], gj = sm.g2[row], gc = sm.hi[kC - 1];
        const float lj = sm.lo[row] * (fabsf(hj) * kLoUnit), hb = sm.hi[32 * quarter];
        // of the products with S and dS'
        const float out_f = p.a.scale * exp_of(hj), in_f = exp_of((gc - hj) + (sm.lo[kC - 1] * (fabsf(gc) * kLoUnit) - lj));
        const float eGC = exp_of(gc);
        // of the 32 columns where quarter > q4
        const float block_f = p.a.scale * exp_of((hb - hj) + (sm.lo[32 * quarter] * (fabsf(hb) * kLoUnit) - lj));
        float kdk = 0.f;  // k . dk, its part from within the chunk
        if (!(ok = warp_wait(&sm.g1, par))) break;
        tc::tc_fence_after();
        // ---- P^T, E^T ------------------------------------------------------
        {
          const uint32_t cs = tl + kColA1 + 32 * quarter;
          unsigned char* erow = reinterpret_cast<unsigned char*>(sm.E[quarter >> 1]) + row * 128;
          float a1[2][16];  // both before the first store: E^T lands on the second one's columns
          if (quarter >= q4) {
#pragma unroll
            for (int b = 0; b < 2; ++b) tc::tmem_ld16(cs + 16 * b, a1[b]);
          }
#pragma unroll
          for (int b = 0; b < 2; ++b) {
            const int c0 = 32 * quarter + 16 * b;
            uint32_t pp[8], ee[8];
            if (quarter < q4) {
#pragma unroll
              for (int e = 0; e < 8; ++e) pp[e] = ee[e] = 0;
            } else {
              float a2[16];
              tc::tmem_ld16(tl + kColA2 + c0, a2);
              tc::tmem_wait_ld();
              const float4* src = reinterpret_cast<const float4*>((quarter > q4 ? sm.r : sm.g2) + c0);
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                const float4 x = src[e];
                float f[4] = {x.x, x.y, x.z, x.w};
                if (quarter > q4) {
#pragma unroll
                  for (int u = 0; u < 4; ++u) f[u] *= block_f;
                } else {
#pragma unroll
                  for (int u = 0; u < 4; ++u) {  // (selects: what lies in the past may not be finite)
                    const int i = 4 * e + u;
                    const bool keep = 16 * b + i >= lane;
                    f[u] = p.a.scale * exp2_approx(f[u] - gj);
                    a1[b][i] = keep ? a1[b][i] : 0.f;
                    a2[i] = keep ? a2[i] : 0.f;
                    f[u] = keep ? f[u] : 0.f;
                  }
                }
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                  const int i = 4 * e + 2 * u;
                  const uint64_t f2 = tc::pack2(f[2 * u], f[2 * u + 1]);
                  float y, z;
                  tc::unpack2(tc::mul2(tc::pack2(a2[i], a2[i + 1]), f2), y, z);
                  ee[i / 2] = pack_bf16(y, z);
                  if constexpr (kDg) {
                    kdk = fmaf(__uint_as_float(ee[i / 2] << 16), a1[b][i], kdk);
                    kdk = fmaf(__uint_as_float(ee[i / 2] & 0xffff0000u), a1[b][i + 1], kdk);
                  }
                  tc::unpack2(tc::mul2(tc::pack2(a1[b][i], a1[b][i + 1]), f2), y, z);
                  pp[i / 2] = pack_bf16(y, z);
                }
              }
            }
            tc::tmem_st8(cs + 8 * b, pp);
            tc::tmem_st8(cs + 16 + 8 * b, ee);
#pragma unroll
            for (int e = 0; e < 2; ++e)
              *reinterpret_cast<uint4*>(erow + (((4 * (quarter & 1) + 2 * b + e) ^ (row & 7)) << 4)) =
                  make_uint4(ee[4 * e], ee[4 * e + 1], ee[4 * e + 2], ee[4 * e + 3]);
          }
          tc::tmem_wait_st();
          tc::fence_proxy_async();
          tc::tc_fence_before();
          tc::mbar_arrive(&sm.pe);
          __syncwarp();
          if (lane == 0) tc::mbar_arrive(&sm.f_empty);
        }
        // ---- the products with the states: row factors ----------------------
        if (!(ok = warp_wait(&sm.g2_, par))) break;
        tc::tc_fence_after();
        float kin = 0.f, sdot = 0.f;
        const unsigned char* krow = tile(kTK) + (K == 128 ? (quarter >> 1) * kTile : 0) + row * 128;
        const unsigned char* qrow = tile(kTQ) + (K == 128 ? (quarter >> 1) * kTile : 0) + row * 128;
        constexpr int kTurns = K / 64;  // of 16 columns, per quarter
        const int p0 = K == 128 ? 4 * (quarter & 1) : 2 * quarter;  // first 16-byte piece of these columns in the row
        const uint64_t of2 = tc::pack2(out_f, out_f), if2 = tc::pack2(in_f, in_f);
#pragma unroll 1
        for (int b = 0; b < kTurns; ++b) {
          float x[16], y[16];
          const uint32_t cq = tl + kColDq + quarter * (K / 4) + 16 * b, ck = tl + kColDk + quarter * (K / 4) + 16 * b;
          tc::tmem_ld16(cq, x);
          tc::tmem_ld16(ck, y);
          tc::tmem_wait_ld();
#pragma unroll
          for (int e = 0; e < 16; e += 2) {
            tc::unpack2(tc::mul2(tc::pack2(x[e], x[e + 1]), of2), x[e], x[e + 1]);
            tc::unpack2(tc::mul2(tc::pack2(y[e], y[e + 1]), if2), y[e], y[e + 1]);
          }
          tc::tmem_st16f(cq, x);
          tc::tmem_st16f(ck, y);
          if constexpr (kDg) kin += dot16(krow, p0 + 2 * b, row, y);
        }
        tc::tmem_wait_st();
        tc::tc_fence_before();
        tc::mbar_arrive(&sm.rmw1);
        if constexpr (kDg) {  // <S, dS'>: this thread's share of the tiles
          const uint4* s4 = reinterpret_cast<const uint4*>(tile(kTS));
          const uint4* d4 = reinterpret_cast<const uint4*>(tile(kTD));
#pragma unroll 2
          for (int e = tid - 128; e < K * V / 8; e += 512) sdot += dot8(s4[e], d4[e]);
          sdot *= eGC;
        }
        release(kTS);
        release(kTD);
        release(kTV);
        release(kTO);
        release(kTK);
        if (!(ok = warp_wait(&sm.g3, par))) break;
        tc::tc_fence_after();
#pragma unroll 1
        for (int b = 0; b < V / 64; ++b) {
          float x[16];
          const uint32_t cv = tl + kColA2 + quarter * (V / 4) + 16 * b;
          tc::tmem_ld16(cv, x);
          tc::tmem_wait_ld();
#pragma unroll
          for (int e = 0; e < 16; e += 2) tc::unpack2(tc::mul2(tc::pack2(x[e], x[e + 1]), if2), x[e], x[e + 1]);
          tc::tmem_st16f(cv, x);
        }
        tc::tmem_wait_st();
        tc::tc_fence_before();
        tc::mbar_arrive(&sm.rmw2);
        // ---- results ---------------------------------------------------------
        if (!(ok = warp_wait(&sm.g4a, par))) break;
        tc::tc_fence_after();
        float xy = -(kdk + kin);
#pragma unroll 1
        for (int z = 0; z < 2; ++z) {  // dq, dk
          __nv_bfloat16* out = static_cast<__nv_bfloat16*>(z ? p.gr.dk : p.gr.dq) + (tok * H + w.h) * K + quarter * (K / 4);
          float* sum = acc + (int64_t)z * kC * K;
#pragma unroll 1
          for (int b = 0; b < kTurns; ++b) {
            float x[16];
            tc::tmem_ld16(tl + (z ? kColDk : kColDq) + quarter * (K / 4) + 16 * b, x);
            tc::tmem_wait_ld();
            if constexpr (kDg) {
              if (z == 0) xy += dot16(qrow, p0 + 2 * b, row, x);
            }
            if (group > 1) {  // this CTA's running sums over the value heads of the group
              if (j > 0) {
#pragma unroll
                for (int e = 0; e < 16; e += 4) {
                  const float4 y = *reinterpret_cast<const float4*>(sum + 16 * b + e);
                  x[e] += y.x; x[e + 1] += y.y; x[e + 2] += y.z; x[e + 3] += y.w;
                }
              }
              if (j + 1 < group) {
#pragma unroll
                for (int e = 0; e < 16; e += 4)
                  *reinterpret_cast<float4*>(sum + 16 * b + e) = make_float4(x[e], x[e + 1], x[e + 2], x[e + 3]);
              }
            }
            if (inside && j + 1 == group) st_32bytes(out + 16 * b, pack8(x), pack8(x + 8));
          }
          __syncwarp();
          if (lane + z == 0) tc::mbar_arrive(&sm.empty[slot_of(kTQ)]);
        }
        tc::tc_fence_before();
        tc::mbar_arrive(&sm.qk_free);
        if constexpr (kDg) {
          if (n > 0 && !(ok = warp_wait(&sm.xy_free, (n - 1) & 1))) break;
          atomicAdd(&sm.xy[quarter >> 1][row], xy);
#pragma unroll
          for (int o = 16; o > 0; o >>= 1) {
            kin += __shfl_xor_sync(0xffffffffu, kin, o);
            sdot += __shfl_xor_sync(0xffffffffu, sdot, o);
          }
          if (lane == 0) {
            sm.part[warp - 4] = kin;
            sm.part[warp + 12] = sdot;
          }
          tc::mbar_arrive(&sm.xy_full);
        }
        if (!(ok = warp_wait(&sm.g4b, par))) break;
        tc::tc_fence_after();
        __nv_bfloat16* out = static_cast<__nv_bfloat16*>(p.gr.dv) + (tok * HV + hv) * V + quarter * (V / 4);
#pragma unroll 1
        for (int b = 0; b < V / 64; ++b) {
          float x[16];
          tc::tmem_ld16(tl + kColA2 + quarter * (V / 4) + 16 * b, x);
          tc::tmem_wait_ld();
          if (inside) st_32bytes(out + 16 * b, pack8(x), pack8(x + 8));
        }
        tc::tc_fence_before();
        tc::mbar_arrive(&sm.dv_free);
      }
    }
  }
  if (!ok) atomicOr(&g_la_fault, 1u);
  tc::tc_fence_before();
  __syncthreads();
  tc::tc_fence_after();
  if (warp == 1) tc::tmem_dealloc(tb, 512);
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

// The driver call above needs the device's context to be current.  A thread
// whose first CUDA work is this call (autograd's, say) has none bound yet.
int bind_context() {
  int dev = 0;
  GDN2_CUDA_TRY(cudaGetDevice(&dev));
  GDN2_CUDA_TRY(cudaSetDevice(dev));
  return 0;
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
  CUtensorMap x, q, y, s;
};

template <int K, bool kOut, bool kStore, bool kBack>
int run_scan(const ScanArgs& p, const ScanMaps& m, cudaStream_t s) {
  constexpr auto kern = la_scan_kernel<K, kOut, kStore, kBack>;
  constexpr size_t bytes = sizeof(ScanSmem<K, kOut>);
  static_assert(bytes <= 227 * 1024, "shared memory of the scan");
  if (int st = smem_opt_in<kern>(bytes)) return st;
  ProfScope ps(kOut ? kKLinAttnScan : kKLinAttnStates, s);
  kern<<<(unsigned)std::min<int64_t>(p.tasks, kLaSms), kOut ? 640 : 256, bytes, s>>>(p, m.x, m.q, m.y, m.s);
  GDN2_LAUNCH_CHECK();
  return 0;
}

// one direction of the scan: the segments' own states and their sum first where the sequences are cut
template <int K, bool kBack>
int scan(ScanArgs& p, const ScanMaps& m, bool store, cudaStream_t s) {
  if (p.seg.multi) {
    p.pre = 1;
    if (int st = run_scan<K, false, false, kBack>(p, m, s)) return st;
    const int64_t KV = p.a.K * p.a.V;
    const int64_t states = p.a.N * p.a.HV, parts = std::min((KV + 511) / 512, std::max<int64_t>(1, 16 * kLaSms / states));
    la_segment_kernel<kBack><<<dim3((unsigned)states, (unsigned)parts), 128, 0, s>>>(p.seg, p.geo, p.a.HV, KV);
    GDN2_LAUNCH_CHECK();
    p.pre = 0;
  }
  if constexpr (kBack) return run_scan<K, false, true, true>(p, m, s);
  else return store ? run_scan<K, true, true, false>(p, m, s) : run_scan<K, true, false, false>(p, m, s);
}

}  // namespace

int la_tc_fwd_launch(const gdn2_linear_attn_args& a, const LaWs& ws, cudaStream_t s) {
  ScanArgs p{a, la_decay(a), la_geom(a, ws), la_segs(a, ws.seg), 0, (int)(a.HV / a.H), 0, (a.flags & GDN2_HAS_H0) ? a.h0 : nullptr,
             (a.flags & GDN2_STORE_FINAL) ? a.ht : nullptr};
  p.tasks = p.seg.entries * a.HV * (a.V / 64);
  if (p.tasks >= (int64_t(1) << 31)) return GDN2_ERR_SHAPE;
  const bool save = a.flags & GDN2_SAVE_FOR_BWD;
  if (int st = bind_context()) return st;
  ScanMaps m;
  if (!token_map(&m.x, a.k, a.K, a.H, a.T, a.B, a.k_stride) || !token_map(&m.q, a.q, a.K, a.H, a.T, a.B, a.q_stride) ||
      !token_map(&m.y, a.v, a.V, a.HV, a.T, a.B, a.v_stride))
    return GDN2_ERR_TENSOR_MAP;
  m.s = m.y;
  if (save && !state_map(&m.s, ws.states16, a.V, la_num_chunks(a) * a.HV * a.K, a.K)) return GDN2_ERR_TENSOR_MAP;
  return a.K == 128 ? scan<128, false>(p, m, save, s) : scan<64, false>(p, m, save, s);
}

namespace {

template <int K, int V, bool kDg>
int run_bwd(const BwdArgs& p, const CUtensorMap (&m)[6], cudaStream_t s) {
  constexpr auto kern = la_bwd_tc_kernel<K, V, kDg>;
  static_assert(sizeof(BwdSmem) <= 227 * 1024, "shared memory of the backward");
  if (int st = smem_opt_in<kern>(sizeof(BwdSmem))) return st;
  ProfScope ps(kKLinAttnBwd, s);
  kern<<<(unsigned)std::min<int64_t>(p.items, kLaSms), 640, sizeof(BwdSmem), s>>>(p, m[0], m[1], m[2], m[3], m[4], m[5]);
  GDN2_LAUNCH_CHECK();
  return 0;
}

template <int K, int V>
int bwd(const BwdArgs& p, const CUtensorMap (&m)[6], cudaStream_t s) {
  return p.gr.dg ? run_bwd<K, V, true>(p, m, s) : run_bwd<K, V, false>(p, m, s);
}

}  // namespace

int la_tc_bwd_launch(const gdn2_linear_attn_args& a, const gdn2_linear_attn_grads& gr, const LaWs& ws,
                     const LaBwdWs& bw, cudaStream_t s) {
  ScanArgs sc{a, la_decay(a), la_geom(a, ws), la_segs(a, bw.seg), 0, (int)(a.HV / a.H), 0, gr.dht, gr.dh0};
  sc.seg.order = ws.seg.order;  // the forward's
  if (sc.seg.cut) {
    sc.seg.map = ws.seg.map;
    sc.seg.first = ws.seg.first;
  }
  sc.tasks = sc.seg.entries * a.HV * (a.V / 64);
  BwdArgs p{a, gr, la_decay(a), la_geom(a, ws), la_num_chunks(a) * a.H, bw.acc, a.decay == GDN2_DECAY_HEAD ? bw.dg : nullptr};
  if (sc.tasks >= (int64_t(1) << 31) || p.items >= (int64_t(1) << 31)) return GDN2_ERR_SHAPE;
  const int64_t ostep[3] = {a.T * a.HV * a.V, a.HV * a.V, a.V}, rows = la_num_chunks(a) * a.HV * a.K;
  if (int st = bind_context()) return st;
  CUtensorMap m[6];  // q, k, v, do, S, dS'
  if (!token_map(&m[0], a.q, a.K, a.H, a.T, a.B, a.q_stride) || !token_map(&m[1], a.k, a.K, a.H, a.T, a.B, a.k_stride) ||
      !token_map(&m[2], a.v, a.V, a.HV, a.T, a.B, a.v_stride) ||
      !token_map(&m[3], gr.dout, a.V, a.HV, a.T, a.B, ostep) || !state_map(&m[4], ws.states16, a.V, rows, a.K) ||
      !state_map(&m[5], bw.dstates16, a.V, rows, a.K))
    return GDN2_ERR_TENSOR_MAP;
  const ScanMaps sm{m[0], m[0], m[3], m[5]};
  if (int st = a.K == 128 ? scan<128, true>(sc, sm, true, s) : scan<64, true>(sc, sm, true, s)) return st;
  if (a.K == 128) return a.V == 128 ? bwd<128, 128>(p, m, s) : bwd<128, 64>(p, m, s);
  return a.V == 128 ? bwd<64, 128>(p, m, s) : bwd<64, 64>(p, m, s);
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
