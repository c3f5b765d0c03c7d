// lora_sm100.cu -- the down projection of the per-row low-rank adapters:
//   h[i,r] = scaling[a_i] * sum_k x[i,k] A[a_i][r,k]     (x unquantized; sums in fp32)
// for the rows i whose adapter a_i is in [0, L). The up projection is part of the linear's
// GEMM (rowsel_sm100.cu), which adds h . B^T before its one rounding.
//
// tcgen05 (kind::f16) on tiles of 128 rows. All of a tile's adapters stand side by side on the
// MMA's N side (rank_pad columns each; a pass takes up to 256 columns, four adapters where the
// tiles are few), and each row keeps the columns of its own; rows never mix, so an adapter's infinities and NaN stay with its rows. When the
// tiles are few, a cluster splits K.
//
// The GEMM's tensor cores take h in x's 16-bit type. h is a sum, and B may bring up what is small
// in it, so it goes with more bits than the type's, as a high and a low part,
// h / hscale = hi + lo / 2^7, at the price of twice the rank in a product that is a few per cent
// of the whole. bf16 has fp32's range (hscale = 1): 2^-16 of each value. f16: hscale, a power of
// two, puts the row's largest value in [2^14, 2^15), and with the low part 2^7 times larger the
// error is 2^-22 of a value down to 2^-23 of the row's largest, and 2^-45 of the largest below (with
// the largest at 1 and a low part of the same scale it was 2^-25 of the largest).
//
// The kernel reads x, ids and A before the dependency wait (the kernel before is the call's
// quantizer, which lets it launch only after its own wait) and writes after it.
#include <cuda.h>
#include <cudaTypedefs.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <mutex>
#include <string>

#include "internal.h"
#include "ptx.cuh"

namespace fp8lin {

__device__ unsigned int g_lora_status;  // watchdog bits (128 = a wait ran out)

namespace lora {

constexpr uint64_t kWaitLimitNs = 4000000000ull;
constexpr uint64_t kDrainLimitNs = 1000000000ull;

struct Params {
  const void *x;
  const void *a;
  const int *ids;
  const float *scaling;
  int dtype;
  int M, K, L, R, rank_pad;
  void *hl;
  float *hscale;
  int4 *plan;      // null: not wanted
  int plan_mixed;
  int split, k_blocks;
  int x_rows;      // rows of x's box
  int cols;        // columns per pass
  uint32_t off_part;
  int tiles, clusters, max_passes;
};

__device__ __forceinline__ bool has_adapter(const Params &p, int id) {
  return static_cast<uint32_t>(id) < static_cast<uint32_t>(p.L);
}

constexpr int ROWS = 128;
constexpr int KB = 64;     // 16-bit elements per K-block: one 128-byte swizzle row
constexpr int COLS = 256;  // columns (adapters x rank_pad) per pass, at most
constexpr int MAX_STAGES = 8;
constexpr int NUM_THREADS = 256;  // producer, MMA, 4 x TMEM, plan, and one more for the row sums
constexpr int MAX_SPLIT = 8;
// dynamic: the ring, cut anew for each item into stages of x_rows + columns rows of 128 bytes,
// then fp32 [ROWS][rank_pad + 4]
constexpr uint32_t SMEM_MAX = 232448 - 4096;  // (the static part is below 4 KB)

__device__ __forceinline__ void record_timeout(volatile int *abort) {
  if (!*abort) {
    atomicOr(&g_lora_status, 128u);
    *abort = 1;
  }
}

// A whole warp waits; copies and MMAs go out from one elected lane of it (operands in uniform
// registers).
__device__ __forceinline__ bool warp_wait(uint32_t bar, uint32_t parity, volatile int *abort,
                                          bool elected) {
  if (__all_sync(0xFFFFFFFFu, ptx::mbar_try_wait(bar, parity))) return true;
  const bool got = ptx::mbar_wait_bounded(bar, parity, abort, kWaitLimitNs);
  if (__all_sync(0xFFFFFFFFu, got)) return true;
  if (elected) record_timeout(abort);
  return false;
}

// The plan of the GEMM's token tiles, by one warp. A run of at least kLoraMixed (32) rows
// crosses a border between blocks of 32 rows, so of a block's runs only the one carried in and
// the one carried on can be long.
__device__ __forceinline__ void make_plan(const Params &p, int lane) {
  int n_one = 0, n_mixed = 0;
  auto emit = [&](int t0, int t1, int a) {
    const int at = a == -2 ? p.plan_mixed + n_mixed : 1 + n_one;
    ++(a == -2 ? n_mixed : n_one);
    if (lane == 0) p.plan[at] = make_int4(t0, t1, a, 0);
  };
  int open = -1, open_end = 0;  // rows of short runs not yet in a tile
  auto flush = [&]() {
    if (open >= 0 && open < open_end) emit(open, open_end, -2);
    open = -1;
  };
  auto add_short = [&](int s, int e) {
    if (s == e) return;
    if (open < 0) open = s;
    open_end = e;
    for (; open_end - open >= kLoraMixed; open += kLoraMixed) emit(open, open + kLoraMixed, -2);
    if (open == open_end) open = -1;
  };
  auto add_run = [&](int s, int e) {
    if (e - s < kLoraMixed) {
      add_short(s, e);
      return;
    }
    flush();
    const int id = __ldg(p.ids + s), a = has_adapter(p, id) ? id : -1;
    const int nt = (e - s + kLoraTileTokens - 1) / kLoraTileTokens;
    const int per = ((e - s + nt - 1) / nt + 31) / 32 * 32;
    for (int t = s; t < e; t += per) emit(t, min(e, t + per), a);
  };
  int start = 0;  // the run carried on
  // Blocks of 32 rows, AHEAD of them at a time, and as many loaded while those are looked at.
  // A row is compared with the one before it by a load of its own; most blocks have no border
  // between runs, which one vote shows for all of them. (The rows before through shuffles and a
  // vote a block: 9216 rows took 24 us, twice as long as all sums; now 11, most of it the loads.)
  constexpr int AHEAD = 32;
  int here[AHEAD], left[AHEAD];
  auto fetch = [&](int b) {
    if (b > 0 && b <= p.M - 32 * AHEAD) {
      const int *q = p.ids + b + lane;
#pragma unroll
      for (int k = 0; k < AHEAD; ++k) {
        here[k] = __ldg(q + 32 * k);
        left[k] = __ldg(q + 32 * k - 1);
      }
      return;
    }
#pragma unroll
    for (int k = 0; k < AHEAD; ++k) {
      const int m = min(b + 32 * k + lane, p.M - 1);  // (a row past the end is no border)
      here[k] = __ldg(p.ids + m);
      left[k] = __ldg(p.ids + (b + 32 * k + lane < p.M ? max(m - 1, 0) : m));
    }
  };
  fetch(0);
  for (int b0 = 0; b0 < p.M; b0 += 32 * AHEAD) {
    uint32_t mine = 0;  // bit k: a run starts at this lane's row of block k
#pragma unroll
    for (int k = 0; k < AHEAD; ++k)
      if (here[k] != left[k]) mine |= 1u << k;
    if (__any_sync(0xFFFFFFFFu, mine != 0)) {  // (different ids may both mean none)
#pragma unroll
      for (int k = 0; k < AHEAD; ++k)
        if (!has_adapter(p, here[k]) && !has_adapter(p, left[k])) mine &= ~(1u << k);
    }
    fetch(b0 + 32 * AHEAD);
    for (uint32_t todo = __reduce_or_sync(0xFFFFFFFFu, mine); todo != 0; todo &= todo - 1) {
      const int k = __ffs(static_cast<int>(todo)) - 1;
      const int b = b0 + 32 * k;
      const uint32_t edges = __ballot_sync(0xFFFFFFFFu, mine >> k & 1u);
      const int first = __ffs(static_cast<int>(edges)) - 1;
      const int last = 31 - __clz(static_cast<int>(edges));
      add_run(start, b + first);
      add_short(b + first, b + last);
      start = b + last;
    }
  }
  add_run(start, p.M);
  flush();
  if (lane == 0) p.plan[0] = make_int4(n_one, n_mixed, 0, 0);
}

// At most how many adapters the 128 rows from m0 have, by a whole warp: exact where an
// adapter's rows lie together.
__device__ __forceinline__ int adapters_at_most(const Params &p, int m0, int lane) {
  int id[ROWS / 32];
#pragma unroll
  for (int j = 0; j < ROWS / 32; ++j) {
    const int m = m0 + 32 * j + lane;
    id[j] = m < p.M ? __ldg(p.ids + m) : -1;
    if (!has_adapter(p, id[j])) id[j] = -1;
  }
  int n = 0, before = -1;  // the last row's of the 32 before
#pragma unroll
  for (int j = 0; j < ROWS / 32; ++j) {
    const uint32_t same = __match_any_sync(0xFFFFFFFFu, id[j]);
    n += __popc(__ballot_sync(0xFFFFFFFFu, id[j] >= 0 && id[j] != before &&
                                               __ffs(static_cast<int>(same)) - 1 == lane));
    before = __shfl_sync(0xFFFFFFFFu, id[j], 31);
  }
  return n;
}

// Two values each as a high part, cut off to the type (up to fp32's largest value a bf16 stays
// finite), and 2^kLoraLowShift times the rest. Both have the value's sign, and where the high part is
// not zero or not finite, nor is the low part: against an infinite B, hi * B + lo * B is what
// the value times B is, and not the NaN of 0 * inf or inf - inf. (A value too small for the
// high part counts as zero there.)
__device__ __forceinline__ void split_16x2(bool f16, float2 w, uint32_t &hi, uint32_t &lo) {
  constexpr float kLow = 1 << kLoraLowShift;
  if (f16) {
    hi = ptx::pack_f16x2_rz(w.x, w.y);
    const float2 h = __half22float2(*reinterpret_cast<const __half2 *>(&hi));
    lo = ptx::pack_f16x2((w.x - h.x) * kLow, (w.y - h.y) * kLow);
  } else {
    hi = ptx::pack_bf16x2_rz(w.x, w.y);
    lo = ptx::pack_bf16x2((w.x - __uint_as_float(hi << 16)) * kLow,
                          (w.y - __uint_as_float(hi & 0xFFFF0000u)) * kLow);
  }
  // the halves that are not zero (as bits 15 and 31), and an infinity's bits
  const uint32_t h = hi & 0x7FFF7FFFu, l = lo & 0x7FFF7FFFu;
  const uint32_t gone = (h + 0x7FFF7FFFu) & ~(l + 0x7FFF7FFFu) & 0x80008000u;
  lo |= gone >> 15 | (gone & hi);
  const uint32_t inf = f16 ? 0x7C00u : 0x7F80u;
  if ((h & 0xFFFFu) == inf) lo = (lo & 0xFFFF0000u) | (hi & 0xFFFFu);
  if (h >> 16 == inf) lo = (lo & 0xFFFFu) | (hi & 0xFFFF0000u);
}

// An item's sums, row by row: the K-splits' parts added in rank order, scaled, and split into
// the two 16-bit parts. CTA `rank` of the S of a cluster has rows rank, rank + S, ..; a warp
// has two rows at a time, a lane values 4 lane .. 4 lane + 3, one 16-byte load from each part
// (4-byte loads took three times as long), all of them before the first is used.
template <int S>
__device__ __forceinline__ void finish_rows(const Params &p, const float *part, int pitch,
                                            const int *live, const float *scaling, int m0,
                                            int rank, int warp, int lane) {
  const bool f16 = p.dtype == kF16;
  uint32_t from[S];
#pragma unroll
  for (int s = 0; s < S; ++s)
    from[s] = S == 1 ? ptx::smem_u32(part) : ptx::map_shared_rank(ptx::smem_u32(part), s);
  const int col = 4 * lane;
  for (int r0 = 2 * warp; rank + r0 * S < ROWS; r0 += 2 * (NUM_THREADS / 32)) {
    int row[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) row[h] = min(rank + (r0 + h) * S, ROWS - 1);
    const bool on[2] = {live[row[0]] != 0, live[row[1]] != 0 && rank + (r0 + 1) * S < ROWS};
    if (!on[0] && !on[1]) continue;  // uniform in the warp
    float4 t[2][S];
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int s = 0; s < S; ++s) {
        const uint32_t at =
            from[s] + static_cast<uint32_t>(row[h] * pitch + min(col, p.rank_pad - 4)) * 4u;
        t[h][s] = S == 1 ? ptx::ld_shared_f32x4(at) : ptx::ld_shared_cluster_v4(at);
      }
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      float v[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int s = 0; s < S; ++s) {
        v[0] += t[h][s].x;
        v[1] += t[h][s].y;
        v[2] += t[h][s].z;
        v[3] += t[h][s].w;
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = col < p.R ? v[i] * scaling[row[h]] : 0.0f;  // R % 8 == 0
      if (!on[h]) continue;
      // f16: the row divided by 2^ex (exact), its largest finite value in [2^14, 2^15)
      int ex = 0;
      if (f16) {
        float top = 0.0f;
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (fabsf(v[i]) <= 3.402823466e38f) top = fmaxf(top, fabsf(v[i]));
#pragma unroll
        for (int d = 16; d > 0; d >>= 1) top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, d));
        if (top > 0.0f)
          ex = max(-126, static_cast<int>(__float_as_uint(top) >> 23) - 127 - 14);
      }
      const float inv = __uint_as_float(static_cast<uint32_t>(127 - ex) << 23);
      if (col < p.rank_pad) {
        uint32_t hi2[2], lo2[2];
#pragma unroll
        for (int i = 0; i < 2; ++i)
          split_16x2(f16, make_float2(v[2 * i] * inv, v[2 * i + 1] * inv), hi2[i], lo2[i]);
        uint32_t *dst = reinterpret_cast<uint32_t *>(p.hl) +
                        static_cast<int64_t>(m0 + row[h]) * p.rank_pad + 2 * lane;
        *reinterpret_cast<uint2 *>(dst) = make_uint2(hi2[0], hi2[1]);
        *reinterpret_cast<uint2 *>(dst + p.rank_pad / 2) = make_uint2(lo2[0], lo2[1]);
      }
      if (lane == 0)
        p.hscale[m0 + row[h]] = __uint_as_float(static_cast<uint32_t>(127 + ex) << 23);
    }
  }
}

// Work comes in items (tile of 128 rows, pass over p.cols columns of its adapters). Item (t, ps)
// is cluster (t + ps) % p.clusters's: a tile of one adapter is its own cluster's only item,
// the passes of a tile of many (decoding requests) spread over the neighbours.
// Bound: with many tiles the reads of x, which the quantizer has left in L2 in part; with few
// the latency of its start, K loop and row sums one after the other (its reads of x and A
// overlap the quantizer).
__global__ void __launch_bounds__(NUM_THREADS, 1)
    down_tile_kernel(const __grid_constant__ CUtensorMap tmap_x,
                     const __grid_constant__ CUtensorMap tmap_a,
                     const __grid_constant__ Params p) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t *smem = reinterpret_cast<uint8_t *>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  const uint32_t sbase = ptx::smem_u32(smem);
  __shared__ alignas(8) uint64_t s_bar[2 * MAX_STAGES + 2];
  __shared__ uint32_t s_slot;
  __shared__ int s_abort;
  __shared__ alignas(16) int s_id[ROWS];  // adapter of each row, -1: none
  __shared__ int s_first[ROWS];  // the row's adapter appears first at this row of the tile
  __shared__ int s_rank[ROWS];   // .. and is this one of the tile's adapters
  __shared__ int s_list[ROWS];   // the tile's adapters
  __shared__ int s_live[ROWS];   // the row's sums are this item's
  __shared__ float s_scaling[ROWS];
  __shared__ int s_count[ROWS / 32];
  __shared__ int s_todo[ROWS];   // pass ps of tile (cluster - ps) may have work
  const uint32_t bar_full = ptx::smem_u32(s_bar);
  const uint32_t bar_empty = bar_full + 8 * MAX_STAGES;
  const uint32_t bar_acc = bar_empty + 8 * MAX_STAGES;
  const uint32_t bar_drain = bar_acc + 8;
  volatile int *abort = &s_abort;
  float *part = reinterpret_cast<float *>(smem + p.off_part);
  const uint32_t x_stage = static_cast<uint32_t>(p.x_rows) * 128;
  // 16 bytes past a multiple of 64: eight rows' 16-byte pieces hit all banks
  const int pitch = p.rank_pad + 4;
  const int per_pass = p.cols / p.rank_pad;

  ptx::grid_launch_dependents();
  const int warp = ptx::uniform(threadIdx.x >> 5), lane = threadIdx.x & 31;
  const int rank = static_cast<int>(ptx::cluster_ctarank());
  const int cluster = static_cast<int>(blockIdx.x) / p.split;
  // the tile whose pass ps is this cluster's (tiles or above: none)
  auto tile_of = [&](int ps) {
    const int t = cluster - ps % p.clusters;
    return t < 0 ? t + p.clusters : t;
  };

  if (threadIdx.x == 0) {
    ptx::prefetch_tmap(&tmap_x);
    ptx::prefetch_tmap(&tmap_a);
    for (int s = 0; s < MAX_STAGES; ++s) {
      ptx::mbar_init(bar_full + 8 * s, 1);
      ptx::mbar_init(bar_empty + 8 * s, 1);
    }
    ptx::mbar_init(bar_acc, 1);
    ptx::mbar_init(bar_drain, 1);
    s_abort = 0;
    ptx::fence_mbar_init();
  }
  if (warp == 1) {
    ptx::tmem_alloc<1>(ptx::smem_u32(&s_slot), COLS);
    ptx::tmem_relinquish<1>();
  }
  for (int ps = warp; ps < p.max_passes; ps += NUM_THREADS / 32) {
    const int t = tile_of(ps);
    const int n = t < p.tiles ? adapters_at_most(p, t * ROWS, lane) : 0;
    if (lane == 0) s_todo[ps] = n > ps * per_pass;
  }
  ptx::tc_fence_before();
  __syncthreads();
  ptx::tc_fence_after();
  const uint32_t tmem = static_cast<uint32_t>(
      ptx::uniform(static_cast<int>(*const_cast<volatile uint32_t *>(&s_slot))));

  const int kb0 = rank * p.k_blocks / p.split;  // (split <= k_blocks)
  const int nkb = (rank + 1) * p.k_blocks / p.split - kb0;
  bool plan_open = p.plan != nullptr && blockIdx.x == 0;  // this CTA's last warp has it to make
  const bool elected = ptx::elect_one();
  uint32_t phases = 0;  // bit s: of stage s, in the producer and the MMA warp
  uint32_t used = 0;       // .. that have been used
  uint32_t items = 0;
  bool ok = true;

  for (int ps = 0; ps < p.max_passes; ++ps) {
    if (s_todo[ps] == 0) continue;
    const int m0 = tile_of(ps) * ROWS;
    // The tile's adapters, in the order of their first rows.
    const int me = threadIdx.x;
    if (me < ROWS) {
      const int id = m0 + me < p.M ? __ldg(p.ids + m0 + me) : -1;
      s_id[me] = has_adapter(p, id) ? id : -1;
      s_scaling[me] = has_adapter(p, id) ? __ldg(p.scaling + id) : 0.0f;
    }
    __syncthreads();
    bool first = false;
    if (me < ROWS) {
      // the lowest row with the same id: within the warp, then among the rows of those before
      const int id = s_id[me];
      int f = (me & ~31) + __ffs(static_cast<int>(__match_any_sync(0xFFFFFFFFu, id))) - 1;
      if (id >= 0) {
#pragma unroll 1
        for (int j = 0; j < (me & ~31); j += 4) {
          const int4 v = *reinterpret_cast<const int4 *>(s_id + j);
          if (v.x == id || v.y == id || v.z == id || v.w == id) {
            f = v.x == id ? j : v.y == id ? j + 1 : v.z == id ? j + 2 : j + 3;
            break;
          }
        }
      }
      first = id >= 0 && f == me;
      s_first[me] = f;
      const uint32_t votes = __ballot_sync(0xFFFFFFFFu, first);
      s_rank[me] = __popc(votes & ((1u << lane) - 1u));
      if (lane == 0) s_count[warp] = __popc(votes);
    }
    __syncthreads();
    int before = 0, distinct = 0;
#pragma unroll
    for (int w = 0; w < ROWS / 32; ++w) {
      if (w < warp) before += s_count[w];
      distinct += s_count[w];
    }
    if (me < ROWS) {
      s_rank[me] += before;
      if (first) s_list[s_rank[me]] = s_id[me];
    }
    __syncthreads();
    const int d0 = ps * per_pass, nd = ptx::uniform(min(per_pass, distinct - d0));
    if (nd <= 0) continue;  // (in the whole cluster)
    if (me < ROWS) {  // (read after the barriers below)
      const int r = s_rank[s_first[me]];
      s_live[me] = s_id[me] >= 0 && r >= d0 && r < d0 + nd;
    }
    // (every item leaves the ring empty)
    const uint32_t tx = x_stage + static_cast<uint32_t>(nd * p.rank_pad) * 128u;
    const int stages = ptx::uniform(static_cast<int>(min(p.off_part / tx, static_cast<uint32_t>(MAX_STAGES))));
    int stage = 0;

    if (warp == 0) {
      for (int i = 0; i < nkb && ok; ++i) {
        if (!(ok = warp_wait(bar_empty + 8 * stage, (phases >> stage & 1u) ^ 1u, abort, elected)))
          break;
        const uint32_t fb = bar_full + 8 * stage;
        const uint32_t dst = sbase + static_cast<uint32_t>(stage) * tx;
        if (elected) {
          ptx::mbar_arrive_expect_tx(fb, tx);
          ptx::tma_load_2d(dst, &tmap_x, (kb0 + i) * KB, m0, fb);
        }
        for (int d = 0; d < nd; ++d) {  // ranks past R read as zero
          const int a = ptx::uniform(s_list[d0 + d]);
          if (elected)
            ptx::tma_load_3d(dst + x_stage + static_cast<uint32_t>(d * p.rank_pad) * 128u, &tmap_a,
                             (kb0 + i) * KB, 0, a, fb);
        }
        phases ^= 1u << stage;
        used |= 1u << stage;
        if (++stage == stages) stage = 0;
      }
    } else if (warp == 1) {
      const uint32_t idesc = ptx::idesc_f16_f32(ROWS, nd * p.rank_pad, p.dtype == kBF16);
      ptx::tc_fence_after();
      for (int i = 0; i < nkb && ok; ++i) {
        if (!(ok = warp_wait(bar_full + 8 * stage, phases >> stage & 1u, abort, elected))) break;
        ptx::tc_fence_after();
        const uint32_t st = sbase + static_cast<uint32_t>(stage) * tx;
        const uint64_t adesc = ptx::sw128_kmajor_desc(st);
        const uint64_t bdesc = ptx::sw128_kmajor_desc(st + x_stage);
        if (elected) {
#pragma unroll
          for (int kk = 0; kk < KB / 16; ++kk)
            ptx::mma_f16<1>(tmem, adesc + 2 * kk, bdesc + 2 * kk, idesc, (i | kk) != 0 ? 1u : 0u);
          ptx::mma_commit(bar_empty + 8 * stage);
        }
        phases ^= 1u << stage;
        if (++stage == stages) stage = 0;
      }
      if (ok && elected) ptx::mma_commit(bar_acc);
    } else if (warp < 6) {
      // TMEM lane = row: keep the columns of the row's own adapter
      const int quarter = warp & 3;
      const int row = quarter * 32 + lane;
      const int mine = s_id[row] >= 0 ? s_rank[s_first[row]] : -1;
      if (ok && !ptx::mbar_wait_bounded(bar_acc, items & 1u, abort, kWaitLimitNs)) {
        record_timeout(abort);
        ok = false;
      }
      ok = __all_sync(0xFFFFFFFFu, ok);
      ptx::tc_fence_after();
      for (int d = 0; d < nd && ok; ++d) {
        const bool keep = mine == d0 + d;
        if (!__any_sync(0xFFFFFFFFu, keep)) continue;
        for (int c = 0; c < p.rank_pad; c += 16) {
          uint32_t r[16];
          ptx::tmem_ld_32x32b_x16(tmem + (static_cast<uint32_t>(quarter * 32) << 16) +
                                      static_cast<uint32_t>(d * p.rank_pad + c),
                                  r);
          ptx::tmem_wait_ld();
          if (keep) {
#pragma unroll
            for (int j = 0; j < 16; j += 4)
              *reinterpret_cast<float4 *>(part + row * pitch + c + j) =
                  make_float4(__uint_as_float(r[j]), __uint_as_float(r[j + 1]),
                              __uint_as_float(r[j + 2]), __uint_as_float(r[j + 3]));
          }
          __syncwarp();  // (the next load is the whole warp's)
        }
      }
      ptx::tc_fence_before();
    } else if (warp == 6 && plan_open) {
      ptx::grid_dependency_wait();
      make_plan(p, lane);
      plan_open = false;
    }
    ++items;

    __syncwarp();
    __syncthreads();
    ptx::cluster_sync();  // every CTA's partial sums are in its shared memory
    ptx::grid_dependency_wait();

    if (*abort == 0) {
      switch (p.split) {
        case 1: finish_rows<1>(p, part, pitch, s_live, s_scaling, m0, rank, warp, lane); break;
        case 2: finish_rows<2>(p, part, pitch, s_live, s_scaling, m0, rank, warp, lane); break;
        case 4: finish_rows<4>(p, part, pitch, s_live, s_scaling, m0, rank, warp, lane); break;
        default: finish_rows<8>(p, part, pitch, s_live, s_scaling, m0, rank, warp, lane);
      }
    }

    // (peers may still be reading this CTA's partial sums, its own warps the lists)
    __syncwarp();
    ptx::cluster_sync();
  }

  ptx::grid_dependency_wait();  // the GEMM's wait for this kernel covers the quantizer too
  if (warp == 6 && plan_open) make_plan(p, lane);
  if (warp == 0) {
    // (after a wait that ran out: no copy may be under way when the CTA ends)
    for (int s = 0; s < MAX_STAGES; ++s)
      if (*abort && (used >> s & 1u))
        ptx::mbar_wait_timeout(bar_empty + 8 * s, (phases >> s & 1u) ^ 1u, kDrainLimitNs);
  } else if (warp == 1 && elected) {
    ptx::mma_commit(bar_drain);
    ptx::mbar_wait_timeout(bar_drain, 0, kDrainLimitNs);
  }
  __syncwarp();
  ptx::tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    ptx::tc_fence_after();
    ptx::tmem_dealloc<1>(tmem, COLS);
  }
}

size_t align256(size_t v) { return (v + 255) / 256 * 256; }

}  // namespace lora

LoraWorkspace lora_workspace(void *base, int64_t M, int64_t R) {
  LoraWorkspace w;
  uint8_t *b = static_cast<uint8_t *>(base);
  const size_t hl = lora::align256(static_cast<size_t>(M) * 2 * lora_rank_pad(R) * 2);
  const size_t sc = lora::align256(static_cast<size_t>(M) * 4);
  w.hl = b;
  w.hscale = reinterpret_cast<float *>(b + hl);
  w.plan = M <= kLoraRowsMaxM ? nullptr : reinterpret_cast<int4 *>(b + hl + sc);
  w.bytes = hl + sc + lora::align256(static_cast<size_t>(lora_plan_max(M)) * sizeof(int4));
  return w;
}

namespace lora {

// Clusters of 1, 2, 4 and 8 CTAs that the GPU holds at once.
struct DownInfo {
  bool ready = false;
  cudaError_t err = cudaSuccess;
  int clusters[MAX_SPLIT + 1] = {};
};

const DownInfo &down_info(const DeviceInfo &dev) {
  static DownInfo info[64];
  static std::mutex mu;
  std::lock_guard<std::mutex> lock(mu);
  DownInfo &di = info[dev.device & 63];
  if (!di.ready) {
    di.ready = true;
    di.err = cudaFuncSetAttribute(down_tile_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                  static_cast<int>(SMEM_MAX));
    di.clusters[1] = dev.sm_count;
    for (int s = 2; s <= MAX_SPLIT && di.err == cudaSuccess; s *= 2) {
      cudaLaunchConfig_t cfg = {};
      cfg.gridDim = dim3(static_cast<unsigned>(dev.sm_count / s * s));
      cfg.blockDim = dim3(NUM_THREADS);
      cfg.dynamicSmemBytes = SMEM_MAX;
      cudaLaunchAttribute attr[1];
      attr[0].id = cudaLaunchAttributeClusterDimension;
      attr[0].val.clusterDim.x = static_cast<unsigned>(s);
      attr[0].val.clusterDim.y = 1;
      attr[0].val.clusterDim.z = 1;
      cfg.attrs = attr;
      cfg.numAttrs = 1;
      di.err = cudaOccupancyMaxActiveClusters(&di.clusters[s], down_tile_kernel, &cfg);
    }
  }
  return di;
}

}  // namespace lora

int launch_lora_down(const LoraArgs &a, cudaStream_t stream) {
  using namespace lora;
  DeviceInfo dev;
  if (!current_device_info(&dev)) return 5;
  const LoraWorkspace w = lora_workspace(a.workspace, a.M, a.R);
  Params p = {};
  p.x = a.x;
  p.a = a.lora_a;
  p.ids = a.ids;
  p.scaling = a.scaling;
  p.dtype = a.dtype;
  p.M = static_cast<int>(a.M);
  p.K = static_cast<int>(a.K);
  p.L = static_cast<int>(a.L);
  p.R = static_cast<int>(a.R);
  p.rank_pad = static_cast<int>(lora_rank_pad(a.R));
  p.hl = w.hl;
  p.hscale = w.hscale;
  p.plan = w.plan;
  p.plan_mixed = static_cast<int>(lora_plan_mixed(a.M));
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[2];
  cudaError_t e;
  p.k_blocks = static_cast<int>((a.K + KB - 1) / KB);
  const int64_t tiles = (a.M + ROWS - 1) / ROWS;
  const DownInfo &di = down_info(dev);
  if (di.err != cudaSuccess) {
    set_error(std::string("fp8_linear_lora: kernel setup: ") + cudaGetErrorString(di.err));
    return 4;
  }
  // K-splits (1, 2, 4 or 8) while there is room for all tiles' clusters, four K-blocks at
  // least for each (64 tokens of 27 adapters, K 4096, the whole call: 29 us, without a split
  // 63; 2000 tokens 79 and 121; 9216 rows, where there is no room for one, the same)
  int split = 1;
  for (int s = 2; s <= MAX_SPLIT && 4 * s <= p.k_blocks + 3; s *= 2)
    if (di.clusters[s] >= tiles) split = s;
  p.split = split;
  // a cluster per tile, and further ones for the passes of tiles with many adapters while CTAs
  // are left over still
  // Few tiles: four adapters a pass, so that more clusters share them (K 4096: 1000 tokens of
  // prompts and decodes, rank 64, 55 us, with three 60, with two 67; 64 tokens, rank 16, 24.4, with
  // eight 26.1; 4096 rows of 8 requests, rank 64, 78, with two 83; only where idle clusters happen to
  // take all further passes, 2000 tokens at rank 64, 82 and with two 78). Many tiles: all columns, so
  // that a tile at the border of two requests takes one pass (16384 rows, rank 128: 347 us, with one
  // adapter a pass 373).
  p.cols = split >= 4 ? std::min(COLS, 4 * p.rank_pad) : COLS;
  const int per_pass = p.cols / p.rank_pad;
  p.tiles = static_cast<int>(tiles);
  p.max_passes = static_cast<int>((std::min<int64_t>(a.L, ROWS) + per_pass - 1) / per_pass);
  p.clusters = static_cast<int>(std::max<int64_t>(
      tiles, std::min<int64_t>(di.clusters[split], tiles * p.max_passes)));
  p.x_rows = static_cast<int>(std::min<int64_t>((a.M + 7) / 8 * 8, ROWS));
  const uint32_t part = ROWS * (static_cast<uint32_t>(p.rank_pad) + 4) * 4;
  p.off_part = (SMEM_MAX - 1024 - part) / 1024 * 1024;
  const CUtensorMapDataType t16 = a.dtype == kF16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16
                                                  : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
  std::string err;
  CUtensorMap tx, ta;
  if (!make_tmap_2d_sw128(&tx, t16, a.x, a.K, a.M, a.K * 2, KB, static_cast<uint32_t>(p.x_rows),
                          &err) ||
      !make_tmap_3d_swizzled(&ta, t16, a.lora_a, a.K, a.R, a.L, a.K * 2, a.R * a.K * 2, KB,
                             static_cast<uint32_t>(p.rank_pad), 128, &err)) {
    set_error("fp8_linear_lora: " + err);
    return 4;
  }
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = static_cast<unsigned>(p.split);
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.stream = stream;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  cfg.gridDim = dim3(static_cast<unsigned>(p.clusters * p.split));
  cfg.blockDim = dim3(NUM_THREADS);
  cfg.dynamicSmemBytes = p.off_part + part + 1024;
  e = cudaLaunchKernelEx(&cfg, down_tile_kernel, tx, ta, p);
  if (e != cudaSuccess) {
    set_error(std::string("fp8_linear_lora: launch failed: ") + cudaGetErrorString(e));
    return 4;
  }
  return 0;
}

cudaError_t read_lora_status(unsigned int *bits, bool clear) {
  cudaError_t e = cudaMemcpyFromSymbol(bits, g_lora_status, sizeof(unsigned int));
  if (e != cudaSuccess) return e;
  if (clear) {
    const unsigned int zero = 0;
    e = cudaMemcpyToSymbol(g_lora_status, &zero, sizeof(unsigned int));
  }
  return e;
}

}  // namespace fp8lin
