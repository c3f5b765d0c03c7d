// rowsel_sm100.cu -- e4m3 linears whose weights depend on the row: rows grouped by expert,
// and one shared projection with a low-rank adapter per row.
//
//   grouped:  out[i,n] = fma(acc[i,n] * xs[i], ws[e,n], bias[e,n]),  e the expert of row i
//   adapters: out[i,n] = fma(acc[i,n] * xs[i], ws[n], bias[n]) + sum_r h[i,r] B[a_i][n,r]
//   acc[i,n] = sum_k e4m3(xq[i,k]) * e4m3(wq[.,n,k])      (fp32, tensor cores)
//
// Both kernels here put the weights on the MMA's M side (D^T = W . X^T): 128 weight rows per
// CTA fill the tensor core's 128 rows whatever the group's size, and a group of few tokens
// only narrows N (a multiple of 16, 32 for a CTA pair), which the instruction descriptor
// gives per tile. A tile is (expert, block of weight rows, block of tokens); token blocks
// never cross an expert's border, and the tokens of a group are split evenly. The table of
// tiles is made by every CTA from the offsets, which are device data.
//
//   persist_kernel<CG, LORA>  persistent CTAs (CG = 2: pairs, 256 weight rows x up to 256
//       tokens; CG = 1: 128 x up to 128, for groups of few rows), TMA ring, two TMEM
//       accumulators, epilogue of one tile under the main loop of the next.
//   split_kernel<LORA, OWN>  when all tiles together do not fill the GPU: a cluster of CTAs per
//       tile splits K; each CTA adds up a share of the tile's rows, of which the others push
//       their partial sums into its shared memory, in rank order (the result does not depend
//       on timing).
//
// Rows outside the experts' ranges are written as zeros. Offsets are clamped to [0, M] and to
// their running maximum, so that no value of them leads outside a tensor.
// Every mbarrier wait is bounded; a wait that runs out sets bit 64 of the device status.
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

__device__ unsigned int g_rowsel_status;  // watchdog bits (64 = a wait ran out)

namespace rowsel {

constexpr int WROWS = 128;  // weight rows per CTA = MMA M (per CTA)
constexpr int BK = 128;     // bytes (= e4m3 elements) per K-block: one 128-byte swizzle row
constexpr int UMMA_K = 32;  // bytes of K per MMA
constexpr int NUM_THREADS = 192;
constexpr int EPI_WARPS = 4;
constexpr uint32_t W_STAGE = WROWS * BK;  // 16 KB
constexpr int X_MAPS = 8;                 // token boxes of 16, 32, .. 128 rows
constexpr int H_MAPS = kLoraTileTokens / 32;  // boxes of the adapters' h: 16, 32, .. 80 rows
constexpr uint64_t kWaitLimitNs = 4000000000ull;
constexpr uint64_t kDrainLimitNs = 1000000000ull;

struct Maps {
  CUtensorMap x[X_MAPS];  // xq [M][K], box 128 B x 16 (i + 1) rows
  CUtensorMap w;          // wq [E][N][K], box 128 B x 128 rows x 1
  CUtensorMap lb;         // lora_b [L][N][R], box 64 (few tokens: sum_width(R)) x 128 rows x 1
  CUtensorMap h[H_MAPS];  // hl [M][2 rank_pad], box 64 x 16 (i + 1) rows
};

struct Params {
  const float *xs;
  const float *ws;
  const void *bias;
  int bias_dtype;
  void *out;
  int out_dtype;
  const int *offsets;  // null: one group of all rows
  int M, N, E;
  int k_blocks;
  int n_wb;        // blocks of weight rows
  int pre_w;       // weights and offsets may be read before the dependency wait (adapters: always)
  // split_kernel
  int split, kps, stages;
  int tok_cap;        // tokens per tile at most
  uint32_t off_ring;  // shared-memory offsets
  uint32_t off_part;
  uint32_t off_lora;
  uint32_t off_tab;
  // adapters
  const int *ids;
  const void *lora_b;
  int lora_dtype;
  int L, R, rank_pad;
  const int4 *plan;  // token tiles (persist_kernel)
  int plan_mixed;    // .. of several adapters: from this entry on
  const void *hl;
  const float *hscale;
  // few tokens, whose down projection is the GEMM's own (split_kernel)
  const void *x;       // [M][K] of lora_dtype
  const void *lora_a;  // [L][R][K]
  const float *scaling;
  int K;
};

__device__ __forceinline__ float load_bias(const void *bias, int dtype, int64_t n) {
  switch (dtype) {
    case kBF16: {
      const uint16_t b = __ldg(reinterpret_cast<const unsigned short *>(bias) + n);
      return __uint_as_float(static_cast<uint32_t>(b) << 16);
    }
    case kF16: return __half2float(__ldg(reinterpret_cast<const __half *>(bias) + n));
    case kF32: return __ldg(reinterpret_cast<const float *>(bias) + n);
    default: return 0.0f;
  }
}

__device__ __forceinline__ void store_out(void *out, int dtype, int64_t i, float v) {
  if (dtype == kF16)
    reinterpret_cast<__half *>(out)[i] = __float2half_rn(v);
  else
    reinterpret_cast<__nv_bfloat16 *>(out)[i] = __float2bfloat16_rn(v);
}

__device__ __forceinline__ void record_timeout(volatile int *abort) {
  if (!*abort) {
    atomicOr(&g_rowsel_status, 64u);
    *abort = 1;
  }
}

// A whole warp waits for a barrier's phase, and goes on converged, as the instructions with
// .aligned (TMEM and matrix loads, matrix stores, barriers) need it. The roles that issue TMA copies and MMAs keep the
// warp converged and issue from one elected lane: in a branch of one lane the operands of each
// copy or MMA go through per-thread registers first, which made an MMA take 125 cycles
// whatever its N and a stage's two copies 400.
__device__ __forceinline__ bool warp_wait(uint32_t bar, uint32_t parity, volatile int *abort,
                                          bool elected) {
  if (__all_sync(0xFFFFFFFFu, ptx::mbar_try_wait(bar, parity))) return true;
  const bool got = ptx::mbar_wait_bounded(bar, parity, abort, kWaitLimitNs);
  if (__all_sync(0xFFFFFFFFu, got)) return true;
  if (elected) record_timeout(abort);
  return false;
}

__device__ __forceinline__ int ceil_div(int a, int b) { return (a + b - 1) / b; }

// The groups' rows and tiles, in shared memory: row[e] .. row[e + 1] are the rows of group e,
// tile[e] its first tile. Called by the whole CTA; ends with a CTA barrier.
__device__ __forceinline__ void build_groups(const Params &p, int tok_max, int *row, int *tile) {
  const int E = p.E;
  if (p.offsets == nullptr) {
    if (threadIdx.x == 0) {
      row[0] = 0;
      row[1] = p.M;
      tile[0] = 0;
      tile[1] = ceil_div(p.M, tok_max) * p.n_wb;
    }
    __syncthreads();
    return;
  }
  for (int i = threadIdx.x; i <= E; i += blockDim.x)
    row[i] = min(max(__ldg(p.offsets + i), 0), p.M);
  __syncthreads();
  if (threadIdx.x < 32) {
    const int lane = threadIdx.x;
    int carry = 0;  // running maximum of the offsets before this chunk
    for (int b = 0; b <= E; b += 32) {
      const int i = b + lane;
      int v = i <= E ? row[i] : 0;
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const int u = __shfl_up_sync(0xFFFFFFFFu, v, d);
        if (lane >= d) v = max(v, u);
      }
      v = max(v, carry);
      if (i <= E) row[i] = v;
      carry = __shfl_sync(0xFFFFFFFFu, v, 31);
    }
    __syncwarp();
    int first = 0;
    for (int b = 0; b <= E; b += 32) {
      const int i = b + lane;
      const int n = i < E ? ceil_div(row[i + 1] - row[i], tok_max) * p.n_wb : 0;
      int v = n;
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const int u = __shfl_up_sync(0xFFFFFFFFu, v, d);
        if (lane >= d) v += u;
      }
      if (i <= E) tile[i] = first + v - n;
      first += __shfl_sync(0xFFFFFFFFu, v, 31);
    }
  }
  __syncthreads();
}

struct Tile {
  int e;       // group
  int wb;      // block of weight rows
  int t0, t1;  // tokens
  int nn;      // MMA N: tokens padded to a multiple of 16 x CG
  int adapter; // of all its tokens, -1: none, -2: several
};

// Tile t of the table; `e` is a group at or before the tile's (advanced to it).
template <int CG>
__device__ __forceinline__ Tile find_tile(const Params &p, int tok_max, const int *row,
                                          const int *tile, int t, int &e) {
  while (tile[e + 1] <= t) ++e;
  Tile q;
  q.e = e;
  const int r0 = row[e], rows = row[e + 1] - r0;
  const int n_tb = ceil_div(rows, tok_max);
  const int per = (ceil_div(rows, n_tb) + 16 * CG - 1) / (16 * CG) * (16 * CG);
  const int l = t - tile[e];
  // The larger operand of the group streams once, the tiles that run side by side share the
  // smaller one through L2.
  int tb;
  if (rows >= p.N) {
    tb = l / p.n_wb;
    q.wb = l - tb * p.n_wb;
  } else {
    q.wb = l / n_tb;
    tb = l - q.wb * n_tb;
  }
  q.t0 = r0 + tb * per;
  q.t1 = min(r0 + rows, q.t0 + per);
  q.nn = (q.t1 - q.t0 + 16 * CG - 1) / (16 * CG) * (16 * CG);
  q.adapter = -1;
  return q;
}

// The tiles of a call with adapters, from the plan: first those of several adapters (they take
// longest, and this way no CTA pair gets a second one before all have one), then the others
// in the order of find_tile. Each step also loads the next tile's entry, which is then at hand
// without a wait.
struct PlanWalk {
  int n_one, first_one, num_tiles;  // token blocks and first tile of one adapter
  int4 next;

  __device__ __forceinline__ int weight_block(const Params &p, int t) const {
    if (t < first_one) return t % p.n_wb;
    return p.M >= p.N ? (t - first_one) % p.n_wb : (t - first_one) / n_one;
  }
  __device__ __forceinline__ void load(const Params &p, int t) {
    if (t >= num_tiles) return;
    const int l = t - first_one;
    next = __ldg(p.plan + (l < 0 ? p.plan_mixed + t / p.n_wb
                                 : 1 + (p.M >= p.N ? l / p.n_wb : l % n_one)));
  }
  __device__ __forceinline__ void start(const Params &p, int t) {
    const int4 head = __ldg(p.plan);
    n_one = head.x;
    first_one = head.y * p.n_wb;
    num_tiles = first_one + n_one * p.n_wb;
    load(p, t);
  }
  template <int CG>
  __device__ __forceinline__ Tile take(const Params &p, int t, int step) {
    Tile q;
    q.e = 0;
    q.wb = weight_block(p, t);
    q.t0 = next.x;
    q.t1 = next.y;
    q.adapter = next.z;
    q.nn = (q.t1 - q.t0 + 16 * CG - 1) / (16 * CG) * (16 * CG);
    load(p, t + step);
    return q;
  }
};

// Zeros to the rows that no group holds; the `n` threads from `first` of every CTA.
__device__ __forceinline__ void zero_rows(const Params &p, const int *row, int first, int n) {
  const int lo = row[0], hi = row[p.E];
  const int todo = lo + p.M - hi;
  uint16_t *out = reinterpret_cast<uint16_t *>(p.out);
  for (int i = blockIdx.x; i < todo; i += gridDim.x) {
    uint16_t *dst = out + static_cast<int64_t>(i < lo ? i : i - lo + hi) * p.N;
    for (int c = static_cast<int>(threadIdx.x) - first; c < p.N; c += n) dst[c] = 0;
  }
}

// ---------------------------------------------------------------- adapters
//
// A tile whose tokens all have one adapter takes it on the tensor cores, as further stages of
// the ring: the adapter's B rows beside the tokens' h, into an accumulator of their own. 64
// 16-bit elements are the 128 bytes of a stage's row: up to rank 32 the high and the low part
// of h share a stage's box, above it each 64 values of the rank take a stage for either part.
// The low part, 2^kLoraLowShift times too large, comes first; the first MMA of the high part divides
// the accumulator by as much.
//
// A tile of tokens of short runs (decoding requests) takes its adapters one after the other,
// each into a window of TMEM columns of its own for all the tile's tokens; their h is loaded
// once and the stages bring B alone. The epilogue keeps the columns of the adapter's own tokens
// while further adapters come in. The columns of the other tokens are never read, so that an
// adapter's infinities stay with its tokens (which one accumulator over tokens masked with
// zeros would not do: 0 * inf).
//
// split_kernel, where the whole call is such tokens and a CTA has few K-blocks, takes the
// adapters on the epilogue warps' own matrix instructions (adapter_sums below), with a ring of
// B boxes that a further warp fills while the K-blocks run. Measured, both ways: 64 tokens of 27
// adapters, 4096 -> 6144, rank 32: 29 us on the warps, 37 in TMEM windows behind the K-blocks of
// one ring (whose order makes the two wait for one another); persist_kernel, 2000 tokens of
// prompts and decodes, 4096 -> 4096, rank 64: 82 us on the warps (0.8 us an adapter, which
// nothing hides in a pair that has one tile), 79 in windows; 16384 rows, rank 128: 351 and 337.

// What an MMA finds in the accumulator: nothing that counts, sums to add to, or the low part's
// sums, to be divided by 2^kLoraLowShift.
enum class Acc { kFresh, kAdd, kShift };

// The stages of an adapter that is a whole tile's: stage(bx, hx, steps, acc) with the columns
// of B and of hl, the 16-element steps and what the accumulator holds; false ends them. (Nested
// counted loops: with the columns computed from a stage's number by division, and MMAs in a loop of
// unknown length, a stage took 0.7 us.)
template <class Stage>
__device__ __forceinline__ bool adapter_stages(int rank_pad, Stage &&stage) {
  if (rank_pad <= 32) return stage(0, 0, rank_pad / 16, Acc::kFresh);
  for (int part = 1; part >= 0; --part)
    for (int bx = 0; bx < rank_pad; bx += 64)
      if (!stage(bx, part * rank_pad + bx, min(4, (rank_pad - bx) / 16),
                 bx != 0 ? Acc::kAdd : part != 0 ? Acc::kFresh : Acc::kShift))
        return false;
  return true;
}

// d = d (as `acc` says) + B . h^T for up to 64 ranks: B at `b`, h at `h`.
template <int CG>
__device__ __forceinline__ void lora_mma(uint32_t d, uint32_t b, uint64_t hdesc, uint32_t idesc,
                                         int steps, Acc acc) {
  const uint64_t bdesc = ptx::sw128_kmajor_desc(b);
#pragma unroll
  for (int kk = 0; kk < 4; ++kk)  // 16 elements: 32 bytes
    if (kk < steps) {
      if (kk == 0 && acc == Acc::kShift)
        ptx::mma_f16_shift<CG, kLoraLowShift>(d, bdesc, hdesc, idesc);
      else
        ptx::mma_f16<CG>(d, bdesc + 2 * kk, hdesc + 2 * kk, idesc,
                         kk == 0 && acc == Acc::kFresh ? 0u : 1u);
    }
}

// A mixed tile's h in shared memory: boxes of 64 columns (`rows` rows of 128 bytes), those of
// the high part and behind them those of the low part; up to rank 32 one box has both.
__device__ __forceinline__ int h_boxes(int rank_pad) {
  return rank_pad <= 32 ? 1 : (rank_pad + 63) / 64 * 2;
}
__device__ __forceinline__ int h_column(int rank_pad, int box) {
  const int half = (rank_pad + 63) / 64;
  return box < half ? box * 64 : rank_pad + (box - half) * 64;
}
// The low part's descriptor offset from the high part's.
__device__ __forceinline__ uint32_t h_low(int rank_pad, int rows) {
  return rank_pad <= 32 ? static_cast<uint32_t>(rank_pad / 8)
                        : static_cast<uint32_t>((rank_pad + 63) / 64 * rows * BK / 16);
}

__device__ __forceinline__ int token_id(const Params &p, int i, int end) {
  const int id = i < end ? __ldg(p.ids + i) : -1;
  return static_cast<uint32_t>(id) < static_cast<uint32_t>(p.L) ? id : -1;
}

// The adapters of up to 32 tokens, by a whole warp with a token a lane: bit l of `leaders` is
// set where token l is the first of its adapter, whose tokens are `same` of that lane.
struct TokenAdapters {
  int id;
  uint32_t same, leaders;

  __device__ __forceinline__ TokenAdapters(const Params &p, int t0, int t1) {
    const int lane = threadIdx.x & 31;
    id = token_id(p, t0 + lane, t1);
    same = __match_any_sync(0xFFFFFFFFu, id);
    leaders = __ballot_sync(0xFFFFFFFFu, id >= 0 && __ffs(static_cast<int>(same)) - 1 == lane);
  }
};

// This lane's row of the TMEM columns base + c of the tokens c in `mask`, to out[c * pitch].
__device__ __forceinline__ void keep_columns(uint32_t base, uint32_t mask, float *out, int pitch) {
  while (mask != 0) {
    const int c0 = __ffs(static_cast<int>(mask)) - 1;
    mask &= mask - 1;
    uint32_t v0, v1 = 0;
    ptx::tmem_ld_32x32b_x1(base + static_cast<uint32_t>(c0), v0);
    int c1 = -1;
    if (mask != 0) {
      c1 = __ffs(static_cast<int>(mask)) - 1;
      mask &= mask - 1;
      ptx::tmem_ld_32x32b_x1(base + static_cast<uint32_t>(c1), v1);
    }
    ptx::tmem_wait_ld();
    out[c0 * pitch] = __uint_as_float(v0);
    if (c1 >= 0) out[c1 * pitch] = __uint_as_float(v1);
  }
}

// The ring of B boxes for adapter_sums: 128 weight rows x 64 ranks (32 or 16 where the rank
// fits), rows of 128, 64 or 32 bytes swizzled over as many; 48 KB of it, so that three to
// eight boxes are under way. A warp of its own fills it (feed_sums), the four epilogue warps
// read it; both go through the tokens eight at a time, through the adapters of eight in the
// order of their first tokens, and through the rank a box at a time. `count` boxes have been
// through the ring.
constexpr uint32_t SUM_RING = 3 * W_STAGE;
constexpr int SUM_SLOTS_MAX = 8;
constexpr int SUM_RANK = 64;
constexpr int SUM_BARS = 2 * SUM_SLOTS_MAX;  // full, empty
__host__ __device__ constexpr int sum_width(int rank) { return rank > 32 ? 64 : rank > 16 ? 32 : 16; }
__device__ __forceinline__ uint32_t sum_slots(int rank) {
  return rank > 32 ? 3u : rank > 16 ? 6u : 8u;
}
struct SumRing {
  uint32_t slots;  // shared-memory addresses
  uint32_t bars;
  volatile int *abort;
  uint32_t n;       // slots
  uint32_t box;     // bytes of one
  uint32_t slot;    // the next, and its phase
  uint32_t phase;
  uint32_t count;

  __device__ __forceinline__ SumRing(const Params &p, uint32_t s, uint32_t b, volatile int *a)
      : slots(s), bars(b), abort(a), n(sum_slots(p.R)),
        box(static_cast<uint32_t>(sum_width(p.R)) * 2u * WROWS), slot(0), phase(0), count(0) {}
  __device__ __forceinline__ uint32_t full() const { return bars + 8 * slot; }
  __device__ __forceinline__ uint32_t empty() const { return bars + 8 * (SUM_SLOTS_MAX + slot); }
  __device__ __forceinline__ void next() {
    ++count;
    if (++slot == n) {
      slot = 0;
      phase ^= 1u;
    }
  }
};

// Lane l of a warp has the adapter of token l % 8 of eight (-1: none); bits 0-7 of the
// result are the tokens whose adapter no earlier one of them has.
__device__ __forceinline__ uint32_t first_tokens(int id) {
  const uint32_t same = __match_any_sync(0xFFFFFFFFu, id) & 0xFFu;
  const int lane = threadIdx.x & 31;
  return __ballot_sync(0xFFFFFFFFu, id >= 0 && lane < 8 && __ffs(static_cast<int>(same)) - 1 == lane) &
         0xFFu;
}

// The boxes for tokens [t0, t1) and weight rows n0 ..; by a whole warp. False when a wait ran
// out (nothing is issued after that).
__device__ __forceinline__ bool feed_sums(const Params &p, const CUtensorMap *map, SumRing &ring,
                                          int t0, int t1, int n0) {
  const int lane = threadIdx.x & 31;
  const bool elected = ptx::elect_one();
  // all of them into L2 first: three to eight boxes under way do not cover a trip to memory
  for (int i = t0; i < t1; i += 32) {
    const int id = token_id(p, i + lane, t1);
    const uint32_t same = __match_any_sync(0xFFFFFFFFu, id);
    if (id >= 0 && __ffs(static_cast<int>(same)) - 1 == lane)
      for (int rc = 0; rc < p.R; rc += SUM_RANK) ptx::tma_prefetch_3d(map, rc, n0, id);
    __syncwarp();
  }
  int next = token_id(p, t0 + (lane & 7), t1);
  for (int i = t0; i < t1; i += 8) {
    const int id = next;
    next = token_id(p, i + 8 + (lane & 7), t1);
    for (uint32_t todo = first_tokens(id); todo != 0; todo &= todo - 1) {
      const int a = __shfl_sync(0xFFFFFFFFu, id, __ffs(static_cast<int>(todo)) - 1);
      for (int rc = 0; rc < p.R; rc += SUM_RANK) {
        if (!warp_wait(ring.empty(), ring.phase ^ 1u, ring.abort, elected)) return false;
        if (elected) {
          ptx::mbar_arrive_expect_tx(ring.full(), ring.box);
          ptx::tma_load_3d(ring.slots + ring.slot * ring.box, map, rc, n0, a, ring.full());
        }
        ring.next();
      }
    }
  }
  return true;
}

// Waits (bounded) until every box issued has landed and been read.
__device__ __forceinline__ void drain_sums(SumRing &ring) {
  for (uint32_t i = min(ring.count, ring.n); i > 0; --i) {
    if (ring.slot == 0) {
      ring.slot = ring.n - 1;
      ring.phase ^= 1u;
    } else {
      --ring.slot;
    }
    ptx::mbar_wait_timeout(ring.empty(), ring.phase, kDrainLimitNs);
  }
}

// Eight tokens' adapters (as token_id gives them) and h, the B operand of their products: h of
// token lane / 4, ranks 16j + 2t, + 1 and 16j + 8 + 2t, + 1, high and low part, t = lane % 4
// (zero past the rank and for tokens without an adapter, whose h is not written).
template <int J>
struct EightTokens {
  int id;
  uint32_t h[J][4];

  __device__ __forceinline__ void load(const Params &p, int i0, int t1) {
    const int lane = threadIdx.x & 31;
    id = token_id(p, i0 + (lane & 7), t1);
    const bool has = __shfl_sync(0xFFFFFFFFu, id, lane >> 2) >= 0;
    const uint32_t *hr = reinterpret_cast<const uint32_t *>(p.hl) +
                         static_cast<int64_t>(i0 + (lane >> 2)) * p.rank_pad + (lane & 3);
#pragma unroll
    for (int j = 0; j < J; ++j) {
      const bool in = has && 16 * j < p.rank_pad;
      h[j][0] = in ? __ldg(hr + 8 * j) : 0u;
      h[j][1] = in ? __ldg(hr + 8 * j + 4) : 0u;
      h[j][2] = in ? __ldg(hr + p.rank_pad / 2 + 8 * j) : 0u;
      h[j][3] = in ? __ldg(hr + p.rank_pad / 2 + 8 * j + 4) : 0u;
    }
  }
};

__device__ __forceinline__ void mma_16x8x16(bool f16, float (&d)[4], const uint32_t (&a)[4],
                                            uint32_t b0, uint32_t b1) {
  if (f16)
    ptx::mma_f16_16x8x16(d, a[0], a[1], a[2], a[3], b0, b1);
  else
    ptx::mma_bf16_16x8x16(d, a[0], a[1], a[2], a[3], b0, b1);
}

// For the eight tokens `now` and the 32 weight rows `quarter` of the boxes: the sums
// sum_r (hi + lo / 2^kLoraLowShift)[token][r] * B[adapter of the token][row][r], as matrix
// fragments: lane 4i + t gets tokens 2t, 2t + 1 of rows i + 8k in s[k]; zero for tokens without an
// adapter. C boxes of 16 J ranks an adapter. By one epilogue warp; false when a wait ran out. The high
// and the low part have accumulators of their own and a box's fragments are read before its
// first MMA, so that the chain of dependent MMAs is J long: in one chain with reads between
// them a box of 32 ranks took 740 cycles.
template <int J, int C>
__device__ __forceinline__ bool adapter_sums(const Params &p, SumRing &ring,
                                             const EightTokens<J * C> &now, int quarter,
                                             float2 (&s)[4]) {
  const int lane = threadIdx.x & 31;
  const bool f16 = p.lora_dtype == kF16;
  const int id = now.id;
#pragma unroll
  for (int k = 0; k < 4; ++k) s[k] = make_float2(0.0f, 0.0f);
  const int id0 = __shfl_sync(0xFFFFFFFFu, id, 2 * (lane & 3));
  const int id1 = __shfl_sync(0xFFFFFFFFu, id, 2 * (lane & 3) + 1);
  // ldmatrix: lane 8m + i has row i + 8 (m % 2) of a 16-row tile, 16-byte column 2j + m / 2;
  // column c of a row lies at c ^ swizzle: address bits 7.. of the row's own (the same for
  // rows 16 apart)
  constexpr uint32_t kRow = 32 * J;  // bytes
  const uint32_t row = static_cast<uint32_t>(quarter * 32 + (lane & 7) + (lane & 8));
  const uint32_t col = static_cast<uint32_t>(lane >> 4);
  const uint32_t swizzle = row * kRow / 128 & (kRow / 16 - 1);
#pragma unroll 1
  for (uint32_t todo = first_tokens(id); todo != 0; todo &= todo - 1) {
    const int a = __shfl_sync(0xFFFFFFFFu, id, __ffs(static_cast<int>(todo)) - 1);
    float d[2][2][4];  // [16-row tile][high, low]
#pragma unroll
    for (int m = 0; m < 2; ++m)
#pragma unroll
      for (int e = 0; e < 8; ++e) d[m][e >> 2][e & 3] = 0.0f;
#pragma unroll
    for (int c = 0; c < C; ++c) {
      if (!warp_wait(ring.full(), ring.phase, ring.abort, lane == 0)) return false;
      const uint32_t box = ring.slots + ring.slot * ring.box + row * kRow;
      uint32_t w[2][J][4];
#pragma unroll
      for (int j = 0; j < J; ++j)
#pragma unroll
        for (int m = 0; m < 2; ++m)
          ptx::ldsm_x4(box + m * 16 * kRow + (((2 * j + col) ^ swizzle) << 4), w[m][j]);
#pragma unroll
      for (int j = 0; j < J; ++j)
#pragma unroll
        for (int m = 0; m < 2; ++m) {
          const uint32_t(&h)[4] = now.h[c * J + j];
          mma_16x8x16(f16, d[m][0], w[m][j], h[0], h[1]);
          mma_16x8x16(f16, d[m][1], w[m][j], h[2], h[3]);
        }
      __syncwarp();
      if (lane == 0) ptx::mbar_arrive(ring.empty());
      ring.next();
    }
    // d[m]: rows i + 16m (0, 1) and i + 16m + 8 (2, 3), tokens 2t (0, 2) and 2t + 1 (1, 3)
    constexpr float kLow = 1.0f / (1 << kLoraLowShift);
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int e = 2 * (k & 1);
      if (id0 == a) s[k].x = fmaf(d[k >> 1][1][e], kLow, d[k >> 1][0][e]);
      if (id1 == a) s[k].y = fmaf(d[k >> 1][1][e + 1], kLow, d[k >> 1][0][e + 1]);
    }
  }
  return true;
}

// All tokens [t0, t1) so, eight at a time: to(i, s) takes the sums of the tokens from t0 + i.
template <int J, int C, class To>
__device__ __forceinline__ bool token_sums(const Params &p, SumRing &ring, int t0, int t1,
                                           int quarter, To &&to) {
  EightTokens<J * C> now;
  now.load(p, t0, t1);
#pragma unroll 1
  for (int i = 0; t0 + i < t1; i += 8) {
    EightTokens<J * C> next;  // (under way meanwhile)
    next.load(p, t0 + i + 8, t1);
    float2 s[4];
    if (!adapter_sums<J, C>(p, ring, now, quarter, s)) return false;
    to(i, s);
    now = next;
  }
  return true;
}

template <class To>
__device__ __forceinline__ bool token_sums(const Params &p, SumRing &ring, int t0, int t1,
                                           int quarter, To &&to) {
  if (p.R > 64) return token_sums<4, 2>(p, ring, t0, t1, quarter, to);
  if (p.R > 32) return token_sums<4, 1>(p, ring, t0, t1, quarter, to);
  if (p.R > 16) return token_sums<2, 1>(p, ring, t0, t1, quarter, to);
  return token_sums<1, 1>(p, ring, t0, t1, quarter, to);
}

// Eight 16-bit values as floats.
__device__ __forceinline__ void unpack8(const uint4 &v, bool f16, float (&f)[8]) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (f16) {
      const float2 t = __half22float2(*reinterpret_cast<const __half2 *>(&w[i]));
      f[2 * i] = t.x;
      f[2 * i + 1] = t.y;
    } else {
      f[2 * i] = __uint_as_float(w[i] << 16);
      f[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
    }
  }
}

__device__ __forceinline__ void epilogue_sync() {
  __syncwarp();
  asm volatile("bar.sync 1, 128;" ::: "memory");
}

// A few tokens' adapters without a down projection of their own (a launch, and a wait for it,
// longer than all of this): the CTAs of the K-split multiply their K ranges of x with those of
// A and push the parts of h to the first of them, which adds them up in rank order and multiplies
// with B. (Not each its own part: where B is infinite, parts of different signs would make a NaN of
// what is an infinity.) CUDA cores, fp32 throughout. Nothing here depends on the quantizer, so it
// comes before the dependency wait. out[m][row] for the tile's 128 rows, in the first CTA; `h`:
// OWN_WORK floats of shared memory, and behind them as many for each CTA.
// Down to here a CTA's values of h times its K-blocks are done before the K-blocks have
// arrived: 4096 -> 4096 (8 K-blocks a CTA), one token, rank 16: 10.3 us against 16.2 with a down
// projection of its own; two tokens 12.4 against 16.8; one token, rank 64: 15.6 against 16.3,
// rank 128: 22.3 against 16.9.
constexpr int OWN_WORK = 384;
__device__ __forceinline__ void own_adapter_sums(const Params &p, int k0, int k1, int n, float *h,
                                                 float *out, int et, int row, int rank,
                                                 uint32_t bar, volatile int *abort) {
  const bool f16 = p.lora_dtype == kF16;
  const int warp = et >> 5, lane = et & 31;
  const int chunks = p.K / 8;  // 16-byte chunks of a row of x or A; K % 16 == 0
  const int c1 = min(k1, p.K) / 8;
  const uint4 *x4 = reinterpret_cast<const uint4 *>(p.x);
  const uint4 *a4 = reinterpret_cast<const uint4 *>(p.lora_a);
  const int n_h = p.M * p.R;
  float *parts = h + OWN_WORK;  // [CTA][n_h]
  const uint32_t to = ptx::map_shared_rank(ptx::smem_u32(parts + rank * n_h), 0);
  // lane m has token m's
  static_assert(kLoraOwnTokens <= 32);
  const int lane_id = token_id(p, lane, p.M);
  const float lane_scaling = lane_id >= 0 ? __ldg(p.scaling + lane_id) : 0.0f;
  bool started = false;  // the first CTA is known to have
  // four values of h at a time (R % 8 == 0: of one token), so that their loads run side by side
#pragma unroll 1
  for (int v = 4 * warp; v < n_h; v += 4 * EPI_WARPS) {
    const int m = v / p.R, r = v - m * p.R;
    const int id = __shfl_sync(0xFFFFFFFFu, lane_id, m);
    float s[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    if (id >= 0) {
#pragma unroll 2
      for (int c = k0 / 8 + lane; c < c1; c += 32) {
        float xv[8];
        uint4 av[4];
#pragma unroll
        for (int i = 0; i < 4; ++i)
          av[i] = __ldg(a4 + (static_cast<int64_t>(id) * p.R + r + i) * chunks + c);
        unpack8(__ldg(x4 + static_cast<int64_t>(m) * chunks + c), f16, xv);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          float f[8];
          unpack8(av[i], f16, f);
#pragma unroll
          for (int j = 0; j < 8; ++j) s[i] = fmaf(xv[j], f[j], s[i]);
        }
      }
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int d = 16; d > 0; d >>= 1) s[i] += __shfl_xor_sync(0xFFFFFFFFu, s[i], d);
    }
    __syncwarp();
    if (!started) ptx::cluster_wait_acquire();
    started = true;
    const float mine = lane == 0 ? s[0] : lane == 1 ? s[1] : lane == 2 ? s[2] : s[3];
    if (lane < 4) ptx::st_shared_cluster_f32(to + static_cast<uint32_t>(v + lane) * 4u, mine);
    __syncwarp();
  }
  if (!started) ptx::cluster_wait_acquire();
  if (lane == 0) ptx::mbar_arrive_cluster(ptx::map_shared_rank(bar, 0));
  if (rank != 0) return;
  if (!ptx::mbar_wait_bounded_cluster(bar, 0, abort, kWaitLimitNs) && lane == 0)
    record_timeout(abort);
  __syncwarp();
  for (int m = 0; m < p.M; ++m) {
    const float sc = __shfl_sync(0xFFFFFFFFu, lane_scaling, m);
    if (et < p.R) {  // (R <= 128)
      float s = 0.0f;
      for (int c = 0; c < p.split; ++c) s += parts[c * n_h + m * p.R + et];
      h[m * p.R + et] = s * sc;
    }
    __syncwarp();
  }
  epilogue_sync();
  const uint16_t *lb = reinterpret_cast<const uint16_t *>(p.lora_b);
#pragma unroll 1
  for (int m = 0; m < p.M; ++m) {
    const int id = __shfl_sync(0xFFFFFFFFu, lane_id, m);
    float s = 0.0f;
    if (id >= 0) {
      const uint4 *b4 = reinterpret_cast<const uint4 *>(
          lb + (static_cast<int64_t>(id) * p.N + min(n, p.N - 1)) * p.R);
#pragma unroll 4
      for (int c = 0; c < p.R / 8; ++c) {
        float f[8];
        unpack8(__ldg(b4 + c), f16, f);
#pragma unroll
        for (int j = 0; j < 8; ++j) s = fmaf(h[m * p.R + 8 * c + j], f[j], s);
      }
    }
    out[m * WROWS + row] = s;
  }
}

// ---------------------------------------------------------------- persistent kernel

// Epilogue staging, per warp: 32 tokens x 32 columns of 16 bits, rows 80 bytes apart (eight
// rows' 16-byte pieces hit all banks once).
constexpr int BOX_PITCH = 80;
constexpr uint32_t BOX_BYTES = 32 * BOX_PITCH;
constexpr int SUM_PITCH = WROWS + 4;

template <int CG, bool LORA>
struct Cfg {
  static constexpr int TOK_MAX = LORA ? kLoraTileTokens : CG == 2 ? 256 : 128;
  static constexpr int X_ROWS = TOK_MAX / CG;  // tokens this CTA loads, at most
  static constexpr uint32_t X_STAGE = X_ROWS * BK;
  static constexpr uint32_t STAGE = W_STAGE + X_STAGE;
  static constexpr int STAGES = LORA ? 7 : 6;
  // TMEM: two accumulators; the adapters' products have a third, which only the epilogue of
  // one tile holds at a time
  static constexpr uint32_t ACC1 = TOK_MAX;
  static constexpr uint32_t ACC_L = 2 * TOK_MAX;
  static constexpr uint32_t TMEM_COLS = CG == 1 && !LORA ? 256 : 512;
  static constexpr uint32_t OFF_PAR = STAGES * STAGE;
  static constexpr uint32_t PAR_WARP = TOK_MAX * 4u * (LORA ? 2u : 1u);  // xs (hscale)
  static constexpr uint32_t OFF_BOX = OFF_PAR + EPI_WARPS * PAR_WARP;
  // the adapters' sums of a tile of several: [kLoraMixed][WROWS], rows 132 floats apart for
  // the fragments' reads
  static constexpr uint32_t OFF_SUM = OFF_BOX + EPI_WARPS * BOX_BYTES;
  static constexpr int WINDOWS = TOK_MAX / kLoraMixed;  // .. of TMEM columns, in ACC_L's place
  // .. and their h: four boxes of this CTA's tokens
  static constexpr uint32_t OFF_H = (OFF_SUM + (LORA ? kLoraMixed * SUM_PITCH * 4u : 0u) + 1023u) &
                                    ~1023u;
  static constexpr uint32_t OFF_TAB = OFF_H + (LORA ? 4u * (kLoraMixed / CG) * BK : 0u);
  static constexpr int TAB = LORA ? 2 : kMaxExperts + 1;
  static constexpr uint32_t OFF_BAR = (OFF_TAB + 2 * TAB * 4 + 7u) & ~7u;
  // full, empty, tfull, tempty, drain, h, windows
  static constexpr uint32_t NUM_BARS = 2 * STAGES + 7 + 2 * WINDOWS;
  static constexpr uint32_t OFF_SLOT = OFF_BAR + NUM_BARS * 8;
  static constexpr uint32_t SMEM_BYTES = OFF_SLOT + 8 + 1024;
  static_assert(STAGE % 1024 == 0, "swizzle atoms need 1024 B alignment");
  static_assert(SMEM_BYTES <= 232448, "shared memory budget");
  static_assert(!LORA || (CG == 2 && 3 * TOK_MAX <= 512), "TMEM budget");
};

template <int CG, bool LORA>
__global__ void __launch_bounds__(NUM_THREADS, 1)
    persist_kernel(const __grid_constant__ Maps maps, const __grid_constant__ Params p) {
  using C = Cfg<CG, LORA>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t *smem = reinterpret_cast<uint8_t *>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  const uint32_t sbase = ptx::smem_u32(smem);
  const uint32_t bar_full = sbase + C::OFF_BAR;
  const uint32_t bar_empty = bar_full + C::STAGES * 8;
  const uint32_t bar_tfull = bar_empty + C::STAGES * 8;
  const uint32_t bar_tempty = bar_tfull + 2 * 8;
  const uint32_t bar_drain = bar_tempty + 2 * 8;
  const uint32_t bar_h = bar_drain + 8;  // full, empty
  const uint32_t bar_wfull = bar_h + 2 * 8;
  const uint32_t bar_wempty = bar_wfull + 8 * C::WINDOWS;
  volatile uint32_t *tmem_slot = reinterpret_cast<volatile uint32_t *>(smem + C::OFF_SLOT);
  volatile int *abort = reinterpret_cast<volatile int *>(smem + C::OFF_SLOT + 4);
  int *g_row = reinterpret_cast<int *>(smem + C::OFF_TAB);
  int *g_tile = g_row + C::TAB;

  const int warp = ptx::uniform(threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  const uint32_t rank = CG == 2 ? ptx::cluster_ctarank() : 0u;  // 0 = leader (issues MMAs)
  const bool leader = rank == 0;
  const int group = blockIdx.x / CG;
  const int n_groups = gridDim.x / CG;

  if (threadIdx.x == 0) {
    ptx::prefetch_tmap(&maps.w);
    for (int s = 0; s < C::STAGES; ++s) {
      ptx::mbar_init(bar_full + 8 * s, 1);
      ptx::mbar_init(bar_empty + 8 * s, 1);
    }
    for (int a = 0; a < 2; ++a) {
      ptx::mbar_init(bar_tfull + 8 * a, 1);
      ptx::mbar_init(bar_tempty + 8 * a, EPI_WARPS * CG);
    }
    ptx::mbar_init(bar_drain, 1);
    ptx::mbar_init(bar_h, 1);
    ptx::mbar_init(bar_h + 8, 1);
    for (int i = 0; i < C::WINDOWS; ++i) {
      ptx::mbar_init(bar_wfull + 8 * i, 1);
      ptx::mbar_init(bar_wempty + 8 * i, EPI_WARPS * CG);
    }
    *abort = 0;
    ptx::fence_mbar_init();
  }
  if (warp == 1) {
    ptx::tmem_alloc<CG>(sbase + C::OFF_SLOT, C::TMEM_COLS);
    ptx::tmem_relinquish<CG>();
  }
  ptx::tc_fence_before();
  __syncthreads();
  if constexpr (CG == 2) ptx::cluster_sync();  // peer barriers initialised before any signal
  ptx::tc_fence_after();
  const uint32_t tmem_base = static_cast<uint32_t>(ptx::uniform(static_cast<int>(*tmem_slot)));

  // Weights and offsets that cannot depend on the kernel before: the first tile's first weight
  // boxes go out at once, their stages armed for the token boxes too.
  int ahead = 0;
  if (!LORA && p.pre_w) {
    build_groups(p, C::TOK_MAX, g_row, g_tile);
    if (warp == 0 && group < g_tile[p.E]) {
      int e = 0;
      const Tile q = find_tile<CG>(p, C::TOK_MAX, g_row, g_tile, group, e);
      const uint32_t tx = CG * W_STAGE + static_cast<uint32_t>(ptx::uniform(q.nn)) * BK;
      const int wz = ptx::uniform(q.e);
      const int wrow = (ptx::uniform(q.wb) * CG + static_cast<int>(rank)) * WROWS;
      const uint32_t fl = CG == 1 ? bar_full : ptx::map_shared_rank(bar_full, 0);
      ahead = min(C::STAGES, p.k_blocks);
      if (ptx::elect_one())
        for (int s = 0; s < ahead; ++s) {
          if (leader) ptx::mbar_arrive_expect_tx(bar_full + 8 * s, tx);
          const uint32_t dst = sbase + static_cast<uint32_t>(s) * C::STAGE;
          if constexpr (CG == 1)
            ptx::tma_load_3d(dst, &maps.w, s * BK, wrow, wz, fl + 8 * s);
          else
            ptx::tma_load_3d_pair(dst, &maps.w, s * BK, wrow, wz, fl + 8 * s);
        }
      __syncwarp();
    }
  }
  ptx::grid_dependency_wait();
  ptx::grid_launch_dependents();
  if (!LORA && !p.pre_w) build_groups(p, C::TOK_MAX, g_row, g_tile);

  PlanWalk plan = {};
  if constexpr (LORA) plan.start(p, group);
  const int num_tiles = LORA ? plan.num_tiles : g_tile[p.E];
  auto tile_at = [&](int t, int &e) -> Tile {
    if constexpr (LORA)
      return plan.template take<CG>(p, t, n_groups);
    else
      return find_tile<CG>(p, C::TOK_MAX, g_row, g_tile, t, e);
  };

  if (warp == 0) {
    // ------------------------------------------------------------ TMA producer
    const bool elected = ptx::elect_one();
    // both CTAs' bytes of a stage complete the leader's barrier
    const uint32_t full_leader = CG == 1 ? bar_full : ptx::map_shared_rank(bar_full, 0);
    int stage = 0;
    uint32_t phase = 0;
    uint32_t issued = 0;
    uint32_t hphase = 0;
    int e = 0;
    bool ok = true;
    for (int t = group; t < num_tiles && ok; t += n_groups) {
      const Tile q = tile_at(t, e);
      const int nn = ptx::uniform(q.nn);
      const int wz = ptx::uniform(q.e);
      const int wrow = (ptx::uniform(q.wb) * CG + static_cast<int>(rank)) * WROWS;
      const int xrow = ptx::uniform(q.t0) + static_cast<int>(rank) * (nn / CG);
      const int mi = nn / CG / 16 - 1;
      const uint32_t tx = CG * W_STAGE + static_cast<uint32_t>(nn) * BK;
      // One stage: the weight box and the token box (mx null: none) at the given coordinates.
      auto load = [&](const CUtensorMap *mw, int wx, int z, const CUtensorMap *mx, int xx) {
        if (!warp_wait(bar_empty + 8 * stage, phase ^ 1u, abort, elected)) return false;
        const uint32_t dst = sbase + static_cast<uint32_t>(stage) * C::STAGE;
        const uint32_t fl = full_leader + 8 * stage;
        if (elected) {
          if (ahead == 0) {
            if (leader)
              ptx::mbar_arrive_expect_tx(bar_full + 8 * stage, mx != nullptr ? tx : CG * W_STAGE);
            if constexpr (CG == 1)
              ptx::tma_load_3d(dst, mw, wx, wrow, z, fl);
            else
              ptx::tma_load_3d_pair(dst, mw, wx, wrow, z, fl);
          }
          if (mx != nullptr) {
            if constexpr (CG == 1)
              ptx::tma_load_2d(dst + W_STAGE, mx, xx, xrow, fl);
            else
              ptx::tma_load_2d_pair(dst + W_STAGE, mx, xx, xrow, fl);
          }
        }
        if (ahead > 0) --ahead;  // (armed, its weights under way)
        ++issued;
        if (++stage == C::STAGES) {
          stage = 0;
          phase ^= 1u;
        }
        return true;
      };
      for (int kb = 0; kb < p.k_blocks && ok; ++kb)
        ok = load(&maps.w, kb * BK, wz, &maps.x[mi], kb * BK);
      if constexpr (LORA) {
        const int adapter = ptx::uniform(q.adapter);
        if (adapter >= 0)
          ok = ok && adapter_stages(p.rank_pad, [&](int bx, int hx, int, Acc) {
                 return load(&maps.lb, bx, adapter, &maps.h[mi], hx);
               });
        if (adapter == -2 && ok) {
          const TokenAdapters ta(p, q.t0, q.t1);
          if (ta.leaders != 0) {
            if (!(ok = warp_wait(bar_h + 8, hphase ^ 1u, abort, elected))) break;
            const int boxes = h_boxes(p.rank_pad);
            if (elected) {
              const uint32_t bytes = static_cast<uint32_t>(nn / CG) * BK;  // (a multiple of 1024)
              const uint32_t hl = ptx::map_shared_rank(bar_h, 0);
              if (leader) ptx::mbar_arrive_expect_tx(bar_h, CG * bytes * static_cast<uint32_t>(boxes));
              for (int i = 0; i < boxes; ++i)
                ptx::tma_load_2d_pair(sbase + C::OFF_H + static_cast<uint32_t>(i) * bytes,
                                      &maps.h[mi], h_column(p.rank_pad, i), xrow, hl);
            }
            hphase ^= 1u;
          }
          for (uint32_t todo = ta.leaders; todo != 0 && ok; todo &= todo - 1) {
            const int a = __shfl_sync(0xFFFFFFFFu, ta.id, __ffs(static_cast<int>(todo)) - 1);
            for (int bx = 0; bx < p.R && ok; bx += 64) ok = load(&maps.lb, bx, a, nullptr, 0);
          }
        }
      }
    }
    // Drain: every load issued here has landed and been consumed.
    if (LORA && !ok) ptx::mbar_wait_timeout(bar_h + 8, hphase ^ 1u, kDrainLimitNs);
    const uint32_t n_drain = issued < C::STAGES ? issued : C::STAGES;
    for (uint32_t i = 0; i < n_drain; ++i) {
      if (stage == 0) {
        stage = C::STAGES - 1;
        phase ^= 1u;
      } else {
        --stage;
      }
      ptx::mbar_wait_timeout(bar_empty + 8 * stage, phase, kDrainLimitNs);
    }
  } else if (warp == 1) {
    // ------------------------------------------------------------ MMA issuer
    if (leader) {
      const bool elected = ptx::elect_one();
      int stage = 0;
      uint32_t phase = 0;
      int window = 0;
      uint32_t wphase = 0, hphase = 0;
      int it = 0;
      int e = 0;
      bool ok = true;
      auto next_stage = [&]() {
        // the stage is reusable (in both CTAs) once its MMAs have read it
        if (elected) {
          if constexpr (CG == 1)
            ptx::mma_commit(bar_empty + 8 * stage);
          else
            ptx::mma_commit_pair_mc(bar_empty + 8 * stage, 0x3);
        }
        if (++stage == C::STAGES) {
          stage = 0;
          phase ^= 1u;
        }
      };
      auto wait = [&](uint32_t bar, uint32_t parity) -> bool {
        if (!warp_wait(bar, parity, abort, elected)) return false;
        ptx::tc_fence_after();
        return true;
      };
      for (int t = group; t < num_tiles; t += n_groups, ++it) {
        const Tile q = tile_at(t, e);
        const int nn = ptx::uniform(q.nn);
        const int acc = it & 1;
        const uint32_t acc_phase = (it >> 1) & 1;
        if (!wait(bar_tempty + 8 * acc, acc_phase ^ 1u)) break;
        const uint32_t d = tmem_base + (acc ? C::ACC1 : 0u);
        const uint32_t idesc = ptx::idesc_e4m3_f32(WROWS * CG, nn);
        for (int kb = 0; kb < p.k_blocks; ++kb) {
          if (!(ok = wait(bar_full + 8 * stage, phase))) break;
          const uint32_t st = sbase + static_cast<uint32_t>(stage) * C::STAGE;
          const uint64_t adesc = ptx::sw128_kmajor_desc(st);
          const uint64_t bdesc = ptx::sw128_kmajor_desc(st + W_STAGE);
          if (elected) {
#pragma unroll
            for (int kk = 0; kk < BK / UMMA_K; ++kk) {
              const uint64_t koff = static_cast<uint64_t>((kk * UMMA_K) >> 4);
              const uint32_t accumulate = (kb | kk) != 0 ? 1u : 0u;
              if constexpr (CG == 1)
                ptx::mma_f8f6f4(d, adesc + koff, bdesc + koff, idesc, accumulate);
              else
                ptx::mma_f8f6f4_pair(d, adesc + koff, bdesc + koff, idesc, accumulate);
            }
          }
          next_stage();
        }
        if constexpr (LORA) {
          const int adapter = ptx::uniform(q.adapter);
          if (ok && adapter != -1) {
            // the third accumulator is free once the epilogue of the tile before has let
            // its own go (the same arrival that this loop waits for one tile later)
            if (it > 0 &&
                !wait(bar_tempty + 8 * (acc ^ 1), static_cast<uint32_t>((it - 1) >> 1) & 1u))
              break;
            const uint32_t id16 = ptx::idesc_f16_f32(WROWS * CG, nn, p.lora_dtype == kBF16);
            if (adapter >= 0) {
              const uint32_t low = p.rank_pad <= 32 ? h_low(p.rank_pad, 0) : 0u;  // (one stage)
              ok = adapter_stages(p.rank_pad, [&](int, int, int steps, Acc acc) {
                if (!wait(bar_full + 8 * stage, phase)) return false;
                const uint32_t st = sbase + static_cast<uint32_t>(stage) * C::STAGE;
                const uint64_t h = ptx::sw128_kmajor_desc(st + W_STAGE);
                if (elected) {
                  lora_mma<CG>(tmem_base + C::ACC_L, st, h + low, id16, steps, acc);
                  if (low != 0) lora_mma<CG>(tmem_base + C::ACC_L, st, h, id16, steps, Acc::kShift);
                }
                next_stage();
                return true;
              });
            } else {
              const TokenAdapters ta(p, q.t0, q.t1);
              const uint32_t low = h_low(p.rank_pad, nn / CG);
              if (ta.leaders != 0) {
                if (!(ok = wait(bar_h, hphase))) break;
                hphase ^= 1u;
              }
              for (int i = __popc(ta.leaders); i > 0 && ok; --i) {
                if (!(ok = wait(bar_wempty + 8 * window, wphase ^ 1u))) break;
                // B's boxes (two above rank 64, in a stage each) with the low part, then with
                // the high part
                const uint32_t d =
                    tmem_base + C::ACC_L + static_cast<uint32_t>(window * kLoraMixed);
                const uint64_t h = ptx::sw128_kmajor_desc(sbase + C::OFF_H);
                const uint64_t h1 = h + static_cast<uint32_t>(nn / CG) * BK / 16;
                if (!(ok = wait(bar_full + 8 * stage, phase))) break;
                const uint32_t b0 = sbase + static_cast<uint32_t>(stage) * C::STAGE;
                uint32_t b1 = 0;
                if (p.R > 64) {
                  const bool wrap = stage + 1 == C::STAGES;
                  const int s1 = wrap ? 0 : stage + 1;
                  if (!(ok = wait(bar_full + 8 * s1, wrap ? phase ^ 1u : phase))) break;
                  b1 = sbase + static_cast<uint32_t>(s1) * C::STAGE;
                }
                if (elected) {
                  const int steps0 = min(4, p.rank_pad / 16), steps1 = p.rank_pad / 16 - 4;
                  lora_mma<CG>(d, b0, h + low, id16, steps0, Acc::kFresh);
                  if (b1 != 0) lora_mma<CG>(d, b1, h1 + low, id16, steps1, Acc::kAdd);
                  lora_mma<CG>(d, b0, h, id16, steps0, Acc::kShift);
                  if (b1 != 0) lora_mma<CG>(d, b1, h1, id16, steps1, Acc::kAdd);
                }
                next_stage();
                if (b1 != 0) next_stage();
                if (ok && elected) ptx::mma_commit_pair_mc(bar_wfull + 8 * window, 0x3);
                if (++window == C::WINDOWS) {
                  window = 0;
                  wphase ^= 1u;
                }
              }
              if (ta.leaders != 0 && elected)  // h may be overwritten
                ptx::mma_commit_pair_mc(bar_h + 8, 0x3);
            }
          }
        }
        if (!ok) break;
        if (elected) {
          if constexpr (CG == 1)
            ptx::mma_commit(bar_tfull + 8 * acc);
          else
            ptx::mma_commit_pair_mc(bar_tfull + 8 * acc, 0x3);
        }
      }
      // No MMA may still be running when the CTAs free TMEM.
      if (elected) {
        if constexpr (CG == 1)
          ptx::mma_commit(bar_drain);
        else
          ptx::mma_commit_pair(bar_drain);
        ptx::mbar_wait_timeout(bar_drain, 0, kDrainLimitNs);
      }
    }
  } else {
    // ------------------------------------------------------------ epilogue
    // TMEM lane = weight row (output column), TMEM column = token. A warp takes its 32
    // columns of 32 tokens at a time as matrix fragments (lane 4i + t: columns i + 8k, tokens
    // 8g + 2t, + 1), transposes them through shared memory (stmatrix) and stores 64-byte
    // pieces of the tokens' rows, 16 bytes a lane.
    const int quarter = warp & 3;
    const int ew = warp - 2;
    float *e_xs = reinterpret_cast<float *>(smem + C::OFF_PAR + ew * C::PAR_WARP);
    float *e_hs = e_xs + C::TOK_MAX;
    float *sum = reinterpret_cast<float *>(smem + C::OFF_SUM);
    int window = 0;
    uint32_t wphase = 0;
    const uint8_t *box = smem + C::OFF_BOX + ew * BOX_BYTES;
    const uint32_t box_st = sbase + C::OFF_BOX + ew * BOX_BYTES +
                            static_cast<uint32_t>((lane & 7) * BOX_PITCH + (lane >> 3) * 16);
    const int fi = lane >> 2, ft = lane & 3;
    const bool wide = p.N % 8 == 0 && reinterpret_cast<uintptr_t>(p.out) % 16 == 0;
    int it = 0;
    int e = 0;
    for (int t = group; t < num_tiles; t += n_groups, ++it) {
      const Tile q = tile_at(t, e);
      const int acc = it & 1;
      const uint32_t acc_phase = (it >> 1) & 1;
      const int cnt = q.t1 - q.t0;
      const int n0 = (q.wb * CG + static_cast<int>(rank)) * WROWS + quarter * 32;
      // all loads at once, then to shared memory: one latency a tile (in a loop that stored
      // each before the next it took 7000 cycles a tile, more than its main loop)
      float w[4], b[4];  // of columns fi + 8k
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int64_t wn = static_cast<int64_t>(q.e) * p.N + min(n0 + fi + 8 * k, p.N - 1);
        w[k] = __ldg(p.ws + wn);
        b[k] = load_bias(p.bias, p.bias_dtype, wn);
      }
      float xs[C::TOK_MAX / 32], hs[C::TOK_MAX / 32];
#pragma unroll
      for (int k = 0; k < C::TOK_MAX / 32; ++k) {
        const int i = 32 * k + lane;
        xs[k] = i < cnt ? __ldg(p.xs + q.t0 + i) : 0.0f;
        hs[k] = LORA && q.adapter >= 0 && i < cnt ? __ldg(p.hscale + q.t0 + i) : 0.0f;
      }
      if (LORA && q.adapter == -2 && token_id(p, q.t0 + lane, q.t1) >= 0)  // (at most 32)
        hs[0] = __ldg(p.hscale + q.t0 + lane);
      __syncwarp();
#pragma unroll
      for (int k = 0; k < C::TOK_MAX / 32; ++k) {
        e_xs[32 * k + lane] = xs[k];
        if constexpr (LORA) e_hs[32 * k + lane] = hs[k];
      }
      __syncwarp();
      if constexpr (LORA) {
        if (q.adapter == -2) {
          // a tile of several adapters: their sums, as they come, to shared memory (a warp
          // writes and reads its own 32 rows; tokens without an adapter: zero)
          const TokenAdapters ta(p, q.t0, q.t1);
          float *mine = sum + quarter * 32 + lane;
          for (uint32_t none = __ballot_sync(0xFFFFFFFFu, ta.id < 0); none != 0; none &= none - 1)
            mine[(__ffs(static_cast<int>(none)) - 1) * SUM_PITCH] = 0.0f;
          bool ok = true;
          for (uint32_t todo = ta.leaders; todo != 0; todo &= todo - 1) {
            const uint32_t mask =
                __shfl_sync(0xFFFFFFFFu, ta.same, __ffs(static_cast<int>(todo)) - 1);
            if (!(ok = warp_wait(bar_wfull + 8 * window, wphase, abort, lane == 0))) break;
            ptx::tc_fence_after();
            keep_columns(tmem_base + (static_cast<uint32_t>(quarter * 32) << 16) + C::ACC_L +
                             static_cast<uint32_t>(window * kLoraMixed),
                         mask, mine, SUM_PITCH);
            ptx::tc_fence_before();
            __syncwarp();
            if (lane == 0)
              ptx::mbar_arrive_cluster_relaxed(ptx::map_shared_rank(bar_wempty + 8 * window, 0));
            if (++window == C::WINDOWS) {
              window = 0;
              wphase ^= 1u;
            }
          }
          if (!ok) break;
          __syncwarp();
        }
      }
      if (!warp_wait(bar_tfull + 8 * acc, acc_phase, abort, lane == 0)) break;
      ptx::tc_fence_after();
      const uint32_t t_row = tmem_base + (static_cast<uint32_t>(quarter * 32) << 16);
      const uint32_t t_acc = t_row + (acc ? C::ACC1 : 0u);
      constexpr uint32_t kHalf = 16u << 16;  // TMEM lanes 16-31 of the quarter
      // (columns all past N: nothing to store)
      for (int c = 0; c < cnt && n0 < p.N; c += 32) {
        __syncwarp();  // the box before has been read
        uint32_t r[2][16];
        ptx::tmem_ld_16x256b_x4(t_acc + static_cast<uint32_t>(c), r[0]);
        ptx::tmem_ld_16x256b_x4(t_acc + kHalf + static_cast<uint32_t>(c), r[1]);
        ptx::tmem_wait_ld();
        float2 v[4][4];  // [g][k]: tokens 8g + 2t, + 1 of column i + 8k
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          const float2 xs = *reinterpret_cast<const float2 *>(e_xs + c + 8 * g + 2 * ft);
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const uint32_t *a = r[k >> 1] + 4 * g + 2 * (k & 1);
            v[g][k] = ptx::fma2(
                ptx::mul2(make_float2(__uint_as_float(a[0]), __uint_as_float(a[1])), xs),
                make_float2(w[k], w[k]), make_float2(b[k], b[k]));
          }
        }
        if constexpr (LORA) {
          if (q.adapter >= 0) {
            ptx::tmem_ld_16x256b_x4(t_row + C::ACC_L + static_cast<uint32_t>(c), r[0]);
            ptx::tmem_ld_16x256b_x4(t_row + C::ACC_L + kHalf + static_cast<uint32_t>(c), r[1]);
            ptx::tmem_wait_ld();
#pragma unroll
            for (int g = 0; g < 4; ++g) {
              const float2 hs = *reinterpret_cast<const float2 *>(e_hs + c + 8 * g + 2 * ft);
#pragma unroll
              for (int k = 0; k < 4; ++k) {
                const uint32_t *a = r[k >> 1] + 4 * g + 2 * (k & 1);
                v[g][k] = ptx::fma2(make_float2(__uint_as_float(a[0]), __uint_as_float(a[1])), hs,
                                    v[g][k]);
              }
            }
          } else if (q.adapter == -2) {  // (one chunk: cnt <= kLoraMixed)
            const float *sr = sum + 2 * ft * SUM_PITCH + quarter * 32 + fi;
#pragma unroll
            for (int g = 0; g < 4; ++g) {
              const float2 hs = *reinterpret_cast<const float2 *>(e_hs + 8 * g + 2 * ft);
#pragma unroll
              for (int k = 0; k < 4; ++k)
                v[g][k] = ptx::fma2(make_float2(sr[8 * g * SUM_PITCH + 8 * k],
                                                sr[(8 * g + 1) * SUM_PITCH + 8 * k]),
                                    hs, v[g][k]);
            }
          }
        }
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          uint32_t o[4];
#pragma unroll
          for (int k = 0; k < 4; ++k)
            o[k] = p.out_dtype == kF16 ? ptx::pack_f16x2(v[g][k].x, v[g][k].y)
                                       : ptx::pack_bf16x2(v[g][k].x, v[g][k].y);
          ptx::stsm_x4_trans(box_st + static_cast<uint32_t>(8 * g * BOX_PITCH), o[0], o[1], o[2],
                             o[3]);
        }
        __syncwarp();
        uint16_t *out = reinterpret_cast<uint16_t *>(p.out) +
                        static_cast<int64_t>(q.t0 + c) * p.N + n0;
        if (wide) {
          const int col = ft * 8;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int m = 8 * i + fi;
            if (c + m < cnt && n0 + col < p.N)
              *reinterpret_cast<uint4 *>(out + static_cast<int64_t>(m) * p.N + col) =
                  *reinterpret_cast<const uint4 *>(box + m * BOX_PITCH + col * 2);
          }
        } else if (n0 + lane < p.N) {
          uint16_t v[32];
#pragma unroll
          for (int m = 0; m < 32; ++m)
            v[m] = *reinterpret_cast<const uint16_t *>(box + m * BOX_PITCH + lane * 2);
          uint16_t *to = out + lane;
#pragma unroll
          for (int m = 0; m < 32; ++m, to += p.N)
            if (c + m < cnt) *to = v[m];
        }
      }
      ptx::tc_fence_before();
      __syncwarp();
      if (lane == 0) {
        if constexpr (CG == 1)
          ptx::mbar_arrive(bar_tempty + 8 * acc);
        else
          ptx::mbar_arrive_cluster_relaxed(ptx::map_shared_rank(bar_tempty + 8 * acc, 0));
      }
    }
    if constexpr (!LORA) zero_rows(p, g_row, 64, 32 * EPI_WARPS);
  }

  __syncwarp();
  ptx::tc_fence_before();
  __syncthreads();
  if constexpr (CG == 2) ptx::cluster_sync();  // the leader's MMAs read the peer's memory
  if (warp == 1) {
    ptx::tc_fence_after();
    ptx::tmem_dealloc<CG>(tmem_base, C::TMEM_COLS);
  }
}

// ---------------------------------------------------------------- split-K kernel

// What bounds it: the latency of a short chain. One expert's row, 2048 -> 1024, 16 experts: 7.3
// us with the quantizer, of which the 2 MB of weights would take 0.6 at the copy rate; 64
// tokens with adapters, 4096 -> 6144: 28 us, three dependent launches, against 7.
constexpr int SPLIT_TOK = 128;   // tokens per tile, at most (with adapters kLoraRowsMaxM)
constexpr int SPLIT_STAGES = 8;  // ring slots, at most
constexpr int SPLIT_MAX = 8;     // CTAs per cluster, at most (portable)
// A tile's set-up and reduction, in K-blocks (half or twice as much: the same times, within
// 2%, at 1 to 64 tokens)
constexpr int SPLIT_COST = 12;
constexpr uint32_t SPLIT_EPI = (2 * SPLIT_TOK + 2 * WROWS) * 4;  // xs, ws, bias, hscale
constexpr uint32_t SPLIT_SMEM = 232448;

// OWN: the adapters by own_adapter_sums. Otherwise a further warp fills the ring of B boxes.
template <bool LORA, bool OWN>
constexpr int split_threads() {
  static_assert(LORA || !OWN);
  return NUM_THREADS + (LORA && !OWN ? 32 : 0);
}

template <bool LORA, bool OWN>
__global__ void __launch_bounds__(split_threads<LORA, OWN>(), 1)
    split_kernel(const __grid_constant__ Maps maps, const __grid_constant__ Params p) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t *smem = reinterpret_cast<uint8_t *>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  const uint32_t sbase = ptx::smem_u32(smem);
  __shared__ alignas(8) uint64_t s_bar[2 * SPLIT_STAGES + 3 + SUM_BARS];
  __shared__ uint32_t s_slot;
  __shared__ int s_abort;
  const uint32_t bar_full = ptx::smem_u32(s_bar);
  const uint32_t bar_empty = bar_full + 8 * SPLIT_STAGES;
  const uint32_t bar_acc = bar_empty + 8 * SPLIT_STAGES;
  const uint32_t bar_drain = bar_acc + 8;
  const uint32_t bar_own = bar_drain + 8;
  const uint32_t bar_sum = bar_own + 8;
  volatile uint32_t *tmem_slot = &s_slot;
  volatile int *abort = &s_abort;
  // partial sums of the rows reduced here: [CTA they come from][token][R rows]
  float *part = reinterpret_cast<float *>(smem + p.off_part);
  float *lora = reinterpret_cast<float *>(smem + p.off_lora);  // [tokens of this CTA][WROWS]
  int *g_row = reinterpret_cast<int *>(smem + p.off_tab);
  int *g_tile = g_row + p.E + 1;
  float *e_xs = reinterpret_cast<float *>(
      smem + ((p.off_tab + static_cast<uint32_t>(p.E + 1) * 8 + 15u) & ~15u));  // [SPLIT_TOK]
  float *e_ws = e_xs + SPLIT_TOK;                              // [WROWS]
  float *e_b = e_ws + WROWS;
  float *e_hs = e_b + WROWS;  // [SPLIT_TOK]

  const int warp = ptx::uniform(threadIdx.x >> 5), lane = threadIdx.x & 31;
  const int rank = static_cast<int>(ptx::cluster_ctarank());
  const int stages = p.stages;
  const uint32_t stage_bytes = W_STAGE + static_cast<uint32_t>(p.tok_cap) * BK;
  uint32_t tmem_cols = 32;
  while (tmem_cols < static_cast<uint32_t>(p.tok_cap)) tmem_cols <<= 1;

  if (threadIdx.x == 0) {
    ptx::prefetch_tmap(&maps.w);
    for (int s = 0; s < stages; ++s) {
      ptx::mbar_init(bar_full + 8 * s, 1);
      ptx::mbar_init(bar_empty + 8 * s, 1);
    }
    ptx::mbar_init(bar_acc, 1);
    ptx::mbar_init(bar_drain, 1);
    if (OWN) ptx::mbar_init(bar_own, static_cast<uint32_t>(p.split) * EPI_WARPS);
    for (int i = 0; i < SUM_SLOTS_MAX; ++i) {
      ptx::mbar_init(bar_sum + 8 * i, 1);
      ptx::mbar_init(bar_sum + 8 * (SUM_SLOTS_MAX + i), EPI_WARPS);
    }
    s_abort = 0;
    ptx::fence_mbar_init();
  }
  const bool pre_w = LORA || p.pre_w;
  if (!pre_w) ptx::grid_dependency_wait();
  build_groups(p, p.tok_cap, g_row, g_tile);
  const int t = blockIdx.x / p.split;
  if (t >= g_tile[p.E]) {  // the whole cluster: fewer tiles than clusters
    if (pre_w) ptx::grid_dependency_wait();
    ptx::grid_launch_dependents();
    zero_rows(p, g_row, 0, blockDim.x);
    return;
  }
  int ge = 0;
  const Tile q = find_tile<1>(p, p.tok_cap, g_row, g_tile, t, ge);
  const int kb0 = rank * p.kps;
  const int nkb = min(p.k_blocks, kb0 + p.kps) - kb0;  // >= 1 (the host's split)
  const int cnt = q.t1 - q.t0;
  const CUtensorMap *mx = &maps.x[ptx::uniform(q.nn) / 16 - 1];
  const uint32_t tx = W_STAGE + static_cast<uint32_t>(ptx::uniform(q.nn)) * BK;

  const int nn = ptx::uniform(q.nn);
  const int we = ptx::uniform(q.e), wrow = ptx::uniform(q.wb) * WROWS, xrow = ptx::uniform(q.t0);
  // The first stages' weight boxes go out at once: before the dependency wait where the
  // weights cannot depend on the kernel before (pre_w).
  if (warp == 0) {
    const int n = min(stages, nkb);
    if (ptx::elect_one())
      for (int i = 0; i < n; ++i) {
        const uint32_t fb = bar_full + 8 * i;
        ptx::mbar_arrive_expect_tx(fb, tx);
        ptx::tma_load_3d(sbase + static_cast<uint32_t>(i) * stage_bytes, &maps.w, (kb0 + i) * BK,
                         wrow, we, fb);
      }
  }
  if (warp == 1) {
    ptx::tmem_alloc<1>(ptx::smem_u32(&s_slot), tmem_cols);
    ptx::tmem_relinquish<1>();
  }
  ptx::tc_fence_before();
  __syncthreads();
  ptx::tc_fence_after();
  const uint32_t tmem = static_cast<uint32_t>(ptx::uniform(static_cast<int>(*tmem_slot)));
  // (waited for before the first push: all CTAs have started)
  ptx::cluster_arrive_release();
  if (OWN && warp >= 2) {
    const int row = (warp & 3) * 32 + lane;
    own_adapter_sums(p, kb0 * BK, (kb0 + nkb) * BK, q.wb * WROWS + row,
                     reinterpret_cast<float *>(smem + p.off_ring), lora, threadIdx.x - 64, row,
                     rank, bar_own, abort);
  }
  // Adapters: the cluster's CTAs share out the tokens, eight at a time (OWN: all of them are the
  // first CTA's).
  const int per_cta = LORA ? ((cnt + 7) / 8 + p.split - 1) / p.split * 8 : 0;
  const int a0 = OWN ? 0 : min(cnt, rank * per_cta);
  const int a1 = OWN ? (rank == 0 ? cnt : 0) : min(cnt, a0 + per_cta);
  // (B and ids are the call's own inputs: their boxes need no wait for the kernel before)
  if (LORA && !OWN && warp == 2 + EPI_WARPS) {
    SumRing ring(p, sbase + p.off_ring, bar_sum, abort);
    feed_sums(p, &maps.lb, ring, q.t0 + a0, q.t0 + a1, q.wb * WROWS);
    drain_sums(ring);
  }
  if (pre_w) ptx::grid_dependency_wait();
  ptx::grid_launch_dependents();

  // rows of the tile that this CTA reduces
  const int R = ((WROWS + p.split - 1) / p.split + 3) & ~3;
  const int r0 = rank * R;
  const int r1 = min(WROWS, r0 + R);
  const int quads = r1 > r0 ? (r1 - r0) >> 2 : 0;
  const int n0 = q.wb * WROWS;

  if (warp == 0) {
    const bool elected = ptx::elect_one();
    int issued = 0;
    int s = 0;
    uint32_t ph = 1;
    for (int i = 0; i < nkb; ++i) {
      const uint32_t fb = bar_full + 8 * s;
      const uint32_t dst = sbase + static_cast<uint32_t>(s) * stage_bytes;
      const bool refill = i >= stages;  // (the first are armed, their weight boxes under way)
      if (refill && !warp_wait(bar_empty + 8 * s, ph, abort, elected)) break;
      if (elected) {
        if (refill) {
          ptx::mbar_arrive_expect_tx(fb, tx);
          ptx::tma_load_3d(dst, &maps.w, (kb0 + i) * BK, wrow, we, fb);
        }
        ptx::tma_load_2d(dst + W_STAGE, mx, (kb0 + i) * BK, xrow, fb);
      }
      ++issued;
      if (++s == stages) {
        s = 0;
        ph ^= 1u;
      }
    }
    for (int i = issued - 1; i >= 0 && i >= issued - stages; --i)
      ptx::mbar_wait_timeout(bar_empty + 8 * (i % stages), static_cast<uint32_t>(i / stages) & 1u,
                             kDrainLimitNs);
  } else if (warp == 1) {
    const bool elected = ptx::elect_one();
    bool ok = true;
    const uint32_t idesc = ptx::idesc_e4m3_f32(WROWS, nn);
    int s = 0;
    uint32_t ph = 0;
    for (int i = 0; i < nkb; ++i) {
      if (!(ok = warp_wait(bar_full + 8 * s, ph, abort, elected))) break;
      ptx::tc_fence_after();
      const uint32_t st = sbase + static_cast<uint32_t>(s) * stage_bytes;
      const uint64_t adesc = ptx::sw128_kmajor_desc(st);
      const uint64_t bdesc = ptx::sw128_kmajor_desc(st + W_STAGE);
      if (elected) {
#pragma unroll
        for (int kk = 0; kk < BK / UMMA_K; ++kk) {
          const uint64_t koff = static_cast<uint64_t>((kk * UMMA_K) >> 4);
          ptx::mma_f8f6f4(tmem, adesc + koff, bdesc + koff, idesc, (i | kk) != 0 ? 1u : 0u);
        }
        ptx::mma_commit(bar_empty + 8 * s);
      }
      if (++s == stages) {
        s = 0;
        ph ^= 1u;
      }
    }
    if (elected) {
      if (ok) ptx::mma_commit(bar_acc);
      ptx::mma_commit(bar_drain);
      ptx::mbar_wait_timeout(bar_drain, 0, kDrainLimitNs);
    }
  } else if (warp < 2 + EPI_WARPS) {
    // xs (adapters: and hscale) of the tokens, weight scales and biases of the rows reduced
    // here
    const int et = threadIdx.x - 64;
    for (int i = et; i < q.nn; i += 128) {
      e_xs[i] = i < cnt ? __ldg(p.xs + q.t0 + i) : 0.0f;
      if constexpr (LORA && !OWN)
        e_hs[i] = token_id(p, q.t0 + i, q.t1) >= 0 ? __ldg(p.hscale + q.t0 + i) : 0.0f;
    }
    for (int i = et; i < r1 - r0; i += 128) {
      const int n = n0 + r0 + i;
      const int64_t wn = static_cast<int64_t>(q.e) * p.N + n;
      e_ws[i] = n < p.N ? __ldg(p.ws + wn) : 0.0f;
      e_b[i] = n < p.N ? load_bias(p.bias, p.bias_dtype, wn) : 0.0f;
    }
    const int quarter = warp & 3;
    const int row = quarter * 32 + lane;
    const int n = n0 + row;
    const float w = LORA && n < p.N ? __ldg(p.ws + n) : 1.0f;
    epilogue_sync();  // xs and hscale are in shared memory
    if constexpr (LORA && !OWN) {
      // (a warp writes and reads back its own rows only; after a wait that ran out, whatever)
      SumRing ring(p, sbase + p.off_ring, bar_sum, abort);
      token_sums(p, ring, q.t0 + a0, q.t0 + a1, quarter, [&](int i, float2(&s)[4]) {
        float *to = lora + (i + 2 * (lane & 3)) * WROWS + quarter * 32 + (lane >> 2);
        const float2 hs = *reinterpret_cast<const float2 *>(e_hs + a0 + i + 2 * (lane & 3));
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          to[8 * k] = s[k].x * hs.x;
          to[8 * k + WROWS] = s[k].y * hs.y;
        }
      });
      __syncwarp();
    }
    // TMEM (lane = weight row, column = token) -> the part of the CTA that reduces the row,
    // fp32: the K-blocks' sums as they are, or with adapters dequantized and added to the
    // adapters' sums
    // (one vote behind the wait; with warp_wait 64 tokens with adapters take 28.8 us, not 28.1)
    const bool ok =
        __all_sync(0xFFFFFFFFu, ptx::mbar_wait_bounded(bar_acc, 0, abort, kWaitLimitNs));
    if (!ok && lane == 0) record_timeout(abort);
    ptx::tc_fence_after();
    if (!OWN) ptx::cluster_wait_acquire();  // (own_adapter_sums has)
    const uint32_t t_row = tmem + (static_cast<uint32_t>(quarter * 32) << 16);
    const uint32_t dst = ptx::map_shared_rank(
        ptx::smem_u32(part) +
            static_cast<uint32_t>(rank * p.tok_cap * R + row % R) * 4u,
        static_cast<uint32_t>(row / R));
#pragma unroll 1
    for (int c = 0; c < q.nn; c += 16) {
      uint32_t r[16];
      if (ok) {
        ptx::tmem_ld_32x32b_x16(t_row + static_cast<uint32_t>(c), r);
        ptx::tmem_wait_ld();
      } else {
#pragma unroll
        for (int j = 0; j < 16; ++j) r[j] = 0u;
      }
#pragma unroll
      for (int j = 0; j < 16; ++j) {
        float v = __uint_as_float(r[j]);
        if constexpr (LORA) {
          v = v * e_xs[c + j] * w;
          if (c + j >= a0 && c + j < a1) v += lora[(c + j - a0) * WROWS + row];
        }
        if (c + j < cnt) ptx::st_shared_cluster_f32(dst + static_cast<uint32_t>((c + j) * R) * 4u, v);
      }
    }
    ptx::tc_fence_before();
  }
  __syncwarp();
  if (warp < 2 || warp >= 2 + EPI_WARPS) ptx::cluster_wait_acquire();

  __syncwarp();
  __syncthreads();
  ptx::cluster_sync();  // the partial sums of this CTA's rows have arrived

  // A task is 4 rows (output columns) of one token: 8 bytes of output.
  const bool wide = p.N % 4 == 0 && reinterpret_cast<uintptr_t>(p.out) % 8 == 0;
  const int step = static_cast<int>(blockDim.x);
  const int step_m = quads > 0 ? step / quads : 0, step_q = step - step_m * quads;
  int m = quads > 0 ? static_cast<int>(threadIdx.x) / quads : cnt;
  int qd = static_cast<int>(threadIdx.x) - m * quads;
#pragma unroll 2
  while (m < cnt) {
    float4 v[SPLIT_MAX];
#pragma unroll
    for (int s = 0; s < SPLIT_MAX; ++s)
      if (s < p.split)
        v[s] = *reinterpret_cast<const float4 *>(part + (s * p.tok_cap + m) * R + 4 * qd);
    float a[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int s = 0; s < SPLIT_MAX; ++s)
      if (s < p.split) {
        a[0] += v[s].x;
        a[1] += v[s].y;
        a[2] += v[s].z;
        a[3] += v[s].w;
      }
    const float xs = e_xs[m];
    const float4 w = *reinterpret_cast<const float4 *>(e_ws + 4 * qd);
    const float4 b = *reinterpret_cast<const float4 *>(e_b + 4 * qd);
    if constexpr (LORA) {
      a[0] += b.x;
      a[1] += b.y;
      a[2] += b.z;
      a[3] += b.w;
    } else {
      a[0] = fmaf(a[0] * xs, w.x, b.x);
      a[1] = fmaf(a[1] * xs, w.y, b.y);
      a[2] = fmaf(a[2] * xs, w.z, b.z);
      a[3] = fmaf(a[3] * xs, w.w, b.w);
    }
    const int n = n0 + r0 + 4 * qd;
    const int64_t o = static_cast<int64_t>(q.t0 + m) * p.N + n;
    if (wide) {
      if (n < p.N)
        *reinterpret_cast<uint2 *>(reinterpret_cast<uint16_t *>(p.out) + o) =
            p.out_dtype == kF16
                ? make_uint2(ptx::pack_f16x2(a[0], a[1]), ptx::pack_f16x2(a[2], a[3]))
                : make_uint2(ptx::pack_bf16x2(a[0], a[1]), ptx::pack_bf16x2(a[2], a[3]));
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (n + i < p.N) store_out(p.out, p.out_dtype, o + i, a[i]);
    }
    m += step_m;
    qd += step_q;
    if (qd >= quads) {
      qd -= quads;
      ++m;
    }
  }
  zero_rows(p, g_row, 0, blockDim.x);

  __syncwarp();
  if (warp == 1) {
    ptx::tc_fence_after();
    ptx::tmem_dealloc<1>(tmem, tmem_cols);
  }
}

// ---------------------------------------------------------------- host side

struct LaunchInfo {
  bool ready = false;
  cudaError_t err = cudaSuccess;
  int max_groups = 0;
};

template <int CG, bool LORA>
LaunchInfo &persist_info(const DeviceInfo &dev) {
  static LaunchInfo info[64];
  static std::mutex mu;
  std::lock_guard<std::mutex> lock(mu);
  LaunchInfo &li = info[dev.device & 63];
  if (!li.ready) {
    li.ready = true;
    li.err = cudaFuncSetAttribute(persist_kernel<CG, LORA>,
                                  cudaFuncAttributeMaxDynamicSharedMemorySize,
                                  static_cast<int>(Cfg<CG, LORA>::SMEM_BYTES));
    li.max_groups = dev.sm_count / CG;
    if (li.err == cudaSuccess && CG == 2) {
      cudaLaunchConfig_t cfg = {};
      cfg.gridDim = dim3(dev.sm_count / CG * CG);
      cfg.blockDim = dim3(NUM_THREADS);
      cfg.dynamicSmemBytes = Cfg<CG, LORA>::SMEM_BYTES;
      cudaLaunchAttribute attr[1];
      attr[0].id = cudaLaunchAttributeClusterDimension;
      attr[0].val.clusterDim.x = CG;
      attr[0].val.clusterDim.y = 1;
      attr[0].val.clusterDim.z = 1;
      cfg.attrs = attr;
      cfg.numAttrs = 1;
      int clusters = 0;
      li.err = cudaOccupancyMaxActiveClusters(&clusters, persist_kernel<CG, LORA>, &cfg);
      if (li.err == cudaSuccess) li.max_groups = std::min(li.max_groups, clusters);
      if (li.err == cudaSuccess && li.max_groups < 1) li.err = cudaErrorInvalidConfiguration;
    }
  }
  return li;
}

int launch_failed(const char *op, cudaError_t e) {
  set_error(std::string(op) + ": launch failed: " + cudaGetErrorString(e));
  return 4;
}

cudaError_t launch(const void *kernel, const Maps &maps, const Params &p, int ctas, int threads,
                   int cluster, size_t smem, cudaStream_t stream) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(ctas));
  cfg.blockDim = dim3(static_cast<unsigned>(threads));
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  int n = 0;
  if (cluster > 0) {
    attr[n].id = cudaLaunchAttributeClusterDimension;
    attr[n].val.clusterDim.x = static_cast<unsigned>(cluster);
    attr[n].val.clusterDim.y = 1;
    attr[n].val.clusterDim.z = 1;
    ++n;
  }
  attr[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[n].val.programmaticStreamSerializationAllowed = 1;
  ++n;
  cfg.attrs = attr;
  cfg.numAttrs = static_cast<unsigned>(n);
  void *args[] = {const_cast<Maps *>(&maps), const_cast<Params *>(&p)};
  return cudaLaunchKernelExC(&cfg, kernel, args);
}

template <int CG, bool LORA>
int launch_persist(const char *op, const Maps &maps, Params &p, int64_t tiles,
                   const DeviceInfo &dev, cudaStream_t stream) {
  LaunchInfo &li = persist_info<CG, LORA>(dev);
  if (li.err != cudaSuccess) return launch_failed(op, li.err);
  const int groups = static_cast<int>(std::min<int64_t>(tiles, li.max_groups));
  const cudaError_t e =
      launch(reinterpret_cast<const void *>(&persist_kernel<CG, LORA>), maps, p, groups * CG,
             NUM_THREADS, CG == 2 ? 2 : 0, Cfg<CG, LORA>::SMEM_BYTES, stream);
  return e == cudaSuccess ? 0 : launch_failed(op, e);
}

// Clusters of each size that the GPU holds at once with one CTA per SM (a size that does not
// divide the SMs of a GPC leaves some of them over).
struct SplitInfo {
  bool ready = false;
  cudaError_t err = cudaSuccess;
  int clusters[SPLIT_MAX + 1] = {};
};

template <bool LORA, bool OWN = false>
SplitInfo &split_info(const DeviceInfo &dev) {
  static SplitInfo info[64];
  static std::mutex mu;
  std::lock_guard<std::mutex> lock(mu);
  SplitInfo &si = info[dev.device & 63];
  if (!si.ready) {
    si.ready = true;
    // (the static barriers take a little of the 227 KB)
    si.err = cudaFuncSetAttribute(split_kernel<LORA, OWN>,
                                  cudaFuncAttributeMaxDynamicSharedMemorySize, SPLIT_SMEM - 1024);
    si.clusters[1] = dev.sm_count;
    for (int s = 2; s <= SPLIT_MAX && si.err == cudaSuccess; ++s) {
      cudaLaunchConfig_t cfg = {};
      cfg.gridDim = dim3(static_cast<unsigned>(dev.sm_count / s * s));
      cfg.blockDim = dim3(split_threads<LORA, OWN>());
      cfg.dynamicSmemBytes = SPLIT_SMEM - 1024;
      cudaLaunchAttribute attr[1];
      attr[0].id = cudaLaunchAttributeClusterDimension;
      attr[0].val.clusterDim.x = static_cast<unsigned>(s);
      attr[0].val.clusterDim.y = 1;
      attr[0].val.clusterDim.z = 1;
      cfg.attrs = attr;
      cfg.numAttrs = 1;
      si.err = cudaOccupancyMaxActiveClusters(&si.clusters[s], split_kernel<LORA, OWN>, &cfg);
    }
  }
  return si;
}

// The K-split that takes the least time: waves of clusters, each as long as its K-blocks and a
// set-up and reduction worth about SPLIT_COST of them; at least two K-blocks a CTA.
int best_split(const SplitInfo &si, int64_t tiles, int k_blocks) {
  int best = 1;
  int64_t least = INT64_MAX;
  for (int s = 1; s <= SPLIT_MAX && s <= std::max(1, k_blocks / 2); ++s) {
    if (si.clusters[s] < 1) continue;
    const int64_t waves = (tiles + si.clusters[s] - 1) / si.clusters[s];
    const int64_t cost = waves * ((k_blocks + s - 1) / s + SPLIT_COST);
    if (cost < least) {
      least = cost;
      best = s;
    }
  }
  return best;
}

template <bool LORA, bool OWN = false>
int launch_split(const char *op, const Maps &maps, Params &p, int tiles, const DeviceInfo &dev,
                 cudaStream_t stream) {
  SplitInfo &si = split_info<LORA, OWN>(dev);
  if (si.err != cudaSuccess) return launch_failed(op, si.err);
  const int best = best_split(si, tiles, p.k_blocks);
  p.kps = (p.k_blocks + best - 1) / best;
  p.split = (p.k_blocks + p.kps - 1) / p.kps;
  const uint32_t stage = W_STAGE + static_cast<uint32_t>(p.tok_cap) * BK;
  const uint32_t rows = static_cast<uint32_t>(((WROWS + p.split - 1) / p.split + 3) & ~3);
  const uint32_t part = static_cast<uint32_t>(p.split * p.tok_cap) * rows * 4;
  const int lora_tok = OWN ? kLoraOwnTokens : (p.tok_cap / 8 + p.split - 1) / p.split * 8;
  const uint32_t lora = LORA ? static_cast<uint32_t>(lora_tok) * WROWS * 4 : 0;
  const uint32_t tab = static_cast<uint32_t>(p.E + 1) * 8 + 16 + SPLIT_EPI;
  const uint32_t ring = OWN ? (1 + SPLIT_MAX) * OWN_WORK * 4u : LORA ? SUM_RING : 0u;
  const uint32_t room = SPLIT_SMEM - 2048 - ring - part - lora - tab;
  p.stages = std::max(1, std::min({static_cast<int>(room / stage), SPLIT_STAGES, p.kps}));
  p.off_ring = static_cast<uint32_t>(p.stages) * stage;
  p.off_part = p.off_ring + ring;
  p.off_lora = p.off_part + part;
  p.off_tab = p.off_lora + lora;
  const size_t smem = p.off_tab + tab + 1024;
  const cudaError_t e = launch(reinterpret_cast<const void *>(&split_kernel<LORA, OWN>), maps, p,
                               tiles * p.split, split_threads<LORA, OWN>(), p.split, smem, stream);
  return e == cudaSuccess ? 0 : launch_failed(op, e);
}

// `n` boxes of tokens: 16, 32, .. 16 n rows.
bool make_common_maps(Maps *m, int n, const uint8_t *xq, const uint8_t *wq, int64_t M, int64_t N,
                      int64_t K, int64_t E, std::string *err) {
  for (int i = 0; i < n; ++i)
    if (!make_tmap_2d_sw128(&m->x[i], CU_TENSOR_MAP_DATA_TYPE_UINT8, xq, K, M, K, BK, 16 * (i + 1),
                            err))
      return false;
  return make_tmap_3d_swizzled(&m->w, CU_TENSOR_MAP_DATA_TYPE_UINT8, wq, K, N, E, K, N * K, BK,
                               WROWS, 128, err);
}

}  // namespace rowsel

namespace {

bool check_device(const char *op, DeviceInfo *dev) {
  if (!current_device_info(dev)) return false;
  if (dev->cc_major == 10) return true;
  set_error(std::string(op) + " needs an sm_100 (B200-class) device; current device is sm_" +
            std::to_string(dev->cc_major) + std::to_string(dev->cc_minor));
  return false;
}

}  // namespace

int launch_grouped(const GroupedArgs &a, cudaStream_t stream) {
  using namespace rowsel;
  const char *op = "fp8_grouped_gemm";
  DeviceInfo dev;
  if (!check_device(op, &dev)) return 5;
  Params p = {};
  p.xs = a.xs;
  p.ws = a.ws;
  p.bias = a.bias;
  p.bias_dtype = a.bias ? a.bias_dtype : kNone;
  p.out = a.out;
  p.out_dtype = a.out_dtype;
  p.offsets = a.offsets;
  p.M = static_cast<int>(a.M);
  p.N = static_cast<int>(a.N);
  p.E = static_cast<int>(a.E);
  p.k_blocks = static_cast<int>((a.K + BK - 1) / BK);
  p.pre_w = a.weights_before_wait ? 1 : 0;
  // Tiles at most, whatever the offsets: every group with rows starts a token block of its own.
  const int64_t live = std::min(a.E, a.M);
  const int64_t wb1 = (a.N + WROWS - 1) / WROWS;
  const int64_t ub1 = wb1 * (live + a.M / SPLIT_TOK);
  if (ub1 > 0x3fffffffLL) {
    set_error(std::string(op) + ": too many output tiles");
    return 2;
  }
  // Few tiles: split K, where that gives every tile two CTAs at least (one alone is faster in
  // the persistent kernel: 512 rows of 4 experts, 2048 x 2048, 17.0 us against 9.4). CTA pairs
  // from 100 rows an expert on: 16 experts of 4096 x 4096 with 64 rows each take 48.3 us with
  // single CTAs and 48.7 with pairs, with 128 rows 55.1 and 52.8, with 256 rows 88.8 and 67.6.
  const SplitInfo &si = split_info<false>(dev);
  if (si.err != cudaSuccess) return launch_failed(op, si.err);
  const bool split = ub1 <= dev.sm_count && best_split(si, ub1, p.k_blocks) > 1;
  const bool pairs = !split && a.M / live >= 100;
  p.tok_cap = split ? static_cast<int>(std::min<int64_t>((a.M + 15) / 16 * 16, SPLIT_TOK)) : 128;
  std::string err;
  Maps maps = {};
  if (!make_common_maps(&maps, p.tok_cap / 16, a.xq, a.wq, a.M, a.N, a.K, a.E, &err)) {
    set_error(std::string(op) + ": " + err);
    return 4;
  }
  p.n_wb = static_cast<int>(wb1);
  if (split) return launch_split<false>(op, maps, p, static_cast<int>(ub1), dev, stream);
  if (!pairs) return launch_persist<1, false>(op, maps, p, ub1, dev, stream);
  const int64_t wb2 = (a.N + 2 * WROWS - 1) / (2 * WROWS);
  p.n_wb = static_cast<int>(wb2);
  return launch_persist<2, false>(op, maps, p, wb2 * (live + a.M / 256), dev, stream);
}

bool lora_own_down(int64_t M, int64_t N, int64_t K, int64_t R) {
  using namespace rowsel;
  DeviceInfo dev;
  if (M > kLoraOwnTokens || !current_device_info(&dev)) return false;
  const SplitInfo &si = split_info<true, true>(dev);
  if (si.err != cudaSuccess) return false;
  const int k_blocks = static_cast<int>((K + BK - 1) / BK);
  const int split = best_split(si, (N + WROWS - 1) / WROWS, k_blocks);
  return M * R * ((k_blocks + split - 1) / split) <= OWN_WORK;
}

int launch_lora_gemm(const LoraArgs &a, cudaStream_t stream) {
  using namespace rowsel;
  const char *op = "fp8_linear_lora";
  DeviceInfo dev;
  if (!check_device(op, &dev)) return 5;
  const LoraWorkspace w = lora_workspace(a.workspace, a.M, a.R);
  const int64_t rp = lora_rank_pad(a.R);
  const bool few = a.M <= kLoraRowsMaxM;
  Params p = {};
  p.xs = a.xs;
  p.ws = a.ws;
  p.bias = a.bias;
  p.bias_dtype = a.bias ? a.bias_dtype : kNone;
  p.out = a.out;
  p.out_dtype = a.out_dtype;
  p.M = static_cast<int>(a.M);
  p.N = static_cast<int>(a.N);
  p.E = 1;
  p.k_blocks = static_cast<int>((a.K + BK - 1) / BK);
  p.ids = a.ids;
  p.lora_b = a.lora_b;
  p.lora_dtype = a.dtype;
  p.L = static_cast<int>(a.L);
  p.R = static_cast<int>(a.R);
  p.rank_pad = static_cast<int>(rp);
  p.x = a.x;
  p.lora_a = a.lora_a;
  p.scaling = a.scaling;
  p.K = static_cast<int>(a.K);
  p.plan = w.plan;
  p.plan_mixed = static_cast<int>(lora_plan_mixed(a.M));
  p.hl = w.hl;
  p.hscale = w.hscale;
  const int rows = few ? WROWS : 2 * WROWS;
  const int64_t wb = (a.N + rows - 1) / rows;
  // the plan's tiles at most (and every product within int32)
  const int64_t tiles =
      wb * (few ? 1 : lora_plan_max(a.M));
  if (tiles > 0x3fffffffLL) {
    set_error(std::string(op) + ": too many output tiles");
    return 2;
  }
  p.n_wb = static_cast<int>(wb);
  p.tok_cap = few ? static_cast<int>((a.M + 15) / 16 * 16) : kLoraTileTokens;
  std::string err;
  Maps maps = {};
  const CUtensorMapDataType t16 = a.dtype == kF16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16
                                                  : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
  bool ok = make_common_maps(&maps, few ? p.tok_cap / 16 : H_MAPS, a.xq, a.wq, a.M, a.N, a.K, 1,
                             &err);
  if (few) {
    const int sw = sum_width(static_cast<int>(a.R));
    ok = ok && make_tmap_3d_swizzled(&maps.lb, t16, a.lora_b, a.R, a.N, a.L, a.R * 2, a.N * a.R * 2,
                                     static_cast<uint32_t>(sw), WROWS, sw * 2, &err);
  } else {
    ok = ok && make_tmap_3d_swizzled(&maps.lb, t16, a.lora_b, a.R, a.N, a.L, a.R * 2, a.N * a.R * 2,
                                     64, WROWS, 128, &err);
    for (int i = 0; ok && i < H_MAPS; ++i)
      ok = make_tmap_2d_sw128(&maps.h[i], t16, w.hl, 2 * rp, a.M, 4 * rp, 64, 16 * (i + 1), &err);
  }
  if (!ok) {
    set_error(std::string(op) + ": " + err);
    return 4;
  }
  if (lora_own_down(a.M, a.N, a.K, a.R))
    return launch_split<true, true>(op, maps, p, static_cast<int>(tiles), dev, stream);
  if (few) return launch_split<true>(op, maps, p, static_cast<int>(tiles), dev, stream);
  return launch_persist<2, true>(op, maps, p, tiles, dev, stream);
}

cudaError_t read_rowsel_status(unsigned int *bits, bool clear) {
  cudaError_t e = cudaMemcpyFromSymbol(bits, g_rowsel_status, sizeof(unsigned int));
  if (e != cudaSuccess) return e;
  if (clear) {
    const unsigned int zero = 0;
    e = cudaMemcpyToSymbol(g_rowsel_status, &zero, sizeof(unsigned int));
  }
  return e;
}

}  // namespace fp8lin
