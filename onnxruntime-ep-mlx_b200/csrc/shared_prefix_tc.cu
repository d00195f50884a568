// shared_prefix_tc_kernel: the tensor-core (tcgen05) pass of b200_shared_prefix_attention.
//
// Work items:
//   * prefix: (key range, kv head, pair of query tiles): every packed token of the batch against one
//     range of the shared prefix, without masks.  All tokens and the g query heads of a kv head are
//     rows of one matrix, so a K/V tile loaded once serves 2 x 128 rows whatever sequences they
//     belong to;
//   * chunk: (sequence, kv head, pair of query tiles) of a long chunk against its own keys, causal.
// Bound by the tensor pipe and the exponentials (4 d flops per row and key); K/V tiles come from L2
// when more than one pair of query tiles reads a range.  Measured alone, bf16, d 128: 256 tokens of 64 / 8
// heads over 16384 keys 162 us (0.85 PFLOP/s, 0.50 of a library matrix product's rate, tensor pipe active 51 %
// of the time); 128 tokens of 32 / 8 heads over 8192 keys 40 us.  The rest is the chain S, softmax, P V of
// a query tile.
//
// A query tile is 128 rows = tile_tokens tokens x g heads.  Roles, joined by mbarriers only:
//   warps 0-3 / 4-7  softmax and epilogue of query tile 0 / 1, one row per thread = tensor-memory lane
//   warp 8           loads Q and K tiles by TMA (8 pages of 16 slots per 128-key tile)
//   warp 9           issues the MMAs: per K/V tile j PV0(j-1), S0(j), PV1(j-1), S1(j), so the tensor
//                    pipe works on one query tile while the other one's softmax runs
//   warp 10          loads V tiles
//   warp 11          takes items and works out what they are, up to two ahead of the others; lets the
//                    own kernel start when the plan is done
// S = Q K^T (both operands in shared memory), O += P V with P in tensor memory over S's columns and V as
// the MN-major operand in the cache's [key][channel] order.  P is one fp16 value per key against fp16
// values (fp16 calls, or bf16 calls on the plan's fp16 copy of the prefix's values) and a hi + lo pair
// of bf16 values against bf16 ones, since one bf16 P costs up to 3e-3 on unit-scale values.  The running
// maximum moves, and O is rescaled, only when it grows by more than 2^8.  Tensor memory: S/P 0 and 1 at
// columns 0 and 128, O 0 and 1 at 256 and 384.  Each item leaves its rows' (m, l, o) in a slab.
// Every wait is bounded; one that runs out sets the status word, the roles drain what they issued,
// tensor memory is freed and the kernel returns.
#include <atomic>
#include <type_traits>

#include "b200_kernels.h"
#include "b200_tcgen05.cuh"
#include "shared_prefix.cuh"

namespace b200 {
namespace {

constexpr int kBM = 128;            // query rows per tile
constexpr int kBN = kPrefixKeys;    // keys per tile
constexpr int kPage = 16;           // slots per TMA box
constexpr int kBoxBytes = 128 * 128;  // [128 rows][64 channels]
constexpr float kLog2e = 1.4426950408889634f;
constexpr int kPolyEvery = 8;       // of so many exponential pairs one is on the FMA pipe (4 or 16: +-1 %)
// Head size 64: O takes half of its 128 columns, single P the other half (columns from S to P).
constexpr uint32_t kPBeside = 256 + 64;

// Two shapes of the kernel.  BESIDE: 160 KB of shared memory and 128 registers per thread at launch (its
// launch bound of 512 threads sets that), so a CTA of the own kernel fits on the SM beside it; for head
// size 128 that leaves one K stage, whose next tile arrives about 900 cycles late.  Otherwise (head size
// 128 only) the SM is this kernel's alone.
template <int D, bool BESIDE>
struct TcLayout {
  static constexpr int kBoxes = D / 64;
  static constexpr int kTile = kBoxes * kBoxBytes;
  static constexpr int kQBuffers = D == 64 ? 2 : 1;  // per query tile
  static constexpr int kKStages = D == 64 ? 3 : BESIDE ? 1 : 2;
  static constexpr int kVStages = D == 64 ? 3 : BESIDE ? 2 : 3;
  static constexpr int kSmemQ = 0;
  static constexpr int kSmemK = 2 * kQBuffers * kTile;
  static constexpr int kSmemV = kSmemK + kKStages * kTile;
  static constexpr int kSmem = kSmemV + kVStages * kTile;
  // setmaxnreg split of the registers per thread at launch
  static constexpr int kBoundThreads = BESIDE ? 512 : 384;
  static constexpr int kLaunchRegs = BESIDE ? 128 : 168;
  static constexpr int kSoftmaxRegs = BESIDE ? 152 : 200, kControlRegs = BESIDE ? 80 : 96;
  static constexpr int kSplitRegs = 2 * 128 * kSoftmaxRegs + 128 * kControlRegs;
  static_assert(kSplitRegs <= 384 * kLaunchRegs, "the register split exceeds the launch allocation");
};

constexpr int kWg = 128;
constexpr int kThreads = 3 * kWg;
constexpr int kLoadWarp = 8, kMmaWarp = 9, kVLoadWarp = 10;  // warp 11: scheduler
constexpr int kSched = 2;  // slots of the item queue
constexpr int kTakers = 2 * kWg / 32 + 3;  // softmax, load, MMA and V load warps

// The whole warp waits for a phase, at most kWaitLimitNs, and not once another role has given up.  The
// roles' code together has to stay in the SM's instruction cache (a role that runs code the others
// have evicted pays hundreds of cycles a line), so the loop stays rolled and is a call where a role has
// the registers for one.
__device__ __forceinline__ bool wait_inline(uint64_t* bar, uint32_t parity, volatile int* failed, int* status) {
  if (__all_sync(0xffffffffu, mbar_try_wait(bar, parity))) return true;
  const uint64_t start = globaltimer_ns();
#pragma unroll 1
  while (!__all_sync(0xffffffffu, mbar_try_wait(bar, parity))) {
    if (__any_sync(0xffffffffu, globaltimer_ns() - start > kWaitLimitNs || *failed != 0)) {
      if (*failed == 0) set_status(status, kStatusTimeout);
      *failed = 1;
      return false;
    }
  }
  return true;
}
__device__ __noinline__ bool wait_call(uint64_t* bar, uint32_t parity, volatile int* failed, int* status) {
  return wait_inline(bar, parity, failed, status);
}
// After a failure, too: a bounded wait for a copy or commit this CTA issued.
__device__ __forceinline__ void wait_drain(uint64_t* bar, uint32_t parity) {
  const uint64_t start = globaltimer_ns();
#pragma unroll 1
  while (!mbar_try_wait(bar, parity))
    if (globaltimer_ns() - start > kWaitLimitNs) return;
}

struct Bars {
  uint64_t q_full[2][2], q_empty[2][2];
  uint64_t k_full[3], k_empty[3], v_full[3], v_empty[3];
  uint64_t s_full[2], p_full[2], o_done[2], pv_done[2];
  uint64_t drain, plan;
  uint64_t sched_full[kSched], sched_empty[kSched];
};

struct Item {
  int stop;                      // no more items
  int chunk, kh, tok0, tok_end;  // tokens [tok0, tok_end) are the sequence's (prefix: the batch's) from the first tile on
  int qpos0;                     // chunk: own position of token tok0
  int k_lo, k_valid;             // first key; keys of the table that hold data
  int k_end;                     // prefix: end of the key range
  int n0, n1, n;                 // K/V tiles of query tile 0, 1, and their maximum
  const int32_t* table;
  int slab;
};

// Item `it` of the list (below 2^31, which the host checked): prefix items ((range, kv head), pair), whose
// neighbours share their K/V tiles in L2, then chunk items.  The whole warp.
__device__ __forceinline__ Item decode_item(const SharedPrefixArgs& a, uint32_t it, uint32_t prefix_items, int lane) {
  Item m{};
  const uint32_t KV = a.p.kv_num_heads;
  const int TQ = a.tile_tokens;
  if (it < prefix_items) {
    const uint32_t r = it / (uint32_t)a.query_pairs, pair = it - r * a.query_pairs;
    const uint32_t range = r / KV;
    m.kh = (int)(r - range * KV);
    m.slab = range;
    m.tok0 = (int)pair * 2 * TQ;
    m.tok_end = a.p.num_tokens;
    m.k_lo = (int)range * a.split_tiles * kBN;
    m.k_valid = a.p.prefix_length;
    m.k_end = min(m.k_valid, m.k_lo + a.split_tiles * kBN);
    m.n0 = (m.k_end - m.k_lo + kBN - 1) / kBN;
    m.n1 = m.tok0 + TQ < m.tok_end ? m.n0 : 0;
    m.n = m.n0;
    m.table = a.p.prefix_block_table;
    return m;
  }
  it -= prefix_items;
  const int pairs = __ldcg(a.seq_pairs + a.p.batch);
  const int nth = (int)(it / KV);
  const int pair_global = pairs - 1 - nth;  // later tiles, which see more keys, first
  m.chunk = 1;
  m.kh = (int)(it - nth * KV);
  int lo = 0, hi = a.p.batch;  // the largest lo with seq_pairs[lo] <= pair_global, 32 candidates at a time
  while (hi - lo > 1) {
    const int step = (hi - lo + 31) / 32, at = lo + lane * step;
    const unsigned le = __ballot_sync(0xffffffffu, at < hi && __ldcg(a.seq_pairs + min(at, a.p.batch)) <= pair_global);
    lo += (__popc(le) - 1) * step;
    hi = min(hi, lo + step);
  }
  const int q0 = (int)(pair_global - __ldcg(a.seq_pairs + lo)) * 2 * TQ;
  const int c0 = a.p.cumulative_sequence_length[lo], c1 = a.p.cumulative_sequence_length[lo + 1];
  const int past = a.p.past_seqlens[lo];
  m.tok0 = c0 + q0;
  m.tok_end = c1;
  m.qpos0 = past + q0;
  m.k_valid = past + c1 - c0;
  m.k_end = m.k_valid;
  const int t1 = c1 - m.tok0;  // tokens from this pair on
  m.n0 = (m.qpos0 + min(TQ, t1) + kBN - 1) / kBN;
  m.n1 = t1 > TQ ? (m.qpos0 + min(2 * TQ, t1) + kBN - 1) / kBN : 0;
  m.n = max(m.n0, m.n1);
  m.table = a.p.block_table + (int64_t)lo * a.p.max_blocks_per_seq;
  m.slab = a.splits;
  return m;
}

__device__ __forceinline__ int tiles_of(const Item& m, int w) { return w ? m.n1 : m.n0; }

// Page `page` of a V stage by plain loads: rows [0, rows) from block `blk` (position pos0 on), zeros
// below, in the TMA's swizzle; then ordered before the tensor core's reads.
template <int D>
__device__ __noinline__ void fill_tail_page(uint8_t* stage, const B200SharedPrefixParams& p, int32_t blk, int pos0, int kh,
                                            int page, int rows, int lane) {
  const bool ok = blk >= 0 && blk < p.num_blocks;
  const int64_t slot0 = (int64_t)blk * p.block_size + pos0 % p.block_size;
  for (int i = lane; i < kPage * (D / 8); i += 32) {
    const int r = i / (D / 8), box = (i % (D / 8)) >> 3, piece = i & 7;
    uint4 v = make_uint4(0, 0, 0, 0);
    if (r < rows && ok)
      v = *reinterpret_cast<const uint4*>(static_cast<const uint8_t*>(p.value_cache) +
                                          (((slot0 + r) * p.kv_num_heads + kh) * D + box * 64) * 2 + piece * 16);
    const int row = page * kPage + r;
    *reinterpret_cast<uint4*>(stage + box * kBoxBytes + row * 128 + ((piece ^ (row & 7)) * 16)) = v;
  }
  fence_proxy_async_smem();
  __syncwarp();
}

// Maxima that keep a NaN: a row whose scores hold one has to end as NaN, and the exponential on the FMA pipe
// alone would drop it.
__device__ __forceinline__ float max3_nan(float a, float b, float c) {
  float d;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
__device__ __forceinline__ float min_nan(float a, float b) {
  float d;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
  return d;
}

// x -> top * tanh(x * to_u), 32 values of a thread; the whole warp.  tanh(u) = u f(u^2) with f a polynomial of
// degree 6, minimax in relative error over |u| <= 1 (fitted with Lawson's algorithm on 4001
// Chebyshev-spaced points, 2000 passes; fp32 evaluation within 1.7e-7): 10 packed instructions for two
// values, where 1 - 2 / (1 + e^(2u)), which takes warps with a larger u, needs two MUFU operations a value.
__device__ __forceinline__ void soft_cap(float (&x)[32], float to_u, float top) {
  float big = 0.f;
#pragma unroll
  for (int i = 0; i < 32; ++i) big = fmaxf(big, fabsf(x[i]));
  if (__all_sync(0xffffffffu, big * fabsf(to_u) <= 1.f)) {
    const float coef[7] = {0.99999994f, -0.333328396f, 0.13325204f, -0.0534570292f, 0.0202899799f, -0.00620337902f, 0.0010410226f};
    const float2 zero = make_float2(0.f, 0.f), scale = make_float2(to_u, to_u), cap = make_float2(top, top);
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const float2 u = tc::fma2(make_float2(x[2 * i], x[2 * i + 1]), scale, zero), t = tc::fma2(u, u, zero);
      float2 f = make_float2(coef[6], coef[6]);
#pragma unroll
      for (int k = 5; k >= 0; --k) f = tc::fma2(f, t, make_float2(coef[k], coef[k]));
      const float2 y = tc::fma2(tc::fma2(u, f, zero), cap, zero);
      x[2 * i] = y.x;
      x[2 * i + 1] = y.y;
    }
  } else {
    const float to_e = 2.f * kLog2e * to_u;
#pragma unroll
    for (int i = 0; i < 32; ++i) {
      const float e = tc::ex2(min_nan(x[i] * to_e, 126.f));
      x[i] = top * (1.f - __fdividef(2.f, 1.f + e));
    }
  }
}

template <typename T, int D, bool BESIDE>
__global__ void __launch_bounds__((TcLayout<D, BESIDE>::kBoundThreads), 1) shared_prefix_tc_kernel(const __grid_constant__ SharedPrefixArgs a,
                                                                        const __grid_constant__ SharedPrefixMaps maps) {
  using L = TcLayout<D, BESIDE>;
  using MMA = mma_op<T>;
  constexpr bool kBF16 = std::is_same<T, __nv_bfloat16>::value;
  constexpr uint32_t kIdQK = tc::idesc_f16(kBM, kBN, kBF16, false, false);
  constexpr uint32_t kIdPV = tc::idesc_f16(kBM, D, kBF16, false, true), kIdPV16 = tc::idesc_f16(kBM, D, false, false, true);
  constexpr int kKStages = L::kKStages, kVStages = L::kVStages;

  extern __shared__ __align__(1024) uint8_t smem[];
  __shared__ __align__(8) Bars bars;
  __shared__ uint32_t tmem_slot;
  __shared__ volatile int s_failed;
  __shared__ volatile uint64_t s_inexact;  // kv heads (bit: head % 64) whose prefix values the fp16 copy does not hold
  __shared__ Item s_items[kSched];

  const B200SharedPrefixParams& p = a.p;
  const uint32_t sbase = smem_u32(smem);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int g = a.group, H = p.num_heads, TQ = a.tile_tokens;

  if (warp == kMmaWarp) tc::alloc(&tmem_slot, 512);
  if (tid == 0) {
    for (int w = 0; w < 2; ++w) {
      for (int i = 0; i < 2; ++i) {
        mbar_init(&bars.q_full[w][i], 1);
        mbar_init(&bars.q_empty[w][i], 1);
      }
      mbar_init(&bars.s_full[w], 1);
      mbar_init(&bars.p_full[w], kWg);
      mbar_init(&bars.o_done[w], 1);
      mbar_init(&bars.pv_done[w], 1);
    }
    for (int i = 0; i < 3; ++i) {
      mbar_init(&bars.k_full[i], 1);
      mbar_init(&bars.k_empty[i], 1);
      mbar_init(&bars.v_full[i], 1);
      mbar_init(&bars.v_empty[i], 1);
    }
    mbar_init(&bars.drain, 1);
    mbar_init(&bars.plan, 1);
    for (int i = 0; i < kSched; ++i) {
      mbar_init(&bars.sched_full[i], 1);
      mbar_init(&bars.sched_empty[i], kTakers);
    }
    fence_mbar_init();
    s_failed = 0;
  }
  tc::fence_before_sync();
  __syncthreads();
  tc::fence_after_sync();
  const uint32_t tmem = tmem_slot;

  // Completion `index` of a barrier, for the whole warp.
  auto wait_softmax = [&](uint64_t* bar, uint32_t index) -> bool {
    return wait_inline(bar, index & 1u, &s_failed, p.device_status);
  };
  auto wait_warp = [&](uint64_t* bar, uint32_t index) -> bool {  // control warps
    return __all_sync(0xffffffffu, mbar_try_wait(bar, index & 1u)) || wait_call(bar, index & 1u, &s_failed, p.device_status);
  };
  auto failed_warp = [&]() -> bool { return __any_sync(0xffffffffu, s_failed != 0); };
  auto drain_idx = [&](uint64_t* bar, uint32_t index) { wait_drain(bar, index & 1u); };
  // The CTA's k-th item, from warp 11.
  auto take_item = [&](uint32_t k, Item& m, auto wait) -> bool {
    const uint32_t slot = k % kSched;
    if (!wait(&bars.sched_full[slot], k / kSched)) return false;
    m = s_items[slot];
    __syncwarp();
    if (lane == 0) mbar_arrive(&bars.sched_empty[slot]);
    return !m.stop;
  };
  // Whether an item's values come from the fp16 copy; waits for the plan (which decides it) at the first
  // prefix item of a call that made the copy.
  bool plan_seen = false;
  auto takes_copy = [&](const Item& m, bool& copy, auto wait) -> bool {
    copy = false;
    if (!a.v_copy || m.chunk) return true;
    if (!plan_seen && !wait(&bars.plan, 0)) return false;
    plan_seen = true;
    copy = !(s_inexact >> (m.kh & 63) & 1);
    return true;
  };

  if (warp >= 2 * (kWg / 32)) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(L::kControlRegs));
    if (warp == kLoadWarp || warp == kVLoadWarp) {
      // ---------------------------------------------------------------- TMA producers
      const bool is_v = warp == kVLoadWarp;
      const uint32_t stages = is_v ? kVStages : kKStages;
      uint64_t* full_bar = is_v ? bars.v_full : bars.k_full;
      uint64_t* empty_bar = is_v ? bars.v_empty : bars.k_empty;
      const CUtensorMap* map = is_v ? &maps.v_map : &maps.k_map;
      const uint32_t ring = is_v ? L::kSmemV : L::kSmemK;
      const uint32_t q_bytes = (uint32_t)(g * TQ * 128 * L::kBoxes);
      uint32_t qc0 = 0, qc1 = 0, c = 0;
      const int oob_z = p.num_blocks * p.block_size;  // past the cache: zero fill
      const int page = (lane % (8 * L::kBoxes)) / L::kBoxes, half = lane % L::kBoxes;
      const bool loader = lane < 8 * L::kBoxes;
      bool ok = true;
      for (uint32_t k = 0; ok && !failed_warp(); ++k) {
        Item m;
        if (!take_item(k, m, wait_warp)) break;
        bool copied = false;
        if (is_v && !(ok = takes_copy(m, copied, wait_warp))) break;
        if (!is_v) {
          for (int w = 0; w < 2 && ok; ++w) {
            if (tiles_of(m, w) == 0) continue;
            const uint32_t qc = w ? qc1 : qc0;
            const uint32_t qb = qc % L::kQBuffers, use = qc / L::kQBuffers;
            if (use > 0 && !(ok = wait_warp(&bars.q_empty[w][qb], use - 1))) break;
            if (lane == 0) mbar_arrive_expect_tx(&bars.q_full[w][qb], q_bytes);
            __syncwarp();
            if (lane < L::kBoxes)
              tma_load_3d(smem + L::kSmemQ + (w * L::kQBuffers + qb) * L::kTile + lane * kBoxBytes, &maps.q_map,
                          &bars.q_full[w][qb], lane * 64, m.kh * g, m.tok0 + w * TQ);
            if (w) qc1 = qc + 1; else qc0 = qc + 1;
          }
        }
        auto block_of = [&](int j) -> int32_t {
          const int pos = m.k_lo + j * kBN + page * kPage;
          return loader && pos < m.k_valid ? __ldg(m.table + pos / p.block_size) : -1;
        };
        if (copied) {  // contiguous rows; TMA fills zeros past the last key
          for (int j = 0; j < m.n && ok; ++j, ++c) {
            const uint32_t st = c % stages;
            if (c >= stages && !(ok = wait_warp(&empty_bar[st], c / stages - 1))) break;
            if (lane == 0) mbar_arrive_expect_tx(&full_bar[st], L::kTile);
            __syncwarp();
            if (lane < L::kBoxes)
              tma_load_3d(smem + ring + st * L::kTile + lane * kBoxBytes, &maps.vc_map, &full_bar[st], lane * 64, m.kh,
                          m.k_lo + j * kBN);
          }
          continue;
        }
        int32_t blk_next = block_of(0);
        for (int j = 0; j < m.n && ok; ++j) {
          const int pos0 = m.k_lo + j * kBN + page * kPage;
          const int32_t blk = blk_next;
          if (j + 1 < m.n) blk_next = block_of(j + 1);  // in flight during the stage wait below
          const bool blk_ok = blk >= 0 && blk < p.num_blocks;
          if (!is_v && loader && pos0 < m.k_valid && !blk_ok) set_status(p.device_status, kStatusBadBlock);
          const int z = blk_ok ? blk * p.block_size + pos0 % p.block_size : oob_z;
          const uint32_t st = c % stages;
          if (c >= stages && !(ok = wait_warp(&empty_bar[st], c / stages - 1))) break;
          // The V page that reaches past the last key: its rows by plain loads, its unused slots zeroed
          // (whatever they hold, NaN included, must not meet P = 0 in the MMA).
          const int valid = min(kBN, m.k_valid - (m.k_lo + j * kBN));
          const int rows = is_v ? valid & (kPage - 1) : 0;
          const int tail_page = valid >> 4;
          if (rows) {
            const int32_t tblk = __shfl_sync(0xffffffffu, blk, L::kBoxes * tail_page);
            const int tpos = __shfl_sync(0xffffffffu, pos0, L::kBoxes * tail_page);
            fill_tail_page<D>(smem + ring + st * L::kTile, p, tblk, tpos, m.kh, tail_page, rows, lane);
          }
          if (lane == 0) mbar_arrive_expect_tx(&full_bar[st], rows ? L::kTile - kPage * 128 * L::kBoxes : L::kTile);
          __syncwarp();
          if (loader && !(rows && page == tail_page))
            tma_load_3d(smem + ring + st * L::kTile + half * kBoxBytes + page * (kPage * 128), map, &full_bar[st],
                        half * 64, m.kh, z);
          ++c;
        }
      }
      for (uint32_t w = 0; w < 2; ++w) {
        const uint32_t qc = w ? qc1 : qc0;
        for (uint32_t i = (qc > L::kQBuffers ? qc - L::kQBuffers : 0); i < qc; ++i)
          drain_idx(&bars.q_full[w][i % L::kQBuffers], i / L::kQBuffers);
      }
      for (uint32_t i = (c > stages ? c - stages : 0); i < c; ++i) drain_idx(&full_bar[i % stages], i / stages);
    } else if (warp == kMmaWarp) {
      // ---------------------------------------------------------------- MMA issuer
      // Its path between two MMAs is what the tensor pipe waits for: one branch around each group of
      // MMAs, descriptors advanced by constants.
      const bool leader = tc::elect_one();
      const uint64_t qdesc = tc::smem_desc(sbase + L::kSmemQ, 16, 1024);
      const uint64_t kdesc = tc::smem_desc(sbase + L::kSmemK, 16, 1024);
      const uint64_t vdesc = tc::smem_desc(sbase + L::kSmemV, kBoxBytes, 1024);
      uint32_t qc0 = 0, qc1 = 0, pc0 = 0, pc1 = 0, kvc = 0;
      bool issued = false, ok = true;
      for (uint32_t k = 0; ok && !failed_warp(); ++k) {
        Item m;
        if (!take_item(k, m, wait_warp)) break;
        bool copied;
        if (!(ok = takes_copy(m, copied, wait_warp))) break;
        const bool pair = kBF16 && !copied;  // P as a hi + lo pair
        const uint32_t id_pv = kBF16 && copied ? kIdPV16 : kIdPV;
#pragma unroll 1
        for (int j = 0; j <= m.n && ok; ++j) {
          const uint32_t ki = kvc + j, vi = ki - 1;
          const uint64_t kd = kdesc + (uint64_t)(ki % kKStages) * (L::kTile >> 4);
          const uint64_t vd = vdesc + (uint64_t)(vi % kVStages) * (L::kTile >> 4);
          bool k_ready = false, v_ready = false;
#pragma unroll 1
          for (int w = 0; w < 2; ++w) {
            const uint32_t pc = w ? pc1 : pc0, qc = w ? qc1 : qc0;
            const int nw = w ? m.n1 : m.n0;
            const bool has_pv = j > 0 && j - 1 < nw, has_s = j < nw;
            auto issue_pv = [&]() -> bool {  // O_w (+)= P_w(j-1) V_(j-1)
              if (!v_ready && !wait_warp(&bars.v_full[vi % kVStages], vi / kVStages)) return false;
              v_ready = true;
              const uint32_t obuf = tmem + 256 + w * 128, add = j > 1;
              if (leader) {
                if (pair) {
                  const uint32_t pbuf = tmem + w * 128;
#pragma unroll
                  for (int kk = 0; kk < kBN / 16; ++kk) {
                    const uint32_t pcol = pbuf + (kk >> 1) * 32 + (kk & 1) * 8;
                    tc::mma_ts(obuf, pcol, vd + (uint64_t)(kk * (2048 >> 4)), kIdPV, kk > 0 ? 1u : add);
                    tc::mma_ts(obuf, pcol + 16, vd + (uint64_t)(kk * (2048 >> 4)), kIdPV, 1u);
                  }
                } else {
                  const uint32_t pbuf = tmem + (D == 64 ? kPBeside : 0) + w * 128;
#pragma unroll
                  for (int kk = 0; kk < kBN / 16; ++kk)
                    tc::mma_ts(obuf, pbuf + (D == 64 ? kk * 8 : (kk >> 1) * 32 + (kk & 1) * 8), vd + (uint64_t)(kk * (2048 >> 4)),
                               id_pv, kk > 0 ? 1u : add);
                }
                tc::commit(&bars.pv_done[w]);
                if (j == nw) tc::commit(&bars.o_done[w]);
              }
              __syncwarp();
              if (w) ++pc1; else ++pc0;
              return true;
            };
            auto issue_s = [&]() -> bool {  // S_w(j) = Q_w K_j^T
              if (!k_ready && !wait_warp(&bars.k_full[ki % kKStages], ki / kKStages)) return false;
              k_ready = true;
              const uint32_t qb = qc % L::kQBuffers;
              if (j == 0 && !wait_warp(&bars.q_full[w][qb], qc / L::kQBuffers)) return false;
              if (leader) {
#pragma unroll
                for (int kk = 0; kk < D / 16; ++kk) {
                  const uint64_t off = (uint64_t)(((kk >> 2) * kBoxBytes + (kk & 3) * 32) >> 4);
                  tc::mma_ss(tmem + w * 128, qdesc + (uint64_t)((w * L::kQBuffers + qb) * (L::kTile >> 4)) + off, kd + off, kIdQK, kk > 0);
                }
                tc::commit(&bars.s_full[w]);
                if (j == nw - 1) tc::commit(&bars.q_empty[w][qb]);
              }
              __syncwarp();
              if (j == nw - 1) {
                if (w) ++qc1; else ++qc0;
              }
              issued = true;
              return true;
            };
            if (has_pv) {
              if (!(ok = wait_warp(&bars.p_full[w], pc))) break;
              tc::fence_after_sync();
            }
            if (D == 64 && !pair) {  // P lies beside S: the next scores do not wait for P V
              if (has_s && !(ok = issue_s())) break;
              if (has_pv && !(ok = issue_pv())) break;
            } else {
              if (has_pv && !(ok = issue_pv())) break;
              if (has_s && !(ok = issue_s())) break;
            }
          }
          if (!ok) break;
          if (leader && j > 0) tc::commit(&bars.v_empty[vi % kVStages]);
          if (leader && k_ready) tc::commit(&bars.k_empty[ki % kKStages]);
        }
        kvc += m.n;
      }
      if (issued) {
        if (leader) tc::commit(&bars.drain);
        drain_idx(&bars.drain, 0);
      }
      __syncwarp();
    } else {
      // ---------------------------------------------------------------- scheduler
      // The first item is the CTA's own and, if it lies in the prefix, needs nothing of the plan, which
      // may still be running then.
      const uint32_t prefix_items = (uint32_t)a.splits * p.kv_num_heads * a.query_pairs;
      bool planned = false;
      uint32_t items = 0;
      for (uint32_t k = 0; !failed_warp(); ++k) {
        const uint32_t slot = k % kSched;
        if (k >= (uint32_t)kSched && !wait_warp(&bars.sched_empty[slot], k / kSched - 1)) break;
        uint32_t it = blockIdx.x;
        if (!planned && (k > 0 || it >= prefix_items)) {
          planned = true;
          // The own kernel needs the plan, not this kernel's results: let it start once the plan is done.
          wait_previous();
          release_dependents();
          items = prefix_items + (uint32_t)__ldcg(a.seq_pairs + p.batch) * p.kv_num_heads;
          if (a.v_copy) {
            uint64_t heads = 0;
            for (int i = lane; i < a.copy_ctas; i += 32) heads |= __ldcg(reinterpret_cast<const unsigned long long*>(a.v_inexact) + i);
            const uint32_t low = __reduce_or_sync(0xffffffffu, (uint32_t)heads), high = __reduce_or_sync(0xffffffffu, (uint32_t)(heads >> 32));
            if (lane == 0) {
              s_inexact = (uint64_t)high << 32 | low;
              mbar_arrive(&bars.plan);
            }
          }
        }
        if (k > 0) {
          uint32_t next = 0;
          if (lane == 0) next = atomicAdd(a.next_item, 1u);
          it = gridDim.x + __shfl_sync(0xffffffffu, next, 0);
        }
        const bool stop = planned && it >= items;
        Item m{};
        if (!stop) m = decode_item(a, it, prefix_items, lane);
        m.stop = stop;
        if (lane == 0) {
          s_items[slot] = m;
          mbar_arrive(&bars.sched_full[slot]);
        }
        __syncwarp();
        if (stop) break;
      }
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(L::kSoftmaxRegs));
    // ------------------------------------------------------------------ softmax + epilogue
    const int w = warp >> 2, row = tid & (kWg - 1);
    const uint32_t lane_off = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t sbuf = tmem + w * 128 + lane_off, obuf = tmem + 256 + w * 128 + lane_off;
    const float qk_scale = p.softcap > 0.f ? p.scale : p.scale * kLog2e;
    const int tl = row / g, hl = row % g;
    uint32_t t = 0, items = 0;
    for (uint32_t k = 0; !failed_warp(); ++k) {
      Item m;
      if (!take_item(k, m, wait_softmax)) break;
      const int nw = tiles_of(m, w);
      if (nw == 0) continue;
      const int tok = m.tok0 + w * TQ + tl;
      const bool row_ok = tl < TQ && tok < m.tok_end;
      // last key the row sees; rows without a token see everything (their results are dropped)
      const int last = m.chunk && row_ok ? m.qpos0 + w * TQ + tl : m.k_end - 1;
      float m_run = -INFINITY, l_run = 0.f;
      bool copied;
      bool ok = takes_copy(m, copied, wait_softmax);
      if (!ok) break;
      for (int j = 0; j < nw; ++j, ++t) {
        if (!(ok = wait_softmax(&bars.s_full[w], t))) break;
        tc::fence_after_sync();
        const int kbase = m.k_lo + j * kBN;
        // Unmasked tiles keep raw scores, the scale goes into the exponent's FMA; others are rewritten
        // in place as scaled log2 values.  Warp-uniform.
        const bool raw = __all_sync(0xffffffffu, kbase + kBN - 1 <= last) && p.softcap <= 0.f && qk_scale > 0.f;
        // P per 32-column chunk: bf16 pairs over the chunk's S (hi halves, then lo halves), single fp16
        // values over the chunk's first 16 columns or, for head size 64, beside S where O leaves room.
        const bool single = !kBF16 || copied;
        const uint32_t pbuf = D == 64 && single ? sbuf + kPBeside : sbuf;
        const int pstep = D == 64 && single ? 16 : 32;
        bool pv_waited = j == 0 || !(D == 64 && single);  // else S of this tile says that P V of the last is done
        auto wait_pv = [&]() -> bool {
          if (pv_waited) return true;
          pv_waited = true;
          if (!wait_softmax(&bars.pv_done[w], t - 1)) return false;
          tc::fence_after_sync();
          return true;
        };
        float2 ls[2];
        // P = 2^(x * scale - m_run) over the tile, every kPolyEvery-th pair on the FMA pipe; returns the
        // largest x * scale.  Each chunk of S is read before P may overwrite it.
        auto exponentials = [&](float scale, auto as_pair) -> float {
          const float mu = m_run == -INFINITY ? 0.f : m_run;
          const float2 ks2 = make_float2(scale, scale), nmu2 = make_float2(-mu, -mu);
          float mx[2] = {-INFINITY, -INFINITY};
          ls[0] = ls[1] = make_float2(0.f, 0.f);
          auto chunk = [&](const float(&x)[32], int c) {
            uint32_t hi[16], lo[16];
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              if (D == 64 && !decltype(as_pair)::value) mx[i & 1] = max3_nan(mx[i & 1], x[2 * i], x[2 * i + 1]);
              const float2 e = tc::fma2(make_float2(x[2 * i], x[2 * i + 1]), ks2, nmu2);
              const float2 pr = i % kPolyEvery == kPolyEvery - 1 ? tc::exp2_poly2(e) : make_float2(tc::ex2(e.x), tc::ex2(e.y));
              ls[i & 1] = tc::add2(ls[i & 1], pr);
              if constexpr (decltype(as_pair)::value) {
                // hi: the upper 16 bits; lo: the exact rest, rounded
                const uint32_t u0 = __float_as_uint(pr.x), u1 = __float_as_uint(pr.y);
                hi[i] = __byte_perm(u0, u1, 0x7632);
                const float2 r = tc::sub2(pr, make_float2(__uint_as_float(u0 & 0xffff0000u), __uint_as_float(u1 & 0xffff0000u)));
                lo[i] = MMA::pack(r.x, r.y);
              } else {
                hi[i] = mma_op<__half>::pack(pr.x, pr.y);
              }
            }
            tc::st16u(pbuf + c * pstep, hi);
            if constexpr (decltype(as_pair)::value) tc::st16u(pbuf + c * 32 + 16, lo);
          };
          float xa[32], xb[32];
          tc::ld32(sbuf, xa);
          tc::wait_ld();
          ok = wait_pv();
#pragma unroll 1
          for (int c = 0; c < kBN / 32; c += 2) {
            tc::ld32(sbuf + (c + 1) * 32, xb);
            chunk(xa, c);
            tc::wait_ld();
            if (c + 2 < kBN / 32) tc::ld32(sbuf + (c + 2) * 32, xa);
            chunk(xb, c + 1);
            tc::wait_ld();
          }
          return max3_nan(mx[0], mx[1], mx[1]) * scale;
        };
        // The running maximum takes in `m_tile`, and O and l follow, where it grows by more than 2^8.
        auto raise_maximum = [&](float m_tile) {
          if (!(m_tile < INFINITY)) l_run = NAN;  // a NaN or +inf among the row's scores
          const float m_new = fmaxf(m_run, m_tile);
          const bool grow = m_new > m_run + 8.0f;
          const float alpha = (grow && m_run != -INFINITY) ? tc::ex2(m_run - m_new) : 1.0f;
          if (grow) {
            l_run *= (m_run == -INFINITY ? 0.f : alpha);
            m_run = m_new;
          }
          if (j > 0 && __any_sync(0xffffffffu, grow && alpha != 1.0f)) {
#pragma unroll 1
            for (int c = 0; c < D / 16; ++c) {
              float r[16];
              tc::ld16(obuf + c * 16, r);
              tc::wait_ld();
#pragma unroll
              for (int i = 0; i < 16; ++i) r[i] *= alpha;
              tc::st16(obuf + c * 16, r);
            }
            tc::wait_st();
          }
        };
        // Where P does not overwrite S, a tile takes one pass with the maximum as it stands: right unless
        // a score exceeds it by more than 2^8, which the pass finds out, and then a second one follows.
        const bool one_pass = D == 64 && single && raw && __all_sync(0xffffffffu, m_run != -INFINITY);
        if (!one_pass) {
          float mx[4];
#pragma unroll
          for (int r = 0; r < 4; ++r) mx[r] = -INFINITY;
          if (raw) {
#pragma unroll
            for (int c = 0; c < kBN / 32; c += 2) {
              float xa[32], xb[32];
              tc::ld32(sbuf + c * 32, xa);
              tc::ld32(sbuf + (c + 1) * 32, xb);
              tc::wait_ld();
#pragma unroll
              for (int i = 0; i < 16; ++i) {
                mx[i & 3] = max3_nan(mx[i & 3], xa[2 * i], xa[2 * i + 1]);
                mx[i & 3] = max3_nan(mx[i & 3], xb[2 * i], xb[2 * i + 1]);
              }
            }
          } else {
            const int vhi = last - kbase;
#pragma unroll 1
            for (int c = 0; c < kBN / 32; ++c) {
              float x[32];
              tc::ld32(sbuf + c * 32, x);
              tc::wait_ld();
              if (p.softcap > 0.f) {
                soft_cap(x, qk_scale / p.softcap, p.softcap * kLog2e);
              } else {
#pragma unroll
                for (int i = 0; i < 32; ++i) x[i] *= qk_scale;
              }
#pragma unroll
              for (int i = 0; i < 32; ++i) x[i] = c * 32 + i <= vhi ? x[i] : -INFINITY;
#pragma unroll
              for (int i = 0; i < 16; ++i) mx[i & 3] = max3_nan(mx[i & 3], x[2 * i], x[2 * i + 1]);
              tc::st32(sbuf + c * 32, x);
            }
            tc::wait_st();
          }
          const float m_tile = max3_nan(max3_nan(mx[0], mx[1], mx[2]), mx[3], mx[3]);
          if (!(ok = wait_pv())) break;
          raise_maximum(raw ? m_tile * qk_scale : m_tile);
        }
#pragma unroll 1
        for (bool again = one_pass;; again = false) {
          const float scale = raw ? qk_scale : 1.0f;
          if (kBF16 && !single) {
            exponentials(scale, std::integral_constant<bool, kBF16>());
            break;
          }
          const float top = exponentials(scale, std::false_type());
          if (!(top < INFINITY)) l_run = NAN;
          if (!again || !ok || !__any_sync(0xffffffffu, top > m_run + 8.0f)) break;
          raise_maximum(top);
        }
        if (!ok) break;
        l_run += (ls[0].x + ls[1].x) + (ls[0].y + ls[1].y);
        tc::wait_st();
        tc::fence_before_sync();
        mbar_arrive(&bars.p_full[w]);
      }
      if (!ok) break;
      if (!wait_softmax(&bars.o_done[w], items++)) break;
      tc::fence_after_sync();
      const int64_t at = (int64_t)m.slab * a.rows + (int64_t)tok * H + m.kh * g + hl;
      // values times 2^11 from the copy: (m, l, o) stands for 2^m l and 2^m o / 2^11, so 11 comes off m and l takes the factor
      if (row_ok) a.slab_ml[at] = copied ? make_float2(m_run - kCopyScaleLog2, l_run * kCopyScale) : make_float2(m_run, l_run);
#pragma unroll
      for (int c = 0; c < D / 32; ++c) {
        float o[32];
        tc::ld32(obuf + c * 32, o);
        tc::wait_ld();
        if (row_ok) {
          float4* dst = reinterpret_cast<float4*>(a.slab_o + at * D + c * 32);
#pragma unroll
          for (int i = 0; i < 8; ++i) dst[i] = make_float4(o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]);
        }
      }
      tc::fence_before_sync();
    }
  }
  tc::fence_before_sync();
  __syncthreads();
  tc::fence_after_sync();
  if (warp == kMmaWarp) tc::dealloc(tmem, 512);
}

template <typename T, int D, bool BESIDE>
cudaError_t launch_shape(const SharedPrefixArgs& a, const SharedPrefixMaps& maps, int num_sms, cudaStream_t stream) {
  using L = TcLayout<D, BESIDE>;
  auto kernel = shared_prefix_tc_kernel<T, D, BESIDE>;
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  static std::atomic<uint32_t> ready[64];  // per device: attributes set and checked
  if (!ready[dev & 63].load(std::memory_order_acquire)) {
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, L::kSmem);
    if (e != cudaSuccess) return e;
    // both kernels' CTAs share an SM only in the largest shared-memory split
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxShared);
    if (e != cudaSuccess) return e;
    cudaFuncAttributes attr;  // setmaxnreg.inc waits until the launch allocation covers the split
    e = cudaFuncGetAttributes(&attr, kernel);
    if (e != cudaSuccess) return e;
    if (attr.numRegs * kThreads < L::kSplitRegs) return cudaErrorInvalidConfiguration;
    ready[dev & 63].store(1, std::memory_order_release);
  }
  return launch_dependent(kernel, dim3(num_sms), dim3(kThreads), L::kSmem, stream, a, maps);
}

template <typename T, int D>
cudaError_t launch_tc_t(const SharedPrefixArgs& a, const SharedPrefixMaps& maps, int num_sms, cudaStream_t stream) {
  if constexpr (D == 128)
    if (!a.beside) return launch_shape<T, D, false>(a, maps, num_sms, stream);
  return launch_shape<T, D, true>(a, maps, num_sms, stream);
}

}  // namespace

cudaError_t launch_shared_prefix_tc(const SharedPrefixArgs& a, const SharedPrefixMaps& maps, int num_sms,
                                    cudaStream_t stream) {
  const bool bf = a.p.act_dtype == B200_DTYPE_BFLOAT16;
  if (a.p.head_size == 64)
    return bf ? launch_tc_t<__nv_bfloat16, 64>(a, maps, num_sms, stream) : launch_tc_t<__half, 64>(a, maps, num_sms, stream);
  return bf ? launch_tc_t<__nv_bfloat16, 128>(a, maps, num_sms, stream) : launch_tc_t<__half, 128>(a, maps, num_sms, stream);
}

}  // namespace b200
