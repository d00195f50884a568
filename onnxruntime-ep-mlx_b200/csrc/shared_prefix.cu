// Causal attention over paged caches for a batch whose sequences share one prefix
// (b200_shared_prefix_attention): the plan and merge kernels of the fast path (shared_prefix.cuh
// gives its structure), the generic kernel, and the launches.
//
// Softmax over a union of key sets: with M the largest m of a row's triples (m, l, o),
//   out = sum 2^(m_i - M) o_i / (sum 2^(m_i - M) l_i + 2^(sink log2 e - M))
//
// shared_prefix_generic_kernel (any head size up to 256, block size, head ratio and alignment): a CTA per
// (token, query head); its warps take the keys of the prefix and the token's own four at a time with an
// fp32 running softmax (m, l, o), and the warps' triples are joined in shared memory.
#include <algorithm>
#include <cmath>

#include "b200_kernels.h"
#include "shared_prefix.cuh"

namespace b200 {
namespace {

constexpr int kGenericWarps = 8;
constexpr int kGenericUnroll = 4;  // keys a warp has in flight

template <typename T, int CH>  // CH channels per lane: head_size <= 32 * CH
__global__ void __launch_bounds__(32 * kGenericWarps) shared_prefix_generic_kernel(const B200SharedPrefixParams p) {
  __shared__ float part_o[kGenericWarps][32 * CH];
  __shared__ float part_m[kGenericWarps], part_l[kGenericWarps];
  const int64_t t = blockIdx.x;
  const int h = blockIdx.y, d = p.head_size, kh = h / (p.num_heads / p.kv_num_heads);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int b = seq_of_token(p.cumulative_sequence_length, p.batch, (int)t);
  const int c0 = p.cumulative_sequence_length[b], c1 = p.cumulative_sequence_length[b + 1];
  const int past = p.past_seqlens[b];
  const int64_t total = (int64_t)past + c1 - c0;
  const bool ok = c0 >= 0 && t >= c0 && t < c1 && c1 <= p.num_tokens && past >= 0 &&
                  total <= (int64_t)p.max_blocks_per_seq * p.block_size;
  if (!ok && threadIdx.x == 0) set_status(p.device_status, past < 0 ? kStatusBadPast : kStatusBadCumulative);
  const int own = ok ? past + (int)(t - c0) + 1 : 0;  // own keys this token sees
  const int64_t keys = (int64_t)p.prefix_length + own;
  const int32_t* table = p.block_table + (int64_t)b * p.max_blocks_per_seq;

  const T* qrow = static_cast<const T*>(p.query) + t * p.query_row_stride + (int64_t)h * d;
  float q[CH], o[CH];
#pragma unroll
  for (int i = 0; i < CH; ++i) {
    q[i] = lane + 32 * i < d ? act<T>::to_f(qrow[lane + 32 * i]) * p.scale : 0.f;
    o[i] = 0.f;
  }
  float m = -INFINITY, l = 0.f;
  for (int64_t j0 = warp * kGenericUnroll; j0 < keys; j0 += kGenericWarps * kGenericUnroll) {
    float k[kGenericUnroll][CH], v[kGenericUnroll][CH], x[kGenericUnroll];
#pragma unroll
    for (int u = 0; u < kGenericUnroll; ++u) {
      const int64_t j = j0 + u;
      const bool mine = j < p.prefix_length;
      const int64_t at = mine ? j : j - p.prefix_length;
      int64_t row = -1;
      if (j < keys) {
        const int32_t blk = mine ? p.prefix_block_table[at / p.block_size] : table[at / p.block_size];
        if (blk < 0 || blk >= p.num_blocks) set_status(p.device_status, kStatusBadBlock);
        else row = (((int64_t)blk * p.block_size + at % p.block_size) * p.kv_num_heads + kh) * d;
      }
      x[u] = 0.f;
#pragma unroll
      for (int i = 0; i < CH; ++i) {
        const bool in = row >= 0 && lane + 32 * i < d;
        k[u][i] = in ? act<T>::to_f(static_cast<const T*>(p.key_cache)[row + lane + 32 * i]) : 0.f;
        v[u][i] = in ? act<T>::to_f(static_cast<const T*>(p.value_cache)[row + lane + 32 * i]) : 0.f;
        x[u] += q[i] * k[u][i];
      }
#pragma unroll
      for (int s = 16; s; s >>= 1) x[u] += __shfl_xor_sync(0xffffffffu, x[u], s);
      if (p.softcap > 0.f) x[u] = p.softcap * tanhf(x[u] / p.softcap);
      if (j >= keys) x[u] = -INFINITY;
    }
    float top = m;
#pragma unroll
    for (int u = 0; u < kGenericUnroll; ++u) top = fmaxf(top, x[u]);
    const float base = top == -INFINITY ? 0.f : top;
    const float f = expf(m - base);
    l *= f;
#pragma unroll
    for (int i = 0; i < CH; ++i) o[i] *= f;
#pragma unroll
    for (int u = 0; u < kGenericUnroll; ++u) {
      const float e = expf(x[u] - base);
      l += e;
#pragma unroll
      for (int i = 0; i < CH; ++i) o[i] += e * v[u][i];
    }
    m = top;
  }
#pragma unroll
  for (int i = 0; i < CH; ++i) part_o[warp][lane + 32 * i] = o[i];
  if (lane == 0) {
    part_m[warp] = m;
    part_l[warp] = l;
  }
  __syncthreads();
  const float sink = p.head_sink ? load_act(p.head_sink, h, p.act_dtype) : -INFINITY;
  float top = sink;
  for (int w = 0; w < kGenericWarps; ++w) top = fmaxf(top, part_m[w]);
  float sum = p.head_sink ? expf(sink - top) : 0.f;
  for (int w = 0; w < kGenericWarps; ++w) {
    if (part_m[w] != -INFINITY) sum += part_l[w] * expf(part_m[w] - top);
    else if (part_l[w] != part_l[w]) sum = part_l[w];  // NaN scores only
  }
  T* out = static_cast<T*>(p.output) + t * p.output_row_stride + (int64_t)h * d;
  for (int c = threadIdx.x; c < d; c += blockDim.x) {
    float acc = 0.f;
    for (int w = 0; w < kGenericWarps; ++w)
      if (part_m[w] != -INFINITY) acc += part_o[w][c] * expf(part_m[w] - top);
    out[c] = act<T>::from_f(sum == 0.f ? 0.f : acc / sum);
  }
}

template <typename T>
void launch_generic_t(const B200SharedPrefixParams& p, cudaStream_t stream) {
  const dim3 grid(p.num_tokens, p.num_heads);
  if (p.head_size <= 64) shared_prefix_generic_kernel<T, 2><<<grid, 32 * kGenericWarps, 0, stream>>>(p);
  else if (p.head_size <= 128) shared_prefix_generic_kernel<T, 4><<<grid, 32 * kGenericWarps, 0, stream>>>(p);
  else shared_prefix_generic_kernel<T, 8><<<grid, 32 * kGenericWarps, 0, stream>>>(p);
}


// ---------------------------------------------------------------------------------------------
// Plan: CTA 0 checks the lengths, routes every sequence and lays out both work lists.  The other CTAs,
// where launched, copy the prefix's bf16 values to fp16 [key][kv head][channel]: with fp16 values the
// tensor-core pass can carry P as one fp16 value instead of a bf16 hi + lo pair, which takes a third of
// its MMA work.  The copy is exact or not used: values go in times kCopyScale, which fp16 holds to the last
// bit for magnitudes from 2^-28 to below 32 and for zero (2^11 puts that window around values of order 0.01
// to 10); a CTA that meets any other value names its kv head, and the tensor-core pass reads that head's
// values from the bf16 pages.  128 sequences 5 us;
// the copy of 16384 keys of 8 heads of 128 channels 18 us (67 MB).  The tensor-core pass starts beside both.
// ---------------------------------------------------------------------------------------------
constexpr int kPlanThreads = 1024;

// Inclusive sums of (x, y) over the block, totals in `total`.
__device__ __forceinline__ int2 block_inclusive_sum(int2 v, int2* warp_sums, int2& total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int x = __shfl_up_sync(0xffffffffu, v.x, o), y = __shfl_up_sync(0xffffffffu, v.y, o);
    if (lane >= o) {
      v.x += x;
      v.y += y;
    }
  }
  if (lane == 31) warp_sums[warp] = v;
  __syncthreads();
  if (warp == 0) {
    int2 s = warp_sums[lane];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int x = __shfl_up_sync(0xffffffffu, s.x, o), y = __shfl_up_sync(0xffffffffu, s.y, o);
      if (lane >= o) {
        s.x += x;
        s.y += y;
      }
    }
    warp_sums[lane] = s;
  }
  __syncthreads();
  if (warp > 0) {
    v.x += warp_sums[warp - 1].x;
    v.y += warp_sums[warp - 1].y;
  }
  total = warp_sums[31];
  __syncthreads();
  return v;
}

__device__ __forceinline__ void copy_prefix_values(const SharedPrefixArgs& a) {
  const B200SharedPrefixParams& p = a.p;
  const int64_t vecs = (int64_t)p.kv_num_heads * p.head_size / 8;  // 16-byte pieces of one key's values
  const int64_t n = vecs * p.prefix_length, step = (int64_t)a.copy_ctas * kPlanThreads;
  __shared__ unsigned long long inexact_heads;
  if (threadIdx.x == 0) inexact_heads = 0;
  __syncthreads();
  auto load = [&](int64_t i) {
    const int64_t key = i / vecs;
    const int32_t blk = __ldg(p.prefix_block_table + key / p.block_size);
    if (blk < 0 || blk >= p.num_blocks) return make_uint4(0, 0, 0, 0);  // the tensor-core kernel reports these
    return __ldg(static_cast<const uint4*>(p.value_cache) + ((int64_t)blk * p.block_size + key % p.block_size) * vecs + (i - key * vecs));
  };
  // bits 15 and 31: a magnitude of 0x4200 (32) and above, or below 0x3180 (2^-28) and not zero
  auto outside_of = [](const uint4& v) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
    uint32_t outside = 0;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const uint32_t m = w[k] & 0x7fff7fffu;
      outside |= (m + 0x3e003e00u) | (~((w[k] | 0x80008000u) - 0x31803180u) & (m + 0x7fff7fffu));
    }
    return outside & 0x80008000u;
  };
  const __nv_bfloat162 factor = __float2bfloat162_rn(kCopyScale);
  const int64_t first = (int64_t)(blockIdx.x - 1) * kPlanThreads + threadIdx.x;
  uint32_t outside = 0;
#pragma unroll 4
  for (int64_t i = first; i < n; i += step) {
    const uint4 v = load(i);
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
    uint32_t o[4];
    outside |= outside_of(v);
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const __nv_bfloat162 x = __hmul2(*reinterpret_cast<const __nv_bfloat162*>(&w[k]), factor);
      const __half2 h = __float22half2_rn(__bfloat1622float2(x));
      o[k] = *reinterpret_cast<const uint32_t*>(&h);
    }
    reinterpret_cast<uint4*>(a.v_copy)[i] = make_uint4(o[0], o[1], o[2], o[3]);
  }
  unsigned long long inexact = 0;
  if (outside)  // rare: which heads (named in the loop above, a call with 8192 keys took 1 us longer)
    for (int64_t i = first; i < n; i += step)
      if (outside_of(load(i))) inexact |= 1ull << ((uint32_t)(i % vecs) / (uint32_t)(p.head_size / 8) & 63u);
  if (inexact) atomicOr(&inexact_heads, inexact);
  __syncthreads();
  if (threadIdx.x == 0) a.v_inexact[blockIdx.x - 1] = inexact_heads;
}

__global__ void __launch_bounds__(kPlanThreads) shared_prefix_plan_kernel(const SharedPrefixArgs a) {
  __shared__ int2 warp_sums[32];
  const B200SharedPrefixParams& p = a.p;
  release_dependents();
  if (blockIdx.x > 0) return copy_prefix_values(a);
  const int tid = threadIdx.x, lane = tid & 31;
  for (int t = tid; t < p.num_tokens; t += kPlanThreads) a.token_info[t] = make_int4(0, -1, 0, 0);
  if (tid == 0) *a.next_item = 0;
  __syncthreads();
  int2 carry = make_int2(0, 0);
  for (int base = 0; base < p.batch; base += kPlanThreads) {
    const int b = base + tid;
    int2 work = make_int2(0, 0);  // 16-key tiles of the own kernel, query-tile pairs of the tensor-core kernel
    int c0 = 0, nq = 0;
    if (b < p.batch) {
      c0 = p.cumulative_sequence_length[b];
      const int c1 = p.cumulative_sequence_length[b + 1], past = p.past_seqlens[b];
      const int64_t total = (int64_t)past + c1 - c0;
      int bits = 0;
      if (c0 < 0 || c0 > c1 || c1 > p.num_tokens || (b == 0 && c0 != 0) || (b == p.batch - 1 && c1 != p.num_tokens))
        bits |= kStatusBadCumulative;
      if (past < 0) bits |= kStatusBadPast;
      if (total > (int64_t)p.max_blocks_per_seq * p.block_size) bits |= kStatusBadCapacity;
      if (bits) set_status(p.device_status, bits);
      if (c0 >= 0 && c0 <= c1 && c1 <= p.num_tokens && past >= 0 && !(bits & kStatusBadCapacity)) nq = c1 - c0;
      if ((int64_t)nq * a.group <= a.own_rows) work.x = nq ? (int)((total + kOwnTile - 1) / kOwnTile) : 0;
      else work.y = (nq + 2 * a.tile_tokens - 1) / (2 * a.tile_tokens);
    }
    int2 total;
    const int2 incl = block_inclusive_sum(work, warp_sums, total);
    const int first = carry.x + incl.x - work.x;
    if (b < p.batch) {
      a.seq_tiles[b] = first;
      a.seq_pairs[b] = carry.y + incl.y - work.y;
    }
    const int4 info = make_int4(c0, nq, first, work.x);
    if (nq <= 32)
      for (int i = 0; i < nq; ++i) a.token_info[c0 + i] = info;
    for (unsigned left = __ballot_sync(0xffffffffu, nq > 32); left; left &= left - 1) {  // long ones: the whole warp
      const int src = __ffs(left) - 1;
      const int4 seq = make_int4(__shfl_sync(0xffffffffu, info.x, src), __shfl_sync(0xffffffffu, info.y, src),
                                 __shfl_sync(0xffffffffu, info.z, src), __shfl_sync(0xffffffffu, info.w, src));
      for (int i = lane; i < seq.y; i += 32) a.token_info[seq.x + i] = seq;
    }
    carry.x += total.x;
    carry.y += total.y;
  }
  if (tid == 0) {
    a.seq_tiles[p.batch] = carry.x;
    a.seq_pairs[p.batch] = carry.y;
  }
}

// ---------------------------------------------------------------------------------------------
// Merge: D / 4 lanes per (token, head) row join the row's triples, BATCH of them in flight.  Bound by the
// slabs' reads, which come from L2 as far as the own keys' stream has left them there, and by the issue of
// instructions: batches of 4 where a row has few triples (whole calls with 4 and 8, medians of four runs in turn: 256
// tokens and at most 3 ranges 362 against 364 us; 31 sequences of drafted tokens 60 against 58, 128 tokens and 9 ranges
// 98.2 against 97.8).
// ---------------------------------------------------------------------------------------------
constexpr int kMergeThreads = 128;
constexpr int kFewRanges = 3;
constexpr float kLog2eMerge = 1.4426950408889634f;

template <typename T, int D, int BATCH>
__global__ void __launch_bounds__(kMergeThreads) shared_prefix_merge_kernel(const SharedPrefixArgs a, int vector_rows) {
  constexpr int kLanes = D / 4;
  const B200SharedPrefixParams& p = a.p;
  const int c = threadIdx.x % kLanes * 4;  // first of this lane's channels
  const int64_t row = (int64_t)blockIdx.x * (kMergeThreads / kLanes) + threadIdx.x / kLanes;
  wait_previous();
  if (row >= a.rows) return;
  const int64_t t = row / p.num_heads;
  const int h = (int)(row - t * p.num_heads);
  // own part: the slab, or `pieces` rows of the own kernel's warps
  const int4 info = __ldcg(a.token_info + t);
  int own = info.y > 0;
  bool cut = false;
  int64_t first_row = 0, next_row = 0;
  if (info.w > 0) {
    const int KV = p.kv_num_heads, kh = h / a.group;
    const OwnRanges ranges((int64_t)__ldcg(a.seq_tiles + p.batch) * KV, a.own_warps);
    const int64_t start = (int64_t)info.z * KV + (int64_t)kh * info.w;
    const int64_t w_first = ranges.warp_of(start);
    own = (int)(ranges.warp_of(start + info.w - 1) - w_first + 1);
    cut = own > 1;
    // a warp's row block 0 holds the piece its range starts with, block 1 its last one
    const int64_t r = (t - info.x) * a.group + h - kh * a.group;
    first_row = (w_first * 2 + (start > ranges.start(w_first) ? 1 : 0)) * a.own_rows + r;
    next_row = (w_first + 1) * 2 * a.own_rows + r;
  }
  const int parts = a.splits + own;
  float top = -INFINITY, sum = 0.f;
  if (p.head_sink) {
    top = act<T>::to_f(static_cast<const T*>(p.head_sink)[h]) * kLog2eMerge;
    sum = 1.f;
  }
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int base = 0; base < parts; base += BATCH) {
    float2 ml[BATCH];
    float4 o[BATCH];
#pragma unroll
    for (int j = 0; j < BATCH; ++j) {
      const int i = base + j, piece = i - a.splits;
      ml[j] = make_float2(-INFINITY, 0.f);
      if (i < parts) {
        const bool warp_row = cut && piece >= 0;
        const int64_t at = !warp_row ? (int64_t)i * a.rows + row
                                     : piece == 0 ? first_row : next_row + (int64_t)(piece - 1) * 2 * a.own_rows;
        ml[j] = __ldcg((warp_row ? a.warp_ml : a.slab_ml) + at);
        o[j] = __ldcg(reinterpret_cast<const float4*>((warp_row ? a.warp_o : a.slab_o) + at * D + c));
      }
    }
    float m = top;
#pragma unroll
    for (int j = 0; j < BATCH; ++j) m = fmaxf(m, ml[j].x);
#pragma unroll
    for (int j = 0; j < BATCH; ++j)
      if (ml[j].y != ml[j].y) sum = ml[j].y;  // NaN scores only: m has stayed at its start
    if (m == -INFINITY) continue;
    const float f = exp2f(top - m);
    top = m;
    sum *= f;
    acc.x *= f; acc.y *= f; acc.z *= f; acc.w *= f;
#pragma unroll
    for (int j = 0; j < BATCH; ++j) {
      if (ml[j].x == -INFINITY) continue;
      const float w = exp2f(ml[j].x - m);
      sum += ml[j].y * w;
      acc.x += w * o[j].x; acc.y += w * o[j].y; acc.z += w * o[j].z; acc.w += w * o[j].w;
    }
  }
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
  T* out = static_cast<T*>(p.output) + t * p.output_row_stride + (int64_t)h * D + c;
  if (vector_rows) {
    *reinterpret_cast<uint2*>(out) = make_uint2(mma_op<T>::pack(acc.x * inv, acc.y * inv), mma_op<T>::pack(acc.z * inv, acc.w * inv));
  } else {
    out[0] = act<T>::from_f(acc.x * inv);
    out[1] = act<T>::from_f(acc.y * inv);
    out[2] = act<T>::from_f(acc.z * inv);
    out[3] = act<T>::from_f(acc.w * inv);
  }
}

template <typename T>
cudaError_t launch_merge_t(const SharedPrefixArgs& a, cudaStream_t stream) {
  const bool vec = (reinterpret_cast<uintptr_t>(a.p.output) | (uintptr_t)(a.p.output_row_stride * 2)) % 8 == 0;
  const int64_t per_cta = kMergeThreads / (a.p.head_size / 4);
  const dim3 grid((unsigned)((a.rows + per_cta - 1) / per_cta)), block(kMergeThreads);
  auto kernel = a.p.head_size == 64
                    ? (a.splits <= kFewRanges ? shared_prefix_merge_kernel<T, 64, 4> : shared_prefix_merge_kernel<T, 64, 8>)
                    : (a.splits <= kFewRanges ? shared_prefix_merge_kernel<T, 128, 4> : shared_prefix_merge_kernel<T, 128, 8>);
  return launch_dependent(kernel, grid, block, 0, stream, a, (int)vec);
}

// ---------------------------------------------------------------------------------------------
// Host side of the fast path
// ---------------------------------------------------------------------------------------------
// Pairs of query tiles up to which head size 128 shares the SMs with the own kernel.  Whole calls shared and
// not (8192 keys, 8 kv heads): 1 pair 49 against 55 us, 2 pairs 94 against 105, 4 pairs 118 against 120, 8
// pairs 209 against 201.  Head size 64 gives up nothing for it and always shares.
constexpr int kBesidePairs = 4;
constexpr int kCopyPairs = 4;  // pairs of query tiles from which the copy of the prefix's values pays

// The shapes the fast path covers; the call also needs 16-byte rows (fast_rows).
bool fast_shape(const B200SharedPrefixParams& p) {
  return (p.head_size == 64 || p.head_size == 128) && p.block_size % kOwnTile == 0 &&
         p.num_heads / p.kv_num_heads <= 128 &&
         // work items are counted in 32 bits: at most 64 ranges and a pair per token, and a pair per sequence
         ((int64_t)64 * p.num_tokens + p.batch) * p.kv_num_heads < INT32_MAX;
}

bool fast_rows(const B200SharedPrefixParams& p) {
  return ((reinterpret_cast<uintptr_t>(p.query) | reinterpret_cast<uintptr_t>(p.key_cache) |
           reinterpret_cast<uintptr_t>(p.value_cache) | (uintptr_t)(p.query_row_stride * 2)) & 15) == 0;
}

// Key ranges of the prefix: the fewest "tile times" over waves of the SMs, where an item costs its
// tiles plus about 2 for its start and end, and a further range costs its rows' triples to write and
// read (about 12 TB/s of traffic against 2.5 us a tile).
void split_prefix(SharedPrefixArgs* a, int num_sms) {
  const B200SharedPrefixParams& p = a->p;
  const int64_t tiles = ((int64_t)p.prefix_length + kPrefixKeys - 1) / kPrefixKeys;
  const int64_t items = (int64_t)p.kv_num_heads * a->query_pairs;
  a->splits = 0;
  a->split_tiles = 1;
  if (tiles == 0 || items == 0) return;
  const double per_range = (double)a->rows * p.head_size * 8 / 12e12 / 2.5e-6;
  double best = 0;
  for (int64_t s = 1; s <= 64 && s <= tiles; ++s) {
    const int64_t per = (tiles + s - 1) / s, n = (tiles + per - 1) / per;
    const double cost = (double)((items * n + num_sms - 1) / num_sms) * (per + 2) + per_range * n;
    if (a->splits == 0 || cost < best) {
      best = cost;
      a->splits = (int)n;
      a->split_tiles = (int)per;
    }
  }
}

// Fills `a` and returns the workspace bytes (0: generic kernel).
size_t layout(const B200SharedPrefixParams& p, int num_sms, SharedPrefixArgs* a) {
  if (!fast_shape(p) || p.num_tokens == 0) return 0;
  a->p = p;
  a->group = p.num_heads / p.kv_num_heads;
  a->tile_tokens = 128 / a->group;
  a->query_pairs = (p.num_tokens + 2 * a->tile_tokens - 1) / (2 * a->tile_tokens);
  // one 8-row MMA tile when a kv head's rows of one token fit and sequences have about one token
  a->own_rows = a->group <= 8 && p.num_tokens <= p.batch ? 8 : 16;
  a->own_warps = num_sms * kOwnCtasPerSm * kOwnWarps;
  a->rows = (int64_t)p.num_tokens * p.num_heads;
  split_prefix(a, num_sms);
  // The copy of the values costs about 4 bytes per value once, and saves every pair of query tiles a
  // third of its MMA work on them.  Whole calls with and without it (8192 prefix keys, 16 own keys, 32 / 8 heads),
  // d 128: 1 pair 43 against 37 us, 2 pairs 52 / 47, 4 pairs 75 / 72, 8 pairs 109 / 110; d 64: 35 / 31, 39 / 41,
  // 52 / 60, 83 / 102.
  const bool copy = p.act_dtype == B200_DTYPE_BFLOAT16 && p.prefix_length > 0 && a->query_pairs >= kCopyPairs;
  a->beside = p.head_size == 64 || a->query_pairs <= kBesidePairs;
  a->copy_ctas = copy ? 2 * num_sms - 1 : 0;
  char* base = static_cast<char*>(p.workspace);
  size_t off = 0;
  auto take = [&](size_t bytes) {
    char* at = base + off;
    off = (off + bytes + 255) / 256 * 256;
    return at;
  };
  const size_t d = p.head_size, slabs = (size_t)a->splits + 1, wrows = (size_t)a->own_warps * 2 * a->own_rows;
  a->next_item = reinterpret_cast<uint32_t*>(take(sizeof(uint32_t)));
  a->seq_tiles = reinterpret_cast<int*>(take(sizeof(int) * ((size_t)p.batch + 1)));
  a->seq_pairs = reinterpret_cast<int*>(take(sizeof(int) * ((size_t)p.batch + 1)));
  a->token_info = reinterpret_cast<int4*>(take(sizeof(int4) * (size_t)p.num_tokens));
  a->slab_ml = reinterpret_cast<float2*>(take(sizeof(float2) * slabs * a->rows));
  a->warp_ml = reinterpret_cast<float2*>(take(sizeof(float2) * wrows));
  a->slab_o = reinterpret_cast<float*>(take(sizeof(float) * slabs * a->rows * d));
  a->warp_o = reinterpret_cast<float*>(take(sizeof(float) * wrows * d));
  a->v_copy = nullptr;
  if (copy) {
    a->v_inexact = reinterpret_cast<uint64_t*>(take(sizeof(uint64_t) * a->copy_ctas));
    a->v_copy = reinterpret_cast<__half*>(take(2 * (size_t)p.prefix_length * p.kv_num_heads * d));
  }
  return off;
}

cudaError_t encode_maps(const SharedPrefixArgs& a, SharedPrefixMaps* maps) {
  const B200SharedPrefixParams& p = a.p;
  const bool bf = p.act_dtype == B200_DTYPE_BFLOAT16;
  const uint64_t d = p.head_size, kv = p.kv_num_heads;
  const uint64_t dims[3] = {d, kv, (uint64_t)p.num_blocks * p.block_size}, strides[2] = {d * 2, kv * d * 2};
  const uint32_t box[3] = {64, 1, kOwnTile};
  const uint64_t q_dims[3] = {d, (uint64_t)p.num_heads, (uint64_t)p.num_tokens};
  const uint64_t q_strides[2] = {d * 2, (uint64_t)p.query_row_stride * 2};
  const uint32_t q_box[3] = {64, (uint32_t)a.group, (uint32_t)a.tile_tokens};
  if (encode_tensor_map(&maps->k_map, bf, 3, p.key_cache, dims, strides, box) ||
      encode_tensor_map(&maps->v_map, bf, 3, p.value_cache, dims, strides, box) ||
      encode_tensor_map(&maps->q_map, bf, 3, p.query, q_dims, q_strides, q_box))
    return cudaErrorInvalidValue;
  if (a.v_copy) {
    const uint64_t c_dims[3] = {d, kv, (uint64_t)p.prefix_length};
    const uint32_t c_box[3] = {64, 1, kPrefixKeys};
    if (encode_tensor_map(&maps->vc_map, false, 3, a.v_copy, c_dims, strides, c_box)) return cudaErrorInvalidValue;
  }
  return cudaSuccess;
}

}  // namespace

size_t shared_prefix_workspace(const B200SharedPrefixParams& p, int num_sms) {
  SharedPrefixArgs a{};
  return layout(p, num_sms, &a);
}

cudaError_t launch_shared_prefix(const B200SharedPrefixParams& p, int num_sms, cudaStream_t stream) {
  SharedPrefixArgs a{};
  if (layout(p, num_sms, &a) == 0 || !fast_rows(p)) {
    if (p.act_dtype == B200_DTYPE_BFLOAT16) launch_generic_t<__nv_bfloat16>(p, stream);
    else launch_generic_t<__half>(p, stream);
    add_launches(1);
    return cudaGetLastError();
  }
  SharedPrefixMaps maps{};
  cudaError_t e = encode_maps(a, &maps);
  if (e != cudaSuccess) return e;
  shared_prefix_plan_kernel<<<1 + a.copy_ctas, kPlanThreads, 0, stream>>>(a);
  e = cudaGetLastError();
  if (e == cudaSuccess) e = launch_shared_prefix_tc(a, maps, num_sms, stream);
  if (e == cudaSuccess) e = launch_shared_prefix_own(a, stream);
  if (e == cudaSuccess)
    e = p.act_dtype == B200_DTYPE_BFLOAT16 ? launch_merge_t<__nv_bfloat16>(a, stream) : launch_merge_t<__half>(a, stream);
  if (e == cudaSuccess) add_launches(4);
  return e;
}

}  // namespace b200
