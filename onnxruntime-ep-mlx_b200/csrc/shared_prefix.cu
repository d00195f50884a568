// Causal attention over paged caches for a batch whose sequences share one prefix
// (b200_shared_prefix_attention).
//
// shared_prefix_generic_kernel: a CTA per (token, query head); its warps take every kWarps-th key
// of the prefix and of the token's own keys with an fp32 running softmax (m, l, o), and the warps'
// triples are joined in shared memory.  Any head size up to 256, block size and head ratio.
#include <algorithm>
#include <cmath>

#include "b200_common.cuh"
#include "layer_kernels.h"

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
  for (int w = 0; w < kGenericWarps; ++w)
    if (part_m[w] != -INFINITY) sum += part_l[w] * expf(part_m[w] - top);
  T* out = static_cast<T*>(p.output) + t * p.output_row_stride + (int64_t)h * d;
  for (int c = threadIdx.x; c < d; c += blockDim.x) {
    float acc = 0.f;
    for (int w = 0; w < kGenericWarps; ++w)
      if (part_m[w] != -INFINITY) acc += part_o[w][c] * expf(part_m[w] - top);
    out[c] = act<T>::from_f(sum > 0.f ? acc / sum : 0.f);
  }
}

template <typename T>
void launch_generic_t(const B200SharedPrefixParams& p, cudaStream_t stream) {
  const dim3 grid(p.num_tokens, p.num_heads);
  if (p.head_size <= 64) shared_prefix_generic_kernel<T, 2><<<grid, 32 * kGenericWarps, 0, stream>>>(p);
  else if (p.head_size <= 128) shared_prefix_generic_kernel<T, 4><<<grid, 32 * kGenericWarps, 0, stream>>>(p);
  else shared_prefix_generic_kernel<T, 8><<<grid, 32 * kGenericWarps, 0, stream>>>(p);
}

}  // namespace

size_t shared_prefix_workspace(const B200SharedPrefixParams&, int) { return 0; }

cudaError_t launch_shared_prefix(const B200SharedPrefixParams& p, int, cudaStream_t stream) {
  if (p.act_dtype == B200_DTYPE_BFLOAT16) launch_generic_t<__nv_bfloat16>(p, stream);
  else launch_generic_t<__half>(p, stream);
  add_launches(1);
  return cudaGetLastError();
}

}  // namespace b200
