// Rotary embedding of new queries and keys with up to four position axes, and the append of keys
// and values to the paged caches, in one pass (b200_rotary_append).
//
//   pair (x0, x1) -> (x0 c - x1 s, x1 c + x0 s) in fp32, rounded once; c, s from row
//   position[axis of the pair] of the tables
//
// Memory bound: every query, key and value row is read once and written once.
#include <algorithm>

#include "b200_common.cuh"
#include "layer_kernels.h"

namespace b200 {
namespace {

__device__ __forceinline__ uint32_t table_hash(int32_t slot) {
  uint32_t x = static_cast<uint32_t>(slot) * 0x9e3779b1u;
  x ^= x >> 15;
  x *= 0x85ebca77u;
  return x ^ (x >> 13);
}

// slot -> last token naming it, in an open-addressing table of `capacity` (a power of two, at
// least twice the tokens) keys, filled with -1 bytes before
__global__ void slot_table_kernel(const int32_t* slots, int n, int64_t slot_count, int* keys, int* last,
                                  uint32_t capacity) {
  const int t = blockIdx.x * blockDim.x + threadIdx.x;
  if (t >= n) return;
  const int32_t slot = slots[t];
  if (slot < 0 || slot >= slot_count) return;
  uint32_t h = table_hash(slot) & (capacity - 1);
  for (uint32_t probe = 0; probe < capacity; ++probe) {
    const int prev = atomicCAS(&keys[h], -1, slot);
    if (prev == -1 || prev == slot) {
      atomicMax(&last[h], t);
      return;
    }
    h = (h + 1) & (capacity - 1);
  }
}

__device__ __forceinline__ int last_token(int32_t slot, int t, const int* keys, const int* last, uint32_t capacity) {
  uint32_t h = table_hash(slot) & (capacity - 1);
  for (uint32_t probe = 0; probe < capacity; ++probe) {
    const int key = keys[h];
    if (key == slot) return last[h];
    if (key == -1) return t;
    h = (h + 1) & (capacity - 1);
  }
  return t;
}

__device__ __forceinline__ int64_t position_of(const B200RotaryAppendParams& p, int axis, int64_t t) {
  const int64_t i = axis * p.position_axis_stride + t * p.position_token_stride;
  return p.position_dtype == B200_DTYPE_INT64 ? static_cast<const int64_t*>(p.position_ids)[i]
                                              : (int64_t) static_cast<const int32_t*>(p.position_ids)[i];
}

__device__ __forceinline__ int axis_of(const B200RotaryAppendParams& p, int pair) {
  int axis = 0, end = p.axis_pairs[0];
#pragma unroll
  for (int a = 1; a < B200_MAX_ROTARY_AXES; ++a) {
    axis += a < p.axes && pair >= end;
    end += a < p.axes ? p.axis_pairs[a] : 0;
  }
  return axis;
}

template <typename T>
__device__ __forceinline__ float table_value(const B200RotaryAppendParams& p, const void* table, int64_t i) {
  return p.table_dtype == B200_DTYPE_FLOAT ? static_cast<const float*>(table)[i]
                                           : act<T>::to_f(static_cast<const T*>(table)[i]);
}

// Channel of half `second` of rotary pair i.
__device__ __forceinline__ int pair_channel(const B200RotaryAppendParams& p, int i, int second) {
  return p.rotary_offset + (p.rotary_interleaved ? 2 * i + second : i + second * (p.rotary_dim / 2));
}

template <typename T>
__device__ __forceinline__ void store_cached(const B200RotaryAppendParams& p, bool is_key, int64_t slot, int head,
                                             int channel, float x) {
  void* cache = is_key ? p.key_cache : p.value_cache;
  const int64_t at = (slot * p.kv_num_heads + head) * p.head_size + channel;
  if (p.cache_dtype == B200_DTYPE_FLOAT8E4M3FN) {
    const float scale = (is_key ? p.k_scale : p.v_scale)[slot / p.block_size * p.kv_num_heads + head];
    static_cast<uint8_t*>(cache)[at] = fp8_code(x, scale);
  } else {
    static_cast<T*>(cache)[at] = act<T>::from_f(x);
  }
}

// One CTA per token, a channel pair or a single channel per thread and step: any head size, offset
// and alignment.
template <typename T>
__global__ void __launch_bounds__(256) rotary_append_kernel(const B200RotaryAppendParams p, const int* keys,
                                                             const int* last, uint32_t capacity) {
  const int64_t t = blockIdx.x;
  const int tid = threadIdx.x, threads = blockDim.x;
  const int d = p.head_size, H = p.num_heads, KV = p.kv_num_heads, half = p.rotary_dim / 2;
  const int32_t slot = p.slot_mapping[t];
  const bool valid = slot >= -1 && (int64_t)slot < (int64_t)p.num_blocks * p.block_size;
  if (!valid && tid == 0) set_status(p.device_status, kStatusBadSlot);
  bool store = valid && slot >= 0;
  if (store) {  // the last token naming the slot writes it
    if (keys) {
      store = last_token(slot, (int)t, keys, last, capacity) == (int)t;
    } else {
      int later = 0;
      for (int64_t u = t + 1 + tid; u < p.num_tokens; u += threads) later |= p.slot_mapping[u] == slot;
      store = !__syncthreads_or(later);
    }
  }
  const T* q = static_cast<const T*>(p.query) + t * p.query_row_stride;
  const T* k = static_cast<const T*>(p.key) + t * p.key_row_stride;
  const T* v = static_cast<const T*>(p.value) + t * p.value_row_stride;
  T* out = static_cast<T*>(p.output) + t * p.output_row_stride;
  for (int i = tid; i < (H + KV) * half; i += threads) {
    const int head = i / half, pair = i % half;
    const int64_t pos = position_of(p, axis_of(p, pair), t);
    float c = 1.f, s = 0.f;
    if (pos >= 0 && pos < p.rotary_positions) {
      c = table_value<T>(p, p.cos_cache, pos * half + pair);
      s = table_value<T>(p, p.sin_cache, pos * half + pair);
    } else {
      set_status(p.device_status, kStatusBadPosition);
    }
    const int c0 = pair_channel(p, pair, 0), c1 = pair_channel(p, pair, 1);
    const T* row = head < H ? q + head * d : k + (head - H) * d;
    const float x0 = act<T>::to_f(row[c0]), x1 = act<T>::to_f(row[c1]);
    const float y0 = x0 * c - x1 * s, y1 = x1 * c + x0 * s;
    if (head < H) {
      out[head * d + c0] = act<T>::from_f(y0);
      out[head * d + c1] = act<T>::from_f(y1);
    } else if (store) {
      store_cached<T>(p, true, slot, head - H, c0, y0);
      store_cached<T>(p, true, slot, head - H, c1, y1);
    }
  }
  const int rest = d - p.rotary_dim;  // channels that do not turn
  for (int i = tid; i < (H + KV) * rest; i += threads) {
    const int head = i / rest, j = i % rest;
    const int c = j < p.rotary_offset ? j : j + p.rotary_dim;
    if (head < H) out[head * d + c] = q[head * d + c];
    else if (store) store_cached<T>(p, true, slot, head - H, c, act<T>::to_f(k[(head - H) * d + c]));
  }
  if (!store) return;
  for (int i = tid; i < KV * d; i += threads) store_cached<T>(p, false, slot, i / d, i % d, act<T>::to_f(v[i]));
}

uint32_t table_capacity(int tokens) {
  uint32_t cap = 64;
  while (cap < 2 * (uint32_t)tokens) cap <<= 1;
  return cap;
}

}  // namespace

size_t rotary_append_workspace(const B200RotaryAppendParams& p) {
  return p.num_tokens > B200_ROTARY_APPEND_SCAN_TOKENS ? 2 * sizeof(int) * (size_t)table_capacity(p.num_tokens) : 0;
}

cudaError_t launch_rotary_append(const B200RotaryAppendParams& p, int, cudaStream_t stream) {
  int *keys = nullptr, *last = nullptr;
  uint32_t cap = 0;
  if (p.num_tokens > B200_ROTARY_APPEND_SCAN_TOKENS) {
    cap = table_capacity(p.num_tokens);
    keys = static_cast<int*>(p.workspace);
    last = keys + cap;
    cudaError_t e = cudaMemsetAsync(keys, 0xff, 2 * sizeof(int) * (size_t)cap, stream);
    if (e != cudaSuccess) return e;
    slot_table_kernel<<<(p.num_tokens + 255) / 256, 256, 0, stream>>>(
        p.slot_mapping, p.num_tokens, (int64_t)p.num_blocks * p.block_size, keys, last, cap);
    add_launches(2);
  }
  if (p.act_dtype == B200_DTYPE_BFLOAT16)
    rotary_append_kernel<__nv_bfloat16><<<p.num_tokens, 256, 0, stream>>>(p, keys, last, cap);
  else
    rotary_append_kernel<__half><<<p.num_tokens, 256, 0, stream>>>(p, keys, last, cap);
  add_launches(1);
  return cudaGetLastError();
}

}  // namespace b200
