// Rotary embedding of new queries and keys with up to four position axes, and the append of keys
// and values to the paged caches, in one pass (b200_rotary_append).
//
//   pair (x0, x1) -> (x0 c - x1 s, x1 c + x0 s) in fp32, rounded once; c, s from row
//   position[axis of the pair] of the tables
//
// Memory bound: every query, key and value row is read once and written once.  Measured, bf16, 128-wide
// heads: 8192 tokens of 32 + 8 + 8 heads with three axes 42 us (201 MB, 0.73 of 6.5 TB/s), 4096 tokens of
// 64 + 8 + 8 heads into an fp8 cache 36 us (160 MB, 0.68), 1001 tokens of 14 + 2 + 2 heads of 64 channels
// 5.4 us, 128 tokens 3.0 us.  The search for later tokens with the same slot is 3.3, 2.4, 1.0 and 0.5 us
// of these; a table filled first costs two launches more.
//
// rotary_append_vec_kernel: a thread owns a unit of 16 channels (two 16-byte pieces: the two halves
// of 8 rotary pairs, or 16 channels that do not turn) and walks the token's heads with it.  The cos and
// sin values of a CTA's tokens, gathered once per pair (axes may change anywhere between pairs), wait in
// shared memory and stay in registers over the heads; the loads of a token's next heads are in flight as
// one is stored (1001 tokens: 6.7 us when they went out in batches).  rotary_append_kernel takes what is
// not aligned to such units.
//
// Of several tokens with one slot the last is stored.  Up to B200_ROTARY_APPEND_SCAN_TOKENS tokens,
// a CTA compares its tokens' slots with every later one (up to 4 tokens per CTA share the reads of
// the list); beyond, where that work grows with the square, a hash table is filled first.
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

// Whether a later token names the same slot, for the TOKENS tokens from t0 on (bit i: token t0 + i).
// A CTA barrier.
template <int TOKENS>
__device__ __forceinline__ int later_same_slot(const B200RotaryAppendParams& p, int64_t t0, const int32_t (&slot)[TOKENS]) {
  const int tid = threadIdx.x, threads = blockDim.x;
  const int32_t* list = p.slot_mapping;
  const int64_t n = p.num_tokens, from = t0 + TOKENS;
  bool hit[TOKENS];
#pragma unroll
  for (int i = 0; i < TOKENS; ++i) {
    hit[i] = false;
#pragma unroll
    for (int j = i + 1; j < TOKENS; ++j) hit[i] |= slot[i] == slot[j];
  }
  auto compare = [&](int32_t other) {
#pragma unroll
    for (int i = 0; i < TOKENS; ++i) hit[i] |= slot[i] == other;
  };
  if (from < n) {  // up to the next 16-byte boundary, whole vectors, the rest
    const int rest = (int)(n - from);
    const int head = min(rest, (int)(-(reinterpret_cast<uintptr_t>(list + from) >> 2) & 3)), vecs = (rest - head) / 4;
    const int32_t* first = list + from;
    const int4* wide = reinterpret_cast<const int4*>(first + head);
    if (tid < head) compare(__ldg(first + tid));
#pragma unroll 4
    for (int v = tid; v < vecs; v += threads) {
      const int4 w = __ldg(wide + v);
      compare(w.x);
      compare(w.y);
      compare(w.z);
      compare(w.w);
    }
    const int tail = head + vecs * 4 + tid;
    if (tail < rest) compare(__ldg(first + tail));
  }
  bool any = false;
#pragma unroll
  for (int i = 0; i < TOKENS; ++i) any |= hit[i];
  if (!__syncthreads_or(any)) return 0;
  int later = 0;
#pragma unroll
  for (int i = 0; i < TOKENS; ++i) later |= (__syncthreads_or(hit[i]) ? 1 : 0) << i;
  return later;
}

template <typename T>
__device__ __forceinline__ void unpack8(const uint4& w, float (&v)[8]) {
  const uint32_t r[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = mma_op<T>::unpack(r[i]);
    v[2 * i] = f.x;
    v[2 * i + 1] = f.y;
  }
}

template <typename T>
__device__ __forceinline__ uint4 pack8(const float (&v)[8]) {
  return make_uint4(mma_op<T>::pack(v[0], v[1]), mma_op<T>::pack(v[2], v[3]), mma_op<T>::pack(v[4], v[5]),
                    mma_op<T>::pack(v[6], v[7]));
}

// 8 e4m3 codes of v / scale, saturating (IEEE division: the bytes b200_kv_append writes).
__device__ __forceinline__ uint2 e4m3x8(const float (&v)[8], float scale) {
  uint32_t w[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const uint32_t lo = __nv_cvt_float2_to_fp8x2(
        make_float2(__fdiv_rn(v[4 * i], scale), __fdiv_rn(v[4 * i + 1], scale)), __NV_SATFINITE, __NV_E4M3);
    const uint32_t hi = __nv_cvt_float2_to_fp8x2(
        make_float2(__fdiv_rn(v[4 * i + 2], scale), __fdiv_rn(v[4 * i + 3], scale)), __NV_SATFINITE, __NV_E4M3);
    w[i] = lo | (hi << 16);
  }
  return make_uint2(w[0], w[1]);
}

constexpr int kVecThreads = 128;

// The cos and sin values of TOKENS tokens from t0 on into shared memory, [token][pair] each (1 and 0
// where a position is out of range).
template <typename T, int TOKENS>
__device__ __forceinline__ void load_turns(const B200RotaryAppendParams& p, int64_t t0, int half, float* cos_s, float* sin_s) {
  bool bad = false;
  for (int j = threadIdx.x; j < TOKENS * half; j += blockDim.x) {
    const int i = TOKENS == 1 ? 0 : j / half, pair = j - i * half;
    if (t0 + i >= p.num_tokens) break;
    const int64_t pos = position_of(p, p.axes == 1 ? 0 : axis_of(p, pair), t0 + i);
    const bool in = pos >= 0 && pos < p.rotary_positions;
    cos_s[j] = in ? table_value<T>(p, p.cos_cache, pos * half + pair) : 1.f;
    sin_s[j] = in ? table_value<T>(p, p.sin_cache, pos * half + pair) : 0.f;
    bad |= !in;
  }
  if (bad) set_status(p.device_status, kStatusBadPosition);
}

// Turn a unit: pairs (a[j], b[j]), or the neighbours of the 16 contiguous channels a, b.
__device__ __forceinline__ void turn(bool interleaved, const float (&c)[8], const float (&s)[8], float (&a)[8], float (&b)[8]) {
  auto pair = [](float& x0, float& x1, float co, float si) {
    const float y0 = x0 * co - x1 * si;
    x1 = x1 * co + x0 * si;
    x0 = y0;
  };
  if (interleaved) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      pair(a[2 * j], a[2 * j + 1], c[j], s[j]);
      pair(b[2 * j], b[2 * j + 1], c[4 + j], s[4 + j]);
    }
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) pair(a[j], b[j], c[j], s[j]);
  }
}

// CTA: TOKENS tokens x heads [blockIdx.y * cta_heads, + cta_heads) of the query, key and value heads in
// that order.  A warp owns one token; a lane owns (unit of `units`, head offset), lanes past the last
// whole head idle.  kBatch heads' loads are in flight: as one is stored, the load kBatch heads on goes out.
template <typename T, bool FP8, int TOKENS>
__global__ void __launch_bounds__(kVecThreads, 5) rotary_append_vec_kernel(const __grid_constant__ B200RotaryAppendParams p,
                                                                            const int* keys, const int* last,
                                                                            uint32_t capacity, int units, int cta_heads) {
  constexpr int kBatch = 4;
  const int64_t t0 = (int64_t)blockIdx.x * TOKENS;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int unit = lane % units, warp_heads = 32 / units;
  const int d = p.head_size, H = p.num_heads, KV = p.kv_num_heads, half = p.rotary_dim / 2;
  const int i = warp % TOKENS;  // this warp's token
  const int head_step = warp_heads * (kVecThreads / 32 / TOKENS);
  const int h_first = blockIdx.y * cta_heads + warp / TOKENS * warp_heads + lane / units;
  const int h_end = min(H + 2 * KV, (int)(blockIdx.y + 1) * cta_heads);
  const bool turns = unit < p.rotary_dim / 16, interleaved = p.rotary_interleaved != 0;
  // first channels of the unit's two pieces in query and key heads
  int ca, cb;
  if (turns) {
    ca = p.rotary_offset + (interleaved ? 16 * unit : 8 * unit);
    cb = interleaved ? ca + 8 : ca + half;
  } else {
    ca = 16 * (unit - p.rotary_dim / 16);
    cb = ca + 8;
    ca += ca < p.rotary_offset ? 0 : p.rotary_dim;
    cb += cb < p.rotary_offset ? 0 : p.rotary_dim;
  }
  const int64_t t = t0 + i;
  const bool active = t < p.num_tokens && lane / units < warp_heads;
  const T* q = static_cast<const T*>(p.query) + t * p.query_row_stride;
  const T* krow = static_cast<const T*>(p.key) + t * p.key_row_stride;
  const T* vrow = static_cast<const T*>(p.value) + t * p.value_row_stride;
  uint4 xa[kBatch], xb[kBatch];
  auto load = [&](int k, int h) {
    const bool value = h >= H + KV;
    const T* row = h < H ? q + h * d : value ? vrow + (h - H - KV) * d : krow + (h - H) * d;
    xa[k] = *reinterpret_cast<const uint4*>(row + (value ? 16 * unit : ca));
    xb[k] = *reinterpret_cast<const uint4*>(row + (value ? 16 * unit + 8 : cb));
  };
#pragma unroll
  for (int k = 0; k < kBatch; ++k)  // in flight during the gather and the search below
    if (active && h_first + k * head_step < h_end) load(k, h_first + k * head_step);
  extern __shared__ float turns_s[];  // cos [TOKENS][half], sin [TOKENS][half]
  load_turns<T, TOKENS>(p, t0, half, turns_s, turns_s + TOKENS * half);
  int32_t slot = -1;
  bool keep = false;
  if (h_end > H) {  // this CTA has rows to store
    int32_t slots[TOKENS];
#pragma unroll
    for (int j = 0; j < TOKENS; ++j) {
      slots[j] = t0 + j < p.num_tokens ? __ldg(p.slot_mapping + t0 + j) : -1;
      if (j == i) slot = slots[j];
    }
    const bool valid = slot >= -1 && (int64_t)slot < (int64_t)p.num_blocks * p.block_size;
    if (!valid && lane == 0) set_status(p.device_status, kStatusBadSlot);
    keep = valid && slot >= 0;
    if (!keys) keep &= !(later_same_slot<TOKENS>(p, t0, slots) >> i & 1);
    else if (keep) keep = last_token(slot, (int)(t0 + i), keys, last, capacity) == (int)(t0 + i);
  }
  __syncthreads();
  if (!active) return;
  float c[8], s[8];
  if (turns) {
    const float4* cp = reinterpret_cast<const float4*>(turns_s + i * half + 8 * unit);
    const float4* sp = reinterpret_cast<const float4*>(turns_s + (TOKENS + i) * half + 8 * unit);
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const float4 cv = cp[j], sv = sp[j];
      c[4 * j] = cv.x; c[4 * j + 1] = cv.y; c[4 * j + 2] = cv.z; c[4 * j + 3] = cv.w;
      s[4 * j] = sv.x; s[4 * j + 1] = sv.y; s[4 * j + 2] = sv.z; s[4 * j + 3] = sv.w;
    }
  }
  T* out = static_cast<T*>(p.output) + t * p.output_row_stride;
  const int64_t at = (int64_t)slot * KV * d;  // cache row of the token
  // the rows that go out as they are or turned: all, or the queries beside an fp8 cache
  const int end = keep && !FP8 ? h_end : min(H, h_end);
  int h0 = h_first;
  for (; h0 < end; h0 += kBatch * head_step) {
#pragma unroll
    for (int k = 0; k < kBatch; ++k) {
      const int h = h0 + k * head_step;
      if (h >= end) break;
      const bool value = h >= H + KV;
      if (turns && !value) {
        float a[8], b[8];
        unpack8<T>(xa[k], a);
        unpack8<T>(xb[k], b);
        turn(interleaved, c, s, a, b);
        xa[k] = pack8<T>(a);
        xb[k] = pack8<T>(b);
      }
      T* row = h < H ? out + h * d : static_cast<T*>(value ? p.value_cache : p.key_cache) + at + (h - H - (value ? KV : 0)) * d;
      *reinterpret_cast<uint4*>(row + (value ? 16 * unit : ca)) = xa[k];
      *reinterpret_cast<uint4*>(row + (value ? 16 * unit + 8 : cb)) = xb[k];
      if (h + kBatch * head_step < end) load(k, h + kBatch * head_step);
    }
  }
  if constexpr (FP8) {  // in batches of their own: the divisions leave no registers for more (39 against 36 us)
    if (!keep) return;
    h0 = h_first + (h_first < H ? (H - h_first + head_step - 1) / head_step * head_step : 0);
    const float* k_scale = p.k_scale + (int64_t)(slot / p.block_size) * KV;
    const float* v_scale = p.v_scale + (int64_t)(slot / p.block_size) * KV;
    for (; h0 < h_end; h0 += kBatch * head_step) {
      float scale[kBatch];
#pragma unroll
      for (int k = 0; k < kBatch; ++k) {
        const int h = h0 + k * head_step;
        if (h >= h_end) break;
        load(k, h);
        scale[k] = __ldg(h >= H + KV ? v_scale + (h - H - KV) : k_scale + (h - H));
      }
#pragma unroll
      for (int k = 0; k < kBatch; ++k) {
        const int h = h0 + k * head_step;
        if (h >= h_end) break;
        const bool value = h >= H + KV;
        float a[8], b[8];
        unpack8<T>(xa[k], a);
        unpack8<T>(xb[k], b);
        if (turns && !value) turn(interleaved, c, s, a, b);
        uint8_t* row = static_cast<uint8_t*>(value ? p.value_cache : p.key_cache) + at + (h - H - (value ? KV : 0)) * d;
        *reinterpret_cast<uint2*>(row + (value ? 16 * unit : ca)) = e4m3x8(a, scale[k]);
        *reinterpret_cast<uint2*>(row + (value ? 16 * unit + 8 : cb)) = e4m3x8(b, scale[k]);
      }
    }
  }
}

// Whether every head splits into 16-byte pieces as the vector kernel reads and writes them.
bool vector_form(const B200RotaryAppendParams& p) {
  const uintptr_t bases = reinterpret_cast<uintptr_t>(p.query) | reinterpret_cast<uintptr_t>(p.key) |
                          reinterpret_cast<uintptr_t>(p.value) | reinterpret_cast<uintptr_t>(p.output) |
                          reinterpret_cast<uintptr_t>(p.key_cache) | reinterpret_cast<uintptr_t>(p.value_cache) |
                          reinterpret_cast<uintptr_t>(p.cos_cache) | reinterpret_cast<uintptr_t>(p.sin_cache);
  const int64_t strides = p.query_row_stride | p.key_row_stride | p.value_row_stride | p.output_row_stride;
  return bases % 16 == 0 && strides % 8 == 0 && p.head_size % 16 == 0 && p.head_size / 16 <= 32 &&
         p.rotary_dim % 16 == 0 && p.rotary_offset % 8 == 0;
}

template <typename T, bool FP8>
void launch_vec(const B200RotaryAppendParams& p, const int* keys, const int* last, uint32_t cap, int num_sms,
                cudaStream_t stream) {
  const int units = p.head_size / 16, heads = p.num_heads + 2 * p.kv_num_heads;
  const size_t turns = sizeof(float) * (size_t)p.rotary_dim;  // cos and sin of one token
  if (p.num_tokens < 16 * num_sms) {
    // Few tokens: a token's heads spread over CTAs, one per lane, while that leaves the SMs at most 8
    // CTAs each, for the shortest chain of loads.
    const int pass = 32 / units * (kVecThreads / 32);
    const unsigned passes = (unsigned)((heads + pass - 1) / pass);
    const bool spread = (int64_t)p.num_tokens * passes <= 8 * (int64_t)num_sms;
    rotary_append_vec_kernel<T, FP8, 1><<<dim3(p.num_tokens, spread ? passes : 1), kVecThreads, turns, stream>>>(
        p, keys, last, cap, units, spread ? pass : heads);
  } else if (p.num_tokens < 48 * num_sms) {  // smaller CTAs fill the last wave better
    rotary_append_vec_kernel<T, FP8, 2><<<dim3((p.num_tokens + 1) / 2), kVecThreads, 2 * turns, stream>>>(
        p, keys, last, cap, units, heads);
  } else {  // 4 tokens share the reads of the slot list
    rotary_append_vec_kernel<T, FP8, 4><<<dim3((p.num_tokens + 3) / 4), kVecThreads, 4 * turns, stream>>>(
        p, keys, last, cap, units, heads);
  }
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

cudaError_t launch_rotary_append(const B200RotaryAppendParams& p, int num_sms, cudaStream_t stream) {
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
  const bool bf = p.act_dtype == B200_DTYPE_BFLOAT16;
  if (vector_form(p)) {
    if (p.cache_dtype == B200_DTYPE_FLOAT8E4M3FN) {
      if (bf) launch_vec<__nv_bfloat16, true>(p, keys, last, cap, num_sms, stream);
      else launch_vec<__half, true>(p, keys, last, cap, num_sms, stream);
    } else {
      if (bf) launch_vec<__nv_bfloat16, false>(p, keys, last, cap, num_sms, stream);
      else launch_vec<__half, false>(p, keys, last, cap, num_sms, stream);
    }
  } else if (bf)
    rotary_append_kernel<__nv_bfloat16><<<p.num_tokens, 256, 0, stream>>>(p, keys, last, cap);
  else
    rotary_append_kernel<__half><<<p.num_tokens, 256, 0, stream>>>(p, keys, last, cap);
  add_launches(1);
  return cudaGetLastError();
}

}  // namespace b200
