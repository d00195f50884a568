// Residual addition + RMS norm, with a 16-bit or fp8 e4m3 output (b200_skip_rms_norm).
//
//   s = x + residual;  y = s / sqrt(mean(s^2) + eps) * weight;  fp8: code = e4m3(y / scale),
//   scale = max|y| / 448 over the row or over a group of channels
//
// Memory bound (about 8 flops per 7 to 8 bytes).  One CTA owns a row and keeps its s in registers
// (ITEMS vectors of VEC channels per thread), so every input is read once and every output written
// once; the sum of squares and a row's maximum cross the CTA through shared memory, and a group of
// channels that lies inside a warp needs shuffles only.  With many rows a CTA walks several and has
// the next row's loads in flight during this row's reductions.  All sums are fp32.
//
// skip_rms_norm_shifted_kernel: rows that start off 16 bytes (odd widths, views), all tensors' alike: the
// vectors stay on 16-byte boundaries and the first and last of a row are taken by elements.  VEC 1 of
// the plain kernel is left for tensors whose rows start off 16 bytes differently.
#include <algorithm>

#include "b200_common.cuh"
#include "layer_kernels.h"

namespace b200 {
namespace {

constexpr float kFp8Max = 448.0f;
constexpr float kAmaxFloor = 1e-12f;  // an all-zero row or group still gets a scale above zero

template <int VEC> struct Raw;
template <> struct Raw<8> { using type = uint4; };
template <> struct Raw<1> { using type = uint16_t; };

template <typename T, int VEC>
__device__ __forceinline__ void unpack(const typename Raw<VEC>::type& raw, float (&v)[VEC]) {
  if constexpr (VEC == 1) {
    v[0] = act<T>::to_f(*reinterpret_cast<const T*>(&raw));
  } else {
    const uint32_t* w = reinterpret_cast<const uint32_t*>(&raw);
#pragma unroll
    for (int i = 0; i < VEC / 2; ++i) {
      const float2 f = mma_op<T>::unpack(w[i]);
      v[2 * i] = f.x;
      v[2 * i + 1] = f.y;
    }
  }
}

template <typename T, int VEC>
__device__ __forceinline__ typename Raw<VEC>::type pack(const float (&v)[VEC]) {
  typename Raw<VEC>::type raw;
  if constexpr (VEC == 1) {
    const T t = act<T>::from_f(v[0]);
    raw = *reinterpret_cast<const uint16_t*>(&t);
  } else {
    uint32_t* w = reinterpret_cast<uint32_t*>(&raw);
#pragma unroll
    for (int i = 0; i < VEC / 2; ++i) w[i] = mma_op<T>::pack(v[2 * i], v[2 * i + 1]);
  }
  return raw;
}

// VEC e4m3 codes of v * inv, saturating, as VEC bytes at dst (aligned to VEC).
template <int VEC>
__device__ __forceinline__ void store_e4m3(uint8_t* dst, const float (&v)[VEC], float inv) {
  if constexpr (VEC == 1) {
    *dst = (uint8_t)__nv_cvt_float_to_fp8(v[0] * inv, __NV_SATFINITE, __NV_E4M3);
  } else {
    uint32_t w[VEC / 4];
#pragma unroll
    for (int i = 0; i < VEC / 4; ++i) {
      const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(v[4 * i] * inv, v[4 * i + 1] * inv), __NV_SATFINITE, __NV_E4M3);
      const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(v[4 * i + 2] * inv, v[4 * i + 3] * inv), __NV_SATFINITE, __NV_E4M3);
      w[i] = lo | (hi << 16);
    }
    *reinterpret_cast<uint2*>(dst) = make_uint2(w[0], w[1]);
  }
}

// Maximum that keeps a NaN.
__device__ __forceinline__ float max_nan(float a, float b) {
  float d;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
  return d;
}

constexpr int kWalkThreads = 512;  // most threads of a walking CTA; its registers are limited for 1024 per SM

// WALK: rows blockIdx.x, + gridDim.x, ..; at most kWalkThreads threads.  Otherwise row blockIdx.x.
template <typename T, int VEC, int ITEMS, bool FP8, bool WALK>
__global__ void __launch_bounds__(WALK ? kWalkThreads : 1024, WALK ? 2 : 1)
    skip_rms_norm_kernel(const __grid_constant__ B200SkipRmsNormParams p) {
  using R = typename Raw<VEC>::type;
  // two of each, by the row's parity: a row's values are still read while the next row's are formed
  __shared__ float warp_sums[2][32];
  __shared__ int group_maxima[FP8 ? 2 : 1][FP8 ? B200_SKIP_RMS_NORM_MAX_HIDDEN / B200_SKIP_RMS_NORM_MIN_GROUP : 1];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, threads = blockDim.x;
  const int n = p.hidden / VEC;
  R xr[ITEMS], rr[ITEMS], wr[ITEMS];
  auto load = [&](int64_t row) {
    const T* x = static_cast<const T*>(p.x) + row * p.x_row_stride;
    const T* res = p.residual ? static_cast<const T*>(p.residual) + row * p.residual_row_stride : nullptr;
#pragma unroll
    for (int k = 0; k < ITEMS; ++k) {
      const int i = tid + k * threads;
      xr[k] = rr[k] = R{};
      if (i < n) {
        xr[k] = __ldcs(reinterpret_cast<const R*>(x + i * VEC));
        if (res) rr[k] = __ldcs(reinterpret_cast<const R*>(res + i * VEC));
      }
    }
  };
  load(blockIdx.x);
#pragma unroll
  for (int k = 0; k < ITEMS; ++k)
    wr[k] = tid + k * threads < n ? __ldg(reinterpret_cast<const R*>(p.weight) + tid + k * threads) : R{};

  int parity = 0;
  for (int64_t row = blockIdx.x; row < p.rows; row += gridDim.x, parity ^= 1) {
    float* warp_sum = warp_sums[parity];
    int* group_max = group_maxima[FP8 ? parity : 0];
    float s[ITEMS][VEC], sum = 0.f;
#pragma unroll
    for (int k = 0; k < ITEMS; ++k) {
      float r[VEC];
      unpack<T, VEC>(xr[k], s[k]);
      unpack<T, VEC>(rr[k], r);
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        s[k][j] += r[j];
        sum += s[k][j] * s[k][j];
      }
    }
    if (WALK && row + gridDim.x < p.rows) load(row + gridDim.x);
    if (p.residual_out) {
      T* ro = static_cast<T*>(p.residual_out) + row * p.residual_out_row_stride;
#pragma unroll
      for (int k = 0; k < ITEMS; ++k)
        if (tid + k * threads < n) *reinterpret_cast<R*>(ro + (tid + k * threads) * VEC) = pack<T, VEC>(s[k]);
    }
    const int groups = FP8 && p.group_size ? (p.hidden + p.group_size - 1) / p.group_size : 1;
    if (FP8)
      for (int i = tid; i < groups; i += threads) group_max[i] = 0;
#pragma unroll
    for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (lane == 0) warp_sum[warp] = sum;
    __syncthreads();
    sum = lane < (threads >> 5) ? warp_sum[lane] : 0.f;
#pragma unroll
    for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    const float rstd = 1.0f / sqrtf(sum / (float)p.hidden + p.epsilon);

#pragma unroll
    for (int k = 0; k < ITEMS; ++k) {
      float w[VEC];
      unpack<T, VEC>(wr[k], w);
#pragma unroll
      for (int j = 0; j < VEC; ++j) s[k][j] = s[k][j] * rstd * w[j];
    }
    if constexpr (!FP8) {
      T* out = static_cast<T*>(p.out) + row * p.out_row_stride;
#pragma unroll
      for (int k = 0; k < ITEMS; ++k)
        if (tid + k * threads < n) *reinterpret_cast<R*>(out + (tid + k * threads) * VEC) = pack<T, VEC>(s[k]);
    } else {
      uint8_t* out = static_cast<uint8_t*>(p.out) + row * p.out_row_stride;
      float* scales = p.scales + row * groups;
      const int group_log2 = __ffs(p.group_size) - 1;
    // lanes of one warp that share a group; a group wider than a warp is joined in shared memory
      const int lanes = p.group_size ? min(32, p.group_size / VEC) : 32;
      const bool in_warp = p.group_size != 0 && p.group_size <= 32 * VEC;
      float amax[ITEMS], row_max = 0.f;
#pragma unroll
      for (int k = 0; k < ITEMS; ++k) {
        float m = 0.f;
        if (tid + k * threads < n) {
#pragma unroll
          for (int j = 0; j < VEC; ++j) m = max_nan(m, fabsf(s[k][j]));
        }
        amax[k] = m;
        row_max = max_nan(row_max, m);
      }
      if (!p.group_size) {
#pragma unroll
        for (int o = 16; o; o >>= 1) row_max = max_nan(row_max, __shfl_xor_sync(0xffffffffu, row_max, o));
        // magnitudes order like their bit patterns, a NaN above all
        if (lane == 0) atomicMax(&group_max[0], __float_as_int(row_max));
        __syncthreads();
        const float scale = max_nan(__int_as_float(group_max[0]), kAmaxFloor) / kFp8Max;
#pragma unroll
        for (int k = 0; k < ITEMS; ++k) amax[k] = scale;
        if (tid == 0) scales[0] = scale;
      } else {
#pragma unroll
        for (int k = 0; k < ITEMS; ++k)
          for (int o = lanes >> 1; o; o >>= 1) amax[k] = max_nan(amax[k], __shfl_xor_sync(0xffffffffu, amax[k], o));
        if (!in_warp) {
#pragma unroll
          for (int k = 0; k < ITEMS; ++k)
            if (lane == 0 && tid + k * threads < n)
              atomicMax(&group_max[(tid + k * threads) * VEC >> group_log2], __float_as_int(amax[k]));
          __syncthreads();
        }
#pragma unroll
        for (int k = 0; k < ITEMS; ++k) {
          const int c = (tid + k * threads) * VEC;
          if (c >= p.hidden) continue;
          const int g = c >> group_log2;
          if (!in_warp) amax[k] = __int_as_float(group_max[g]);
          amax[k] = max_nan(amax[k], kAmaxFloor) / kFp8Max;
          if (c == g << group_log2) scales[g] = amax[k];
        }
      }
#pragma unroll
      for (int k = 0; k < ITEMS; ++k)
        if (tid + k * threads < n) store_e4m3<VEC>(out + (tid + k * threads) * VEC, s[k], 1.0f / amax[k]);
    }
  }
}

// Rows whose first elements all lie `shift` elements past a 16-byte boundary (the same for every row of a
// CTA: the grid is a multiple of 8).  Vector v holds row elements 8 v - shift .. + 7.
template <typename T, int ITEMS, bool FP8, bool WALK>
__global__ void __launch_bounds__(WALK ? kWalkThreads : 1024, WALK && ITEMS <= 2 ? 2 : 1)
    skip_rms_norm_shifted_kernel(const __grid_constant__ B200SkipRmsNormParams p) {
  __shared__ float warp_sums[2][32];
  __shared__ int group_maxima[FP8 ? 2 : 1][FP8 ? B200_SKIP_RMS_NORM_MAX_HIDDEN / B200_SKIP_RMS_NORM_MIN_GROUP : 1];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, threads = blockDim.x, h = p.hidden;
  const int shift = (int)((reinterpret_cast<uintptr_t>(static_cast<const T*>(p.x) + blockIdx.x * p.x_row_stride) & 15) / 2);
  const int n = (shift + h + 7) / 8;
  auto first = [&](int k) { return (tid + k * threads) * 8 - shift; };  // row element of the k-th vector's start
  auto store_vector = [&](T* row, int e, const uint4& v) {
    if (e >= 0 && e + 8 <= h) {
      *reinterpret_cast<uint4*>(row + e) = v;
      return;
    }
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (e + j >= 0 && e + j < h) reinterpret_cast<uint16_t*>(row)[e + j] = (uint16_t)(w[j / 2] >> (j % 2 * 16));
  };
  uint4 xr[ITEMS], rr[ITEMS], wr[ITEMS];
  auto load = [&](int64_t row) {
    const T* x = static_cast<const T*>(p.x) + row * p.x_row_stride;
    const T* res = p.residual ? static_cast<const T*>(p.residual) + row * p.residual_row_stride : nullptr;
#pragma unroll
    for (int k = 0; k < ITEMS; ++k) {
      xr[k] = rr[k] = make_uint4(0, 0, 0, 0);
      if (tid + k * threads < n) {
        // a vector at a row's edge is loaded whole, too: its 16 bytes hold an element of the row, so they
        // lie in the same allocation; what is not the row's is dropped when s is formed
        xr[k] = __ldcs(reinterpret_cast<const uint4*>(x + first(k)));
        if (res) rr[k] = __ldcs(reinterpret_cast<const uint4*>(res + first(k)));
      }
    }
  };
  load(blockIdx.x);
#pragma unroll
  for (int k = 0; k < ITEMS; ++k) {  // the weights lie off the rows' boundaries: by elements, once
    uint32_t w[4] = {0, 0, 0, 0};
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (first(k) + j >= 0 && first(k) + j < h)
        w[j / 2] |= (uint32_t)__ldg(static_cast<const uint16_t*>(p.weight) + first(k) + j) << (j % 2 * 16);
    wr[k] = make_uint4(w[0], w[1], w[2], w[3]);
  }
  const int groups = FP8 && p.group_size ? (h + p.group_size - 1) / p.group_size : 1;
  const int group_log2 = p.group_size ? __ffs(p.group_size) - 1 : 31;

  int parity = 0;
  for (int64_t row = blockIdx.x; row < p.rows; row += gridDim.x, parity ^= 1) {
    float* warp_sum = warp_sums[parity];
    int* group_max = group_maxima[FP8 ? parity : 0];
    float s[ITEMS][8], sum = 0.f;
#pragma unroll
    for (int k = 0; k < ITEMS; ++k) {
      float r[8];
      unpack<T, 8>(xr[k], s[k]);
      unpack<T, 8>(rr[k], r);
#pragma unroll
      for (int j = 0; j < 8; ++j) s[k][j] += r[j];
      if (first(k) < 0 || first(k) + 8 > h) {
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (first(k) + j < 0 || first(k) + j >= h) s[k][j] = 0.f;
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) sum += s[k][j] * s[k][j];
    }
    if (WALK && row + gridDim.x < p.rows) load(row + gridDim.x);
    if (p.residual_out) {
      T* ro = static_cast<T*>(p.residual_out) + row * p.residual_out_row_stride;
#pragma unroll
      for (int k = 0; k < ITEMS; ++k)
        if (tid + k * threads < n) store_vector(ro, first(k), pack<T, 8>(s[k]));
    }
    if (FP8)
      for (int i = tid; i < groups; i += threads) group_max[i] = 0;
#pragma unroll
    for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (lane == 0) warp_sum[warp] = sum;
    __syncthreads();
    sum = lane < (threads >> 5) ? warp_sum[lane] : 0.f;
#pragma unroll
    for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    const float rstd = 1.0f / sqrtf(sum / (float)h + p.epsilon);
#pragma unroll
    for (int k = 0; k < ITEMS; ++k) {
      float w[8];
      unpack<T, 8>(wr[k], w);
#pragma unroll
      for (int j = 0; j < 8; ++j) s[k][j] = s[k][j] * rstd * w[j];
    }
    if constexpr (!FP8) {
      T* out = static_cast<T*>(p.out) + row * p.out_row_stride;
#pragma unroll
      for (int k = 0; k < ITEMS; ++k)
        if (tid + k * threads < n) store_vector(out, first(k), pack<T, 8>(s[k]));
    } else {
      uint8_t* out = static_cast<uint8_t*>(p.out) + row * p.out_row_stride;
      float* scales = p.scales + row * groups;
      // Elements outside the row are zeros here.  A vector meets at most two groups (one without groups),
      // a warp's 256 channels a few: the largest magnitude of each.
      if (!p.group_size) {
        float m = 0.f;
#pragma unroll
        for (int k = 0; k < ITEMS; ++k)
#pragma unroll
          for (int j = 0; j < 8; ++j) m = max_nan(m, fabsf(s[k][j]));
        // magnitudes order like their bit patterns, a NaN above all
        const int top = __reduce_max_sync(0xffffffffu, __float_as_int(m));
        if (lane == 0) atomicMax(&group_max[0], top);
      } else {
#pragma unroll
        for (int k = 0; k < ITEMS; ++k) {
          const int e = first(k), e_warp = e - lane * 8;
          if (e_warp >= h) continue;
          const int g0 = max(e, 0) >> group_log2, next = (g0 + 1 << group_log2) - e;  // first element of group g0 + 1
          float m0 = 0.f, m1 = 0.f;
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const float y = fabsf(s[k][j]);
            m0 = j < next ? max_nan(m0, y) : m0;
            m1 = j < next ? m1 : max_nan(m1, y);
          }
          const int g_end = min(e_warp + 255, h - 1) >> group_log2;
          for (int g = max(e_warp, 0) >> group_log2; g <= g_end; ++g) {
            const int top = __reduce_max_sync(0xffffffffu, __float_as_int(g == g0 ? m0 : g == g0 + 1 ? m1 : 0.f));
            if (lane == 0) atomicMax(&group_max[g], top);
          }
        }
      }
      __syncthreads();
      for (int i = tid; i < groups; i += threads) scales[i] = max_nan(__int_as_float(group_max[i]), kAmaxFloor) / kFp8Max;
#pragma unroll
      for (int k = 0; k < ITEMS; ++k) {
        const int e = first(k);
        if (tid + k * threads >= n) continue;
        const int g0 = max(e, 0) >> group_log2, g1 = min(e + 7, h - 1) >> group_log2, next = (g1 << group_log2) - e;
        const float inv0 = 1.0f / (max_nan(__int_as_float(group_max[g0]), kAmaxFloor) / kFp8Max);
        const float inv1 = g1 == g0 ? inv0 : 1.0f / (max_nan(__int_as_float(group_max[g1]), kAmaxFloor) / kFp8Max);
        float y[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) y[j] = s[k][j] * (j < next ? inv0 : inv1);
        if (e >= 0 && e + 8 <= h) {
          store_e4m3<8>(out + e, y, 1.0f);
        } else {
#pragma unroll
          for (int j = 0; j < 8; ++j)
            if (e + j >= 0 && e + j < h) out[e + j] = (uint8_t)__nv_cvt_float_to_fp8(y[j], __NV_SATFINITE, __NV_E4M3);
        }
      }
    }
  }
}

template <typename T, int ITEMS, bool WALK>
void launch_shifted_items(const B200SkipRmsNormParams& p, int vectors, int num_sms, cudaStream_t stream) {
  const int threads = (vectors + 32 * ITEMS - 1) / (32 * ITEMS) * 32;
  // walking CTAs keep the rows' shift: the grid is a multiple of 8
  const int grid = WALK ? std::max(8, num_sms * std::max(1, 1024 / threads) / 8 * 8) : p.rows;
  if (p.out_dtype == B200_DTYPE_FLOAT8E4M3FN)
    skip_rms_norm_shifted_kernel<T, ITEMS, true, WALK><<<grid, threads, 0, stream>>>(p);
  else
    skip_rms_norm_shifted_kernel<T, ITEMS, false, WALK><<<grid, threads, 0, stream>>>(p);
}

template <typename T>
void launch_shifted(const B200SkipRmsNormParams& p, int num_sms, cudaStream_t stream) {
  const int vectors = (p.hidden + 14) / 8;  // at the largest shift
  if (p.rows > 4 * num_sms && p.rows >= 16 && vectors <= 3 * kWalkThreads) {
    if (vectors <= 128) launch_shifted_items<T, 1, true>(p, vectors, num_sms, stream);
    else if (vectors <= 2 * kWalkThreads) launch_shifted_items<T, 2, true>(p, vectors, num_sms, stream);
    else launch_shifted_items<T, 3, true>(p, vectors, num_sms, stream);
  } else if (vectors <= 1024) {
    launch_shifted_items<T, 1, false>(p, vectors, num_sms, stream);
  } else {
    launch_shifted_items<T, 5, false>(p, vectors, num_sms, stream);
  }
}

template <typename T, int VEC, int ITEMS, bool WALK>
void launch_items(const B200SkipRmsNormParams& p, int num_sms, cudaStream_t stream) {
  const int threads = (p.hidden / VEC + 32 * ITEMS - 1) / (32 * ITEMS) * 32;
  const int grid = WALK ? std::min(p.rows, num_sms * std::max(1, 1024 / threads)) : p.rows;
  if (p.out_dtype == B200_DTYPE_FLOAT8E4M3FN)
    skip_rms_norm_kernel<T, VEC, ITEMS, true, WALK><<<grid, threads, 0, stream>>>(p);
  else
    skip_rms_norm_kernel<T, VEC, ITEMS, false, WALK><<<grid, threads, 0, stream>>>(p);
}

// Few rows: as many threads as there are vectors, for the shortest row.  Many rows: two vectors per thread
// in CTAs that walk, 1024 threads per SM (960 and 768 were up to 30 % slower at 8192 channels).
template <typename T, int VEC>
void launch_vec(const B200SkipRmsNormParams& p, int num_sms, cudaStream_t stream) {
  const int n = p.hidden / VEC;
  if (p.rows > 4 * num_sms && n <= 2 * kWalkThreads) {
    if (n <= 128) launch_items<T, VEC, 1, true>(p, num_sms, stream);
    else launch_items<T, VEC, 2, true>(p, num_sms, stream);
  } else if (n <= 1024) {
    launch_items<T, VEC, 1, false>(p, num_sms, stream);
  } else if (n <= 4096) {
    launch_items<T, VEC, 4, false>(p, num_sms, stream);
  } else if constexpr (VEC == 1) {
    launch_items<T, VEC, 32, false>(p, num_sms, stream);
  }
}

template <typename T>
void launch_type(const B200SkipRmsNormParams& p, int num_sms, cudaStream_t stream) {
  // where the rows of each tensor start: elements past a multiple of 8, for row 0 and from row to row
  const int out_size = p.out_dtype == p.dtype ? 2 : 1;
  struct Rows {
    uintptr_t base;
    int64_t stride;
  } const tensors[] = {{reinterpret_cast<uintptr_t>(p.x) / 2, p.x_row_stride},
                       {reinterpret_cast<uintptr_t>(p.out) / out_size, p.out_row_stride},
                       {reinterpret_cast<uintptr_t>(p.residual) / 2, p.residual_row_stride},
                       {reinterpret_cast<uintptr_t>(p.residual_out) / 2, p.residual_out_row_stride}};
  const bool given[] = {true, true, p.residual != nullptr, p.residual_out != nullptr};
  bool alike = true, aligned = reinterpret_cast<uintptr_t>(p.weight) % 16 == 0 && p.hidden % 8 == 0;
  for (int i = 0; i < 4; ++i) {
    if (!given[i]) continue;
    alike &= (tensors[i].base - tensors[0].base) % 8 == 0 && (p.rows == 1 || (tensors[i].stride - tensors[0].stride) % 8 == 0);
    aligned &= tensors[i].base % 8 == 0 && (p.rows == 1 || tensors[i].stride % 8 == 0);
  }
  if (aligned) launch_vec<T, 8>(p, num_sms, stream);
  else if (alike) launch_shifted<T>(p, num_sms, stream);
  else launch_vec<T, 1>(p, num_sms, stream);
}

}  // namespace

cudaError_t launch_skip_rms_norm(const B200SkipRmsNormParams& p, int num_sms, cudaStream_t stream) {
  if (p.dtype == B200_DTYPE_BFLOAT16) launch_type<__nv_bfloat16>(p, num_sms, stream);
  else launch_type<__half>(p, num_sms, stream);
  add_launches(1);
  return cudaGetLastError();
}

}  // namespace b200
