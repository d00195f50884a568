// Residual addition + RMS norm, with a 16-bit or fp8 e4m3 output (b200_skip_rms_norm).
//
//   s = x + residual;  y = s / sqrt(mean(s^2) + eps) * weight;  fp8: code = e4m3(y / scale),
//   scale = max|y| / 448 over the row or over a group of channels
//
// Memory bound (about 8 flops per 7 to 8 bytes); what comes next is the issue of instructions, so the
// arithmetic is on packed fp32 pairs and a row's fixed work (reductions, square root, divisions) is short:
// 16384 x 4096 in groups of 128 went from 92 to 78 us with that.  A row's s stays in registers (ITEMS
// vectors of VEC channels per thread), so every input is read once and every output written once.  All
// sums are fp32; a row's or group's maximum crosses warps through shared memory.
//
// Who owns a row (launch_vec): a CTA with few rows (latency: a short row for each thread), with many rows
// a warp up to 1024 channels (no barriers) and a CTA beyond; those walk over rows and have the next row's
// loads in flight during this row's reductions.
//
// skip_rms_norm_shifted_kernel: rows that start off 16 bytes (odd widths, views), all tensors' alike: the
// vectors lie on 16-byte boundaries and the elements before and after them are taken singly.  VEC 1 of
// the plain kernel is left for tensors whose rows start off 16 bytes differently.
//
// Measured, bf16 (MB moved, share of 6.5 TB/s): 16384 x 4096 to fp8 rows 77 us (470 MB, 0.94), in groups
// of 128 78 us; 16384 x 512 to bf16 9.4 us (67 MB); 16384 x 513 10.1 us; 4096 x 16384 to bf16 87 us
// (537 MB, 0.95), 4096 x 12289 69 us (403 MB, 0.90); 200 x 256 1.9 us, the launch.
#include <algorithm>

#include "b200_common.cuh"
#include "b200_tcgen05.cuh"
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

// VEC e4m3 codes of v, saturating, as VEC bytes at dst (aligned to VEC).
template <int VEC>
__device__ __forceinline__ void store_e4m3(uint8_t* dst, const float (&v)[VEC]) {
  if constexpr (VEC == 1) {
    *dst = (uint8_t)__nv_cvt_float_to_fp8(v[0], __NV_SATFINITE, __NV_E4M3);
  } else {
    uint32_t w[VEC / 4];
#pragma unroll
    for (int i = 0; i < VEC / 4; ++i) {
      const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(v[4 * i], v[4 * i + 1]), __NV_SATFINITE, __NV_E4M3);
      const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(v[4 * i + 2], v[4 * i + 3]), __NV_SATFINITE, __NV_E4M3);
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
__device__ __forceinline__ float max_nan(float a, float b, float c) {
  float d;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}

// The arithmetic on VEC channels, two to an instruction.
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  float2 d;
  asm("{\n\t.reg .b64 ra, rb, rd;\n\tmov.b64 ra, {%2, %3};\n\tmov.b64 rb, {%4, %5};\n\t"
      "mul.rn.f32x2 rd, ra, rb;\n\tmov.b64 {%0, %1}, rd;\n\t}"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}
template <int VEC, typename F1, typename F2>
__device__ __forceinline__ void each(float (&a)[VEC], F1 one, F2 two) {
  if constexpr (VEC == 1) {
    a[0] = one(a[0], 0);
  } else {
#pragma unroll
    for (int j = 0; j < VEC; j += 2) {
      const float2 y = two(make_float2(a[j], a[j + 1]), j);
      a[j] = y.x;
      a[j + 1] = y.y;
    }
  }
}
template <int VEC>
__device__ __forceinline__ void add(float (&a)[VEC], const float (&b)[VEC]) {
  each<VEC>(a, [&](float x, int) { return x + b[0]; },
            [&](float2 x, int j) { return tc::add2(x, make_float2(b[j], b[j + 1])); });
}
template <int VEC>
__device__ __forceinline__ void multiply(float (&a)[VEC], const float (&b)[VEC]) {
  each<VEC>(a, [&](float x, int) { return x * b[0]; }, [&](float2 x, int j) { return mul2(x, make_float2(b[j], b[j + 1])); });
}
template <int VEC>
__device__ __forceinline__ void scale_by(float (&a)[VEC], float f) {
  each<VEC>(a, [&](float x, int) { return x * f; }, [&](float2 x, int) { return mul2(x, make_float2(f, f)); });
}
template <int VEC>
__device__ __forceinline__ void add_squares(float2& sum, const float (&a)[VEC]) {
  if constexpr (VEC == 1) {
    sum.x += a[0] * a[0];
  } else {
#pragma unroll
    for (int j = 0; j < VEC; j += 2) sum = tc::fma2(make_float2(a[j], a[j + 1]), make_float2(a[j], a[j + 1]), sum);
  }
}
template <int VEC>
__device__ __forceinline__ float max_magnitude(float m, const float (&a)[VEC]) {
  if constexpr (VEC == 1) {
    m = max_nan(m, fabsf(a[0]));
  } else {
#pragma unroll
    for (int j = 0; j < VEC; j += 2) m = max_nan(m, fabsf(a[j]), fabsf(a[j + 1]));
  }
  return m;
}

// scale of a row's or group's largest magnitude, and what a value is multiplied with before it is rounded
// (the division is within 2 units in the last place, far below a code's step)
__device__ __forceinline__ float scale_of(float amax) { return max_nan(amax, kAmaxFloor) * (1.0f / kFp8Max); }
__device__ __forceinline__ float inverse(float scale) { return __fdividef(1.0f, scale); }

// Who owns a row.
enum Owner {
  kOneRow,   // CTA: row blockIdx.x
  kWalkCta,  // CTA: rows blockIdx.x, + gridDim.x, ..
  kWalkWarp  // warp w of all: rows w, + all warps, ..
};
constexpr int kWalkThreads = 512;  // most threads of a walking CTA; its registers are limited for 1024 per SM
constexpr int kWarpRowWarps = 8;   // warps of a CTA whose warps own rows
constexpr int kWarpRowVectors = 128;  // longest row of a warp

constexpr int max_threads(Owner owner) { return owner == kOneRow ? 1024 : owner == kWalkCta ? kWalkThreads : 32 * kWarpRowWarps; }
// CTAs per SM that the registers are limited for
constexpr int min_ctas(Owner owner, int items) { return owner == kOneRow ? 1 : owner == kWalkCta ? (items <= 2 ? 2 : 1) : items == 1 ? 4 : items == 2 ? 3 : 2; }

// A row's threads, its shared values and what they wait with.
template <Owner OWNER, bool FP8>
struct RowShared {
  static constexpr int kWidest = OWNER == kWalkWarp ? kWarpRowVectors * 8 + 7 : B200_SKIP_RMS_NORM_MAX_HIDDEN;
  static constexpr int kRows = OWNER == kWalkWarp ? kWarpRowWarps : 1;
  // two of each, by the row's parity: a row's values are still read while the next row's are formed
  float warp_sums[2][32];
  int group_maxima[kRows][FP8 ? 2 : 1][FP8 ? (kWidest + B200_SKIP_RMS_NORM_MIN_GROUP - 1) / B200_SKIP_RMS_NORM_MIN_GROUP : 1];
};
template <Owner OWNER>
__device__ __forceinline__ void sync_row() {
  if constexpr (OWNER == kWalkWarp) __syncwarp();
  else __syncthreads();
}
// Sum over a row's threads, in all of them, and a row barrier.
template <Owner OWNER>
__device__ __forceinline__ float row_sum(float sum, float* warp_sum) {
#pragma unroll
  for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  if constexpr (OWNER == kWalkWarp) {
    __syncwarp();
  } else {
    const int lane = threadIdx.x & 31;
    if (lane == 0) warp_sum[threadIdx.x >> 5] = sum;
    __syncthreads();
    sum = lane < (blockDim.x >> 5) ? warp_sum[lane] : 0.f;
#pragma unroll
    for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  }
  return sum;
}

template <typename T, int VEC, int ITEMS, bool FP8, Owner OWNER>
__global__ void __launch_bounds__(max_threads(OWNER), min_ctas(OWNER, ITEMS))
    skip_rms_norm_kernel(const __grid_constant__ B200SkipRmsNormParams p) {
  using R = typename Raw<VEC>::type;
  constexpr bool WARP = OWNER == kWalkWarp;
  __shared__ RowShared<OWNER, FP8> shared;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int tid = WARP ? lane : threadIdx.x, threads = WARP ? 32 : blockDim.x;
  const int64_t first_row = WARP ? (int64_t)blockIdx.x * kWarpRowWarps + warp : blockIdx.x;
  const int64_t row_step = WARP ? (int64_t)gridDim.x * kWarpRowWarps : gridDim.x;
  if (first_row >= p.rows) return;
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
  load(first_row);
  auto load_weights = [&]() {
#pragma unroll
    for (int k = 0; k < ITEMS; ++k)
      wr[k] = tid + k * threads < n ? __ldg(reinterpret_cast<const R*>(p.weight) + tid + k * threads) : R{};
  };
  constexpr bool kWeightsLate = OWNER == kOneRow && ITEMS >= 4;  // not beside x and residual in 64 registers
  if (!kWeightsLate) load_weights();

  const float inv_h = 1.0f / (float)p.hidden;
  int parity = 0;
  for (int64_t row = first_row; row < p.rows; row += row_step, parity ^= 1) {
    int* group_max = shared.group_maxima[WARP ? warp : 0][FP8 ? parity : 0];
    float s[ITEMS][VEC];
    float2 sums = make_float2(0.f, 0.f);
#pragma unroll
    for (int k = 0; k < ITEMS; ++k) {
      float r[VEC];
      unpack<T, VEC>(xr[k], s[k]);
      unpack<T, VEC>(rr[k], r);
      add<VEC>(s[k], r);
      add_squares<VEC>(sums, s[k]);
    }
    if (OWNER != kOneRow && row + row_step < p.rows) load(row + row_step);
    if (kWeightsLate) load_weights();
    if (p.residual_out) {
      T* ro = static_cast<T*>(p.residual_out) + row * p.residual_out_row_stride;
#pragma unroll
      for (int k = 0; k < ITEMS; ++k)
        if (tid + k * threads < n) *reinterpret_cast<R*>(ro + (tid + k * threads) * VEC) = pack<T, VEC>(s[k]);
    }
    const int groups = FP8 && p.group_size ? (p.hidden + p.group_size - 1) / p.group_size : 1;
    if (FP8)
      for (int i = tid; i < groups; i += threads) group_max[i] = 0;
    const float sum = row_sum<OWNER>(sums.x + sums.y, shared.warp_sums[parity]);
    const float rstd = rsqrtf(sum * inv_h + p.epsilon);

#pragma unroll
    for (int k = 0; k < ITEMS; ++k) {
      float w[VEC];
      unpack<T, VEC>(wr[k], w);
      scale_by<VEC>(s[k], rstd);
      multiply<VEC>(s[k], w);
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
        // s is zero past the row's end, and NaN there only if it is all over the row
        amax[k] = max_magnitude<VEC>(0.f, s[k]);
        row_max = max_nan(row_max, amax[k]);
      }
      if (!p.group_size) {
        // magnitudes order like their bit patterns, a NaN above all
        int top = __reduce_max_sync(0xffffffffu, __float_as_int(row_max));
        if (!WARP) {
          if (lane == 0) atomicMax(&group_max[0], top);
          __syncthreads();
          top = group_max[0];
        }
        const float scale = scale_of(__int_as_float(top)), inv = inverse(scale);
#pragma unroll
        for (int k = 0; k < ITEMS; ++k) amax[k] = inv;
        if (tid == 0) scales[0] = scale;
      } else {
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          if (o >= lanes) break;
#pragma unroll
          for (int k = 0; k < ITEMS; ++k) amax[k] = max_nan(amax[k], __shfl_xor_sync(0xffffffffu, amax[k], o));
        }
        if (!in_warp) {
#pragma unroll
          for (int k = 0; k < ITEMS; ++k)
            if (lane == 0 && tid + k * threads < n)
              atomicMax(&group_max[(tid + k * threads) * VEC >> group_log2], __float_as_int(amax[k]));
          sync_row<OWNER>();
        }
#pragma unroll
        for (int k = 0; k < ITEMS; ++k) {
          const int c = (tid + k * threads) * VEC;
          if (c >= p.hidden) continue;
          const int g = c >> group_log2;
          if (!in_warp) amax[k] = __int_as_float(group_max[g]);
          const float scale = scale_of(amax[k]);
          if (c == g << group_log2) scales[g] = scale;
          amax[k] = inverse(scale);
        }
      }
#pragma unroll
      for (int k = 0; k < ITEMS; ++k)
        if (tid + k * threads < n) {
          scale_by<VEC>(s[k], amax[k]);
          store_e4m3<VEC>(out + (tid + k * threads) * VEC, s[k]);
        }
    }
  }
}

// Rows that all start the same number of elements before a 16-byte boundary, as those that a CTA or warp
// walks to do (a multiple of 8 rows further on): `head` elements up to the boundary, n whole vectors, and
// the rest.  A thread holds ITEMS vectors and, the first few, one of the at most 14 single elements.
template <typename T, int ITEMS, bool FP8, Owner OWNER>
__global__ void __launch_bounds__(max_threads(OWNER), min_ctas(OWNER, ITEMS))
    skip_rms_norm_shifted_kernel(const __grid_constant__ B200SkipRmsNormParams p) {
  constexpr bool WARP = OWNER == kWalkWarp;
  __shared__ RowShared<OWNER, FP8> shared;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, h = p.hidden;
  const int tid = WARP ? lane : threadIdx.x, threads = WARP ? 32 : blockDim.x;
  const int64_t first_row = WARP ? (int64_t)blockIdx.x * kWarpRowWarps + warp : blockIdx.x;
  const int64_t row_step = WARP ? (int64_t)gridDim.x * kWarpRowWarps : gridDim.x;
  if (first_row >= p.rows) return;
  const int head = min(h, (int)(-(reinterpret_cast<uintptr_t>(static_cast<const T*>(p.x) + first_row * p.x_row_stride) / 2) & 7));
  const int n = (h - head) / 8;
  const bool single = tid < h - 8 * n;
  const int es = tid < head ? tid : 8 * n + tid;              // the single element
  auto first = [&](int k) { return head + (tid + k * threads) * 8; };  // first element of the k-th vector
  auto valid = [&](int k) { return tid + k * threads < n; };

  uint4 xr[ITEMS], rr[ITEMS], wr[ITEMS];
  uint16_t x1 = 0, r1 = 0, w1 = 0;
  auto load = [&](int64_t row) {
    const T* x = static_cast<const T*>(p.x) + row * p.x_row_stride;
    const T* res = p.residual ? static_cast<const T*>(p.residual) + row * p.residual_row_stride : nullptr;
#pragma unroll
    for (int k = 0; k < ITEMS; ++k) {
      xr[k] = rr[k] = make_uint4(0, 0, 0, 0);
      if (valid(k)) {
        xr[k] = __ldcs(reinterpret_cast<const uint4*>(x + first(k)));
        if (res) rr[k] = __ldcs(reinterpret_cast<const uint4*>(res + first(k)));
      }
    }
    if (single) {
      x1 = __ldcs(reinterpret_cast<const uint16_t*>(x) + es);
      if (res) r1 = __ldcs(reinterpret_cast<const uint16_t*>(res) + es);
    }
  };
  load(first_row);
  const uint16_t* weight = static_cast<const uint16_t*>(p.weight);
#pragma unroll
  for (int k = 0; k < ITEMS; ++k) {  // the weights lie off the rows' boundaries: by elements, once
    uint32_t w[4] = {0, 0, 0, 0};
    if (valid(k)) {
#pragma unroll
      for (int j = 0; j < 8; ++j) w[j / 2] |= (uint32_t)__ldg(weight + first(k) + j) << (j % 2 * 16);
    }
    wr[k] = make_uint4(w[0], w[1], w[2], w[3]);
  }
  if (single) w1 = __ldg(weight + es);
  const int groups = FP8 && p.group_size ? (h + p.group_size - 1) / p.group_size : 1;
  const int group_log2 = p.group_size ? __ffs(p.group_size) - 1 : 30;

  const float inv_h = 1.0f / (float)h;
  int parity = 0;
  for (int64_t row = first_row; row < p.rows; row += row_step, parity ^= 1) {
    int* group_max = shared.group_maxima[WARP ? warp : 0][FP8 ? parity : 0];
    float s[ITEMS][8], s1[1], t1[1];
    float2 sums = make_float2(0.f, 0.f);
#pragma unroll
    for (int k = 0; k < ITEMS; ++k) {
      float r[8];
      unpack<T, 8>(xr[k], s[k]);
      unpack<T, 8>(rr[k], r);
      add<8>(s[k], r);
      add_squares<8>(sums, s[k]);
    }
    unpack<T, 1>(x1, s1);
    unpack<T, 1>(r1, t1);
    add<1>(s1, t1);
    add_squares<1>(sums, s1);
    if (OWNER != kOneRow && row + row_step < p.rows) load(row + row_step);
    if (p.residual_out) {
      T* ro = static_cast<T*>(p.residual_out) + row * p.residual_out_row_stride;
#pragma unroll
      for (int k = 0; k < ITEMS; ++k)
        if (valid(k)) *reinterpret_cast<uint4*>(ro + first(k)) = pack<T, 8>(s[k]);
      if (single) ro[es] = act<T>::from_f(s1[0]);
    }
    if (FP8)
      for (int i = tid; i < groups; i += threads) group_max[i] = 0;
    const float sum = row_sum<OWNER>(sums.x + sums.y, shared.warp_sums[parity]);
    const float rstd = rsqrtf(sum * inv_h + p.epsilon);
#pragma unroll
    for (int k = 0; k < ITEMS; ++k) {
      float w[8];
      unpack<T, 8>(wr[k], w);
      scale_by<8>(s[k], rstd);
      multiply<8>(s[k], w);
    }
    unpack<T, 1>(w1, t1);
    s1[0] = s1[0] * rstd * t1[0];
    if constexpr (!FP8) {
      T* out = static_cast<T*>(p.out) + row * p.out_row_stride;
#pragma unroll
      for (int k = 0; k < ITEMS; ++k)
        if (valid(k)) *reinterpret_cast<uint4*>(out + first(k)) = pack<T, 8>(s[k]);
      if (single) out[es] = act<T>::from_f(s1[0]);
    } else {
      uint8_t* out = static_cast<uint8_t*>(p.out) + row * p.out_row_stride;
      float* scales = p.scales + row * groups;
      // magnitudes order like their bit patterns, a NaN above all
      if (!p.group_size) {
        float m = fabsf(s1[0]);
#pragma unroll
        for (int k = 0; k < ITEMS; ++k) m = max_magnitude<8>(m, s[k]);
        const int top = __reduce_max_sync(0xffffffffu, __float_as_int(m));
        if (lane == 0) atomicMax(&group_max[0], top);
      } else {
        if (single) atomicMax(&group_max[es >> group_log2], __float_as_int(fabsf(s1[0])));
        // A vector meets at most two groups.
#pragma unroll
        for (int k = 0; k < ITEMS; ++k) {
          if (!valid(k)) continue;
          const int e = first(k);
          const int g0 = e >> group_log2, next = (g0 + 1 << group_log2) - e;  // first element of group g0 + 1
          float m0 = max_magnitude<8>(0.f, s[k]), m1 = 0.f;
          if (next < 8) {
            m0 = 0.f;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
              const float y = fabsf(s[k][j]);
              m0 = j < next ? max_nan(m0, y) : m0;
              m1 = j < next ? m1 : max_nan(m1, y);
            }
          }
          atomicMax(&group_max[g0], __float_as_int(m0));
          if (next < 8) atomicMax(&group_max[g0 + 1], __float_as_int(m1));
        }
      }
      sync_row<OWNER>();
      if (!p.group_size) {
        const float scale = scale_of(__int_as_float(group_max[0])), inv = inverse(scale);
        if (tid == 0) scales[0] = scale;
#pragma unroll
        for (int k = 0; k < ITEMS; ++k) scale_by<8>(s[k], inv);
        s1[0] *= inv;
      } else {
        for (int i = tid; i < groups; i += threads) scales[i] = scale_of(__int_as_float(group_max[i]));
#pragma unroll
        for (int k = 0; k < ITEMS; ++k) {
          if (!valid(k)) continue;
          const int g0 = first(k) >> group_log2, next = (g0 + 1 << group_log2) - first(k);
          const float inv = inverse(scale_of(__int_as_float(group_max[g0])));
          if (next >= 8) {
            scale_by<8>(s[k], inv);
          } else {
            const float inv1 = inverse(scale_of(__int_as_float(group_max[g0 + 1])));
#pragma unroll
            for (int j = 0; j < 8; ++j) s[k][j] *= j < next ? inv : inv1;
          }
        }
        if (single) s1[0] *= inverse(scale_of(__int_as_float(group_max[es >> group_log2])));
      }
#pragma unroll
      for (int k = 0; k < ITEMS; ++k)
        if (valid(k)) store_e4m3<8>(out + first(k), s[k]);
      if (single) store_e4m3<1>(out + es, s1);
    }
  }
}

template <typename T, int VEC, int ITEMS, Owner OWNER, bool SHIFTED>
void launch_items(const B200SkipRmsNormParams& p, int vectors, int num_sms, cudaStream_t stream) {
  const int threads = OWNER == kWalkWarp ? 32 * kWarpRowWarps : std::max(32, (vectors + 32 * ITEMS - 1) / (32 * ITEMS) * 32);
  int grid = p.rows;
  if (OWNER == kWalkCta) grid = std::max(8, num_sms * (ITEMS <= 2 ? std::max(1, 1024 / threads) : 1) / 8 * 8);  // keeps the rows' shift
  if (OWNER == kWalkWarp) grid = num_sms * min_ctas(OWNER, ITEMS);
  const bool fp8 = p.out_dtype == B200_DTYPE_FLOAT8E4M3FN;
  if constexpr (SHIFTED) {
    if (fp8) skip_rms_norm_shifted_kernel<T, ITEMS, true, OWNER><<<grid, threads, 0, stream>>>(p);
    else skip_rms_norm_shifted_kernel<T, ITEMS, false, OWNER><<<grid, threads, 0, stream>>>(p);
  } else {
    if (fp8) skip_rms_norm_kernel<T, VEC, ITEMS, true, OWNER><<<grid, threads, 0, stream>>>(p);
    else skip_rms_norm_kernel<T, VEC, ITEMS, false, OWNER><<<grid, threads, 0, stream>>>(p);
  }
}

// Many rows: 16384 x 256 to fp8 rows takes 6.0 us with a warp per row and took 9.5 us with a CTA per row;
// CTAs of two vectors per thread, 1024 threads per SM (960 and 768 were up to 30 % slower at 8192
// channels), or of four and 512 threads: 4096 x 16384 87 us, 109 us in CTAs of one row each.
template <typename T, int VEC, bool SHIFTED>
void launch_vec(const B200SkipRmsNormParams& p, int num_sms, cudaStream_t stream) {
  const int n = p.hidden / VEC;  // vectors of a row, at most
  const bool many = p.rows > 4 * num_sms && p.rows >= 16;
  if (many && n <= kWarpRowVectors) {
    if (n <= 32) launch_items<T, VEC, 1, kWalkWarp, SHIFTED>(p, n, num_sms, stream);
    else if (n <= 64) launch_items<T, VEC, 2, kWalkWarp, SHIFTED>(p, n, num_sms, stream);
    else launch_items<T, VEC, 4, kWalkWarp, SHIFTED>(p, n, num_sms, stream);
  } else if (many && n <= 2 * kWalkThreads) {
    launch_items<T, VEC, 2, kWalkCta, SHIFTED>(p, n, num_sms, stream);
  } else if (VEC == 8 && many && n <= 4 * kWalkThreads) {
    launch_items<T, 8, 4, kWalkCta, SHIFTED>(p, n, num_sms, stream);
  } else if (n <= 1024) {
    launch_items<T, VEC, 1, kOneRow, SHIFTED>(p, n, num_sms, stream);
  } else if (VEC == 8 || n <= 4096) {
    launch_items<T, VEC, 4, kOneRow, SHIFTED>(p, n, num_sms, stream);
  } else if constexpr (VEC == 1) {
    launch_items<T, VEC, 32, kOneRow, SHIFTED>(p, n, num_sms, stream);
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
  if (aligned) launch_vec<T, 8, false>(p, num_sms, stream);
  else if (alike) launch_vec<T, 8, true>(p, num_sms, stream);
  else launch_vec<T, 1, false>(p, num_sms, stream);
}

}  // namespace

cudaError_t launch_skip_rms_norm(const B200SkipRmsNormParams& p, int num_sms, cudaStream_t stream) {
  if (p.dtype == B200_DTYPE_BFLOAT16) launch_type<__nv_bfloat16>(p, num_sms, stream);
  else launch_type<__half>(p, num_sms, stream);
  add_launches(1);
  return cudaGetLastError();
}

}  // namespace b200
