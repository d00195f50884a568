// C ABI of the decoder-layer operators (include/b200_layer.h): argument checks, defaults and the
// status word.  Every check runs before anything touches the device.
#include <cmath>
#include <exception>
#include <initializer_list>
#include <string>

#include "b200_kernels.h"
#include "layer_kernels.h"

namespace {

using b200::set_error;

bool is_act(int dt) { return dt == B200_DTYPE_FLOAT16 || dt == B200_DTYPE_BFLOAT16; }

int invalid(const char* op, const std::string& what) {
  return set_error(B200_ERR_INVALID_ARGUMENT, std::string(op) + ": " + what);
}

int unsupported(const char* op, const std::string& what) {
  return set_error(B200_ERR_UNSUPPORTED, std::string(op) + ": " + what);
}

int launched(const char* op, cudaError_t e) {
  if (e == cudaSuccess) return B200_OK;
  return set_error(B200_ERR_CUDA, std::string(op) + ": CUDA error: " + cudaGetErrorString(e));
}

int sm_count(int32_t asked) {
  if (asked > 0) return asked;
  static int cached[64] = {0};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 148;
  if (cached[dev] == 0) {
    int n = 0;
    if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || n <= 0) n = 148;
    cached[dev] = n;
  }
  return cached[dev];
}

template <typename F>
int guarded(const char* op, F&& body) {
  try {
    return body();
  } catch (const std::exception& e) {
    return set_error(B200_ERR_FAIL, std::string(op) + ": " + e.what());
  } catch (...) {
    return set_error(B200_ERR_FAIL, std::string(op) + ": unknown failure");
  }
}

int64_t dense(int64_t stride, int64_t width) { return stride ? stride : width; }

// Whether every address (NULL passes) is a multiple of its element's size.
bool aligned(std::initializer_list<const void*> addresses, size_t size) {
  uintptr_t bits = 0;
  for (const void* a : addresses) bits |= reinterpret_cast<uintptr_t>(a);
  return bits % size == 0;
}

// B200_OK for a workspace of at least `need` bytes whose address is a multiple of `align`.
int check_workspace(const char* op, const char* size_call, const void* workspace, size_t bytes, size_t need, size_t align) {
  if (!need) return B200_OK;
  if (!workspace || bytes < need)
    return set_error(B200_ERR_WORKSPACE, std::string(op) + ": workspace missing or smaller than " + size_call + "()");
  if (reinterpret_cast<uintptr_t>(workspace) % align)
    return set_error(B200_ERR_WORKSPACE, std::string(op) + ": workspace must be aligned to " + std::to_string(align) + " bytes");
  return B200_OK;
}

// ---- skip RMS norm
constexpr const char* kNorm = "SkipRmsNorm";

int check_norm(B200SkipRmsNormParams* p) {
  if (p->rows < 0 || p->hidden <= 0) return invalid(kNorm, "rows >= 0 and hidden > 0");
  if (p->hidden > B200_SKIP_RMS_NORM_MAX_HIDDEN) return unsupported(kNorm, "hidden above 32768 is not implemented");
  if (!is_act(p->dtype)) return invalid(kNorm, "x must be fp16 or bf16");
  const bool fp8 = p->out_dtype == B200_DTYPE_FLOAT8E4M3FN;
  if (!fp8 && p->out_dtype != p->dtype) return invalid(kNorm, "out must be x's type or fp8 e4m3");
  if (!(p->epsilon >= 0.f) || std::isinf(p->epsilon)) return invalid(kNorm, "epsilon must be finite and non-negative");
  const int g = p->group_size;
  if (!fp8 && g != 0) return invalid(kNorm, "group_size needs an fp8 output");
  if (g != 0 && (g < B200_SKIP_RMS_NORM_MIN_GROUP || g > B200_SKIP_RMS_NORM_MAX_GROUP || (g & (g - 1))))
    return invalid(kNorm, "group_size must be 0 or a power of two from 32 to 1024");
  p->x_row_stride = dense(p->x_row_stride, p->hidden);
  p->residual_row_stride = dense(p->residual_row_stride, p->hidden);
  p->out_row_stride = dense(p->out_row_stride, p->hidden);
  p->residual_out_row_stride = dense(p->residual_out_row_stride, p->hidden);
  for (int64_t s : {p->x_row_stride, p->residual_row_stride})
    if (s < 0) return invalid(kNorm, "negative row stride");
  if (p->rows > 1 && (p->out_row_stride < p->hidden || (p->residual_out && p->residual_out_row_stride < p->hidden)))
    return invalid(kNorm, "output rows overlap");
  if (p->rows == 0) return B200_OK;
  if (!p->x || !p->weight || !p->out) return invalid(kNorm, "x, weight and out are required");
  if (fp8 && !p->scales) return invalid(kNorm, "an fp8 output requires scales");
  if (fp8 && (p->out == p->x || p->out == p->residual || p->out == p->residual_out))
    return invalid(kNorm, "an fp8 output cannot share a 16-bit tensor's memory");
  if (p->out == p->residual_out) return invalid(kNorm, "out and residual_out must differ");
  if (!aligned({p->x, p->residual, p->weight, p->residual_out, fp8 ? nullptr : p->out}, 2) || !aligned({p->scales}, 4))
    return invalid(kNorm, "a tensor is not aligned to its elements");
  return B200_OK;
}

// ---- rotary append
constexpr const char* kRope = "RotaryAppend";

int check_rope_shapes(const B200RotaryAppendParams* p) {
  if (p->num_heads <= 0 || p->kv_num_heads <= 0 || p->head_size <= 0)
    return invalid(kRope, "num_heads, kv_num_heads and head_size must be positive");
  if (p->num_tokens < 0) return invalid(kRope, "num_tokens must not be negative");
  if (p->num_tokens > (1 << 29)) return unsupported(kRope, "more than 2^29 tokens");
  return B200_OK;
}

int check_rope(B200RotaryAppendParams* p) {
  if (int rc = check_rope_shapes(p)) return rc;
  if (p->num_blocks <= 0 || p->block_size <= 0) return invalid(kRope, "caches require positive block geometry");
  if ((int64_t)p->num_blocks * p->block_size > INT32_MAX) return unsupported(kRope, "cache slot count exceeds int32");
  if (!is_act(p->act_dtype)) return invalid(kRope, "query, key and value must be fp16 or bf16");
  const bool fp8 = p->cache_dtype == B200_DTYPE_FLOAT8E4M3FN;
  if (!fp8 && p->cache_dtype != p->act_dtype) return invalid(kRope, "the cache must have the activations' type or fp8 e4m3");
  if (p->table_dtype != p->act_dtype && p->table_dtype != B200_DTYPE_FLOAT)
    return invalid(kRope, "cos_cache and sin_cache must have the activations' type or fp32");
  if (p->position_dtype != B200_DTYPE_INT32 && p->position_dtype != B200_DTYPE_INT64)
    return invalid(kRope, "position_ids must be int32 or int64");
  if (p->rotary_dim <= 0 || p->rotary_dim % 2 || p->rotary_offset < 0 || p->rotary_dim > p->head_size ||
      p->rotary_offset > p->head_size - p->rotary_dim)
    return invalid(kRope, "rotary_dim must be even and rotary_offset + rotary_dim must not exceed head_size");
  if (p->rotary_positions <= 0) return invalid(kRope, "cos_cache and sin_cache must not be empty");
  if (p->axes < 1 || p->axes > B200_MAX_ROTARY_AXES) return invalid(kRope, "axes must be 1 to 4");
  int64_t pairs = 0;
  for (int a = 0; a < p->axes; ++a) {
    if (p->axis_pairs[a] < 0) return invalid(kRope, "axis_pairs must not be negative");
    pairs += p->axis_pairs[a];
  }
  if (pairs != p->rotary_dim / 2) return invalid(kRope, "axis_pairs must sum to rotary_dim / 2");
  const int64_t q = (int64_t)p->num_heads * p->head_size, kv = (int64_t)p->kv_num_heads * p->head_size;
  if (q > INT32_MAX || kv > INT32_MAX) return unsupported(kRope, "a token's row exceeds int32");
  p->query_row_stride = dense(p->query_row_stride, q);
  p->key_row_stride = dense(p->key_row_stride, kv);
  p->value_row_stride = dense(p->value_row_stride, kv);
  p->output_row_stride = dense(p->output_row_stride, q);
  if (!p->position_token_stride) p->position_token_stride = 1;
  if (p->num_tokens > 1 && p->output_row_stride < q) return invalid(kRope, "output rows overlap");
  if (p->num_tokens == 0) return B200_OK;
  if (!p->query || !p->key || !p->value || !p->output || !p->key_cache || !p->value_cache || !p->position_ids ||
      !p->cos_cache || !p->sin_cache || !p->slot_mapping)
    return invalid(kRope, "missing required tensor");
  if (fp8 && (!p->k_scale || !p->v_scale)) return invalid(kRope, "fp8 caches require k_scale and v_scale");
  if (!aligned({p->query, p->key, p->value, p->output}, 2) || !aligned({p->key_cache, p->value_cache}, fp8 ? 1 : 2) ||
      !aligned({p->cos_cache, p->sin_cache}, p->table_dtype == B200_DTYPE_FLOAT ? 4 : 2) ||
      !aligned({p->position_ids}, p->position_dtype == B200_DTYPE_INT64 ? 8 : 4) ||
      !aligned({p->slot_mapping, p->k_scale, p->v_scale, p->device_status}, 4))
    return invalid(kRope, "a tensor is not aligned to its elements");
  return B200_OK;
}

// ---- shared prefix attention
constexpr const char* kPrefix = "SharedPrefixAttention";
constexpr int kMaxSms = 1024;

int check_prefix_shapes(B200SharedPrefixParams* p) {
  if (p->num_heads <= 0 || p->kv_num_heads <= 0 || p->num_heads % p->kv_num_heads != 0)
    return invalid(kPrefix, "bad num_heads/kv_num_heads");
  if (p->head_size <= 0) return invalid(kPrefix, "head_size must be positive");
  if (p->head_size > B200_SHARED_PREFIX_MAX_HEAD_SIZE) return unsupported(kPrefix, "head_size above 256 is not implemented");
  if (p->num_heads > 65535) return unsupported(kPrefix, "more than 65535 heads");
  if (!is_act(p->act_dtype)) return invalid(kPrefix, "query and caches must be fp16 or bf16");
  if (p->num_blocks <= 0 || p->block_size <= 0) return invalid(kPrefix, "caches require positive block geometry");
  if ((int64_t)p->num_blocks * p->block_size > INT32_MAX) return unsupported(kPrefix, "cache slot count exceeds int32");
  if (p->num_tokens < 0 || p->batch < (p->num_tokens > 0) || p->max_blocks_per_seq < 0)
    return invalid(kPrefix, "batch must be positive, num_tokens and max_blocks_per_seq not negative");
  if (p->prefix_length < 0 || p->prefix_blocks < 0 ||
      p->prefix_length > (int64_t)p->prefix_blocks * p->block_size)
    return invalid(kPrefix, "prefix_length exceeds prefix_block_table");
  if ((int64_t)p->prefix_length + (int64_t)p->max_blocks_per_seq * p->block_size > INT32_MAX)
    return unsupported(kPrefix, "a sequence's keys exceed int32");
  // grids and the workspace are counted from it in 32 bits
  if (p->num_sms > kMaxSms) return invalid(kPrefix, "num_sms exceeds " + std::to_string(kMaxSms));
  return B200_OK;
}

int check_prefix(B200SharedPrefixParams* p) {
  if (int rc = check_prefix_shapes(p)) return rc;
  if (!std::isfinite(p->scale)) return invalid(kPrefix, "scale must be finite");
  if (!(p->softcap >= 0.f) || std::isinf(p->softcap)) return invalid(kPrefix, "softcap must be finite and non-negative");
  const int64_t width = (int64_t)p->num_heads * p->head_size;
  p->query_row_stride = dense(p->query_row_stride, width);
  p->output_row_stride = dense(p->output_row_stride, width);
  if (p->num_tokens > 1 && p->output_row_stride < width) return invalid(kPrefix, "output rows overlap");
  if (p->num_tokens == 0) return B200_OK;
  if (!p->query || !p->key_cache || !p->value_cache || !p->output || !p->cumulative_sequence_length ||
      !p->past_seqlens || !p->block_table || (p->prefix_length > 0 && !p->prefix_block_table))
    return invalid(kPrefix, "missing required tensor");
  if (!aligned({p->query, p->key_cache, p->value_cache, p->head_sink, p->output}, 2) ||
      !aligned({p->cumulative_sequence_length, p->past_seqlens, p->block_table, p->prefix_block_table, p->device_status}, 4))
    return invalid(kPrefix, "a tensor is not aligned to its elements");
  if (p->scale == 0.f) p->scale = 1.0f / std::sqrt((float)p->head_size);
  return B200_OK;
}

// Clears what was read and nothing that was set since.
__global__ void clear_bits_kernel(int32_t* status, int bits) { atomicAnd(status, ~bits); }

}  // namespace

extern "C" {

size_t b200_layer_struct_size(int32_t which) {
  switch (which) {
    case 0: return sizeof(B200SkipRmsNormParams);
    case 1: return sizeof(B200RotaryAppendParams);
    case 2: return sizeof(B200SharedPrefixParams);
    default: return 0;
  }
}

int b200_skip_rms_norm(const B200SkipRmsNormParams* params, void* stream) {
  if (!params) return invalid(kNorm, "null params");
  return guarded(kNorm, [&] {
    B200SkipRmsNormParams p = *params;
    if (int rc = check_norm(&p)) return rc;
    if (p.rows == 0) return B200_OK;
    return launched(kNorm, b200::launch_skip_rms_norm(p, sm_count(0), static_cast<cudaStream_t>(stream)));
  });
}

int b200_rotary_append_workspace_size(const B200RotaryAppendParams* params, size_t* bytes) {
  if (!params || !bytes) return invalid(kRope, "null params or bytes pointer");
  if (int rc = check_rope_shapes(params)) return rc;
  *bytes = b200::rotary_append_workspace(*params);
  return B200_OK;
}

int b200_rotary_append(const B200RotaryAppendParams* params, void* stream) {
  if (!params) return invalid(kRope, "null params");
  return guarded(kRope, [&] {
    B200RotaryAppendParams p = *params;
    if (int rc = check_rope(&p)) return rc;
    if (p.num_tokens == 0) return B200_OK;
    const size_t need = b200::rotary_append_workspace(p);
    if (int rc = check_workspace(kRope, "b200_rotary_append_workspace_size", p.workspace, p.workspace_bytes, need, sizeof(int)))
      return rc;
    return launched(kRope, b200::launch_rotary_append(p, sm_count(0), static_cast<cudaStream_t>(stream)));
  });
}

int b200_shared_prefix_attention_workspace_size(const B200SharedPrefixParams* params, size_t* bytes) {
  if (!params || !bytes) return invalid(kPrefix, "null params or bytes pointer");
  B200SharedPrefixParams p = *params;
  if (int rc = check_prefix_shapes(&p)) return rc;
  *bytes = b200::shared_prefix_workspace(p, sm_count(p.num_sms));
  return B200_OK;
}

int b200_shared_prefix_attention(const B200SharedPrefixParams* params, void* stream) {
  if (!params) return invalid(kPrefix, "null params");
  return guarded(kPrefix, [&] {
    B200SharedPrefixParams p = *params;
    if (int rc = check_prefix(&p)) return rc;
    if (p.num_tokens == 0) return B200_OK;
    const int sms = sm_count(p.num_sms);
    const size_t need = b200::shared_prefix_workspace(p, sms);
    if (int rc = check_workspace(kPrefix, "b200_shared_prefix_attention_workspace_size", p.workspace, p.workspace_bytes,
                                 need, 16))  // 16-byte accesses and a TMA source
      return rc;
    return launched(kPrefix, b200::launch_shared_prefix(p, sms, static_cast<cudaStream_t>(stream)));
  });
}

int b200_layer_read_status(int32_t* device_status, void* stream_ptr) {
  if (!device_status || !aligned({device_status}, 4))
    return set_error(B200_ERR_INVALID_ARGUMENT, "layer status: no status word, or a misaligned one");
  cudaStream_t stream = static_cast<cudaStream_t>(stream_ptr);
  int bits = 0;
  cudaError_t e = cudaMemcpyAsync(&bits, device_status, sizeof(int), cudaMemcpyDeviceToHost, stream);
  if (e == cudaSuccess) e = cudaStreamSynchronize(stream);
  if (e != cudaSuccess) return launched("layer status", e);
  if (bits == 0) return B200_OK;
  clear_bits_kernel<<<1, 1, 0, stream>>>(device_status, bits);
  b200::add_launches(1);
  if ((e = cudaGetLastError()) != cudaSuccess) return launched("layer status", e);
  if (bits & (b200::kStatusBadCumulative | b200::kStatusBadPast | b200::kStatusBadCapacity))
    return set_error(B200_ERR_FAIL, "SharedPrefixAttention: inconsistent cumulative lengths, past lengths or block table");
  if (bits & b200::kStatusBadBlock)
    return set_error(B200_ERR_FAIL, "SharedPrefixAttention: block table contains an invalid physical block");
  if (bits & b200::kStatusBadSlot)
    return set_error(B200_ERR_FAIL, "RotaryAppend: slot_mapping must contain -1 or valid physical cache slots");
  if (bits & b200::kStatusBadPosition)
    return set_error(B200_ERR_FAIL, "RotaryAppend: rotary position exceeds the cos/sin cache");
  if (bits & b200::kStatusTimeout)
    return set_error(B200_ERR_DEVICE, "SharedPrefixAttention: a device wait timed out (TMA copy did not complete)");
  return set_error(B200_ERR_DEVICE, "layer status: device status " + std::to_string(bits));
}

}  // extern "C"
