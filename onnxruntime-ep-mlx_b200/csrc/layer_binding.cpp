// CPython binding of the decoder-layer operators for torch tensors (module onnxruntime_ep_b200._layer).
//
// A decode step makes these calls once or more per layer on a few tokens, where the host's time is the
// call's time: the checks of shapes, types and strides, the outputs' allocation and the call of the C ABI
// (include/b200_layer.h) take about half as long here as through ctypes.  layer.py has the public
// functions and their documentation.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/ATen.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include <atomic>
#include <map>
#include <memory>
#include <mutex>
#include <string>
#include <utility>
#include <vector>

#include "b200_layer.h"

namespace {

using at::ScalarType;
using at::Tensor;

PyObject* g_error_class = nullptr;  // onnxruntime_ep_b200.B200Error

struct Failure {
  int code;
  std::string message;
};

[[noreturn]] void bad(const char* op, const std::string& what) {
  throw Failure{B200_ERR_INVALID_ARGUMENT, std::string(op) + ": " + what};
}

void checked(int code) {
  if (code != B200_OK) throw Failure{code, b200_last_error()};
}

// Run `body`, turning its C++ exceptions into Python ones.
template <typename F>
PyObject* guarded(F&& body) {
  try {
    return body();
  } catch (const Failure& f) {
    PyObject* e = PyObject_CallFunction(g_error_class, "is", f.code, f.message.c_str());
    if (e) {
      PyErr_SetObject(g_error_class, e);
      Py_DECREF(e);
    }
  } catch (const std::exception& e) {
    if (!PyErr_Occurred()) PyErr_SetString(PyExc_RuntimeError, e.what());
  } catch (...) {
    if (!PyErr_Occurred()) PyErr_SetString(PyExc_RuntimeError, "layer binding: unknown failure");
  }
  return nullptr;
}

const Tensor& tensor(const char* op, const char* name, PyObject* o) {
  if (!THPVariable_Check(o)) bad(op, std::string(name) + " must be a tensor");
  return THPVariable_Unpack(o);
}

int32_t integer(const char* op, const char* name, PyObject* o) {
  PyObject* index = PyNumber_Index(o);
  long long v = -1;
  int overflow = 0;
  if (index) {
    v = PyLong_AsLongLongAndOverflow(index, &overflow);
    Py_DECREF(index);
  }
  if (!index || overflow || v < INT32_MIN || v > INT32_MAX) {
    PyErr_Clear();
    bad(op, std::string(name) + " must be a 32-bit integer");
  }
  return (int32_t)v;
}

float number(const char* op, const char* name, PyObject* o) {
  const double v = PyFloat_AsDouble(o);
  if (v == -1.0 && PyErr_Occurred()) {
    PyErr_Clear();
    bad(op, std::string(name) + " must be a number");
  }
  return (float)v;
}

int dtype_of(ScalarType t) {
  switch (t) {
    case at::kHalf: return B200_DTYPE_FLOAT16;
    case at::kBFloat16: return B200_DTYPE_BFLOAT16;
    case at::kFloat: return B200_DTYPE_FLOAT;
    case at::kFloat8_e4m3fn: return B200_DTYPE_FLOAT8E4M3FN;
    case at::kInt: return B200_DTYPE_INT32;
    case at::kLong: return B200_DTYPE_INT64;
    default: return 0;
  }
}

std::string shape_text(at::IntArrayRef shape) {
  std::string s = "[";
  for (size_t i = 0; i < shape.size(); ++i) s += (i ? ", " : "") + std::to_string(shape[i]);
  return s + "]";
}

bool on(const Tensor& t, int device) { return t.is_cuda() && t.get_device() == device; }

// Row stride of a [rows, width] tensor with contiguous rows.
int64_t rows(const char* op, const char* name, const Tensor& t, int64_t n, int64_t width, ScalarType type, int device) {
  if (t.scalar_type() != type || !on(t, device) || t.dim() != 2 || t.size(0) != n || t.size(1) != width)
    bad(op, std::string(name) + " must be a " + shape_text({n, width}) + " tensor of " + at::toString(type) + " on cuda:" +
                std::to_string(device));
  if (width > 1 && t.stride(1) != 1) bad(op, std::string(name) + " rows must be contiguous");
  if (n <= 1) return width;
  if (t.stride(0) == 0) bad(op, std::string(name) + " must not be a broadcast row");  // the C ABI reads 0 as dense
  return t.stride(0);
}

// Address of a contiguous tensor.
template <typename P = void>
P* dense(const char* op, const char* name, const Tensor& t, at::IntArrayRef shape, ScalarType type, int device) {
  if (t.scalar_type() != type || !on(t, device) || t.sizes() != shape || !t.is_contiguous())
    bad(op, std::string(name) + " must be a contiguous " + shape_text(shape) + " tensor of " + at::toString(type) +
                " on cuda:" + std::to_string(device));
  return static_cast<P*>(t.data_ptr());
}

int device_of(const char* op, const Tensor& t) {
  if (!t.is_cuda()) bad(op, "tensors must be on a CUDA device");
  return t.get_device();
}

Tensor empty(at::IntArrayRef shape, ScalarType type, int device) {
  return at::detail::empty_cuda(shape, type, c10::Device(c10::kCUDA, (c10::DeviceIndex)device), std::nullopt);
}

// Status word per (device, stream), zeroed once: calls only set bits, b200_layer_read_status clears them.
// Calls on different streams never share one, so a call's report goes to nobody else; a captured call reports
// to the stream that it was captured on.  Words come in blocks, so that a capture on a stream without a word
// gets one without an allocation.
constexpr int kBlockWords = 1024;
using StreamWords = std::map<std::pair<int, cudaStream_t>, int32_t*>;
StreamWords& stream_words() {
  static auto* words = new StreamWords;  // until exit, like the blocks below
  return *words;
}
int32_t* status_word(const char* op, int device, cudaStream_t stream) {
  static auto* blocks = new std::map<int, std::pair<std::vector<Tensor>, int>>;  // device -> blocks, words used
  StreamWords& words = stream_words();
  const auto it = words.find({device, stream});
  if (it != words.end()) return it->second;
  auto& [kept, used] = (*blocks)[device];
  if (used == (int)kept.size() * kBlockWords) {
    cudaStreamCaptureStatus status;
    C10_CUDA_CHECK(cudaStreamIsCapturing(stream, &status));
    if (status != cudaStreamCaptureStatusNone) bad(op, "the first call on a device cannot be captured: make one before");
    Tensor block = empty({kBlockWords}, at::kInt, device);
    block.zero_();
    C10_CUDA_CHECK(cudaStreamSynchronize(stream));  // zeroed before any other stream uses it
    kept.push_back(std::move(block));
  }
  int32_t* word = static_cast<int32_t*>(kept.back().data_ptr()) + used % kBlockWords;
  ++used;
  return words[{device, stream}] = word;
}

// Captures whose graphs, and all that was instantiated from them, are gone.  Filled by the CUDA driver's
// threads, which may not make CUDA calls then.
struct Ended {
  std::atomic<bool> any{false};
  std::mutex mutex;
  std::vector<unsigned long long> captures;
};
Ended& ended() {
  static auto* e = new Ended;  // until exit
  return *e;
}

// Scratch of a stream's eager calls, or of the calls that one capture took from a stream: either follow one
// another, and calls that may overlap never share it.  A graph is replayed wherever and whenever its owner
// likes, so each capture has buffers of its own.  They live as long as the graph and its instances; one that
// became too small is kept, since earlier calls of the capture use it.
struct Scratch {
  bool captured = false;
  std::vector<Tensor> buffers;  // the last one is the current one
};
using StreamScratch = std::map<std::pair<int, cudaStream_t>, Scratch>;

void forget_ended(std::map<unsigned long long, StreamScratch>& captures) {
  Ended& e = ended();
  if (!e.any.load(std::memory_order_acquire)) return;
  const std::lock_guard<std::mutex> lock(e.mutex);
  for (const auto id : e.captures) captures.erase(id);
  e.captures.clear();
  e.any.store(false, std::memory_order_release);
}

// `id` joins the ended captures when its graph and the last instance are destroyed.
void tell_end(unsigned long long id, cudaGraph_t graph) {
  auto note = std::make_unique<unsigned long long>(id);
  cudaUserObject_t object;
  C10_CUDA_CHECK(cudaUserObjectCreate(
      &object, note.get(),
      [](void* p) {
        const std::unique_ptr<unsigned long long> note(static_cast<unsigned long long*>(p));
        try {
          Ended& e = ended();
          const std::lock_guard<std::mutex> lock(e.mutex);
          e.captures.push_back(*note);
          e.any.store(true, std::memory_order_release);
        } catch (...) {  // the buffers stay until exit
        }
      },
      1, cudaUserObjectNoDestructorSync));
  note.release();
  const cudaError_t e = cudaGraphRetainUserObject(graph, object, 1, cudaGraphUserObjectMove);
  if (e != cudaSuccess) cudaUserObjectRelease(object, 1);
  C10_CUDA_CHECK(e);
}

Scratch& scratch(int device, cudaStream_t stream) {
  static auto* eager = new StreamScratch;  // both until exit
  static auto* captures = new std::map<unsigned long long, StreamScratch>;
  forget_ended(*captures);
  cudaStreamCaptureStatus status;
  C10_CUDA_CHECK(cudaStreamIsCapturing(stream, &status));
  if (status != cudaStreamCaptureStatusActive) return (*eager)[{device, stream}];
  unsigned long long id = 0;
  cudaGraph_t graph = nullptr;
  C10_CUDA_CHECK(cudaStreamGetCaptureInfo_v2(stream, &status, &id, &graph, nullptr, nullptr));
  if (captures->find(id) == captures->end()) tell_end(id, graph);
  Scratch& own = (*captures)[id][{device, stream}];
  own.captured = true;
  return own;
}

// Run an operator with a workspace: the caller's, or the stream's or capture's own, grown where too small.
template <typename P>
void run_with_workspace(const char* op, P* p, PyObject* workspace, int device, cudaStream_t stream,
                        int (*size)(const P*, size_t*), int (*run)(const P*, void*)) {
  if (workspace != Py_None) {
    const Tensor& w = tensor(op, "workspace", workspace);
    if (w.scalar_type() != at::kByte || !on(w, device) || !w.is_contiguous())
      throw Failure{B200_ERR_WORKSPACE, std::string(op) + ": workspace must be a contiguous uint8 tensor on the caches' device"};
    p->workspace = w.data_ptr();
    p->workspace_bytes = w.numel();
    return checked(run(p, stream));
  }
  Scratch& own = scratch(device, stream);
  auto& buffers = own.buffers;
  p->workspace = buffers.empty() ? nullptr : buffers.back().data_ptr();
  p->workspace_bytes = buffers.empty() ? 0 : buffers.back().numel();
  const int code = run(p, stream);
  size_t need = 0;
  if (code != B200_ERR_WORKSPACE || size(p, &need) != B200_OK || need <= p->workspace_bytes) return checked(code);
  if (!own.captured) buffers.clear();  // the allocator hands it to later work of this stream only
  buffers.push_back(empty({(int64_t)std::max<size_t>({need, (size_t)1 << 20, 2 * p->workspace_bytes})}, at::kByte, device));
  p->workspace = buffers.back().data_ptr();
  p->workspace_bytes = buffers.back().numel();
  checked(run(p, stream));
}

PyObject* tuple_of(std::initializer_list<PyObject*> items) {
  PyObject* t = PyTuple_New(items.size());
  Py_ssize_t i = 0;
  for (PyObject* o : items) PyTuple_SET_ITEM(t, i++, o);
  return t;
}

PyObject* shared(PyObject* o) {
  Py_INCREF(o);
  return o;
}

// An output tensor given by the caller, or a new one.
PyObject* given_or(PyObject* given, Tensor&& made) { return given != Py_None ? shared(given) : THPVariable_Wrap(std::move(made)); }

bool arguments(const char* name, Py_ssize_t got, Py_ssize_t want) {
  if (got == want) return true;
  PyErr_Format(PyExc_TypeError, "%s takes %zd arguments (%zd given)", name, want, got);
  return false;
}

// x, residual, weight, epsilon, fp8, group_size, output, scales, residual_output
PyObject* skip_rms_norm(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (!arguments("skip_rms_norm", n, 9)) return nullptr;
  return guarded([&] {
    constexpr const char* op = "SkipRmsNorm";
    const Tensor& x = tensor(op, "x", args[0]);
    const ScalarType type = x.scalar_type();
    if ((type != at::kHalf && type != at::kBFloat16) || x.dim() != 2) bad(op, "x must be a [rows, hidden] tensor of fp16 or bf16");
    const int64_t count = x.size(0), hidden = x.size(1);
    if (count > INT32_MAX || hidden > INT32_MAX) bad(op, "x is too large");
    const int device = device_of(op, x);
    const bool fp8 = args[4] == Py_True;
    const ScalarType out_type = fp8 ? at::kFloat8_e4m3fn : type;
    B200SkipRmsNormParams p{};
    p.rows = (int32_t)count;
    p.hidden = (int32_t)hidden;
    p.dtype = dtype_of(type);
    p.out_dtype = dtype_of(out_type);
    p.epsilon = number(op, "epsilon", args[3]);
    p.group_size = integer(op, "group_size", args[5]);
    p.x_row_stride = rows(op, "x", x, count, hidden, type, device);
    p.x = x.data_ptr();
    if (args[1] != Py_None) {
      const Tensor& r = tensor(op, "residual", args[1]);
      p.residual_row_stride = rows(op, "residual", r, count, hidden, type, device);
      p.residual = r.data_ptr();
    }
    p.weight = dense(op, "weight", tensor(op, "weight", args[2]), {hidden}, type, device);
    const c10::cuda::CUDAGuard guard((c10::DeviceIndex)device);
    Tensor out, scales, sum;
    auto take = [&](const char* name, PyObject* given, ScalarType t, Tensor& made, int64_t* stride) -> void* {
      if (given == Py_None) {
        made = empty({count, hidden}, t, device);
        return made.data_ptr();
      }
      const Tensor& o = tensor(op, name, given);
      *stride = rows(op, name, o, count, hidden, t, device);
      return o.data_ptr();
    };
    p.out = take("output", args[6], out_type, out, &p.out_row_stride);
    p.residual_out = take("residual_output", args[8], type, sum, &p.residual_out_row_stride);
    if (fp8) {
      const int64_t groups = p.group_size > 0 ? (hidden + p.group_size - 1) / p.group_size : 1;
      if (args[7] == Py_None) {
        scales = empty({count, groups}, at::kFloat, device);
        p.scales = static_cast<float*>(scales.data_ptr());
      } else {
        p.scales = dense<float>(op, "scales", tensor(op, "scales", args[7]), {count, groups}, at::kFloat, device);
      }
    }
    checked(b200_skip_rms_norm(&p, c10::cuda::getCurrentCUDAStream((c10::DeviceIndex)device).stream()));
    PyObject* o = given_or(args[6], std::move(out));
    PyObject* s = given_or(args[8], std::move(sum));
    return fp8 ? tuple_of({o, given_or(args[7], std::move(scales)), s}) : tuple_of({o, s});
  });
}

// query, key, value, key_cache, value_cache, position_ids, cos_cache, sin_cache, slot_mapping, num_heads,
// kv_num_heads, axis_sections, rotary_interleaved, rotary_offset, k_scale, v_scale, output, workspace
PyObject* rotary_append(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (!arguments("rotary_append", n, 18)) return nullptr;
  return guarded([&] {
    constexpr const char* op = "RotaryAppend";
    const Tensor& q = tensor(op, "query", args[0]);
    const ScalarType type = q.scalar_type();
    if ((type != at::kHalf && type != at::kBFloat16) || q.dim() != 2) bad(op, "query must be a [tokens, hidden] tensor of fp16 or bf16");
    const Tensor& kc = tensor(op, "key_cache", args[3]);
    B200RotaryAppendParams p{};
    const int64_t H = p.num_heads = integer(op, "num_heads", args[9]), KV = p.kv_num_heads = integer(op, "kv_num_heads", args[10]);
    if (kc.dim() != 4 || kc.size(2) != KV) bad(op, "key_cache must be [blocks, block_size, kv_num_heads, head_size]");
    const int64_t nt = q.size(0), blocks = kc.size(0), block_size = kc.size(1), d = kc.size(3);
    if (nt > INT32_MAX || blocks > INT32_MAX || block_size > INT32_MAX || d > INT32_MAX) bad(op, "a dimension is too large");
    const int device = device_of(op, q);
    p.num_tokens = (int32_t)nt;
    p.num_blocks = (int32_t)blocks;
    p.block_size = (int32_t)block_size;
    p.head_size = (int32_t)d;
    p.act_dtype = dtype_of(type);
    p.query = q.data_ptr();
    if (args[1] == Py_None && args[2] == Py_None) {
      p.query_row_stride = p.key_row_stride = p.value_row_stride = rows(op, "packed query", q, nt, (H + 2 * KV) * d, type, device);
      p.key = static_cast<const char*>(p.query) + 2 * H * d;
      p.value = static_cast<const char*>(p.query) + 2 * (H + KV) * d;
    } else if (args[1] == Py_None || args[2] == Py_None) {
      bad(op, "key and value must be given together");
    } else {
      const Tensor &k = tensor(op, "key", args[1]), &v = tensor(op, "value", args[2]);
      p.query_row_stride = rows(op, "query", q, nt, H * d, type, device);
      p.key_row_stride = rows(op, "key", k, nt, KV * d, type, device);
      p.value_row_stride = rows(op, "value", v, nt, KV * d, type, device);
      p.key = k.data_ptr();
      p.value = v.data_ptr();
    }
    const ScalarType cache = kc.scalar_type();
    if (cache != type && cache != at::kFloat8_e4m3fn) bad(op, "the cache must have the activations' type or fp8 e4m3");
    p.cache_dtype = dtype_of(cache);
    p.key_cache = dense(op, "key_cache", kc, kc.sizes(), cache, device);
    p.value_cache = dense(op, "value_cache", tensor(op, "value_cache", args[4]), kc.sizes(), cache, device);
    if (cache != type) {
      if (args[14] == Py_None || args[15] == Py_None) bad(op, "fp8 caches require k_scale and v_scale");
      p.k_scale = dense<float>(op, "k_scale", tensor(op, "k_scale", args[14]), {blocks, KV}, at::kFloat, device);
      p.v_scale = dense<float>(op, "v_scale", tensor(op, "v_scale", args[15]), {blocks, KV}, at::kFloat, device);
    }
    const Tensor& cos = tensor(op, "cos_cache", args[6]);
    const ScalarType table = cos.scalar_type();
    if ((table != type && table != at::kFloat) || cos.dim() != 2 || cos.size(0) > INT32_MAX || cos.size(1) > INT32_MAX / 2)
      bad(op, "cos_cache must be [positions, rotary_dim / 2] of the activations' type or fp32");
    p.table_dtype = dtype_of(table);
    p.rotary_positions = (int32_t)cos.size(0);
    p.rotary_dim = (int32_t)(2 * cos.size(1));
    p.cos_cache = dense(op, "cos_cache", cos, cos.sizes(), table, device);
    p.sin_cache = dense(op, "sin_cache", tensor(op, "sin_cache", args[7]), cos.sizes(), table, device);
    p.rotary_interleaved = integer(op, "rotary_interleaved", args[12]);
    p.rotary_offset = integer(op, "rotary_offset", args[13]);
    const c10::cuda::CUDAGuard guard((c10::DeviceIndex)device);
    const Tensor& given_pos = tensor(op, "position_ids", args[5]);
    const ScalarType index = given_pos.scalar_type();
    const int64_t rank = given_pos.dim();
    if ((index != at::kInt && index != at::kLong) || rank < 1 || rank > 2 || given_pos.size(rank - 1) != nt || !on(given_pos, device))
      bad(op, "position_ids must be an int32 or int64 [tokens] or [axes, tokens] tensor on cuda:" + std::to_string(device));
    // the C ABI reads a token stride of 0 as 1
    const Tensor pos = nt > 1 && given_pos.stride(rank - 1) == 0 ? given_pos.contiguous() : given_pos;
    p.position_dtype = dtype_of(index);
    p.position_ids = pos.data_ptr();
    p.position_token_stride = pos.stride(rank - 1);
    p.position_axis_stride = rank == 2 ? pos.stride(0) : 0;
    const int64_t axes = rank == 2 ? pos.size(0) : 1;
    int64_t named = 1;
    p.axis_pairs[0] = (int32_t)cos.size(1);
    if (args[11] != Py_None) {
      named = PySequence_Check(args[11]) ? PySequence_Size(args[11]) : -1;
      PyErr_Clear();
      for (int64_t i = 0; i < named && i < B200_MAX_ROTARY_AXES; ++i) {
        PyObject* item = PySequence_GetItem(args[11], i);
        if (!item) PyErr_Clear(), bad(op, "axis_sections must be a sequence of integers");
        try {
          p.axis_pairs[i] = integer(op, "axis_sections", item);
        } catch (...) {
          Py_DECREF(item);
          throw;
        }
        Py_DECREF(item);
      }
    }
    if (named != axes || axes > B200_MAX_ROTARY_AXES)
      bad(op, "axis_sections must name the pairs of each of the " + std::to_string(axes) + " position axes (at most 4)");
    p.axes = (int32_t)axes;
    p.slot_mapping = dense<int32_t>(op, "slot_mapping", tensor(op, "slot_mapping", args[8]), {nt}, at::kInt, device);
    Tensor out;
    if (args[16] == Py_None) {
      out = empty({nt, H * d}, type, device);
      p.output = out.data_ptr();
    } else {
      const Tensor& o = tensor(op, "output", args[16]);
      p.output_row_stride = rows(op, "output", o, nt, H * d, type, device);
      p.output = o.data_ptr();
    }
    cudaStream_t stream = c10::cuda::getCurrentCUDAStream((c10::DeviceIndex)device).stream();
    p.device_status = status_word(op, device, stream);
    if (nt <= B200_ROTARY_APPEND_SCAN_TOKENS) checked(b200_rotary_append(&p, stream));
    else run_with_workspace(op, &p, args[17], device, stream, b200_rotary_append_workspace_size, b200_rotary_append);
    return tuple_of({given_or(args[16], std::move(out)), shared(args[3]), shared(args[4])});
  });
}

// query, key_cache, value_cache, cumulative_sequence_length, past_seqlens, block_table, prefix_block_table,
// prefix_length, num_heads, kv_num_heads, scale, softcap, head_sink, output, workspace, num_sms
PyObject* shared_prefix_attention(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (!arguments("shared_prefix_attention", n, 16)) return nullptr;
  return guarded([&] {
    constexpr const char* op = "SharedPrefixAttention";
    const Tensor& q = tensor(op, "query", args[0]);
    const ScalarType type = q.scalar_type();
    if ((type != at::kHalf && type != at::kBFloat16) || q.dim() != 2) bad(op, "query must be a [tokens, hidden] tensor of fp16 or bf16");
    const Tensor& kc = tensor(op, "key_cache", args[1]);
    B200SharedPrefixParams p{};
    const int64_t H = p.num_heads = integer(op, "num_heads", args[8]), KV = p.kv_num_heads = integer(op, "kv_num_heads", args[9]);
    if (kc.dim() != 4 || kc.size(2) != KV) bad(op, "key_cache must be [blocks, block_size, kv_num_heads, head_size]");
    const int64_t nt = q.size(0), d = kc.size(3);
    const int device = device_of(op, q);
    p.query_row_stride = rows(op, "query", q, nt, H * d, type, device);
    p.query = q.data_ptr();
    p.key_cache = dense(op, "key_cache", kc, kc.sizes(), type, device);
    p.value_cache = dense(op, "value_cache", tensor(op, "value_cache", args[2]), kc.sizes(), type, device);
    const Tensor& table = tensor(op, "block_table", args[5]);
    if (table.dim() != 2) bad(op, "block_table must be [batch, blocks]");
    const int64_t batch = table.size(0);
    if (std::max({nt, kc.size(0), kc.size(1), d, batch + 1, table.size(1)}) > INT32_MAX) bad(op, "a dimension is too large");
    p.block_table = dense<int32_t>(op, "block_table", table, table.sizes(), at::kInt, device);
    p.past_seqlens = dense<int32_t>(op, "past_seqlens", tensor(op, "past_seqlens", args[4]), {batch}, at::kInt, device);
    p.cumulative_sequence_length = dense<int32_t>(op, "cumulative_sequence_length",
                                                  tensor(op, "cumulative_sequence_length", args[3]), {batch + 1}, at::kInt, device);
    if (args[6] != Py_None) {
      const Tensor& pt = tensor(op, "prefix_block_table", args[6]);
      if (pt.numel() > INT32_MAX) bad(op, "a dimension is too large");
      p.prefix_blocks = (int32_t)pt.numel();
      p.prefix_block_table = dense<int32_t>(op, "prefix_block_table", pt, {pt.numel()}, at::kInt, device);
    }
    if (args[12] != Py_None) p.head_sink = dense(op, "head_sink", tensor(op, "head_sink", args[12]), {H}, type, device);
    p.head_size = (int32_t)d;
    p.scale = number(op, "scale", args[10]);
    p.softcap = number(op, "softcap", args[11]);
    p.act_dtype = dtype_of(type);
    p.num_tokens = (int32_t)nt;
    p.batch = (int32_t)batch;
    p.num_blocks = (int32_t)kc.size(0);
    p.block_size = (int32_t)kc.size(1);
    p.max_blocks_per_seq = (int32_t)table.size(1);
    p.prefix_length = integer(op, "prefix_length", args[7]);
    p.num_sms = integer(op, "num_sms", args[15]);
    const c10::cuda::CUDAGuard guard((c10::DeviceIndex)device);
    Tensor out;
    if (args[13] == Py_None) {
      out = empty({nt, H * d}, type, device);
      p.output = out.data_ptr();
    } else {
      const Tensor& o = tensor(op, "output", args[13]);
      p.output_row_stride = rows(op, "output", o, nt, H * d, type, device);
      p.output = o.data_ptr();
    }
    cudaStream_t stream = c10::cuda::getCurrentCUDAStream((c10::DeviceIndex)device).stream();
    p.device_status = status_word(op, device, stream);
    run_with_workspace(op, &p, args[14], device, stream, b200_shared_prefix_attention_workspace_size,
                       b200_shared_prefix_attention);
    return given_or(args[13], std::move(out));
  });
}

// device index -> None; raises what the current stream's calls on it reported since the last time
PyObject* read_status(PyObject*, PyObject* arg) {
  return guarded([&]() -> PyObject* {
    const int device = integer("layer status", "device", arg);
    const c10::cuda::CUDAGuard guard((c10::DeviceIndex)device);
    cudaStream_t stream = c10::cuda::getCurrentCUDAStream((c10::DeviceIndex)device).stream();
    const auto it = stream_words().find({device, stream});
    if (it != stream_words().end()) checked(b200_layer_read_status(it->second, stream));
    Py_RETURN_NONE;
  });
}

PyObject* set_error_class(PyObject*, PyObject* cls) {
  Py_INCREF(cls);
  g_error_class = cls;
  Py_RETURN_NONE;
}

PyMethodDef kMethods[] = {
    {"skip_rms_norm", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)(void)>(skip_rms_norm)), METH_FASTCALL, nullptr},
    {"rotary_append", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)(void)>(rotary_append)), METH_FASTCALL, nullptr},
    {"shared_prefix_attention", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)(void)>(shared_prefix_attention)),
     METH_FASTCALL, nullptr},
    {"read_status", read_status, METH_O, nullptr},
    {"set_error_class", set_error_class, METH_O, nullptr},
    {nullptr, nullptr, 0, nullptr}};

PyModuleDef kModule = {PyModuleDef_HEAD_INIT, "_layer", "Binding of include/b200_layer.h for torch tensors.", -1, kMethods,
                       nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__layer(void) { return PyModule_Create(&kModule); }
