// The native side of nibble_b200/kv_cache.py: checks tensors, allocates outputs and workspaces from the caching allocator, and
// hands pointers plus the current stream of the tensors' device to the C ABI.  Every violation is a TORCH_CHECK, i.e. a
// RuntimeError.  (Messages hold no numbers: with this image's compiler, formatting one through a stream crashes.)  Nothing here takes
// part in autograd: a call whose input asks for a gradient, or carries a forward-mode tangent, is refused.
#include "kv_module.h"

#include <ATen/ATen.h>
#include <ATen/MemoryOverlap.h>
#include <ATen/cuda/CUDAContext.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/core/AutogradState.h>
#include <c10/core/GradMode.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <algorithm>
#include <cstdlib>
#include <cstring>
#include <optional>

#include "../../include/w4a16_b200.h"

namespace w4a16 {
namespace {

const at::Tensor& tensor_of(PyObject* object, const char* name) {
    TORCH_CHECK(THPVariable_Check(object), name, " must be a tensor");
    const at::Tensor& t = THPVariable_Unpack(object);
    TORCH_CHECK(t.is_cuda(), name, " must be a CUDA tensor");
    TORCH_CHECK(!(t.requires_grad() && c10::GradMode::is_enabled()),
                name, " requires a gradient, which this operator does not form; detach it or use torch.no_grad()");
    TORCH_CHECK(!(at::isFloatingType(t.scalar_type()) && c10::AutogradState::get_tls_state().get_fw_grad_mode() && t._fw_grad(/*level=*/0).defined()),
                name, " carries a tangent of forward-mode differentiation, which this operator does not pass on");
    return t;
}
std::optional<at::Tensor> optional_of(PyObject* object, const char* name) {
    if (object == Py_None) return std::nullopt;
    return tensor_of(object, name);
}
int64_t integer_of(PyObject* object) {
    const int64_t value = PyLong_AsLongLong(object);
    if (PyErr_Occurred() != nullptr) throw python_error();
    return value;
}
double number_of(PyObject* object) {
    const double value = PyFloat_AsDouble(object);
    if (PyErr_Occurred() != nullptr) throw python_error();
    return value;
}
void check_count(Py_ssize_t count, Py_ssize_t wanted, const char* what) {
    TORCH_CHECK(count == wanted, what, " takes another number of arguments");
}
void check_status(int status, const char* what) {
    TORCH_CHECK(status == W4A16_OK, what, " failed: ", w4a16_status_string(status));
}

at::ScalarType dtype_of(int32_t type) { return type == W4A16_TYPE_BF16 ? at::kBFloat16 : at::kHalf; }

// A cache as Python holds it: one buffer and its sizes.
struct Cache {
    at::Tensor memory;
    w4a16_kv8_cache parts;
};
constexpr int kCacheArguments = 6;
Cache cache_of(PyObject* const* args) {
    Cache cache;
    cache.memory = tensor_of(args[0], "the cache");
    check_status(w4a16_kv8_cache_describe(cache.memory.data_ptr(), static_cast<size_t>(cache.memory.nbytes()), integer_of(args[1]),
                                          integer_of(args[2]), integer_of(args[3]), integer_of(args[4]),
                                          static_cast<int32_t>(integer_of(args[5])), &cache.parts),
                 "QuantizedKVCache");
    return cache;
}

// Numbers of one type, [batch, tokens, heads, head_dim] in any order of the first three.
w4a16_rows rows_of(const at::Tensor& t, const at::Device& device, at::ScalarType dtype, const char* name) {
    TORCH_CHECK(t.device() == device, name, " must be on the same device");
    TORCH_CHECK(t.scalar_type() == dtype, name, dtype == at::kHalf ? " must have dtype torch.float16" : " must have dtype torch.bfloat16");
    TORCH_CHECK(t.dim() == 4, name, " must have shape [batch, tokens, heads, head_dim]");
    TORCH_CHECK(t.stride(3) == 1 || t.numel() == 0, "the last dimension of ", name, " must be contiguous");
    return w4a16_rows{t.data_ptr(), t.stride(0), t.stride(1), t.stride(2)};
}

const int64_t* words_of(const at::Tensor& t, const at::Device& device, int64_t count, const char* name) {
    TORCH_CHECK(t.device() == device, name, " must be on the same device");
    TORCH_CHECK(t.scalar_type() == at::kLong && t.is_contiguous(), name, " must be a contiguous int64 tensor");
    TORCH_CHECK(t.numel() == count, name, " has the wrong number of elements");
    return t.const_data_ptr<int64_t>();
}

w4a16_rotary_spec spec_of(const at::Tensor& inv_freq, const at::Device& device, int64_t head_dim, double scale, bool interleaved) {
    TORCH_CHECK(inv_freq.device() == device, "inv_freq must be on the same device");
    TORCH_CHECK(inv_freq.scalar_type() == at::kFloat && inv_freq.is_contiguous() && inv_freq.dim() == 1,
                "inv_freq must be a contiguous 1-d float32 tensor");
    TORCH_CHECK(inv_freq.numel() >= 1 && 2 * inv_freq.numel() <= head_dim, "inv_freq must have between 1 and head_dim / 2 elements");
    return w4a16_rotary_spec{inv_freq.const_data_ptr<float>(), static_cast<int32_t>(2 * inv_freq.numel()), interleaved ? 1 : 0,
                             static_cast<float>(scale)};
}

w4a16_stream_t current_stream() { return reinterpret_cast<w4a16_stream_t>(at::cuda::getCurrentCUDAStream().stream()); }

// (what nibble_b200.cuda.programmatic_launch_enabled() says; asked here, since looking it up in Python shows in a call of 5 us)
uint32_t launch_flags() {
    const char* knob = std::getenv("W4A16_PDL");
    return knob != nullptr && std::strcmp(knob, "1") == 0 ? W4A16_FLAG_PROGRAMMATIC_LAUNCH : 0u;
}

bool truth_of(PyObject* object) {
    const int value = PyObject_IsTrue(object);
    if (value < 0) throw python_error();
    return value != 0;
}

// Whether integers i_d, |i_d| < sizes[d], can make sum i_d * strides[d] equal to `offset`; strides falling from `dim` on.  True where
// finding out would take long, as with strides that do not nest.
bool reachable(const int64_t (&sizes)[4], const int64_t (&strides)[4], int dim, int64_t offset) {
    if (dim == 4) return offset == 0;
    int64_t within = 0;                                  // what the dimensions behind this one reach
    for (int d = dim + 1; d < 4; ++d) within += (sizes[d] - 1) * strides[d];
    const int64_t stride = strides[dim], most = sizes[dim] - 1;
    if (most == 0 || stride == 0) return reachable(sizes, strides, dim + 1, offset);
    // i * stride from offset - within to offset + within
    int64_t low = offset - within, high = offset + within;
    low = low >= 0 ? (low + stride - 1) / stride : -(-low / stride);
    high = high >= 0 ? high / stride : -((-high + stride - 1) / stride);
    low = std::max(low, -most);
    high = std::min(high, most);
    if (high - low > 3) return true;
    for (int64_t i = low; i <= high; ++i) {
        if (reachable(sizes, strides, dim + 1, offset - i * stride)) return true;
    }
    return false;
}

// Whether two tensors of the same sizes go from number to number by the same strides (those of dimensions with one entry say nothing).
bool same_strides(const at::Tensor& a, const at::Tensor& b) {
    for (int64_t d = 0; d < a.dim(); ++d) {
        if (a.size(d) > 1 && a.stride(d) != b.stride(d)) return false;
    }
    return true;
}

// Whether two tensors of the same sizes (four dimensions at most) and 16-bit type may share memory: by their extents, and where those
// meet and the strides are the same, as of two parts of a fused row, exactly.
bool may_share(const at::Tensor& a, const at::Tensor& b) {
    if (a.numel() == 0) return false;
    auto past = [](const at::Tensor& t) {
        int64_t numbers = 1;
        for (int64_t d = 0; d < t.dim(); ++d) numbers += (t.size(d) - 1) * t.stride(d);
        return reinterpret_cast<uintptr_t>(t.const_data_ptr()) + static_cast<uintptr_t>(numbers) * 2;
    };
    const auto begin_a = reinterpret_cast<uintptr_t>(a.const_data_ptr()), begin_b = reinterpret_cast<uintptr_t>(b.const_data_ptr());
    if (past(a) <= begin_b || past(b) <= begin_a) return false;
    if (!same_strides(a, b) || (begin_a - begin_b) % 2 != 0) return true;
    int64_t sizes[4] = {1, 1, 1, 1}, strides[4] = {0, 0, 0, 0};
    int order[4] = {0, 1, 2, 3};
    std::sort(order, order + a.dim(), [&](int x, int y) { return a.stride(x) > a.stride(y); });
    for (int64_t d = 0; d < a.dim(); ++d) {
        sizes[d] = a.size(order[d]);
        strides[d] = a.stride(order[d]);
    }
    return reachable(sizes, strides, 0, (static_cast<int64_t>(begin_a) - static_cast<int64_t>(begin_b)) / 2);
}

}  // namespace

// rotary(x, positions, inv_freq, scale, interleaved, out or None) -> Tensor
PyObject* rotary(PyObject*, PyObject* const* args, Py_ssize_t count) {
    HANDLE_TH_ERRORS
    check_count(count, 6, "rotary");
    const at::Tensor& x = tensor_of(args[0], "x");
    const at::Tensor& positions = tensor_of(args[1], "positions");
    const at::Tensor& inv_freq = tensor_of(args[2], "inv_freq");
    const double scale = number_of(args[3]);
    const bool interleaved = truth_of(args[4]);
    std::optional<at::Tensor> given = optional_of(args[5], "out");
    const uint32_t flags = launch_flags();
    TORCH_CHECK(x.dim() >= 2 && x.dim() <= 4, "x must have shape [heads, head_dim], [tokens, heads, head_dim] or [batch, tokens, heads, head_dim]");
    TORCH_CHECK(x.scalar_type() == at::kHalf || x.scalar_type() == at::kBFloat16, "x must have dtype torch.float16 or torch.bfloat16");
    TORCH_CHECK(x.size(-1) >= 2 && x.size(-1) <= 256 && x.size(-1) % 2 == 0, "head_dim must be even, between 2 and 256");
    TORCH_CHECK(x.size(-2) <= INT32_MAX, "too many heads");
    TORCH_CHECK(positions.sizes() == x.sizes().slice(0, x.dim() - 2), "positions must have the shape of x without heads and head_dim");
    const w4a16_rotary_spec spec = spec_of(inv_freq, x.device(), x.size(-1), scale, interleaved);
    const c10::cuda::CUDAGuard guard(x.device());
    at::Tensor out;
    bool in_place = false;
    if (given.has_value()) {
        out = *given;
        TORCH_CHECK(out.device() == x.device() && out.scalar_type() == x.scalar_type(), "out must be on the device of x and of its dtype");
        TORCH_CHECK(out.sizes() == x.sizes(), "out must have the shape of x");
        at::assert_no_internal_overlap(out);
        in_place = out.data_ptr() == x.data_ptr() && same_strides(out, x);
        TORCH_CHECK(in_place || !may_share(out, x), "out must be x itself or share no memory with it");
    } else {
        out = at::detail::empty_cuda(x.sizes(), x.scalar_type(), x.device(), c10::nullopt);
    }
    TORCH_CHECK(x.numel() == 0 || (x.stride(-1) == 1 && out.stride(-1) == 1), "the last dimension of x and out must be contiguous");
    // (as [batch, tokens, heads, head_dim], dimensions that are not there having one entry)
    const int64_t missing = 4 - x.dim();
    auto size = [&](int64_t dim) { return dim < missing ? 1 : x.size(dim - missing); };
    auto rows = [&](const at::Tensor& t) {
        auto stride = [&](int64_t dim) { return dim < missing ? 0 : t.stride(dim - missing); };
        return w4a16_rows{t.data_ptr(), stride(0), stride(1), stride(2)};
    };
    const w4a16_rows from = rows(x), to = in_place ? from : rows(out);
    const int64_t* at_positions = words_of(positions, x.device(), size(0) * size(1), "positions");
    if (x.numel() > 0) {
        pybind11::gil_scoped_release unlocked;
        check_status(w4a16_rotary(&spec, &from, &to, size(0), size(1), static_cast<int32_t>(size(2)),
                                  static_cast<int32_t>(size(3)), at_positions,
                                  x.scalar_type() == at::kBFloat16 ? W4A16_TYPE_BF16 : W4A16_TYPE_F16, flags, current_stream()),
                     "apply_rotary");
    }
    // (so that autograd, and whoever else goes by versions, sees that a tensor given as `out` has changed)
    if (given.has_value() && !out.is_inference()) out.unsafeGetTensorImpl()->bump_version();
    return THPVariable_Wrap(std::move(out));
    END_HANDLE_TH_ERRORS
}

// kv8_bytes(batch, kv_heads, max_len, head_dim) -> int
PyObject* kv8_bytes(PyObject*, PyObject* const* args, Py_ssize_t count) {
    HANDLE_TH_ERRORS
    check_count(count, 4, "kv8_bytes");
    return PyLong_FromSize_t(w4a16_kv8_cache_bytes(integer_of(args[0]), integer_of(args[1]), integer_of(args[2]), integer_of(args[3])));
    END_HANDLE_TH_ERRORS
}

// kv8_append(cache..., k, v, start, counts or None, inv_freq or None, rope_scale, interleaved, q or None) -> turned q or None
PyObject* kv8_append(PyObject*, PyObject* const* args, Py_ssize_t count) {
    HANDLE_TH_ERRORS
    check_count(count, kCacheArguments + 8, "kv8_append");
    const Cache cache = cache_of(args);
    args += kCacheArguments;
    const at::Tensor& k = tensor_of(args[0], "k");
    const at::Tensor& v = tensor_of(args[1], "v");
    const at::Tensor& start = tensor_of(args[2], "start");
    const std::optional<at::Tensor> counts = optional_of(args[3], "counts");
    const std::optional<at::Tensor> inv_freq = optional_of(args[4], "inv_freq");
    const double rope_scale = number_of(args[5]);
    const bool interleaved = truth_of(args[6]);
    const std::optional<at::Tensor> q = optional_of(args[7], "q");
    const uint32_t flags = launch_flags();
    const at::Device device = cache.memory.device();
    const at::ScalarType dtype = dtype_of(cache.parts.type);
    const w4a16_rows k_rows = rows_of(k, device, dtype, "k"), v_rows = rows_of(v, device, dtype, "v");
    const int64_t tokens = k.size(1);
    TORCH_CHECK(k.size(0) == cache.parts.batch && k.size(2) == cache.parts.kv_heads && k.size(3) == cache.parts.head_dim,
                "k must have shape [batch, tokens, kv_heads, head_dim] of the cache");
    TORCH_CHECK(v.sizes() == k.sizes(), "v must have the shape of k");
    const int64_t* starts = words_of(start, device, cache.parts.batch, "start");
    const int64_t* counted = counts.has_value() ? words_of(*counts, device, cache.parts.batch, "counts") : nullptr;
    TORCH_CHECK(!q.has_value() || inv_freq.has_value(), "q is turned along with the keys, which takes inv_freq");
    const c10::cuda::CUDAGuard guard(device);
    w4a16_rotary_spec spec{};
    w4a16_rows q_rows{}, turned_rows{};
    at::Tensor turned;
    if (inv_freq.has_value()) spec = spec_of(*inv_freq, device, cache.parts.head_dim, rope_scale, interleaved);
    if (q.has_value()) {
        q_rows = rows_of(*q, device, dtype, "q");
        TORCH_CHECK(q->size(0) == k.size(0) && q->size(1) == tokens && q->size(3) == k.size(3) && q->size(2) > 0,
                    "q must have shape [batch, tokens, q_heads, head_dim]");
        TORCH_CHECK(q->size(2) <= INT32_MAX, "too many heads");
        turned = at::detail::empty_cuda(q->sizes(), dtype, device, c10::nullopt);
        turned_rows = rows_of(turned, device, dtype, "q");
    }
    if (tokens > 0) {
        pybind11::gil_scoped_release unlocked;
        check_status(w4a16_kv8_append(&cache.parts, &k_rows, &v_rows, tokens, starts, counted, inv_freq.has_value() ? &spec : nullptr,
                                      q.has_value() ? &q_rows : nullptr, q.has_value() ? &turned_rows : nullptr,
                                      q.has_value() ? static_cast<int32_t>(q->size(2)) : 0, flags, current_stream()),
                     "QuantizedKVCache.append");
    }
    if (!q.has_value()) Py_RETURN_NONE;
    return THPVariable_Wrap(std::move(turned));
    END_HANDLE_TH_ERRORS
}

// kv8_read(cache..., lengths, first or None, tokens) -> (k, v)
PyObject* kv8_read(PyObject*, PyObject* const* args, Py_ssize_t count) {
    HANDLE_TH_ERRORS
    check_count(count, kCacheArguments + 3, "kv8_read");
    const Cache cache = cache_of(args);
    args += kCacheArguments;
    const at::Tensor& lengths = tensor_of(args[0], "lengths");
    const std::optional<at::Tensor> first = optional_of(args[1], "first");
    const int64_t tokens = integer_of(args[2]);
    const uint32_t flags = launch_flags();
    TORCH_CHECK(tokens >= 0, "tokens must not be negative");
    const at::Device device = cache.memory.device();
    const int64_t* length = words_of(lengths, device, cache.parts.batch, "lengths");
    const int64_t* begin = first.has_value() ? words_of(*first, device, cache.parts.batch, "first") : nullptr;
    const c10::cuda::CUDAGuard guard(device);
    const int64_t shape[] = {cache.parts.batch, tokens, cache.parts.kv_heads, cache.parts.head_dim};
    at::Tensor k = at::detail::empty_cuda(shape, dtype_of(cache.parts.type), device, c10::nullopt);
    at::Tensor v = at::detail::empty_cuda(shape, dtype_of(cache.parts.type), device, c10::nullopt);
    if (tokens > 0) {
        pybind11::gil_scoped_release unlocked;
        check_status(w4a16_kv8_read(&cache.parts, length, begin, tokens, k.data_ptr(), v.data_ptr(), flags, current_stream()),
                     "QuantizedKVCache.read");
    }
    PyObject* first_half = THPVariable_Wrap(std::move(k));
    PyObject* second_half = first_half == nullptr ? nullptr : THPVariable_Wrap(std::move(v));
    PyObject* both = second_half == nullptr ? nullptr : PyTuple_Pack(2, first_half, second_half);
    Py_XDECREF(first_half);
    Py_XDECREF(second_half);
    return both;
    END_HANDLE_TH_ERRORS
}

// kv8_attention(cache..., q, lengths, counts or None, softmax_scale) -> Tensor
PyObject* kv8_attention(PyObject*, PyObject* const* args, Py_ssize_t count) {
    HANDLE_TH_ERRORS
    check_count(count, kCacheArguments + 4, "kv8_attention");
    const Cache cache = cache_of(args);
    args += kCacheArguments;
    const at::Tensor& q = tensor_of(args[0], "q");
    const at::Tensor& lengths = tensor_of(args[1], "lengths");
    const std::optional<at::Tensor> counts = optional_of(args[2], "counts");
    const double softmax_scale = number_of(args[3]);
    const uint32_t flags = launch_flags();
    const at::Device device = cache.memory.device();
    const at::ScalarType dtype = dtype_of(cache.parts.type);
    const w4a16_rows q_rows = rows_of(q, device, dtype, "q");
    TORCH_CHECK(q.size(0) == cache.parts.batch && q.size(3) == cache.parts.head_dim, "q must have shape [batch, tokens, q_heads, head_dim]");
    TORCH_CHECK(q.size(2) > 0 && q.size(2) <= INT32_MAX && q.size(2) % cache.parts.kv_heads == 0,
                "the query heads must be a multiple of the cache's key/value heads");
    const int64_t* length = words_of(lengths, device, cache.parts.batch, "lengths");
    const int64_t* counted = counts.has_value() ? words_of(*counts, device, cache.parts.batch, "counts") : nullptr;
    const c10::cuda::CUDAGuard guard(device);
    at::Tensor out = at::detail::empty_cuda(q.sizes(), dtype, device, c10::nullopt);
    if (q.numel() > 0) {
        pybind11::gil_scoped_release unlocked;
        const auto heads = static_cast<int32_t>(q.size(2));
        const size_t wanted = w4a16_kv8_attention_workspace_bytes(&cache.parts, heads, q.size(1));
        at::Tensor workspace;
        if (wanted > 0) workspace = at::detail::empty_cuda({static_cast<int64_t>(wanted)}, at::kByte, device, c10::nullopt);
        check_status(w4a16_kv8_attention(&cache.parts, &q_rows, out.data_ptr(), heads, q.size(1), length, counted,
                                         static_cast<float>(softmax_scale), wanted > 0 ? workspace.data_ptr() : nullptr, wanted, flags,
                                         current_stream()),
                     "QuantizedKVCache.attention");
    }
    return THPVariable_Wrap(std::move(out));
    END_HANDLE_TH_ERRORS
}

}  // namespace w4a16
