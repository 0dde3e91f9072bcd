// Operator calls on torch tensors, natively: module `_torch_call`, used by ops.py.
//
// Every operator of the C-ABI becomes a vectorcall that takes the C function's arguments in order -- tensors (or None, or
// what pinned() returns) where it takes pointers, numbers elsewhere -- without the trailing stream, which is torch's current one.
// Conversion and checks are generated from the C signature.  The same call through ctypes spent 9 us of host time on a
// launch of 2.7 us (stream object 2.9 us, 0.3 us per pointer object); this way it is 3.5 us.
//
// The functions are looked up in the library that lib.py has loaded (bind), so a build of it with other kernels is called
// through the same module.  torch supplies memory and the stream; no torch type crosses the C-ABI.
#include <torch/csrc/autograd/python_variable.h>

#include <ATen/core/CachingHostAllocator.h>
#include <ATen/hip/EmptyTensor.h>
#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/utils/object_ptr.h>

#include <dlfcn.h>

#include <tuple>
#include <type_traits>
#include <utility>

#include "../../../include/cpmcu_amd.h"

namespace {

const char* (*g_last_error)(void) = nullptr;

template <typename Body>
auto without_gil(Body body) {
    struct Released {
        PyThreadState* state = PyEval_SaveThread();
        ~Released() { PyEval_RestoreThread(state); }
    } released;
    return body();
}

// Every entry of the module goes through one of these.  Asking a tensor for its memory or its layout throws where it has none (vmapped,
// fake, meta or sparse tensors), as do streams without a device: that is Python's RuntimeError, and must not cross the interpreter's C frames.
template <typename Body>
PyObject* guarded(Body body) {
    try {
        return body();
    } catch (const c10::Error& e) {
        PyErr_SetString(PyExc_RuntimeError, e.what_without_backtrace());
    } catch (const std::exception& e) {
        PyErr_SetString(PyExc_RuntimeError, e.what());
    } catch (...) {
        PyErr_SetString(PyExc_RuntimeError, "an exception of unknown type");
    }
    return nullptr;
}
template <PyObject* (*F)(PyObject*, PyObject* const*, Py_ssize_t)>
PyObject* entry(PyObject* self, PyObject* const* args, Py_ssize_t nargs) {
    return guarded([&] { return F(self, args, nargs); });
}
template <PyObject* (*F)(PyObject*, PyObject*)>
PyObject* entry(PyObject* self, PyObject* arg) {
    return guarded([&] { return F(self, arg); });
}

// The name of pinned()'s capsules.
constexpr const char* kPinned = "cpmcu pinned memory";

// One C argument from one Python object; false with a Python error set.
template <typename T>
bool convert(PyObject* o, T* out) {
    if constexpr (std::is_pointer_v<T>) {
        if (o == Py_None) {
            *out = nullptr;
            return true;
        }
        if (THPVariable_Check(o)) {
            const at::Tensor& t = THPVariable_Unpack(o);
            if (!t.is_cuda() || !t.is_contiguous()) {
                PyErr_SetString(PyExc_AssertionError, "device-resident contiguous tensor required");
                return false;
            }
            *out = reinterpret_cast<T>(t.data_ptr());
            return true;
        }
        // (a bare number is no address: only what pinned() has looked at stands for memory that is not a device tensor's)
        if (!PyCapsule_IsValid(o, kPinned)) {
            PyErr_Format(PyExc_TypeError, "a tensor or None required, not %.100s", Py_TYPE(o)->tp_name);
            return false;
        }
        *out = reinterpret_cast<T>(PyCapsule_GetPointer(o, kPinned));
        return true;
    } else if constexpr (std::is_floating_point_v<T>) {
        *out = static_cast<T>(PyFloat_AsDouble(o));
    } else if constexpr (std::is_same_v<T, int>) {
        const long v = PyLong_AsLong(o);
        if (v < INT32_MIN || v > INT32_MAX) {
            PyErr_SetString(PyExc_OverflowError, "integer argument outside 32 bits");
            return false;
        }
        *out = static_cast<int>(v);
    } else {
        *out = static_cast<T>(PyLong_AsSize_t(o));
    }
    return !PyErr_Occurred();
}

// torch's current stream.  torch's default stream is HIP's null stream, which the library has to be told apart from "its own
// blocking stream": every launch on a blocking stream is ordered behind the null stream by a marker packet, 7-8 us between two
// launches (append of 9 rows in a row: 10.5 us each, 3 on the null stream itself).
void* current_stream(c10::DeviceIndex device = -1) {
    void* const st = reinterpret_cast<void*>(c10::hip::getCurrentHIPStream(device).stream());
    return st ? st : CPMCU_STREAM_LEGACY;
}

PyObject* status(int rc) {
    if (rc == CPMCU_OK) Py_RETURN_NONE;
    PyErr_SetString(rc == CPMCU_ERR_INVALID_ARGUMENT ? PyExc_ValueError : PyExc_RuntimeError, g_last_error());
    return nullptr;
}

template <typename Fn>
struct Caller;
template <typename R, typename... A>
struct Caller<R (*)(A...)> {
    using Args = std::tuple<A...>;
    static constexpr size_t kAll = sizeof...(A);
    // a status-returning function whose last argument is void* takes the stream there
    static constexpr bool kStream = std::is_same_v<R, int> && std::is_same_v<std::tuple_element_t<kAll - 1, Args>, void*>;
    static constexpr size_t kGiven = kAll - (kStream ? 1 : 0);

    template <size_t... I>
    static bool fill(Args& a, PyObject* const* args, std::index_sequence<I...>) {
        return (convert(args[I], &std::get<I>(a)) && ...);
    }
    static PyObject* call(R (*fn)(A...), PyObject* const* args, Py_ssize_t nargs) {
        if (nargs != static_cast<Py_ssize_t>(kGiven)) {
            PyErr_Format(PyExc_TypeError, "%zd arguments given, %zd expected", nargs, static_cast<Py_ssize_t>(kGiven));
            return nullptr;
        }
        Args a;
        if (!fill(a, args, std::make_index_sequence<kGiven>{})) return nullptr;
        if constexpr (kStream) std::get<kAll - 1>(a) = current_stream();
        const R r = without_gil([&] { return std::apply(fn, a); });
        if constexpr (std::is_same_v<R, int>) return status(r);
        else return PyLong_FromSize_t(r);
    }
};

#define CPMCU_TORCH_CALLS(X)                                                                                              \
    X(kv_append) X(rope_table) X(rope_apply) X(gather_rows) X(head_weight_tile) X(head_workspace_bytes)                   \
    X(frspec_head_topk) X(lm_head_argmax) X(log_softmax_sliced) X(log_softmax_workspace_bytes) X(topk)                    \
    X(topk_workspace_bytes) X(remap) X(tree_accept) X(kv_compact) X(accept_commit) X(verify_tail) X(verify_tail_inplace)  \
    X(draft_tree_begin) X(draft_tree_extend) X(draft_tree_finish) X(draft_tree_finish_root) X(int8_weight_tile)

#define X(name)                                                                                                    \
    decltype(&cpmcu_##name) fn_##name = nullptr;                                                                   \
    PyObject* call_##name(PyObject*, PyObject* const* args, Py_ssize_t nargs) {                                    \
        return Caller<decltype(&cpmcu_##name)>::call(fn_##name, args, nargs);                                      \
    }
CPMCU_TORCH_CALLS(X)
#undef X

// The one operator with host-side results: (num_partials, partial_stride).
decltype(&cpmcu_lm_head_partials) fn_lm_head_partials = nullptr;
PyObject* call_lm_head_partials(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
    if (nargs != 11) {
        PyErr_Format(PyExc_TypeError, "%zd arguments given, 11 expected", nargs);
        return nullptr;
    }
    const void *hidden, *w;
    int layout, n, V, H, apply_scale, num = 0, stride = 0;
    float scale;
    void *logits, *ws;
    size_t ws_bytes;
    if (!(convert(args[0], &hidden) && convert(args[1], &w) && convert(args[2], &layout) && convert(args[3], &n) && convert(args[4], &V) &&
          convert(args[5], &H) && convert(args[6], &apply_scale) && convert(args[7], &scale) && convert(args[8], &logits) &&
          convert(args[9], &ws) && convert(args[10], &ws_bytes)))
        return nullptr;
    void* const st = current_stream();
    const int rc =
        without_gil([&] { return fn_lm_head_partials(hidden, w, layout, n, V, H, apply_scale, scale, logits, ws, ws_bytes, &num, &stride, st); });
    if (rc != CPMCU_OK) return status(rc);
    return Py_BuildValue("ii", num, stride);
}

// A condition on the caller's tensors; false with an AssertionError set.
bool expect(bool ok, const char* what) {
    if (!ok) PyErr_SetString(PyExc_AssertionError, what);
    return ok;
}
const at::Tensor* tensor_or_null(PyObject* o) { return THPVariable_Check(o) ? &THPVariable_Unpack(o) : nullptr; }

// kv_append_rows(k_pool, v_pool, block_table, k_new, v_new, kv_len, Hkv): rows and types from the tensors.
PyObject* call_kv_append_rows(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
    if (nargs != 7) {
        PyErr_Format(PyExc_TypeError, "%zd arguments given, 7 expected", nargs);
        return nullptr;
    }
    void *k_pool, *v_pool;
    const int32_t *table, *kv_len;
    const void *k_new, *v_new;
    int Hkv;
    if (!(convert(args[0], &k_pool) && convert(args[1], &v_pool) && convert(args[2], &table) && convert(args[3], &k_new) &&
          convert(args[4], &v_new) && convert(args[5], &kv_len) && convert(args[6], &Hkv)))
        return nullptr;
    const at::Tensor *k = tensor_or_null(args[3]), *v = tensor_or_null(args[4]), *len = tensor_or_null(args[5]);
    if (!expect(k && v && len && k->dim() >= 1, "kv_append: tensors required") ||
        !expect(k->scalar_type() == at::kHalf && v->scalar_type() == at::kHalf && len->scalar_type() == at::kInt, "kv_append: element types") ||
        !expect(k->numel() == k->size(0) * Hkv * CPMCU_HEAD_DIM && v->numel() == k->numel(), "kv_append: shapes of the rows"))
        return nullptr;
    const int T = static_cast<int>(k->size(0));
    void* const st = current_stream();
    return status(without_gil([&] { return fn_kv_append(k_pool, v_pool, table, k_new, v_new, kv_len, T, Hkv, st); }));
}

// tree_attention_rows(q, k_pool, v_pool, block_table, kv_len, max_kv_len, k_new, v_new, rope, block_window_size, mask, mask_k_range, Hkv,
// scale, out, workspace, num_splits): shapes from the tensors.  None, or the bytes needed where the workspace is too small.
decltype(&cpmcu_tree_attention_window) fn_tree_attention_window = nullptr;
decltype(&cpmcu_tree_attention_workspace_bytes) fn_tree_attention_workspace_bytes = nullptr;
PyObject* call_tree_attention_rows(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
    if (nargs != 17) {
        PyErr_Format(PyExc_TypeError, "%zd arguments given, 17 expected", nargs);
        return nullptr;
    }
    const void *q, *k_new, *v_new;
    void *k_pool, *v_pool, *out, *ws;
    const int32_t *table, *kv_len;
    const float* rope;
    const uint64_t* mask;
    int max_kv_len, window, mask_k_range, Hkv, splits;
    float scale;
    if (!(convert(args[0], &q) && convert(args[1], &k_pool) && convert(args[2], &v_pool) && convert(args[3], &table) && convert(args[4], &kv_len) &&
          convert(args[5], &max_kv_len) && convert(args[6], &k_new) && convert(args[7], &v_new) && convert(args[8], &rope) &&
          convert(args[9], &window) && convert(args[10], &mask) && convert(args[11], &mask_k_range) && convert(args[12], &Hkv) &&
          convert(args[13], &scale) && convert(args[14], &out) && convert(args[15], &ws) && convert(args[16], &splits)))
        return nullptr;
    const at::Tensor *tq = tensor_or_null(args[0]), *len = tensor_or_null(args[4]), *tk = tensor_or_null(args[6]), *tv = tensor_or_null(args[7]),
                     *tr = tensor_or_null(args[8]), *tm = tensor_or_null(args[10]), *tw = tensor_or_null(args[15]);
    if (!expect(tq && len && tq->dim() == 3 && tq->size(2) == CPMCU_HEAD_DIM && tq->scalar_type() == at::kHalf, "tree_attention: q is [T, Hq, 128] of 16-bit floats") ||
        !expect(len->scalar_type() == at::kInt, "tree_attention: kv_len is int32"))
        return nullptr;
    const int64_t T = tq->size(0), Hq = tq->size(1);
    int W = 0;
    if (tm) {
        if (!expect((tm->scalar_type() == at::kLong || tm->scalar_type() == at::kUInt64) && T > 0 && tm->numel() % T == 0, "tree_attention: mask of 64-bit words, rows alike"))
            return nullptr;
        W = static_cast<int>(tm->numel() / T);
    }
    if (tk && !expect(tv && tk->scalar_type() == at::kHalf && tv->scalar_type() == at::kHalf && tk->numel() == T * Hkv * CPMCU_HEAD_DIM && tv->numel() == tk->numel(),
                      "tree_attention: k_new and v_new are [T, Hkv, 128] of 16-bit floats"))
        return nullptr;
    if (tr && !expect(tr->scalar_type() == at::kFloat && tr->numel() == T * CPMCU_HEAD_DIM, "tree_attention: rope is [T, 64, 2] of floats")) return nullptr;
    const size_t need = fn_tree_attention_workspace_bytes(static_cast<int>(T), static_cast<int>(Hq), Hkv, max_kv_len);
    const size_t have = tw ? static_cast<size_t>(tw->nbytes()) : 0;
    if (have < need) return PyLong_FromSize_t(need);
    void* const st = current_stream();
    return status(without_gil([&] {
        return fn_tree_attention_window(q, k_pool, v_pool, table, kv_len, max_kv_len, k_new, v_new, rope, window, mask, W, mask_k_range,
                                        static_cast<int>(T), static_cast<int>(Hq), Hkv, scale, out, ws, have, splits, st);
    }));
}

// ---- batches: operators whose tensors may be views of wider rows; types, shapes and the device are checked here ----

// The tensors of a call: on the current device, whose current stream the call goes to.  Null or false with an AssertionError set.
struct Call {
    c10::DeviceIndex device = -1;  // (asked for with the first device tensor: there may be none)
    const at::Tensor* strided(PyObject* o, at::ScalarType type, const char* what) {
        const at::Tensor* t = tensor_or_null(o);
        if (t && t->is_cuda() && t->scalar_type() == type) {
            if (device < 0) device = c10::hip::current_device();
            if (t->device().index() == device) return t;
        }
        PyErr_Format(PyExc_AssertionError, "%s on the current device required", what);
        return nullptr;
    }
    const at::Tensor* dense(PyObject* o, at::ScalarType type, const char* what) {
        const at::Tensor* t = strided(o, type, what);
        return t && expect(t->is_contiguous(), "device-resident contiguous tensor required") ? t : nullptr;
    }
    void* stream() const { return current_stream(device); }
};
int32_t* ints(const at::Tensor* t) { return static_cast<int32_t*>(t->data_ptr()); }
at::Tensor new_tensor(const at::Tensor& like, at::ScalarType type, at::IntArrayRef sizes) { return at::detail::empty_cuda(sizes, type, like.device(), std::nullopt); }
// n values of a one-dimensional tensor, from `at` on, as a tensor of their own on the same memory.
at::Tensor part_of(const at::Tensor& whole, int64_t at, int64_t n) {
    auto impl = c10::make_intrusive<c10::TensorImpl>(c10::Storage(whole.storage()), whole.key_set(), whole.dtype());
    impl->set_storage_offset(at);
    impl->set_sizes_contiguous(n);
    return at::Tensor(std::move(impl));
}
bool integer(PyObject* o, int* out) { return convert(o, out); }

decltype(&cpmcu_batch_tables) fn_batch_tables = nullptr;
decltype(&cpmcu_rope_rows) fn_rope_rows = nullptr;
decltype(&cpmcu_kv_append_slots) fn_kv_append_slots = nullptr;
decltype(&cpmcu_quantize_rows) fn_quantize_rows = nullptr;
decltype(&cpmcu_int8_linear) fn_int8_linear = nullptr;
decltype(&cpmcu_int8_weight_bytes) fn_int8_weight_bytes = nullptr;

bool arguments(Py_ssize_t nargs, Py_ssize_t expected) {
    if (nargs != expected) PyErr_Format(PyExc_TypeError, "%zd arguments given, %zd expected", nargs, expected);
    return nargs == expected;
}

// batch_tables(kv_lens, new_lens, block_tables, held, free_pages, counts, max_rows): (kv_lens, held, counts, row_offsets, positions, slots, state).
// One allocation (six cost 2.5 us of host time more), each part on 16 bytes; state is the first three as they lie in it, counts, held, kv_lens.
PyObject* call_batch_tables(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
    if (!arguments(nargs, 7)) return nullptr;
    Call call;
    const at::Tensor* t[6];
    for (int i = 0; i < 6; ++i)
        if (!(t[i] = call.dense(args[i], at::kInt, "batch_tables: int32 tensors"))) return nullptr;
    int max_rows;
    if (!integer(args[6], &max_rows)) return nullptr;
    const at::Tensor &tables = *t[2], &stack = *t[4];
    const int64_t B = t[0]->numel();
    if (!expect(tables.dim() == 2 && tables.size(0) == B && t[1]->numel() == B && t[3]->numel() == B && t[5]->numel() == 2,
                "batch_tables: lengths and held pages are [B], the tables [B, max_blocks], the counts [2]") ||
        !expect(B <= INT32_MAX && tables.size(1) <= INT32_MAX && stack.numel() <= INT32_MAX, "batch_tables: sizes beyond 32 bits"))
        return nullptr;
    const int64_t rows = max_rows > 0 ? max_rows : 0, sizes[6] = {2, B, B, B + 1, rows, rows};
    int64_t at[7] = {0};
    for (int i = 0; i < 6; ++i) at[i + 1] = at[i] + (sizes[i] + 3) / 4 * 4;
    const at::Tensor whole = new_tensor(*t[0], at::kInt, at::IntArrayRef(&at[6], 1));
    int32_t* const out = ints(&whole);
    void* const st = call.stream();
    const int rc = without_gil([&] {
        return fn_batch_tables(ints(t[0]), ints(t[1]), static_cast<int>(B), ints(t[2]), static_cast<int>(tables.size(1)), ints(t[3]), ints(t[4]), static_cast<int>(stack.numel()),
                               ints(t[5]), out + at[2], out + at[1], out, out + at[3], out + at[4], out + at[5], max_rows, st);
    });
    if (rc != CPMCU_OK) return status(rc);
    THPObjectPtr result(PyTuple_New(7));
    if (!result) return nullptr;
    const int order[6] = {2, 1, 0, 3, 4, 5};
    for (int i = 0; i < 7; ++i) {
        PyObject* o = THPVariable_Wrap(i < 6 ? part_of(whole, at[order[i]], sizes[order[i]]) : part_of(whole, 0, at[3]));
        if (!o) return nullptr;
        PyTuple_SET_ITEM(result.get(), i, o);
    }
    return result.release();
}

// Rows of heads, [n, heads, D] of 16-bit floats whose heads follow each other; rows may be further apart.
struct HeadRows {
    void* at = nullptr;
    int64_t stride = 0, n = 0, heads = 0, dim = 0;
};
bool head_rows(Call& call, PyObject* o, const char* what, HeadRows* r) {
    const at::Tensor* t = call.strided(o, at::kHalf, what);
    if (!t) return false;
    if (t->dim() != 3 || t->size(0) > INT32_MAX || t->size(1) > INT32_MAX || t->size(2) > INT32_MAX ||
        (t->numel() > 0 && (t->stride(2) != 1 || (t->size(1) > 1 && t->stride(1) != t->size(2))))) {
        PyErr_Format(PyExc_AssertionError, "%s: [n, heads, D] with the heads of a row one after the other required", what);
        return false;
    }
    *r = HeadRows{t->data_ptr(), t->size(0) > 1 ? t->stride(0) : t->size(1) * t->size(2), t->size(0), t->size(1), t->size(2)};
    return true;
}
bool alike(const HeadRows& a, const HeadRows& b) { return a.n == b.n && a.heads == b.heads && a.dim == b.dim; }

// rope_rows(q, k, positions, inv_freq, interleaved, magnitude, transposed, q_out, k_out): k and k_out may be None.
PyObject* call_rope_rows(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
    if (!arguments(nargs, 9)) return nullptr;
    Call call;
    HeadRows q, k, q_out, k_out;
    int interleaved, transposed;
    float magnitude;
    if (!head_rows(call, args[0], "rope_rows: q of 16-bit floats", &q) || !head_rows(call, args[7], "rope_rows: q_out of 16-bit floats", &q_out) ||
        (args[1] != Py_None && (!head_rows(call, args[1], "rope_rows: k of 16-bit floats", &k) || !head_rows(call, args[8], "rope_rows: k_out of 16-bit floats", &k_out))))
        return nullptr;
    const at::Tensor *pos = call.dense(args[2], at::kInt, "rope_rows: int32 positions"), *freq = pos ? call.dense(args[3], at::kFloat, "rope_rows: float32 inv_freq") : nullptr;
    if (!freq || !integer(args[4], &interleaved) || !convert(args[5], &magnitude) || !integer(args[6], &transposed)) return nullptr;
    if (!expect(alike(q, q_out) && alike(k, k_out) && (args[1] == Py_None || (k.n == q.n && k.dim == q.dim)), "rope_rows: q, k and their results differ in shape") ||
        !expect(pos->numel() == q.n && freq->numel() <= INT32_MAX / 2, "rope_rows: a position for each row required"))
        return nullptr;
    void* const st = call.stream();
    return status(without_gil([&] {
        return fn_rope_rows(ints(pos), static_cast<const float*>(freq->data_ptr()), static_cast<int>(2 * freq->numel()), interleaved, magnitude, transposed, q.at, q.stride, q_out.at,
                            q_out.stride, static_cast<int>(q.heads), k.at, k.stride, k_out.at, k_out.stride, static_cast<int>(k.heads), static_cast<int>(q.dim), static_cast<int>(q.n), st);
    }));
}

// kv_append_slots(k_pool, v_pool, k, v, slots, q, q_out, positions, inv_freq, interleaved, magnitude): q and q_out, positions and inv_freq may be None.
PyObject* call_kv_append_slots(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
    if (!arguments(nargs, 11)) return nullptr;
    Call call;
    const char* const pools = "kv_append_slots: pools of 16-bit floats";
    const at::Tensor *k_pool = call.dense(args[0], at::kHalf, pools), *v_pool = k_pool ? call.dense(args[1], at::kHalf, pools) : nullptr;
    HeadRows k, v, q, q_out;
    if (!v_pool || !head_rows(call, args[2], "kv_append_slots: k of 16-bit floats", &k) || !head_rows(call, args[3], "kv_append_slots: v of 16-bit floats", &v) ||
        (args[5] != Py_None && (!head_rows(call, args[5], "kv_append_slots: q of 16-bit floats", &q) || !head_rows(call, args[6], "kv_append_slots: q_out of 16-bit floats", &q_out))))
        return nullptr;
    const at::Tensor *slots = call.dense(args[4], at::kInt, "kv_append_slots: int32 slots"), *pos = nullptr, *freq = nullptr;
    if (!slots || (args[7] != Py_None && !(pos = call.dense(args[7], at::kInt, "kv_append_slots: int32 positions"))) ||
        (args[8] != Py_None && !(freq = call.dense(args[8], at::kFloat, "kv_append_slots: float32 inv_freq"))))
        return nullptr;
    int interleaved;
    float magnitude;
    if (!integer(args[9], &interleaved) || !convert(args[10], &magnitude)) return nullptr;
    if (!expect(k_pool->dim() == 4 && k_pool->size(2) == CPMCU_PAGE_SIZE && k_pool->size(3) == CPMCU_HEAD_DIM && v_pool->dim() == 4 && v_pool->size(0) == k_pool->size(0) &&
                    v_pool->size(1) == k_pool->size(1) && v_pool->size(2) == CPMCU_HEAD_DIM && v_pool->size(3) == CPMCU_PAGE_SIZE && k_pool->size(0) <= INT32_MAX,
                "kv_append_slots: pools are [pages, Hkv, 256, 128] and [pages, Hkv, 128, 256]") ||
        !expect(alike(k, v) && k.heads == k_pool->size(1) && k.dim == CPMCU_HEAD_DIM && slots->numel() == k.n, "kv_append_slots: k and v are [n, Hkv, 128], slots [n]") ||
        !expect(alike(q, q_out) && (args[5] == Py_None || (q.n == k.n && q.dim == CPMCU_HEAD_DIM)), "kv_append_slots: q and q_out are [n, Hq, 128]") ||
        !expect((pos != nullptr) == (freq != nullptr) && (!pos || pos->numel() == k.n) && (!freq || freq->numel() <= CPMCU_HEAD_DIM), "kv_append_slots: positions [n] and inv_freq go together"))
        return nullptr;
    void* const st = call.stream();
    return status(without_gil([&] {
        return fn_kv_append_slots(k_pool->data_ptr(), v_pool->data_ptr(), static_cast<int>(k_pool->size(0)), ints(slots), k.at, k.stride, v.at, v.stride, static_cast<int>(k.n),
                                  static_cast<int>(k.heads), pos ? ints(pos) : nullptr, freq ? static_cast<const float*>(freq->data_ptr()) : nullptr,
                                  freq ? static_cast<int>(2 * freq->numel()) : 0, interleaved, magnitude, q.at, q.stride, q_out.at, q_out.stride, static_cast<int>(q.heads), st);
    }));
}

// quantize_rows(x): (xq [n, K rounded up to 64] of int8, scales [n])
PyObject* call_quantize_rows(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
    if (!arguments(nargs, 1)) return nullptr;
    Call call;
    const at::Tensor* x = call.strided(args[0], at::kHalf, "quantize_rows: rows of 16-bit floats");
    if (!x || !expect(x->dim() == 2 && (x->numel() == 0 || x->size(1) == 1 || x->stride(1) == 1) && x->size(0) <= INT32_MAX && x->size(1) <= INT32_MAX - 64, "quantize_rows: [n, K] with whole rows required"))
        return nullptr;
    const int64_t n = x->size(0), K = x->size(1), sizes[2] = {n, (K + 63) / 64 * 64};
    at::Tensor xq = new_tensor(*x, at::kChar, at::IntArrayRef(sizes, 2)), scales = new_tensor(*x, at::kFloat, at::IntArrayRef(sizes, 1));
    if (n == 0 || K == 0) return expect(K > 0, "quantize_rows: rows without values") ? Py_BuildValue("NN", THPVariable_Wrap(xq), THPVariable_Wrap(scales)) : nullptr;
    void* const st = call.stream();
    const int rc = without_gil([&] {
        return fn_quantize_rows(x->data_ptr(), n > 1 ? x->stride(0) : K, static_cast<int>(n), static_cast<int>(K), static_cast<int8_t*>(xq.data_ptr()), static_cast<float*>(scales.data_ptr()), st);
    });
    if (rc != CPMCU_OK) return status(rc);
    return Py_BuildValue("NN", THPVariable_Wrap(std::move(xq)), THPVariable_Wrap(std::move(scales)));
}

// Whether a tensor is as large as a weight [V, K] is when it is tiled (the bytes pass 32 bits); never where there is no such weight.
bool tiled_from(const at::Tensor& w, int V, int K) {
    const size_t bytes = fn_int8_weight_bytes(V, K);
    return bytes > 0 && static_cast<size_t>(w.numel()) == bytes;
}

// int8_weight_fits(w_tiled, V, K): the check that int8_linear makes, for any tensor.
PyObject* call_int8_weight_fits(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
    if (!arguments(nargs, 3)) return nullptr;
    const at::Tensor* w = tensor_or_null(args[0]);
    int V, K;
    if (!expect(w, "int8_weight_fits: tensor required") || !integer(args[1], &V) || !integer(args[2], &K)) return nullptr;
    return PyBool_FromLong(w->scalar_type() == at::kChar && tiled_from(*w, V, K));
}

// int8_linear(xq, x_scales, w_tiled, w_scales, V, K, out or None): out [n, V]
PyObject* call_int8_linear(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
    if (!arguments(nargs, 7)) return nullptr;
    Call call;
    const at::Tensor* t[4];
    for (int i = 0; i < 4; ++i)
        if (!(t[i] = call.dense(args[i], i % 2 ? at::kFloat : at::kChar, i % 2 ? "int8_linear: float32 scales" : "int8_linear: int8 rows and weights"))) return nullptr;
    int V, K;
    if (!integer(args[4], &V) || !integer(args[5], &K)) return nullptr;
    const at::Tensor& xq = *t[0];
    if (!expect(V >= 1 && K >= 1 && xq.dim() == 2 && xq.size(1) == (int64_t{K} + 63) / 64 * 64 && xq.size(0) <= INT32_MAX && t[1]->numel() == xq.size(0),
                "int8_linear: rows are [n, K rounded up to 64], with a scale each") ||
        !expect(t[3]->numel() == V && tiled_from(*t[2], V, K), "int8_linear: the weight is tiled from [V, K], with a scale for each channel"))
        return nullptr;
    const int64_t n = xq.size(0), sizes[2] = {n, V};
    at::Tensor made;
    const at::Tensor* out;
    if (args[6] == Py_None) {
        made = new_tensor(xq, at::kHalf, at::IntArrayRef(sizes, 2));
        out = &made;
    } else if (!(out = call.dense(args[6], at::kHalf, "int8_linear: out of 16-bit floats")) || !expect(out->dim() == 2 && out->size(0) == n && out->size(1) == V, "int8_linear: out is [n, V]")) {
        return nullptr;
    }
    if (n > 0) {
        void* const st = call.stream();
        const int rc = without_gil([&] {
            return fn_int8_linear(static_cast<const int8_t*>(xq.data_ptr()), static_cast<const float*>(t[1]->data_ptr()), static_cast<const int8_t*>(t[2]->data_ptr()),
                                  static_cast<const float*>(t[3]->data_ptr()), static_cast<int>(n), V, K, out->data_ptr(), st);
        });
        if (rc != CPMCU_OK) return status(rc);
    }
    if (args[6] != Py_None) {
        Py_INCREF(args[6]);
        return args[6];
    }
    return THPVariable_Wrap(std::move(made));
}

// Attention of a batch's rows over its pages: (q, k_pool, v_pool, block_tables, row_offsets or None, positions, scale, out).  The workspace is the call's own,
// as the results are: calls on several streams, and captured ones, share nothing.
decltype(&cpmcu_batch_prompt_attention) fn_prompt_attention = nullptr;
decltype(&cpmcu_batch_prompt_attention_workspace_bytes) fn_prompt_attention_workspace_bytes = nullptr;
decltype(&cpmcu_batch_decode_attention) fn_decode_attention = nullptr;
decltype(&cpmcu_batch_decode_attention_workspace_bytes) fn_decode_attention_workspace_bytes = nullptr;
template <bool PROMPT>
PyObject* batch_attention(PyObject* const* args, Py_ssize_t nargs) {
    if (!arguments(nargs, 8)) return nullptr;
    Call call;
    HeadRows q, out;
    const char* const pools = "batch attention: pools of 16-bit floats";
    if (!head_rows(call, args[0], "batch attention: q of 16-bit floats", &q) || !head_rows(call, args[7], "batch attention: out of 16-bit floats", &out)) return nullptr;
    const at::Tensor *k_pool = call.dense(args[1], at::kHalf, pools), *v_pool = k_pool ? call.dense(args[2], at::kHalf, pools) : nullptr, *offsets = nullptr;
    const at::Tensor *tables = v_pool ? call.strided(args[3], at::kInt, "batch attention: int32 block_tables") : nullptr,
                     *pos = tables ? call.dense(args[5], at::kInt, "batch attention: int32 positions") : nullptr;
    float scale;
    if (!pos || ((PROMPT || args[4] != Py_None) && !(offsets = call.dense(args[4], at::kInt, "batch attention: int32 row_offsets"))) || !convert(args[6], &scale)) return nullptr;
    if (!expect(k_pool->dim() == 4 && k_pool->size(2) == CPMCU_PAGE_SIZE && k_pool->size(3) == CPMCU_HEAD_DIM && v_pool->dim() == 4 && v_pool->size(0) == k_pool->size(0) &&
                    v_pool->size(1) == k_pool->size(1) && v_pool->size(2) == CPMCU_HEAD_DIM && v_pool->size(3) == CPMCU_PAGE_SIZE && k_pool->size(0) <= INT32_MAX && k_pool->size(1) <= INT32_MAX,
                "batch attention: pools are [pages, Hkv, 256, 128] and [pages, Hkv, 128, 256]") ||
        !expect(alike(q, out) && q.dim == CPMCU_HEAD_DIM && pos->numel() == q.n, "batch attention: q and out are [n, Hq, 128], positions [n]") ||
        !expect(tables->dim() == 2 && (tables->numel() == 0 || tables->size(1) == 1 || tables->stride(1) == 1) && tables->size(0) <= INT32_MAX && tables->size(1) <= INT32_MAX && (!offsets || offsets->numel() == tables->size(0) + 1),
                "batch attention: block_tables are [B, max_blocks] with whole rows, row_offsets [B + 1]"))
        return nullptr;
    const int B = static_cast<int>(tables->size(0)), M = static_cast<int>(tables->size(1)), n = static_cast<int>(q.n), Hq = static_cast<int>(q.heads), Hkv = static_cast<int>(k_pool->size(1));
    int64_t bytes = 0;
    if constexpr (PROMPT) bytes = static_cast<int64_t>(fn_prompt_attention_workspace_bytes(B, M, n, Hq, Hkv));
    else bytes = static_cast<int64_t>(fn_decode_attention_workspace_bytes(B, M, Hq, Hkv));
    at::Tensor ws;
    if (n > 0 && bytes > 0) ws = new_tensor(*tables, at::kByte, at::IntArrayRef(&bytes, 1));
    void* const st = call.stream();
    return status(without_gil([&] {
        const auto fn = PROMPT ? fn_prompt_attention : fn_decode_attention;
        return fn(q.at, q.stride, k_pool->data_ptr(), v_pool->data_ptr(), static_cast<int>(k_pool->size(0)), ints(tables), B > 1 ? tables->stride(0) : M, M, offsets ? ints(offsets) : nullptr, ints(pos), B, n, Hq, Hkv,
                  scale, out.at, out.stride, ws.defined() ? ws.data_ptr() : nullptr, static_cast<size_t>(bytes), st);
    }));
}
PyObject* call_prompt_attention(PyObject*, PyObject* const* args, Py_ssize_t nargs) { return batch_attention<true>(args, nargs); }
PyObject* call_decode_attention(PyObject*, PyObject* const* args, Py_ssize_t nargs) { return batch_attention<false>(args, nargs); }

// adjust_logits(logits, penalties, tokens, lens, requests, bias_ids, bias_values, allowed, draft_ids, tree_mask, out, want_ids): ids [n] or None.  All but
// logits and out may be None.
decltype(&cpmcu_adjust_logits) fn_adjust_logits = nullptr;
decltype(&cpmcu_adjust_logits_workspace_bytes) fn_adjust_logits_workspace_bytes = nullptr;
PyObject* call_adjust_logits(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
    if (!arguments(nargs, 12)) return nullptr;
    Call call;
    const at::Tensor* rows[2];
    for (int i = 0; i < 2; ++i) {
        rows[i] = call.strided(args[i ? 10 : 0], at::kHalf, "adjust_logits: rows of 16-bit floats");
        if (!rows[i]) return nullptr;
        if (!expect(rows[i]->dim() == 2 && (rows[i]->numel() == 0 || rows[i]->size(1) == 1 || rows[i]->stride(1) == 1) && rows[i]->size(0) <= INT32_MAX && rows[i]->size(1) <= INT32_MAX,
                    "adjust_logits: [n, V] with whole rows required"))
            return nullptr;
    }
    const at::Tensor &in = *rows[0], &out = *rows[1];
    const int64_t n = in.size(0), V = in.size(1), words = (V + 31) / 32;
    if (!expect(out.size(0) == n && out.size(1) == V, "adjust_logits: out is [n, V]")) return nullptr;
    const at::Tensor* t[9] = {};  // args 1 to 9
    const at::ScalarType types[9] = {at::kFloat, at::kInt, at::kInt, at::kInt, at::kInt, at::kFloat, at::kInt, at::kInt, at::kLong};
    const char* const what[9] = {"adjust_logits: float32 penalties", "adjust_logits: int32 tokens", "adjust_logits: int32 lens", "adjust_logits: int32 requests", "adjust_logits: int32 bias_ids",
                                 "adjust_logits: float32 bias_values", "adjust_logits: int32 allowed", "adjust_logits: int32 draft_ids", "adjust_logits: int64 tree_mask"};
    for (int i = 0; i < 9; ++i)
        if (args[1 + i] != Py_None && !(t[i] = i == 6 ? call.strided(args[1 + i], types[i], what[i]) : call.dense(args[1 + i], types[i], what[i]))) return nullptr;
    const at::Tensor *penalties = t[0], *tokens = t[1], *lens = t[2], *requests = t[3], *bias_ids = t[4], *bias_values = t[5], *allowed = t[6], *draft_ids = t[7], *tree_mask = t[8];
    const int64_t R = penalties ? penalties->numel() / 3 : bias_ids && bias_ids->dim() == 2 ? bias_ids->size(0) : 0;
    if (!expect(!penalties || (penalties->dim() == 2 && penalties->size(1) == 3), "adjust_logits: penalties are [R, 3]") ||
        !expect((tokens != nullptr) == (lens != nullptr) && (!tokens || (penalties && tokens->dim() == 2 && tokens->size(0) == R && lens->numel() == R)),
                "adjust_logits: tokens [R, L] and lens [R] go together, with penalties") ||
        !expect(!requests || requests->numel() == n, "adjust_logits: requests are [n]") ||
        !expect((bias_ids != nullptr) == (bias_values != nullptr) && (!bias_ids || (bias_ids->dim() == 2 && bias_ids->size(0) == R && bias_values->sizes() == bias_ids->sizes())),
                "adjust_logits: bias_ids and bias_values are [R, biases]") ||
        !expect(!allowed || (allowed->dim() == 2 && allowed->size(0) == n && allowed->size(1) == words && (words == 1 || n == 0 || allowed->stride(1) == 1)),
                "adjust_logits: allowed is [n, ceil(V / 32)] with whole rows") ||
        !expect((draft_ids != nullptr) == (tree_mask != nullptr) && (!draft_ids || (draft_ids->numel() == n && tree_mask->dim() == 2 && tree_mask->size(0) == n)),
                "adjust_logits: draft_ids [n] and tree_mask [n, words] go together") ||
        !expect(R <= INT32_MAX && (!tokens || tokens->size(1) <= INT32_MAX) && (!bias_ids || bias_ids->size(1) <= INT32_MAX) && (!tree_mask || tree_mask->size(1) <= INT32_MAX),
                "adjust_logits: sizes beyond 32 bits"))
        return nullptr;
    const bool no_text = tokens && tokens->size(1) == 0, no_bias = bias_ids && bias_ids->size(1) == 0;
    const int want = PyObject_IsTrue(args[11]);
    if (want < 0) return nullptr;
    // (ids is the caller's to keep, so the workspace is memory of its own)
    at::Tensor ids, ws;
    int64_t bytes = 0;
    if (want) {
        bytes = V > 0 ? static_cast<int64_t>(fn_adjust_logits_workspace_bytes(static_cast<int>(n), static_cast<int>(V))) : 0;
        ids = new_tensor(in, at::kInt, at::IntArrayRef(&n, 1));
        if (bytes > 0) ws = new_tensor(in, at::kByte, at::IntArrayRef(&bytes, 1));
    }
    const auto i32 = [](const at::Tensor* x) { return x ? ints(x) : nullptr; };
    const auto f32 = [](const at::Tensor* x) { return x ? static_cast<const float*>(x->data_ptr()) : nullptr; };
    void* const st = call.stream();
    const int rc = without_gil([&] {
        return fn_adjust_logits(in.data_ptr(), n > 1 ? in.stride(0) : V, static_cast<int>(n), static_cast<int>(V), f32(penalties), no_text ? nullptr : i32(tokens), no_text ? nullptr : i32(lens),
                                static_cast<int>(R), tokens ? static_cast<int>(tokens->size(1)) : 0, i32(requests), no_bias ? nullptr : i32(bias_ids), no_bias ? nullptr : f32(bias_values),
                                bias_ids ? static_cast<int>(bias_ids->size(1)) : 0, allowed ? static_cast<const uint32_t*>(allowed->data_ptr()) : nullptr, allowed && n > 1 ? allowed->stride(0) : words,
                                i32(draft_ids), tree_mask ? static_cast<const uint64_t*>(tree_mask->data_ptr()) : nullptr, tree_mask ? static_cast<int>(tree_mask->size(1)) : 0, out.data_ptr(),
                                n > 1 ? out.stride(0) : V, want ? ints(&ids) : nullptr, ws.defined() ? ws.data_ptr() : nullptr, static_cast<size_t>(bytes), st);
    });
    if (rc != CPMCU_OK) return status(rc);
    if (!want) Py_RETURN_NONE;
    return THPVariable_Wrap(std::move(ids));
}

// empty(like, dtype, rows, cols, dtype, rows, cols, ...): uninitialised [rows, cols] tensors ([rows] where cols is 0) on like's
// device, as a tuple.  dtype: 'h' 16-bit float, 'f' fp32, 'i' int32, 'l' int64.
PyObject* empty(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
    if (nargs < 4 || (nargs - 1) % 3 != 0 || !THPVariable_Check(args[0])) {
        PyErr_SetString(PyExc_TypeError, "empty(tensor, dtype, rows, cols, ...) expected");
        return nullptr;
    }
    if (!expect(THPVariable_Unpack(args[0]).is_cuda(), "device-resident contiguous tensor required")) return nullptr;
    const Py_ssize_t n = (nargs - 1) / 3;
    THPObjectPtr out(PyTuple_New(n));
    if (!out) return nullptr;
    const auto device = THPVariable_Unpack(args[0]).device();
    for (Py_ssize_t i = 0; i < n; ++i) {
        const char* code = PyUnicode_AsUTF8(args[1 + 3 * i]);
        const long rows = PyLong_AsLong(args[2 + 3 * i]), cols = PyLong_AsLong(args[3 + 3 * i]);
        if (PyErr_Occurred()) return nullptr;
        const auto type = code[0] == 'h' ? at::kHalf : code[0] == 'f' ? at::kFloat : code[0] == 'l' ? at::kLong : at::kInt;
        const int64_t sizes[2] = {rows, cols};
        PyObject* t = THPVariable_Wrap(at::detail::empty_cuda(at::IntArrayRef(sizes, cols ? 2 : 1), type, device, std::nullopt));
        if (!t) return nullptr;
        PyTuple_SET_ITEM(out.get(), i, t);
    }
    return out.release();
}

// pinned(tensor): a contiguous pinned host tensor's memory, in the place of a device tensor, for a call on the current stream: the GPU writes
// it through the mapped address.  The allocator is told of the stream, so that a tensor dropped before the work is done is not
// given to somebody else ahead of it (device memory is reused in stream order by itself).
PyObject* pinned(PyObject*, PyObject* o) {
    if (!THPVariable_Check(o)) {
        PyErr_SetString(PyExc_TypeError, "pinned(tensor) expected");
        return nullptr;
    }
    const at::Tensor& t = THPVariable_Unpack(o);
    if (!expect(t.is_contiguous() && t.is_pinned(), "device-resident or pinned contiguous tensor required")) return nullptr;
    at::getHostAllocator(at::kCUDA)->record_event(t.data_ptr(), t.storage().data_ptr().get_context(), c10::hip::getCurrentHIPStreamMasqueradingAsCUDA().unwrap());
    return PyCapsule_New(t.data_ptr(), kPinned, nullptr);
}

// synchronize(): waits for torch's current stream.
PyObject* synchronize(PyObject*, PyObject*) {
    const auto stream = c10::hip::getCurrentHIPStream();
    without_gil([&] { stream.synchronize(); });
    Py_RETURN_NONE;
}

// bind(handle): the library's functions, from the handle lib.py loaded it under.
PyObject* bind(PyObject*, PyObject* handle) {
    void* h = PyLong_AsVoidPtr(handle);
    if (PyErr_Occurred()) return nullptr;
    auto find = [&](const char* name, auto* slot) {
        *slot = reinterpret_cast<std::remove_pointer_t<decltype(slot)>>(dlsym(h, name));
        if (!*slot) PyErr_Format(PyExc_ImportError, "the library does not export %s", name);
        return *slot != nullptr;
    };
    bool ok = find("cpmcu_last_error", &g_last_error) && find("cpmcu_lm_head_partials", &fn_lm_head_partials) &&
              find("cpmcu_tree_attention_window", &fn_tree_attention_window) &&
              find("cpmcu_tree_attention_workspace_bytes", &fn_tree_attention_workspace_bytes) && find("cpmcu_batch_tables", &fn_batch_tables) &&
              find("cpmcu_rope_rows", &fn_rope_rows) && find("cpmcu_kv_append_slots", &fn_kv_append_slots) &&
              find("cpmcu_quantize_rows", &fn_quantize_rows) && find("cpmcu_int8_linear", &fn_int8_linear) &&
              find("cpmcu_int8_weight_bytes", &fn_int8_weight_bytes) && find("cpmcu_batch_prompt_attention", &fn_prompt_attention) &&
              find("cpmcu_batch_prompt_attention_workspace_bytes", &fn_prompt_attention_workspace_bytes) && find("cpmcu_batch_decode_attention", &fn_decode_attention) &&
              find("cpmcu_batch_decode_attention_workspace_bytes", &fn_decode_attention_workspace_bytes) && find("cpmcu_adjust_logits", &fn_adjust_logits) &&
              find("cpmcu_adjust_logits_workspace_bytes", &fn_adjust_logits_workspace_bytes);
#define X(name) ok = ok && find("cpmcu_" #name, &fn_##name);
    CPMCU_TORCH_CALLS(X)
#undef X
    if (!ok) return nullptr;
    Py_RETURN_NONE;
}

#define ENTRY(name, fn) {name, reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(static_cast<PyObject* (*)(PyObject*, PyObject* const*, Py_ssize_t)>(entry<fn>))), METH_FASTCALL, nullptr},
#define X(name) ENTRY(#name, call_##name)
PyMethodDef g_methods[] = {
    CPMCU_TORCH_CALLS(X)
    X(lm_head_partials)
    X(kv_append_rows)
    X(tree_attention_rows)
    X(batch_tables)
    X(rope_rows)
    X(kv_append_slots)
    X(quantize_rows)
    X(int8_linear)
    X(int8_weight_fits)
    X(prompt_attention)
    X(decode_attention)
    X(adjust_logits)
    ENTRY("empty", empty)
    {"pinned", entry<pinned>, METH_O, nullptr},
    {"synchronize", entry<synchronize>, METH_NOARGS, nullptr},
    {"bind", entry<bind>, METH_O, nullptr},
    {nullptr, nullptr, 0, nullptr}};
#undef X
#undef ENTRY
PyModuleDef g_module = {PyModuleDef_HEAD_INIT, "_torch_call", "The library's operators on torch tensors.", -1, g_methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

extern "C" __attribute__((visibility("default"))) PyObject* PyInit__torch_call(void) { return PyModule_Create(&g_module); }
