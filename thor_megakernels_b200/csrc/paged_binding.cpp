// Python entry points of the paged cache (thor_megakernels_b200/paged.py) as a CPython module: argument checks on
// torch tensors, the structs of include/b200_megakernel.h, and the call into libb200mk.so.  A decode step makes two of
// these calls per layer, and their kernels take 3 to 5 us at small sizes: through ctypes the host needed 11 to 14 us
// for each, here a few.  The library's functions are handed over as addresses (init), so that this module links
// against nothing of the framework.
//
// Every function returns what it made, or an int: a non-zero return code of the library, or -1 when the device has no
// error word yet (the caller makes one and calls again).

#include <Python.h>

#include <ATen/core/Tensor.h>
#include <ATen/ops/empty.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <optional>

#include "../../include/b200_megakernel.h"

namespace {

using AppendFn = int (*)(const MkPagedCache *, const MkPagedBatch *, const MkPagedAppend *, void *);
using AttentionFn = int (*)(const MkPagedCache *, const MkPagedBatch *, const MkPagedAttention *, void *);
using WorkspaceFn = int64_t (*)(const MkPagedCache *, const MkPagedBatch *, int32_t);

AppendFn g_append = nullptr;
AttentionFn g_attention = nullptr;
WorkspaceFn g_workspace = nullptr;
constexpr int kDevices = 64;
int32_t *g_error_word[kDevices] = {};

#define REFUSE(...)                                \
    do {                                           \
        PyErr_Format(PyExc_ValueError, __VA_ARGS__); \
        return false;                              \
    } while (0)

// The tensor behind an argument; null for None.
bool read_tensor(PyObject *o, const char *name, bool optional, const at::Tensor *&t) {
    t = nullptr;
    if (o == Py_None) {
        if (optional) return true;
        REFUSE("%s is missing", name);
    }
    if (!THPVariable_Check(o)) REFUSE("%s must be a tensor", name);
    t = &THPVariable_Unpack(o);
    if (!t->defined() || t->layout() != at::kStrided) REFUSE("%s must be a dense tensor", name);
    return true;
}

bool read_cache(PyObject *const *a, PyObject *ks_obj, PyObject *vs_obj, MkPagedCache &c, int &device) {
    const at::Tensor *k, *v, *ks, *vs;
    if (!read_tensor(a[0], "k_pages", false, k) || !read_tensor(a[1], "v_pages", false, v) || !read_tensor(ks_obj, "k_scales", true, ks) ||
        !read_tensor(vs_obj, "v_scales", true, vs))
        return false;
    if (!k->is_cuda() || !v->is_cuda()) REFUSE("k_pages and v_pages must be CUDA tensors");
    device = k->get_device();
    if (device >= kDevices) REFUSE("more devices than the framework serves");
    if (k->dim() != 4 || v->sizes() != k->sizes() || v->strides() != k->strides() || v->scalar_type() != k->scalar_type() || v->get_device() != device)
        REFUSE("k_pages and v_pages must be [pages, kv_heads, page_size, head_dim] tensors of one type, shape and layout on one device");
    const int64_t pages = k->size(0), heads = k->size(1), size = k->size(2), dim = k->size(3);
    c = MkPagedCache{};
    if (k->scalar_type() == at::kFloat8_e4m3fn) {
        c.format = MK_CACHE_E4M3;
        const char *names[2] = {"k_scales", "v_scales"};
        const at::Tensor *scales[2] = {ks, vs};
        for (int i = 0; i < 2; ++i)
            if (!scales[i] || scales[i]->scalar_type() != at::kFloat || scales[i]->dim() != 2 || scales[i]->size(0) != pages ||
                scales[i]->size(1) != heads || !scales[i]->is_contiguous() || !scales[i]->is_cuda() || scales[i]->get_device() != device)
                REFUSE("%s must be a contiguous fp32 [pages, kv_heads] tensor on the cache's device", names[i]);
        c.k_scales = ks->mutable_data_ptr<float>();
        c.v_scales = vs->mutable_data_ptr<float>();
    } else if (k->scalar_type() == at::kBFloat16) {
        if (ks || vs) REFUSE("a bf16 cache has no scales");
        c.format = MK_CACHE_BF16;
    } else {
        REFUSE("the cache must be bf16 or float8_e4m3fn");
    }
    if (k->stride(3) != 1 && dim > 1) REFUSE("head_dim must be the dense dimension of the pages");
    if (pages > INT32_MAX || heads > INT32_MAX || size > INT32_MAX || dim > INT32_MAX) REFUSE("the cache has too many pages");
    c.k_pages = k->mutable_data_ptr();
    c.v_pages = v->mutable_data_ptr();
    // the pitch of a dimension of one element is never used; it only has to be a valid one
    c.slot_stride = k->stride(2);
    c.head_stride = heads == 1 ? size * c.slot_stride : k->stride(1);
    c.page_stride = pages == 1 ? std::max(heads * c.head_stride, size * c.slot_stride) : k->stride(0);
    c.num_pages = (int32_t)pages; c.num_kv_heads = (int32_t)heads; c.page_size = (int32_t)size; c.head_dim = (int32_t)dim;
    return true;
}

bool is_int_vector(const at::Tensor &t, int64_t n, int device) {
    return t.scalar_type() == at::kInt && t.is_cuda() && t.get_device() == device && t.dim() == 1 && t.size(0) == n && t.is_contiguous();
}

bool read_batch(PyObject *table_obj, PyObject *where_obj, const char *where_name, PyObject *cu_obj, int64_t tokens, int device, MkPagedBatch &b) {
    const at::Tensor *table, *where, *cu;
    if (!read_tensor(table_obj, "page_table", false, table) || !read_tensor(where_obj, where_name, false, where) ||
        !read_tensor(cu_obj, "cu_tokens", true, cu))
        return false;
    if (table->dim() != 2 || table->scalar_type() != at::kInt || !table->is_cuda() || table->get_device() != device ||
        (table->size(1) > 1 && table->stride(1) != 1))
        REFUSE("page_table must be an int32 [sequences, columns] tensor with dense rows on the cache's device");
    const int64_t seqs = table->size(0), columns = table->size(1);
    if (!is_int_vector(*where, seqs, device)) REFUSE("%s must be a contiguous int32 vector of %lld elements on the cache's device", where_name, (long long)seqs);
    if (cu && !is_int_vector(*cu, seqs + 1, device))
        REFUSE("cu_tokens must be a contiguous int32 vector of %lld elements on the cache's device", (long long)seqs + 1);
    if (!cu && seqs && tokens % seqs) REFUSE("%lld rows do not divide over %lld sequences; give cu_tokens", (long long)tokens, (long long)seqs);
    if (seqs > INT32_MAX || columns > INT32_MAX || tokens > INT32_MAX) REFUSE("too many rows, sequences or columns");
    b = MkPagedBatch{};
    b.page_table = table->const_data_ptr<int>();
    b.table_stride = seqs == 1 ? columns : table->stride(0);
    b.positions = where->const_data_ptr<int>();
    b.cu_tokens = cu ? cu->const_data_ptr<int>() : nullptr;
    b.error_word = g_error_word[device];
    b.seqs = (int32_t)seqs; b.tokens = (int32_t)tokens; b.max_pages = (int32_t)columns;
    return true;
}

// bf16 rows [tokens, heads, dim]; a pitch that is never used (one token, one head) need not be a valid one.
bool read_rows(const at::Tensor &t, const char *name, int64_t heads, int64_t tokens, int64_t dim, int device, int64_t &token_pitch, int64_t &head_pitch) {
    if (t.dim() != 3 || t.scalar_type() != at::kBFloat16 || !t.is_cuda() || t.get_device() != device || t.size(2) != dim ||
        (heads >= 0 && t.size(1) != heads) || (tokens >= 0 && t.size(0) != tokens) || (dim > 1 && t.stride(2) != 1))
        REFUSE("%s must be a bf16 [tokens, heads, %lld] tensor with dense rows on the cache's device, as many rows and heads as the others", name,
               (long long)dim);
    if (t.size(1) > INT32_MAX) REFUSE("%s has too many heads", name);
    token_pitch = t.size(0) > 1 ? t.stride(0) : 0;
    head_pitch = t.size(1) > 1 ? t.stride(1) : 0;
    return true;
}

// `out` itself, or a new tensor of `like`'s shape
bool read_output(PyObject *obj, const char *name, const at::Tensor &like, int device, at::Tensor &out) {
    const at::Tensor *given;
    if (!read_tensor(obj, name, true, given)) return false;
    if (!given) {
        out = at::empty(like.sizes(), like.options().requires_grad(false), at::MemoryFormat::Contiguous);
        return true;
    }
    if (given->scalar_type() != at::kBFloat16 || !given->is_cuda() || given->get_device() != device || given->sizes() != like.sizes() ||
        !given->is_contiguous())
        REFUSE("%s must be a contiguous bf16 tensor of the queries' shape on the cache's device", name);
    out = *given;
    return true;
}

PyObject *give(PyObject *given, const at::Tensor &made) {
    if (given != Py_None) return Py_NewRef(given);
    return THPVariable_Wrap(made);
}

struct OnDevice {   // the device of a call as the current one, left alone where it is already
    std::optional<c10::cuda::CUDAGuard> guard;
    explicit OnDevice(int device) {
        if (c10::cuda::current_device() != device) guard.emplace((c10::DeviceIndex)device);
    }
};
void *stream_of(int device) { return c10::cuda::getCurrentCUDAStream((c10::DeviceIndex)device).stream(); }

// Whether two tensors' memory, from the first element to the last, overlaps.
bool overlap(const at::Tensor &a, const at::Tensor &b) {
    if (!a.numel() || !b.numel()) return false;
    const auto bytes = [](const at::Tensor &t) {
        int64_t last = 0;
        for (int64_t i = 0; i < t.dim(); ++i) last += (t.size(i) - 1) * t.stride(i);
        return (last + 1) * (int64_t)t.element_size();
    };
    const char *pa = (const char *)a.const_data_ptr(), *pb = (const char *)b.const_data_ptr();
    return pa < pb + bytes(b) && pb < pa + bytes(a);
}

// k, v, k_pages, v_pages, page_table, start, q, q_out, rope_cos, rope_sin, half_layout, k_scales, v_scales, cu_tokens
PyObject *append(PyObject *, PyObject *const *a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (n != 14) return PyErr_Format(PyExc_TypeError, "append: %zd arguments", n);
    MkPagedCache c;
    MkPagedBatch b;
    MkPagedAppend args = {};
    int device;
    const at::Tensor *k, *v, *q, *cos, *sin;
    at::Tensor q_out;
    if (!read_cache(a + 2, a[11], a[12], c, device) || !read_tensor(a[0], "k", false, k) || !read_tensor(a[1], "v", false, v) ||
        !read_tensor(a[6], "q", true, q) || !read_tensor(a[8], "rope_cos", true, cos) || !read_tensor(a[9], "rope_sin", true, sin) ||
        !read_rows(*k, "k", c.num_kv_heads, -1, c.head_dim, device, args.k_token_stride, args.k_head_stride))
        return nullptr;
    const int64_t tokens = k->size(0);
    if (!read_rows(*v, "v", c.num_kv_heads, tokens, c.head_dim, device, args.v_token_stride, args.v_head_stride) ||
        !read_batch(a[4], a[5], "start", a[13], tokens, device, b))
        return nullptr;
    if (!cos != !sin) return PyErr_Format(PyExc_ValueError, "rope_cos and rope_sin go together");
    for (const at::Tensor *t : {cos, sin})
        if (t && (t->scalar_type() != at::kFloat || t->dim() != 2 || t->sizes() != cos->sizes() || !t->is_contiguous() || !t->is_cuda() ||
                  t->get_device() != device || t->size(0) > INT32_MAX || t->size(1) > INT32_MAX))
            return PyErr_Format(PyExc_ValueError, "rope_cos and rope_sin must be contiguous fp32 [positions, rot] tensors on the cache's device");
    if (cos) {
        args.rope_cos = cos->const_data_ptr<float>();
        args.rope_sin = sin->const_data_ptr<float>();
        args.rope_positions = (int32_t)cos->size(0);
        args.rot_dim = (int32_t)cos->size(1);
    }
    if (q) {
        if (!read_rows(*q, "q", -1, tokens, c.head_dim, device, args.q_token_stride, args.q_head_stride) ||
            !read_output(a[7], "q_out", *q, device, q_out))
            return nullptr;
        if (a[7] != Py_None) {
            const bool in_place = q_out.const_data_ptr() == q->const_data_ptr() && q->is_contiguous();
            if (overlap(q_out, *k) || overlap(q_out, *v) || (!in_place && overlap(q_out, *q)))
                return PyErr_Format(PyExc_ValueError, "q_out may be q itself, but overlap neither it in another way nor k or v");
        }
        args.q = q->const_data_ptr();
        args.q_out = q_out.mutable_data_ptr();
        args.num_q_heads = (int32_t)q->size(1);
    } else if (a[7] != Py_None) {
        return PyErr_Format(PyExc_ValueError, "q_out without q");
    }
    if (tokens > 0) {
        if (!b.error_word) return PyLong_FromLong(-1);
        args.k = k->const_data_ptr();
        args.v = v->const_data_ptr();
        args.half_layout = a[10] == Py_True;
        OnDevice on(device);
        if (const int code = g_append(&c, &b, &args, stream_of(device))) return PyLong_FromLong(code);
    }
    if (!q) Py_RETURN_NONE;
    return give(a[7], q_out);
    END_HANDLE_TH_ERRORS
}

// q, k_pages, v_pages, page_table, lengths, scale, k_scales, v_scales, cu_tokens, out, workspace
PyObject *attention(PyObject *, PyObject *const *a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (n != 11) return PyErr_Format(PyExc_TypeError, "attention: %zd arguments", n);
    MkPagedCache c;
    MkPagedBatch b;
    MkPagedAttention args = {};
    int device;
    const at::Tensor *q, *given;
    at::Tensor out, workspace;
    if (!read_cache(a + 1, a[6], a[7], c, device) || !read_tensor(a[0], "q", false, q) ||
        !read_rows(*q, "q", -1, -1, c.head_dim, device, args.q_token_stride, args.q_head_stride) ||
        !read_batch(a[3], a[4], "lengths", a[8], q->size(0), device, b) || !read_tensor(a[10], "workspace", true, given) ||
        !read_output(a[9], "out", *q, device, out))
        return nullptr;
    const double scale = a[5] == Py_None ? 1.0 / std::sqrt((double)c.head_dim) : PyFloat_AsDouble(a[5]);
    if (scale == -1.0 && PyErr_Occurred()) return nullptr;
    if (a[9] != Py_None && overlap(out, *q)) return PyErr_Format(PyExc_ValueError, "out must not overlap q");
    if (q->size(0) == 0) return give(a[9], out);
    if (!b.error_word) return PyLong_FromLong(-1);
    args.q = q->const_data_ptr();
    args.out = out.mutable_data_ptr();
    args.num_q_heads = (int32_t)q->size(1);
    args.scale = (float)scale;
    OnDevice on(device);
    if (given) {
        if (!given->is_cuda() || given->get_device() != device || !given->is_contiguous())
            return PyErr_Format(PyExc_ValueError, "workspace must be a contiguous tensor on the cache's device");
        args.workspace = given->mutable_data_ptr();
        args.workspace_bytes = (int64_t)given->nbytes();
    } else {
        args.workspace_bytes = g_workspace(&c, &b, args.num_q_heads);
        if (args.workspace_bytes < 0) return PyLong_FromLong(MK_ERR_UNSUPPORTED);
        if (args.workspace_bytes > 0) {
            workspace = at::empty({args.workspace_bytes}, q->options().dtype(at::kByte).requires_grad(false));
            args.workspace = workspace.mutable_data_ptr();
        }
    }
    if (const int code = g_attention(&c, &b, &args, stream_of(device))) return PyLong_FromLong(code);
    return give(a[9], out);
    END_HANDLE_TH_ERRORS
}

// q, k_pages, v_pages, page_table, lengths, k_scales, v_scales, cu_tokens -> bytes as a float (an int is an error)
PyObject *attention_workspace(PyObject *, PyObject *const *a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (n != 8) return PyErr_Format(PyExc_TypeError, "attention_workspace: %zd arguments", n);
    MkPagedCache c;
    MkPagedBatch b;
    int device;
    int64_t token_pitch, head_pitch;
    const at::Tensor *q;
    if (!read_cache(a + 1, a[5], a[6], c, device) || !read_tensor(a[0], "q", false, q) ||
        !read_rows(*q, "q", -1, -1, c.head_dim, device, token_pitch, head_pitch) || !read_batch(a[3], a[4], "lengths", a[7], q->size(0), device, b))
        return nullptr;
    if (q->size(0) == 0) return PyFloat_FromDouble(0.0);
    if (!b.error_word) return PyLong_FromLong(-1);
    OnDevice on(device);
    const int64_t bytes = g_workspace(&c, &b, (int32_t)q->size(1));
    if (bytes < 0) return PyLong_FromLong(MK_ERR_UNSUPPORTED);
    return PyFloat_FromDouble((double)bytes);
    END_HANDLE_TH_ERRORS
}

// What this module was built from; build.py looks for it in the file.
__attribute__((used)) const char built_from[] = MK_BINDING_TAG;

// addresses of mk_paged_append, mk_paged_attention, mk_paged_attention_workspace; the library's mk_abi_sizeof of the four structs
PyObject *init(PyObject *, PyObject *const *a, Py_ssize_t n) {
    if (n != 7) return PyErr_Format(PyExc_TypeError, "init: %zd arguments", n);
    const size_t sizes[4] = {sizeof(MkPagedCache), sizeof(MkPagedBatch), sizeof(MkPagedAppend), sizeof(MkPagedAttention)};
    for (int i = 0; i < 4; ++i)
        if (PyLong_AsLong(a[3 + i]) != (long)sizes[i])
            return PyErr_Occurred() ? nullptr : PyErr_Format(PyExc_RuntimeError, "libb200mk.so and _paged_binding.so differ in their structs; build both anew");
    g_append = (AppendFn)PyLong_AsVoidPtr(a[0]);
    g_attention = (AttentionFn)PyLong_AsVoidPtr(a[1]);
    g_workspace = (WorkspaceFn)PyLong_AsVoidPtr(a[2]);
    if (PyErr_Occurred()) return nullptr;
    Py_RETURN_NONE;
}

// device index, address of its error word
PyObject *set_error_word(PyObject *, PyObject *const *a, Py_ssize_t n) {
    if (n != 2) return PyErr_Format(PyExc_TypeError, "set_error_word: %zd arguments", n);
    const long device = PyLong_AsLong(a[0]);
    void *word = PyLong_AsVoidPtr(a[1]);
    if (PyErr_Occurred()) return nullptr;
    if (device < 0 || device >= kDevices) return PyErr_Format(PyExc_ValueError, "device %ld", device);
    g_error_word[device] = (int32_t *)word;
    Py_RETURN_NONE;
}

PyMethodDef methods[] = {
    {"append", (PyCFunction)(void (*)(void))append, METH_FASTCALL, nullptr},
    {"attention", (PyCFunction)(void (*)(void))attention, METH_FASTCALL, nullptr},
    {"attention_workspace", (PyCFunction)(void (*)(void))attention_workspace, METH_FASTCALL, nullptr},
    {"init", (PyCFunction)(void (*)(void))init, METH_FASTCALL, nullptr},
    {"set_error_word", (PyCFunction)(void (*)(void))set_error_word, METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr},
};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_paged_binding", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__paged_binding() { return PyModule_Create(&module); }
