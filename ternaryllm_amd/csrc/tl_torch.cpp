// The short way from a torch call to a product: what ops.spmm and ops.mlp_gate_up do in Python, for the plain calls (ordinary
// tensors on the weight's device, one of the library's types, rows or one K-major matrix, no workspace or one that is there).
// A call that is anything else gets None, and Python's general path, which also words the errors.
//
// Bound by the host: one fp16 row 4096 x 4096 is 4 us of kernel; through Python's checks, ctypes and stream objects the call took
// 18.6 us, this way 7.1 (another launch before it has ended; 2.5 us of it are the launch).
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/ATen.h>
#include <c10/core/DeviceGuard.h>
#include <c10/core/GradMode.h>
#include <c10/hip/HIPStream.h>
#include <hip/hip_runtime_api.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/function.h>
#include <torch/csrc/autograd/functions/accumulate_grad.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/autograd/saved_variable.h>
#include <torch/csrc/autograd/variable.h>

#include <cmath>
#include <mutex>
#include <unordered_set>
#include <vector>

#include "ternary_spmm.h"

namespace {

// The library's entry points, as Python loaded it (init).
decltype(&tl_spmm) g_spmm;
decltype(&tl_spmm_workspace) g_workspace;
decltype(&tl_mlp_gate_up) g_gate_up;
decltype(&tl_mlp_gate_up_few) g_gate_up_few;
decltype(&tl_rope_heads) g_rope_heads;
decltype(&tl_rope_to_pages) g_rope_to_pages;
decltype(&tl_read_pages) g_read_pages;
decltype(&tl_paged_attention_workspace) g_attention_workspace;
decltype(&tl_paged_attention) g_attention;
decltype(&tl_paged_attention_shared_workspace) g_shared_workspace;
decltype(&tl_paged_attention_shared) g_shared;
decltype(&tl_teacher_entries) g_teacher;
decltype(&tl_head_loss_workspace) g_loss_workspace;
decltype(&tl_head_loss) g_loss;
decltype(&tl_head_loss_backward) g_loss_backward;
decltype(&tl_last_error) g_last_error;
PyObject* g_workspaces;  // {(device index, stream): uint8 tensor}: the scratch of ops

int type_code(const at::Tensor& t)
{
    return t.scalar_type() == at::kHalf ? TL_F16 : t.scalar_type() == at::kFloat ? TL_F32 : -1;
}

// A tensor with no class, mode or wrapper of its own between the caller and its memory; null for None and for anything else.
const at::Tensor* plain(PyObject* o)
{
    if (!THPVariable_CheckExact(o)) return nullptr;
    const at::Tensor& t = THPVariable_Unpack(o);
    return t.layout() == at::kStrided && t.is_cuda() && !t.is_neg() && !t.is_conj() && t.has_storage() ? &t : nullptr;
}

struct Rows {
    int64_t M = 0, ld = 0;
    int layout = TL_X_ROW_MAJOR;
};

// x as the library's activations of K rows of a weight: [.., K] in uniform rows, or, kmajor, [K, M] or [1, K, M].
bool geometry(const at::Tensor& x, int64_t K, bool kmajor, Rows* r)
{
    const int64_t dims = x.dim();
    if (dims < 1 || dims > 3) return false;
    if (kmajor) {
        if (dims < 2 || (dims == 3 && x.size(0) != 1) || x.size(-2) != K || x.stride(-1) != 1) return false;
        r->M = x.size(-1);
        r->ld = K > 1 ? x.stride(-2) : std::max<int64_t>(r->M, 1);
        r->layout = TL_X_K_MAJOR;
        return r->M > 0;
    }
    if (x.size(-1) != K || (dims != 2 && !x.is_contiguous()) || x.stride(-1) != 1) return false;
    r->M = dims == 1 ? 1 : dims == 2 ? x.size(0) : x.size(0) * x.size(1);
    r->ld = dims == 2 && r->M > 1 ? x.stride(0) : std::max<int64_t>(K, 1);
    return r->M > 0;
}

bool scale_fits(PyObject* o, const at::Tensor** scale, int64_t N, c10::Device device)
{
    *scale = nullptr;
    if (o == Py_None) return true;
    const at::Tensor* s = plain(o);
    if (!s || s->device() != device || s->numel() != N || !s->is_contiguous() || type_code(*s) < 0) return false;
    *scale = s;
    return true;
}

// The call's workspace (kept until the call has been made, whatever another thread does to the dict): false where Python has
// to make one first.
bool workspace(const tl_layout_header* header, const Rows& r, int x_type, c10::Device device, void* stream, at::Tensor* ws)
{
    int64_t need = 0;
    if (g_workspace(header, r.M, x_type, r.layout, &need) != TL_OK) return false;
    if (need == 0) return true;
    PyObject* key = Py_BuildValue("(iK)", (int)device.index(), (unsigned long long)(uintptr_t)stream);
    if (!key) throw python_error();
    PyObject* found = PyDict_GetItemWithError(g_workspaces, key);  // borrowed
    Py_DECREF(key);
    if (!found && PyErr_Occurred()) throw python_error();
    if (!found || !THPVariable_Check(found)) return false;
    const at::Tensor& t = THPVariable_Unpack(found);
    if (t.numel() < need) return false;
    *ws = t;
    return true;
}

void* current_stream(c10::Device device) { return c10::hip::getCurrentHIPStream(device.index()).stream(); }

at::Tensor output(const at::Tensor& x, const Rows& r, int64_t N, bool kmajor)
{
    c10::SmallVector<int64_t, 3> shape(x.sizes().begin(), x.sizes().end());
    if (kmajor) shape[shape.size() - 2] = r.M;
    shape.back() = N;
    return at::empty(shape, x.options().requires_grad(false));
}

const tl_layout_header* header_at(PyObject* address) { return static_cast<const tl_layout_header*>(PyLong_AsVoidPtr(address)); }

// product(header address, blob, x, scale or None, kmajor or None: x of K values a row is rows) -> tensor or None
PyObject* product(PyObject*, PyObject* const* args, Py_ssize_t count)
{
    HANDLE_TH_ERRORS
    if (count != 5) {
        PyErr_SetString(PyExc_TypeError, "product takes five arguments");
        return nullptr;
    }
    const tl_layout_header* header = header_at(args[0]);
    const at::Tensor *blob = plain(args[1]), *x = plain(args[2]), *scale;
    const bool kmajor = args[4] == Py_None ? header && x && x->dim() > 0 && x->size(-1) != header->inners : args[4] == Py_True;
    Rows r;
    if (!header || !blob || !x || x->device() != blob->device() || type_code(*x) < 0 || !geometry(*x, header->inners, kmajor, &r) ||
        !scale_fits(args[3], &scale, header->columns, x->device()))
        Py_RETURN_NONE;
    const c10::DeviceGuard guard(x->device());
    void* stream = current_stream(x->device());
    at::Tensor ws;
    const int type = type_code(*x);
    if (!workspace(header, r, type, x->device(), stream, &ws)) Py_RETURN_NONE;
    at::Tensor y = output(*x, r, header->columns, kmajor);
    int rc;
    {
        const pybind11::gil_scoped_release no_gil;
        rc = g_spmm(header, blob->data_ptr(), x->data_ptr(), type, r.layout, r.ld, r.M, y.data_ptr(), type, header->columns,
                    scale ? scale->data_ptr() : nullptr, scale ? type_code(*scale) : TL_F32, ws.defined() ? ws.data_ptr() : nullptr,
                    ws.defined() ? ws.numel() : 0, stream);
    }
    if (rc != TL_OK) Py_RETURN_NONE;
    return THPVariable_Wrap(std::move(y));
    END_HANDLE_TH_ERRORS
}

// gate_up(gate header, gate blob, up header, up blob, x, gate scale, up scale) -> silu(gate) * up, or None
PyObject* gate_up(PyObject*, PyObject* const* args, Py_ssize_t count)
{
    HANDLE_TH_ERRORS
    if (count != 7) {
        PyErr_SetString(PyExc_TypeError, "gate_up takes seven arguments");
        return nullptr;
    }
    const tl_layout_header *g = header_at(args[0]), *u = header_at(args[2]);
    const at::Tensor *gb = plain(args[1]), *ub = plain(args[3]), *x = plain(args[4]), *gs, *us;
    Rows r;
    if (!g || !u || !gb || !ub || !x || x->device() != gb->device() || x->device() != ub->device() || type_code(*x) < 0 ||
        g->inners != u->inners || g->columns != u->columns || g->tile_rows != u->tile_rows || !geometry(*x, g->inners, false, &r) ||
        !scale_fits(args[5], &gs, g->columns, x->device()) || !scale_fits(args[6], &us, g->columns, x->device()) ||
        (gs == nullptr) != (us == nullptr) || (gs && type_code(*gs) != type_code(*us)))
        Py_RETURN_NONE;
    const bool few = r.M <= 48;
    if (few && (r.M < 2 || !g->off_codes || !u->off_codes)) Py_RETURN_NONE;
    const c10::DeviceGuard guard(x->device());
    void* stream = current_stream(x->device());
    at::Tensor ws;
    const int type = type_code(*x), scale_type = gs ? type_code(*gs) : TL_F32;
    if (!few && !workspace(g, r, type, x->device(), stream, &ws)) Py_RETURN_NONE;
    at::Tensor h = output(*x, r, g->columns, false);
    int rc;
    {
        const pybind11::gil_scoped_release no_gil;
        const void *gsp = gs ? gs->data_ptr() : nullptr, *usp = us ? us->data_ptr() : nullptr;
        rc = few ? g_gate_up_few(g, gb->data_ptr(), u, ub->data_ptr(), x->data_ptr(), type, TL_X_ROW_MAJOR, r.ld, r.M, h.data_ptr(), type, g->columns,
                                 gsp, usp, scale_type, TL_ACT_SILU_GATE, stream)
                 : g_gate_up(g, gb->data_ptr(), u, ub->data_ptr(), x->data_ptr(), type, TL_X_ROW_MAJOR, r.ld, r.M, h.data_ptr(), type, g->columns,
                             gsp, usp, scale_type, TL_ACT_SILU_GATE, ws.defined() ? ws.data_ptr() : nullptr, ws.defined() ? ws.numel() : 0, stream);
    }
    if (rc != TL_OK) Py_RETURN_NONE;
    return THPVariable_Wrap(std::move(h));
    END_HANDLE_TH_ERRORS
}

// ---- a paged cache: what ops.rope_heads, rope_to_pages, read_pages and paged_attention do for plain calls.  One token's heads
// rotated took 36 us through Python's checks and structures.

int64_t step(const at::Tensor& t, int d) { return t.size(d) > 1 ? t.stride(d) : 0; }

bool absent(PyObject* o) { return o == Py_None; }

// Whether a derivative is asked for, backward or forward, which Python refuses.
bool differentiated(std::initializer_list<const at::Tensor*> tensors)
{
    const bool backward = c10::GradMode::is_enabled(), forward = c10::AutogradState::get_tls_state().get_fw_grad_mode();
    for (const at::Tensor* t : tensors)
        if ((backward && t->requires_grad()) || (forward && t->_fw_grad(0).defined())) return true;
    return false;
}

// x [tokens, heads, head_dim] on `device`, of type `type`, its rows' last dimension in one piece; y where it goes (null: pages).
bool head_rows(const at::Tensor& x, const at::Tensor* y, PyObject* norm, tl_head_rows* r)
{
    if (x.dim() != 3 || x.stride(2) != 1 || x.numel() == 0 || differentiated({&x})) return false;
    const at::Tensor* w = nullptr;
    if (!absent(norm)) {
        w = plain(norm);
        if (!w || w->dim() != 1 || w->size(0) != x.size(2) || w->scalar_type() != x.scalar_type() || w->device() != x.device() || !w->is_contiguous() || differentiated({w})) return false;
    }
    *r = tl_head_rows{x.data_ptr(), step(x, 0), step(x, 1), y ? y->data_ptr() : nullptr, y ? step(*y, 0) : 0, y ? step(*y, 1) : 0,
                      w ? w->data_ptr() : nullptr, (int32_t)x.size(1)};
    return true;
}

// An output that is not given, or is the operand itself.
bool output_rows(PyObject* given, PyObject* operand, const at::Tensor& x, at::Tensor* y)
{
    if (given == operand) *y = x;
    else if (absent(given)) *y = at::empty(x.sizes(), x.options().requires_grad(false));
    else return false;
    return true;
}

bool rotation(PyObject* frequencies, PyObject* positions, PyObject* factor, PyObject* interleaved, PyObject* eps, const at::Tensor& like, tl_rotation* r)
{
    const double f = PyFloat_AsDouble(factor), e = PyFloat_AsDouble(eps);
    const int pairs_side_by_side = PyObject_IsTrue(interleaved);
    if (PyErr_Occurred()) {
        PyErr_Clear();
        return false;
    }
    *r = tl_rotation{nullptr, nullptr, 0, 0, (float)f, (float)e};
    if (absent(frequencies)) return true;
    const at::Tensor* t = plain(frequencies);
    if (!t || t->dim() != 1 || t->scalar_type() != at::kDouble || t->device() != like.device() || !t->is_contiguous() || differentiated({t})) return false;
    r->frequencies = static_cast<const double*>(t->data_ptr());
    r->pairs = (int32_t)t->numel();
    r->interleaved = pairs_side_by_side;
    if (absent(positions)) return true;
    const at::Tensor* p = plain(positions);
    if (!p || p->dim() != 1 || p->size(0) != like.size(0) || p->scalar_type() != at::kLong || p->device() != like.device() || !p->is_contiguous()) return false;
    r->positions = static_cast<const int64_t*>(p->data_ptr());
    return true;
}

const at::Tensor* member(PyObject* tuple, int i) { return absent(PyTuple_GET_ITEM(tuple, i)) ? nullptr : plain(PyTuple_GET_ITEM(tuple, i)); }

// ops.Pages and ops.PageBatch as the library's structures.
bool pages_and_batch(PyObject* pages, PyObject* batch, c10::Device device, tl_pages* p, tl_page_batch* b, int64_t* most_rows)
{
    if (!PyTuple_Check(pages) || PyTuple_GET_SIZE(pages) != 4 || !PyTuple_Check(batch) || PyTuple_GET_SIZE(batch) != 4) return false;
    const at::Tensor *k = member(pages, 0), *v = member(pages, 1), *ke = member(pages, 2), *ve = member(pages, 3);
    if (!k || !v || k->dim() != 4 || k->numel() == 0 || k->sizes() != v->sizes() || k->strides() != v->strides() || k->stride(3) != 1 ||
        k->scalar_type() != v->scalar_type() || k->device() != device || v->device() != device || differentiated({k, v}))
        return false;
    const bool bytes = k->scalar_type() == at::kFloat8_e4m3fn;
    if (!bytes && k->scalar_type() != at::kHalf) return false;
    if (bytes) {
        for (const at::Tensor* e : {ke, ve})
            if (!e || e->dim() != 3 || e->sizes() != k->sizes().slice(0, 3) || e->scalar_type() != at::kByte || !e->is_contiguous() || e->device() != device) return false;
    } else if (!absent(PyTuple_GET_ITEM(pages, 2)) || !absent(PyTuple_GET_ITEM(pages, 3))) {
        return false;
    }
    const at::Tensor *table = member(batch, 0), *starts = member(batch, 1), *lengths = member(batch, 2);
    for (const at::Tensor* t : {table, starts, lengths})
        if (!t || t->scalar_type() != at::kInt || t->device() != device || t->numel() == 0) return false;
    if (table->dim() != 2 || starts->dim() != 1 || lengths->dim() != 1 || starts->size(0) != table->size(0) + 1 || lengths->size(0) != table->size(0) ||
        step(*table, 1) > 1 || step(*starts, 0) > 1 || step(*lengths, 0) > 1)
        return false;
    *most_rows = PyLong_AsLongLong(PyTuple_GET_ITEM(batch, 3));
    if (PyErr_Occurred()) {
        PyErr_Clear();
        return false;
    }
    const int64_t any = k->size(2) * k->size(3);   // (a dimension of one entry has no stride of its own)
    auto stride = [&](int d) { return k->size(d) > 1 ? k->stride(d) : any; };
    *p = tl_pages{k->data_ptr(), v->data_ptr(), bytes ? ke->data_ptr() : nullptr, bytes ? ve->data_ptr() : nullptr, stride(0), stride(1), stride(2), k->size(0),
                  (int32_t)k->size(2), (int32_t)k->size(1), (int32_t)k->size(3), bytes ? TL_E4M3 : TL_F16};
    *b = tl_page_batch{static_cast<const int32_t*>(table->data_ptr()), static_cast<const int32_t*>(starts->data_ptr()),
                       static_cast<const int32_t*>(lengths->data_ptr()), table->size(0) > 1 ? table->stride(0) : table->size(1), (int32_t)table->size(1),
                       (int32_t)table->size(0)};
    return true;
}

PyObject* pair_of(at::Tensor a, at::Tensor b)
{
    PyObject* both = PyTuple_New(2);
    if (!both) throw python_error();
    PyTuple_SET_ITEM(both, 0, THPVariable_Wrap(std::move(a)));
    PyTuple_SET_ITEM(both, 1, THPVariable_Wrap(std::move(b)));
    return both;
}

// rope_heads(q, k, positions, frequencies, factor, interleaved, q_norm, k_norm, eps, q_out, k_out) -> (q, k) or None
PyObject* rope_heads(PyObject*, PyObject* const* a, Py_ssize_t count)
{
    HANDLE_TH_ERRORS
    if (count != 11) {
        PyErr_SetString(PyExc_TypeError, "rope_heads takes eleven arguments");
        return nullptr;
    }
    const at::Tensor *q = plain(a[0]), *k = plain(a[1]);
    tl_rotation turn;
    if (!q || !k || q->dim() != 3 || k->dim() != 3 || type_code(*q) < 0 || k->scalar_type() != q->scalar_type() || k->device() != q->device() ||
        k->size(0) != q->size(0) || k->size(2) != q->size(2) || (!absent(a[3]) && absent(a[2])) || !rotation(a[3], a[2], a[4], a[5], a[8], *q, &turn))
        Py_RETURN_NONE;
    const c10::DeviceGuard guard(q->device());
    at::Tensor q_out, k_out;
    tl_head_rows qr, kr;
    if (a[0] == a[1] || !output_rows(a[9], a[0], *q, &q_out) || !output_rows(a[10], a[1], *k, &k_out) || !head_rows(*q, &q_out, a[6], &qr) || !head_rows(*k, &k_out, a[7], &kr))
        Py_RETURN_NONE;
    // (in place on one of two views of the same rows: Python looks at where they lie)
    if ((a[9] == a[0] || a[10] == a[1]) && q->storage().data() == k->storage().data()) Py_RETURN_NONE;
    void* stream = current_stream(q->device());
    int rc;
    {
        const pybind11::gil_scoped_release no_gil;
        rc = g_rope_heads(&qr, &kr, type_code(*q), q->size(0), (int)q->size(2), &turn, stream);
    }
    if (rc != TL_OK) Py_RETURN_NONE;
    return pair_of(std::move(q_out), std::move(k_out));
    END_HANDLE_TH_ERRORS
}

// rope_to_pages(q, k, v, pages, batch, frequencies, positions, factor, interleaved, q_norm, k_norm, eps) -> q or None
PyObject* rope_to_pages(PyObject*, PyObject* const* a, Py_ssize_t count)
{
    HANDLE_TH_ERRORS
    if (count != 12) {
        PyErr_SetString(PyExc_TypeError, "rope_to_pages takes twelve arguments");
        return nullptr;
    }
    const at::Tensor *q = plain(a[0]), *k = plain(a[1]), *v = plain(a[2]);
    tl_rotation turn;
    tl_pages p;
    tl_page_batch b;
    int64_t most;
    if (!q || !k || !v || q->dim() != 3 || k->dim() != 3 || type_code(*k) < 0 || q->scalar_type() != k->scalar_type() || v->scalar_type() != k->scalar_type() ||
        q->device() != k->device() || v->device() != k->device() || q->size(0) != k->size(0) || q->size(2) != k->size(2) || v->sizes() != k->sizes() ||
        !rotation(a[5], a[6], a[7], a[8], a[11], *k, &turn) || !pages_and_batch(a[3], a[4], k->device(), &p, &b, &most) || p.kv_heads != k->size(1) ||
        p.head_dim != k->size(2))
        Py_RETURN_NONE;
    const c10::DeviceGuard guard(k->device());
    at::Tensor q_out = at::empty(q->sizes(), q->options().requires_grad(false));
    tl_head_rows qr, kr, vr;
    if (!head_rows(*q, &q_out, a[9], &qr) || !head_rows(*k, nullptr, a[10], &kr) || !head_rows(*v, nullptr, Py_None, &vr)) Py_RETURN_NONE;
    void* stream = current_stream(k->device());
    int rc;
    {
        const pybind11::gil_scoped_release no_gil;
        rc = g_rope_to_pages(&qr, &kr, &vr, type_code(*k), k->size(0), &turn, &p, &b, stream);
    }
    if (rc != TL_OK) Py_RETURN_NONE;
    return THPVariable_Wrap(std::move(q_out));
    END_HANDLE_TH_ERRORS
}

// read_pages(pages, batch, tokens, fp16) -> (k, v) or None
PyObject* read_pages(PyObject*, PyObject* const* a, Py_ssize_t count)
{
    HANDLE_TH_ERRORS
    if (count != 4) {
        PyErr_SetString(PyExc_TypeError, "read_pages takes four arguments");
        return nullptr;
    }
    const at::Tensor* k = PyTuple_Check(a[0]) && PyTuple_GET_SIZE(a[0]) == 4 ? member(a[0], 0) : nullptr;
    const int64_t tokens = PyLong_AsLongLong(a[2]);
    if (PyErr_Occurred()) PyErr_Clear();
    tl_pages p;
    tl_page_batch b;
    int64_t most;
    if (!k || tokens <= 0 || !pages_and_batch(a[0], a[1], k->device(), &p, &b, &most)) Py_RETURN_NONE;
    const c10::DeviceGuard guard(k->device());
    const bool half = a[3] == Py_True;
    at::Tensor both = at::empty({2, tokens, p.kv_heads, p.head_dim}, k->options().dtype(half ? at::kHalf : at::kFloat).requires_grad(false));
    at::Tensor k_out = both.select(0, 0), v_out = both.select(0, 1);
    void* stream = current_stream(k->device());
    int rc;
    {
        const pybind11::gil_scoped_release no_gil;
        rc = g_read_pages(&p, &b, tokens, half ? TL_F16 : TL_F32, k_out.data_ptr(), v_out.data_ptr(), (int64_t)p.kv_heads * p.head_dim, p.head_dim, stream);
    }
    if (rc != TL_OK) Py_RETURN_NONE;
    return pair_of(std::move(k_out), std::move(v_out));
    END_HANDLE_TH_ERRORS
}

// Groups of the batch's sequences that begin alike; false where they are none of a plain call.
bool prefix_of(PyObject* prefix, const tl_page_batch& b, c10::Device device, tl_page_prefix* p)
{
    if (!PyTuple_Check(prefix) || PyTuple_GET_SIZE(prefix) != 3) return false;
    const long long most = absent(PyTuple_GET_ITEM(prefix, 2)) ? -1 : PyLong_AsLongLong(PyTuple_GET_ITEM(prefix, 2));
    if (PyErr_Occurred()) {
        PyErr_Clear();
        return false;
    }
    const at::Tensor *groups = member(prefix, 0), *shared = member(prefix, 1);
    for (const at::Tensor* t : {groups, shared})
        if (!t || t->scalar_type() != at::kInt || t->device() != device || t->numel() == 0 || t->dim() != 1 || !t->is_contiguous()) return false;
    if (shared->numel() != b.seqs || groups->numel() > INT32_MAX) return false;
    *p = tl_page_prefix{static_cast<const int32_t*>(groups->data_ptr()), static_cast<const int32_t*>(shared->data_ptr()), (int32_t)(groups->numel() - 1),
                        (int32_t)std::min<long long>(std::max<long long>(most, -1), INT32_MAX)};
    return true;
}

// paged_attention(q, pages, batch, scale or None, out or None, prefix or None) -> out or None
PyObject* paged_attention(PyObject*, PyObject* const* a, Py_ssize_t count)
{
    HANDLE_TH_ERRORS
    if (count != 6) {
        PyErr_SetString(PyExc_TypeError, "paged_attention takes six arguments");
        return nullptr;
    }
    const at::Tensor* q = plain(a[0]);
    tl_pages p;
    tl_page_batch b;
    int64_t most, need;
    if (!q || q->dim() != 3 || q->numel() == 0 || q->stride(2) != 1 || q->scalar_type() != at::kHalf || differentiated({q}) || !pages_and_batch(a[1], a[2], q->device(), &p, &b, &most) ||
        p.head_dim != q->size(2))
        Py_RETURN_NONE;
    const int64_t tokens = q->size(0), width = q->size(1) * q->size(2);
    const double scale = absent(a[3]) ? 1.0 / std::sqrt((double)q->size(2)) : PyFloat_AsDouble(a[3]);
    if (PyErr_Occurred()) {
        PyErr_Clear();
        Py_RETURN_NONE;
    }
    const c10::DeviceGuard guard(q->device());
    const at::Tensor* given = absent(a[4]) ? nullptr : plain(a[4]);
    if (!absent(a[4]) && (!given || given->dim() != 2 || given->size(0) != tokens || given->size(1) != width || given->scalar_type() != at::kHalf ||
                          given->device() != q->device() || !given->is_contiguous() || differentiated({given}) || given->storage().data() == q->storage().data()))
        Py_RETURN_NONE;
    tl_page_prefix prefix;
    const bool grouped = !absent(a[5]);
    if (grouped && !prefix_of(a[5], b, q->device(), &prefix)) Py_RETURN_NONE;
    if ((grouped ? g_shared_workspace(tokens, (int)q->size(1), &p, &b, &prefix, most, &need)
                 : g_attention_workspace(tokens, (int)q->size(1), &p, &b, most, &need)) != TL_OK)
        Py_RETURN_NONE;
    at::Tensor out = given ? *given : at::empty({tokens, width}, q->options().requires_grad(false));
    at::Tensor ws = at::empty({need}, q->options().dtype(at::kByte).requires_grad(false));
    void* stream = current_stream(q->device());
    int rc;
    {
        const pybind11::gil_scoped_release no_gil;
        if (grouped) {
            rc = g_shared(q->data_ptr(), step(*q, 0), step(*q, 1), TL_F16, tokens, (int)q->size(1), &p, &b, &prefix, most, (float)scale, out.data_ptr(),
                          ws.data_ptr(), need, stream);
        } else {
            rc = g_attention(q->data_ptr(), step(*q, 0), step(*q, 1), TL_F16, tokens, (int)q->size(1), &p, &b, most, (float)scale, out.data_ptr(), ws.data_ptr(),
                             need, stream);
        }
    }
    if (rc != TL_OK) Py_RETURN_NONE;
    return THPVariable_Wrap(std::move(out));
    END_HANDLE_TH_ERRORS
}

// ---- a head's losses.  Forty rows' loss and gradients took the host 184 us through an autograd function of Python's, for 100 us of kernels.

// What is wanted of the rows: targets, or a teacher's entries (and what those were made into).
struct Wanted {
    at::Tensor targets, entries, shares, known;
    int64_t ignore = 0;
    float temperature = 1.f;
    tl_loss_target call() const
    {
        if (targets.defined()) return tl_loss_target{static_cast<const int64_t*>(targets.data_ptr()), ignore, nullptr, nullptr, nullptr, 1, 1.f};
        return tl_loss_target{nullptr, 0, static_cast<const int32_t*>(entries.data_ptr()), static_cast<const float*>(shares.data_ptr()),
                              static_cast<const float*>(known.data_ptr()), (int32_t)entries.size(1), temperature};
    }
};

int64_t row_step(const at::Tensor& x) { return x.size(0) > 1 ? x.stride(0) : std::max<int64_t>(x.size(1), 1); }

at::Tensor bytes_on(const at::Tensor& like, int64_t bytes) { return at::empty({bytes}, like.options().dtype(at::kByte).requires_grad(false)); }

// The backward pass of a loss, once.
struct HeadLossBackward : torch::autograd::Node {
    tl_layout_header header;
    at::Tensor blob, codes, lse;
    Wanted wanted;                         // (its targets are `targets`, whose later changes are noticed)
    torch::autograd::SavedVariable x_, scale_, targets_;
    bool has_scale, has_targets;
    std::mutex mutex_;

    std::string name() const override { return "HeadLossBackward"; }

    void release_variables() override
    {
        const std::lock_guard<std::mutex> lock(mutex_);
        x_.reset_data(), scale_.reset_data(), targets_.reset_data();
        lse.reset();
        wanted = Wanted();
    }

    torch::autograd::variable_list apply(torch::autograd::variable_list&& grads) override
    {
        const std::lock_guard<std::mutex> lock(mutex_);
        torch::autograd::variable_list out(2);
        if (!grads[0].defined()) return out;
        const at::Tensor x = x_.unpack(), scale = has_scale ? scale_.unpack() : at::Tensor();   // (raises if they were changed or are gone)
        Wanted w = wanted;
        if (has_targets) w.targets = targets_.unpack();
        at::Tensor dx, ds;
        {
            const at::AutoGradMode no_grad(false);
            const c10::DeviceGuard guard(x.device());
            const at::Tensor grad = grads[0].detach().to(at::kFloat).contiguous();
            if (task_should_compute_output(0)) dx = at::empty(x.sizes(), x.options().requires_grad(false));
            if (has_scale && task_should_compute_output(1)) ds = at::empty(scale.sizes(), scale.options().requires_grad(false));
            const tl_loss_target target = w.call();
            const int type = type_code(x);
            int64_t need = 0;
            TORCH_CHECK(g_loss_workspace(&header, x.size(0), type, &target, 1, &need) == TL_OK, g_last_error());
            const at::Tensor ws = bytes_on(x, need);
            TORCH_CHECK(g_loss_backward(&header, blob.data_ptr(), codes.defined() ? codes.data_ptr() : nullptr, x.data_ptr(), type, row_step(x), x.size(0),
                                        has_scale ? scale.data_ptr() : nullptr, has_scale ? type_code(scale) : TL_F32, &target,
                                        static_cast<const float*>(lse.data_ptr()), static_cast<const float*>(grad.data_ptr()),
                                        dx.defined() ? dx.data_ptr() : nullptr, x.size(1), ds.defined() ? ds.data_ptr() : nullptr, ws.data_ptr(), need,
                                        current_stream(x.device())) == TL_OK,
                        g_last_error());
        }
        if (c10::GradMode::is_enabled()) {     // (a graph of the gradients is asked for: they have none, which whoever follows it to an operand is told)
            const std::shared_ptr<torch::autograd::Node> once(
                new torch::autograd::Error("the losses of a head are differentiable once", torch::autograd::collect_next_edges(x, scale, grads[0])),
                torch::autograd::deleteNode);
            for (at::Tensor* d : {&dx, &ds})
                if (d->defined()) torch::autograd::set_history(*d, once);
        }
        out[0] = dx, out[1] = ds;
        return out;
    }
};

// What accumulates a leaf's gradient belongs to the stream on which a graph first asked for it, and is the same in every graph of the leaf while one lives: a
// captured backward pass would wait for that stream, which ends the capture in a thread of the engine's, and the process.  So a call whose operands lead to one of another
// stream is refused.
void refuse_captured(void* stream, std::initializer_list<const at::Tensor*> operands)
{
    hipStreamCaptureStatus capture = hipStreamCaptureStatusNone;
    if (hipStreamIsCapturing(static_cast<hipStream_t>(stream), &capture) != hipSuccess || capture == hipStreamCaptureStatusNone) return;
    std::vector<torch::autograd::Node*> left;
    std::unordered_set<torch::autograd::Node*> seen;
    auto look = [&](torch::autograd::Node* node, c10::DeviceIndex device) {
        if (!node || !seen.insert(node).second) return;
        if (!dynamic_cast<torch::autograd::AccumulateGrad*>(node)) {
            left.push_back(node);
            return;
        }
        const auto of = node->stream();
        TORCH_CHECK(of && of->id() == c10::hip::getCurrentHIPStream(device).id(),
                    "a graph of the same leaf lives outside of the captured one: let go of it first, or take a new leaf");
    };
    for (const at::Tensor* t : operands) {
        if (!t) continue;
        const c10::DeviceIndex device = t->device().index();
        look(t->is_leaf() ? torch::autograd::impl::try_get_grad_accumulator(*t).get() : t->grad_fn().get(), device);
        while (!left.empty()) {
            torch::autograd::Node* node = left.back();
            left.pop_back();
            for (const torch::autograd::Edge& e : node->next_edges()) look(e.function.get(), device);
        }
    }
}

// capturable(x): raises for a leaf that a captured backward pass must not reach
PyObject* capturable(PyObject*, PyObject* o)
{
    HANDLE_TH_ERRORS
    const at::Tensor* x = plain(o);
    if (x && x->requires_grad()) refuse_captured(current_stream(x->device()), {x});
    Py_RETURN_NONE;
    END_HANDLE_TH_ERRORS
}

// head_loss(header address, blob, transposed codes or None, x, scale or None, targets or None, ignore, ids or None, logits or None, temperature)
// -> losses, None for a call that is not a plain one, or the library's status
PyObject* head_loss(PyObject*, PyObject* const* a, Py_ssize_t count)
{
    HANDLE_TH_ERRORS
    if (count != 10) {
        PyErr_SetString(PyExc_TypeError, "head_loss takes ten arguments");
        return nullptr;
    }
    const tl_layout_header* header = header_at(a[0]);
    const at::Tensor *blob = plain(a[1]), *codes = absent(a[2]) ? nullptr : plain(a[2]), *x = plain(a[3]), *scale;
    const double temperature = PyFloat_AsDouble(a[9]);
    const long long ignore = PyLong_AsLongLong(a[6]);
    if (PyErr_Occurred()) {
        PyErr_Clear();
        Py_RETURN_NONE;
    }
    if (!header || !blob || !x || (!absent(a[2]) && (!codes || codes->device() != blob->device())) || x->device() != blob->device() || type_code(*x) < 0 ||
        x->dim() != 2 || x->size(0) == 0 || x->size(1) != header->inners || (x->size(1) > 1 && x->stride(1) != 1) || row_step(*x) < x->size(1) ||
        !scale_fits(a[4], &scale, header->columns, x->device()) || (scale && scale->dim() != 1))
        Py_RETURN_NONE;
    const int64_t rows = x->size(0);
    const bool backward = c10::GradMode::is_enabled(), forward = c10::AutogradState::get_tls_state().get_fw_grad_mode();
    const bool by_x = backward && x->requires_grad(), by_scale = backward && scale && scale->requires_grad();
    if ((by_x && !codes) || (forward && (x->_fw_grad(0).defined() || (scale && scale->_fw_grad(0).defined())))) Py_RETURN_NONE;
    Wanted wanted;
    const at::Tensor *ids = nullptr, *logits = nullptr;
    if (!absent(a[5])) {
        const at::Tensor* t = plain(a[5]);
        if (!t || t->dim() != 1 || t->size(0) != rows || t->scalar_type() != at::kLong || t->device() != x->device() || !t->is_contiguous()) Py_RETURN_NONE;
        wanted.targets = *t;
        wanted.ignore = ignore;
    } else {
        ids = plain(a[7]), logits = plain(a[8]);
        if (!ids || !logits || ids->dim() != 2 || ids->size(0) != rows || ids->size(1) == 0 || logits->sizes() != ids->sizes() || ids->scalar_type() != at::kLong ||
            type_code(*logits) < 0 || ids->device() != x->device() || logits->device() != x->device() || differentiated({logits}))
            Py_RETURN_NONE;
        for (const at::Tensor* t : {ids, logits})
            if ((t->size(1) > 1 && t->stride(1) != 1) || row_step(*t) < t->size(1)) Py_RETURN_NONE;
    }
    const c10::DeviceGuard guard(x->device());
    void* stream = current_stream(x->device());
    if (by_x || by_scale) refuse_captured(stream, {by_x ? x : nullptr, by_scale ? scale : nullptr});
    const auto floats = x->options().dtype(at::kFloat).requires_grad(false);
    at::Tensor loss = at::empty({rows}, floats), lse = at::empty({rows + 1}, floats);
    const int type = type_code(*x);
    int rc = TL_OK;
    if (ids) {
        wanted.entries = at::empty(ids->sizes(), floats.dtype(at::kInt));
        wanted.shares = at::empty(ids->sizes(), floats);
        wanted.known = at::empty({rows}, floats);
        wanted.temperature = (float)temperature;
        rc = g_teacher(static_cast<const int64_t*>(ids->data_ptr()), row_step(*ids), logits->data_ptr(), type_code(*logits), row_step(*logits), rows,
                       (int)ids->size(1), (int)header->columns, (float)temperature, static_cast<int32_t*>(wanted.entries.data_ptr()),
                       static_cast<float*>(wanted.shares.data_ptr()), static_cast<float*>(wanted.known.data_ptr()), stream);
    }
    if (rc == TL_OK) {
        const tl_loss_target target = wanted.call();
        int64_t need = 0;
        rc = g_loss_workspace(header, rows, type, &target, 0, &need);
        if (rc == TL_OK) {
            const at::Tensor ws = bytes_on(*x, need);
            const pybind11::gil_scoped_release no_gil;
            rc = g_loss(header, blob->data_ptr(), x->data_ptr(), type, row_step(*x), rows, scale ? scale->data_ptr() : nullptr, scale ? type_code(*scale) : TL_F32,
                        &target, static_cast<float*>(loss.data_ptr()), static_cast<float*>(lse.data_ptr()), ws.data_ptr(), need, stream);
        }
    }
    if (rc != TL_OK) return PyLong_FromLong(rc);
    if (by_x || by_scale) {
        const std::shared_ptr<HeadLossBackward> node(new HeadLossBackward(), torch::autograd::deleteNode);
        node->header = *header;
        node->blob = *blob, node->lse = lse;
        if (codes) node->codes = *codes;
        node->x_ = torch::autograd::SavedVariable(*x, false);
        node->has_scale = scale != nullptr;
        if (scale) node->scale_ = torch::autograd::SavedVariable(*scale, false);
        node->has_targets = wanted.targets.defined();
        if (node->has_targets) node->targets_ = torch::autograd::SavedVariable(wanted.targets, false);
        node->wanted = wanted;
        node->wanted.targets.reset();
        node->set_next_edges(torch::autograd::collect_next_edges(*x, scale ? *scale : at::Tensor()));
        torch::autograd::set_history(loss, node);
    }
    return THPVariable_Wrap(std::move(loss));
    END_HANDLE_TH_ERRORS
}

// init(addresses of the library's entry points in the order of g_*, the scratch dict)
PyObject* init(PyObject*, PyObject* args)
{
    PyObject *addresses, *dict;
    constexpr Py_ssize_t kEntries = 16;
    if (!PyArg_ParseTuple(args, "O!O!", &PyTuple_Type, &addresses, &PyDict_Type, &dict)) return nullptr;
    if (PyTuple_GET_SIZE(addresses) != kEntries) {
        PyErr_SetString(PyExc_TypeError, "init takes the address of each entry point");
        return nullptr;
    }
    Py_ssize_t i = 0;
    auto take = [&](auto& entry) { entry = reinterpret_cast<std::decay_t<decltype(entry)>>(PyLong_AsVoidPtr(PyTuple_GET_ITEM(addresses, i++))); };
    take(g_spmm), take(g_workspace), take(g_gate_up), take(g_gate_up_few);
    take(g_rope_heads), take(g_rope_to_pages), take(g_read_pages), take(g_attention_workspace), take(g_attention);
    take(g_shared_workspace), take(g_shared), take(g_teacher), take(g_loss_workspace), take(g_loss), take(g_loss_backward), take(g_last_error);
    if (PyErr_Occurred()) return nullptr;
    Py_INCREF(dict);
    g_workspaces = dict;
    Py_RETURN_NONE;
}

PyMethodDef g_methods[] = {
    {"init", init, METH_VARARGS, "addresses of the library's entry points, and the scratch buffers"},
    {"product", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(product)), METH_FASTCALL, "x @ W * scale, or None"},
    {"gate_up", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(gate_up)), METH_FASTCALL, "silu(x @ Wg) * (x @ Wu), or None"},
    {"rope_heads", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(rope_heads)), METH_FASTCALL, "heads normalised and rotated, or None"},
    {"rope_to_pages", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(rope_to_pages)), METH_FASTCALL, "the same into pages, or None"},
    {"read_pages", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(read_pages)), METH_FASTCALL, "rows out of pages, or None"},
    {"paged_attention", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(paged_attention)), METH_FASTCALL, "attention over pages, or None"},
    {"head_loss", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(head_loss)), METH_FASTCALL, "what a head's rows are worth, None, or a status"},
    {"capturable", capturable, METH_O, "refuses a leaf whose gradient must not be captured"},
    {nullptr, nullptr, 0, nullptr},
};
PyModuleDef g_module = {PyModuleDef_HEAD_INIT, "_tl_torch", nullptr, -1, g_methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__tl_torch(void) { return PyModule_Create(&g_module); }
