// The serving operators as a CPython module (vall_e_amd._serving): checks of the tensors, the result's allocation, the current stream and
// the C call, in C++.  A step of a serving loop calls these per layer on a handful of rows; through ctypes the checks and argument
// conversions took 6 of a call's 10 us on the host, twice the kernel launch itself (rope_kv_paged 10.5 us, here 4.0).
// Everything on the device is behind include/valle_hip.h; this file holds no device code.
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>
#include <ATen/hip/EmptyTensor.h>
#include <c10/hip/HIPFunctions.h>
#include <c10/hip/HIPStream.h>
#include "../../include/valle_hip.h"

namespace {

PyObject* g_error = nullptr;            // vall_e_amd._lib.ValleHipError
constexpr int64_t HEAD = 64;

struct HipError : std::runtime_error { using std::runtime_error::runtime_error; };

#define NEED(cond, ...) TORCH_CHECK_VALUE(cond, __VA_ARGS__)

const at::Tensor& tensor(PyObject* o, const char* name) {
    TORCH_CHECK_TYPE(THPVariable_Check(o), name, ": a tensor is needed");
    return THPVariable_Unpack(o);
}
const at::Tensor* maybe(PyObject* o, const char* name) { return o == Py_None ? nullptr : &tensor(o, name); }
int64_t whole(PyObject* o, const char* name) {
    const int64_t v = PyLong_AsLongLong(o);
    if (v == -1 && PyErr_Occurred()) throw python_error();
    NEED(v >= INT32_MIN && v <= INT32_MAX, name, ": ", v, " is out of range");
    return v;
}

std::string shape_of(const at::Tensor& t) {
    std::ostringstream s;
    s << t.scalar_type() << " " << t.sizes() << " on " << t.device() << (t.is_contiguous() ? "" : " (not contiguous)");
    return s.str();
}

int gpu_of(const at::Tensor& t, const char* what) {
    if (!t.is_cuda()) throw HipError(std::string(what) + " needs GPU tensors; there is no CPU fallback");
    return t.get_device();
}
int dtype_of(const at::Tensor& t) {
    if (t.scalar_type() == at::kBFloat16) return VALLE_BF16;
    if (t.scalar_type() == at::kFloat) return VALLE_F32;
    throw HipError(std::string("dtype ") + c10::toString(t.scalar_type()) + " is not built (float32 and bfloat16 are)");
}
bool on(const at::Tensor& t, int dev) { return t.is_cuda() && t.get_device() == dev; }

// a contiguous whole-number tensor of the given shape on the call's GPU
template <typename T = int32_t>
T* ints(const at::Tensor& t, const char* name, int dev, std::initializer_list<int64_t> shape) {
    const auto type = sizeof(T) == 8 ? at::kLong : at::kInt;
    NEED(t.scalar_type() == type && on(t, dev) && t.sizes() == at::IntArrayRef(shape) && t.is_contiguous(),
         name, ": contiguous ", type, " tensor of shape ", at::IntArrayRef(shape), " on GPU ", dev, " needed, got ", shape_of(t));
    return static_cast<T*>(t.data_ptr());
}

// [rows][heads][64] with the heads packed: any row stride that keeps rows 16-byte aligned, a copy otherwise
struct Heads { at::Tensor held; void* p; int64_t stride, rows, heads; };
bool packed_heads(const at::Tensor& t) {
    return t.stride(2) == 1 && (t.stride(1) == HEAD || t.size(1) == 1) && t.stride(0) % 8 == 0 && t.stride(0) >= 0 && reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0;
}
Heads heads(const at::Tensor& t, const char* name, int dev, at::ScalarType type, int64_t rows) {
    NEED(t.dim() == 3 && t.size(2) == HEAD && (rows < 0 || t.size(0) == rows), name, ": shape (rows", rows < 0 ? std::string() : " = " + std::to_string(rows),
         ", heads, ", HEAD, ") needed, got ", t.sizes());
    TORCH_CHECK_TYPE(t.scalar_type() == type, name, " is ", t.scalar_type(), ", ", type, " needed");
    NEED(on(t, dev), name, " is on ", t.device(), ", GPU ", dev, " needed");
    if (packed_heads(t)) return {at::Tensor(), t.data_ptr(), t.stride(0), t.size(0), t.size(1)};
    at::Tensor c = t.clone(at::MemoryFormat::Contiguous);
    return {c, c.data_ptr(), t.size(1) * HEAD, t.size(0), t.size(1)};
}
at::Tensor fresh(at::IntArrayRef shape, at::ScalarType type, int dev) {
    return at::detail::empty_cuda(shape, type, c10::Device(c10::DeviceType::CUDA, static_cast<c10::DeviceIndex>(dev)), std::nullopt);
}
// the result: a new tensor like q, or the caller's
at::Tensor result(PyObject* given, const at::Tensor& q, int dev) {
    if (given == Py_None) return fresh(q.sizes(), q.scalar_type(), dev);
    const at::Tensor& o = tensor(given, "out");
    NEED(o.sizes() == q.sizes() && o.scalar_type() == q.scalar_type() && on(o, dev) && packed_heads(o), "out: like q ", shape_of(q),
         ", heads packed, rows 16-byte aligned; got ", shape_of(o));
    return o;
}

bool page_size_ok(int64_t p) { return p == 16 || p == 32 || p == 64 || p == 128 || p == 256; }
// pages [n_pages][kv_heads][page][64] (layers: one more dimension in front), contiguous inside a layer
void pools(const at::Tensor& k, const at::Tensor& v, int dev, at::ScalarType type, bool layers) {
    TORCH_CHECK_TYPE(k.scalar_type() == type && v.scalar_type() == type, "caches are ", k.scalar_type(), " / ", v.scalar_type(), ", ", type, " needed");
    const int d = layers ? 1 : 0;
    NEED(k.dim() == 4 + d && v.sizes() == k.sizes() && k.size(3 + d) == HEAD && page_size_ok(k.size(2 + d)) && k.numel() > 0, "caches: two pools of ",
         layers ? "(n_layers, " : "(", "n_pages, kv_heads, page_size 16 | 32 | 64 | 128 | 256, 64), got ", k.sizes(), ", ", v.sizes());
    NEED(on(k, dev) && on(v, dev), "caches on ", k.device(), " / ", v.device(), ", GPU ", dev, " needed");
    for (const at::Tensor* c : {&k, &v}) {
        int64_t want = 1;
        for (int i = 3 + d; i >= d; --i) {
            NEED(c->stride(i) == want || c->size(i) == 1, "the pages of a layer must be contiguous");
            want *= c->size(i);
        }
        if (layers) NEED(c->size(0) == 1 || (c->stride(0) >= want && c->stride(0) == k.stride(0)), "both pools' layers must lie equally far apart");
    }
}

void check(int rc) {
    if (rc != VALLE_OK) {
        const char* msg = valle_last_error();
        throw HipError("libvalle_hip error " + std::to_string(rc) + ": " + (msg ? msg : "?"));
    }
}
struct NoLock {                          // the interpreter's lock is released while this lives
    PyThreadState* state = PyEval_SaveThread();
    ~NoLock() { PyEval_RestoreThread(state); }
};
struct OnDevice {
    c10::DeviceIndex was, dev;
    explicit OnDevice(int d) : was(c10::hip::current_device()), dev(static_cast<c10::DeviceIndex>(d)) {
        if (was != dev) c10::hip::set_device(dev);
    }
    ~OnDevice() {
        if (was != dev) (void)hipSetDevice(was);
    }
};
// f(current stream of the GPU) with that GPU current
template <typename F>
void launch(int dev, F&& f) {
    void* stream = c10::hip::getCurrentHIPStream(static_cast<c10::DeviceIndex>(dev)).stream();
    int rc;
    {
        NoLock unlocked;
        OnDevice current(dev);
        rc = f(stream);
    }
    check(rc);
}

#define TRY HANDLE_TH_ERRORS try {
#define CATCH } catch (const HipError& e) { PyErr_SetString(g_error ? g_error : PyExc_RuntimeError, e.what()); return nullptr; } END_HANDLE_TH_ERRORS
#define ARGS(n) TORCH_CHECK_TYPE(nargs == (n), "_serving: ", n, " arguments needed, got ", nargs)

// (len_old, len_new, parents | None, block_table, n_blocks, n_blocks_out, free_list, free_count, free_count_out, status, cu_rows, slots,
//  positions, tree_mask, ticket, page_size)
PyObject* page_plan(PyObject*, PyObject* const* a, Py_ssize_t nargs) {
    TRY
    ARGS(16);
    const at::Tensor& tab = tensor(a[3], "block_table");
    const int dev = gpu_of(tab, "PageTable.plan");
    NEED(tab.dim() == 2, "block_table: (requests, max_blocks) needed");
    const int64_t B = tab.size(0), width = tab.size(1);
    const at::Tensor &fl = tensor(a[6], "free_list"), &slots = tensor(a[11], "slots");
    NEED(fl.dim() == 1 && slots.dim() == 1, "free_list and slots have one dimension");
    const int64_t pages = fl.size(0), rows = slots.size(0);
    NEED(B <= INT32_MAX && width <= INT32_MAX && pages <= INT32_MAX && rows <= INT32_MAX, "tables of more than 2^31 entries");
    const at::Tensor* par = maybe(a[2], "parents");
    const int32_t* lo = ints(tensor(a[0], "len_old"), "len_old", dev, {B});
    const int32_t* ln = ints(tensor(a[1], "len_new"), "len_new", dev, {B});
    const int32_t* pp = par ? ints(*par, "parents", dev, {rows}) : nullptr;
    int64_t* mask = ints<int64_t>(tensor(a[13], "tree_mask"), "tree_mask", dev, {rows});
    int32_t* tp = ints(tab, "block_table", dev, {B, width});
    const int32_t *nb = ints(tensor(a[4], "n_blocks"), "n_blocks", dev, {B}), *fc = ints(tensor(a[7], "free_count"), "free_count", dev, {1});
    int32_t *nbo = ints(tensor(a[5], "n_blocks_out"), "n_blocks_out", dev, {B}), *fco = ints(tensor(a[8], "free_count_out"), "free_count_out", dev, {1});
    int32_t *flp = ints(fl, "free_list", dev, {pages}), *st = ints(tensor(a[9], "status"), "status", dev, {B}), *cu = ints(tensor(a[10], "cu_rows"), "cu_rows", dev, {B + 1});
    int32_t *sp = ints(slots, "slots", dev, {rows}), *ps = ints(tensor(a[12], "positions"), "positions", dev, {rows});
    int32_t* ticket = ints(tensor(a[14], "ticket"), "ticket", dev, {1});
    const int page = whole(a[15], "page_size");
    launch(dev, [&](void* s) { return valle_page_plan_masked(lo, ln, B, page, tp, width, nb, nbo, flp, pages, fc, fco, st, cu, sp, ps, rows, pp, mask, ticket, s); });
    Py_RETURN_NONE;
    CATCH
}

// (q, k, v, positions, rope, slots, k_cache, v_cache, out | None) -> out
PyObject* rope_kv_paged(PyObject*, PyObject* const* a, Py_ssize_t nargs) {
    TRY
    ARGS(9);
    const at::Tensor &q = tensor(a[0], "q"), &rope = tensor(a[4], "rope"), &kc = tensor(a[6], "k_cache"), &vc = tensor(a[7], "v_cache");
    const int dev = gpu_of(q, "rope_kv_paged"), dt = dtype_of(q);
    const auto type = q.scalar_type();
    pools(kc, vc, dev, type, false);
    const Heads qh = heads(q, "q", dev, type, -1);
    const Heads kh = heads(tensor(a[1], "k"), "k", dev, type, qh.rows), vh = heads(tensor(a[2], "v"), "v", dev, type, qh.rows);
    NEED(kh.heads == kc.size(1) && vh.heads == kc.size(1), "k, v have ", kh.heads, ", ", vh.heads, " heads, the cache ", kc.size(1));
    NEED(rope.scalar_type() == at::kFloat && on(rope, dev) && rope.dim() == 3 && rope.size(0) > 0 && rope.size(0) <= INT32_MAX && rope.size(1) == HEAD / 2 &&
         rope.size(2) == 2 && rope.is_contiguous(), "rope: contiguous float32 (positions, 32, 2) table on GPU ", dev, " needed, got ", shape_of(rope));
    const int32_t *pos = ints(tensor(a[3], "positions"), "positions", dev, {qh.rows}), *slots = ints(tensor(a[5], "slots"), "slots", dev, {qh.rows});
    const at::Tensor out = result(a[8], q, dev);
    if (qh.rows) {
        NEED(qh.rows <= INT32_MAX && qh.heads <= INT32_MAX && kc.size(0) <= INT32_MAX, "rope_kv_paged: sizes beyond 2^31");
        launch(dev, [&](void* s) {
            return valle_rope_kv_paged(qh.p, qh.stride, kh.p, kh.stride, vh.p, vh.stride, out.data_ptr(), out.stride(0), pos, static_cast<const float*>(rope.data_ptr()),
                                       rope.size(0), slots, qh.rows, qh.heads, kc.size(1), HEAD, kc.data_ptr(), vc.data_ptr(), kc.size(0), kc.size(2), dt, s);
        });
    }
    if (a[8] != Py_None) { Py_INCREF(a[8]); return a[8]; }
    return THPVariable_Wrap(out);
    CATCH
}

// (q, k_cache, v_cache, block_table, ctx_len, cu_rows, tree_mask | None, max_nodes | None, max_ctx | None, softmax_scale, out | None) -> out
PyObject* attn_tree(PyObject*, PyObject* const* a, Py_ssize_t nargs) {
    TRY
    ARGS(11);
    const at::Tensor &q = tensor(a[0], "q"), &kc = tensor(a[1], "k_cache"), &vc = tensor(a[2], "v_cache"), &tab = tensor(a[3], "block_table");
    const int dev = gpu_of(q, "attn_tree"), dt = dtype_of(q);
    const auto type = q.scalar_type();
    pools(kc, vc, dev, type, false);
    const Heads qh = heads(q, "q", dev, type, -1);
    NEED(tab.dim() == 2, "block_table: (requests, max_blocks) needed, got ", tab.sizes());
    const int64_t B = tab.size(0), width = tab.size(1), hkv = kc.size(1), page = kc.size(2);
    NEED(qh.heads % hkv == 0, qh.heads, " heads over ", hkv, " kv heads");
    const int64_t nodes = a[7] == Py_None ? std::max<int64_t>(1, std::min<int64_t>(64, qh.rows)) : whole(a[7], "max_nodes");
    NEED(nodes > 0 && nodes <= 64, "max_nodes ", nodes, ": 1 .. 64");
    const int64_t ctx_hint = a[8] == Py_None ? std::min<int64_t>(width * page, INT32_MAX) : whole(a[8], "max_ctx");
    const double scale = PyFloat_AsDouble(a[9]);
    if (scale == -1.0 && PyErr_Occurred()) throw python_error();
    const int32_t *tp = ints(tab, "block_table", dev, {B, width}), *ctx = ints(tensor(a[4], "ctx_len"), "ctx_len", dev, {B});
    const int32_t* cu = ints(tensor(a[5], "cu_rows"), "cu_rows", dev, {B + 1});
    const at::Tensor* mt = maybe(a[6], "tree_mask");
    const int64_t* mask = mt ? ints<int64_t>(*mt, "tree_mask", dev, {qh.rows}) : nullptr;
    const at::Tensor out = result(a[10], q, dev);
    if (qh.rows && B) {
        NEED(qh.rows <= INT32_MAX && qh.heads <= INT32_MAX && B <= INT32_MAX && width <= INT32_MAX && kc.size(0) <= INT32_MAX, "attn_tree: sizes beyond 2^31");
        const size_t need = valle_attn_tree_workspace_bytes(qh.rows, B, nodes, ctx_hint, qh.heads, hkv, dt);
        at::Tensor ws;                                       // of this call: two streams or graphs never share it
        if (need) ws = fresh({static_cast<int64_t>(need)}, at::kByte, dev);
        launch(dev, [&](void* s) {
            return valle_attn_tree(qh.p, qh.stride, kc.data_ptr(), vc.data_ptr(), kc.size(0), page, tp, width, ctx, cu, mask, out.data_ptr(), out.stride(0), qh.rows, B,
                                   nodes, ctx_hint, qh.heads, hkv, HEAD, static_cast<float>(scale), dt, need ? ws.data_ptr() : nullptr, need, s);
        });
    }
    if (a[10] != Py_None) { Py_INCREF(a[10]); return a[10]; }
    return THPVariable_Wrap(out);
    CATCH
}

// (k_cache, v_cache, block_table, ctx_len, path, n_accept, n_blocks | None, status | None) -> new lengths
PyObject* kv_commit(PyObject*, PyObject* const* a, Py_ssize_t nargs) {
    TRY
    ARGS(8);
    const at::Tensor &kc = tensor(a[0], "k_cache"), &vc = tensor(a[1], "v_cache"), &tab = tensor(a[2], "block_table"), &path = tensor(a[4], "path");
    const int dev = gpu_of(kc, "kv_commit"), dt = dtype_of(kc);
    pools(kc, vc, dev, kc.scalar_type(), true);
    NEED(tab.dim() == 2 && path.dim() == 2 && path.size(1) > 0 && path.size(1) <= 64, "block_table (requests, max_blocks) and path (requests, 1 .. 64) needed, got ",
         tab.sizes(), ", ", path.sizes());
    const int64_t B = tab.size(0), width = tab.size(1), wide = path.size(1);
    const int32_t *tp = ints(tab, "block_table", dev, {B, width}), *ctx = ints(tensor(a[3], "ctx_len"), "ctx_len", dev, {B});
    const int32_t *pp = ints(path, "path", dev, {B, wide}), *acc = ints(tensor(a[5], "n_accept"), "n_accept", dev, {B});
    const at::Tensor *nb = maybe(a[6], "n_blocks"), *st = maybe(a[7], "status");
    const int32_t *nbp = nb ? ints(*nb, "n_blocks", dev, {B}) : nullptr, *sp = st ? ints(*st, "status", dev, {B}) : nullptr;
    const at::Tensor out = fresh({B}, at::kInt, dev);
    if (B) {
        NEED(B <= INT32_MAX && width <= INT32_MAX && kc.size(0) <= INT32_MAX && kc.size(1) <= INT32_MAX, "kv_commit: sizes beyond 2^31");
        launch(dev, [&](void* s) {
            return valle_paged_kv_commit_served(kc.data_ptr(), vc.data_ptr(), kc.size(0), kc.stride(0), tp, width, kc.size(1), kc.size(3), ctx, nbp, sp, pp, wide, acc,
                                                static_cast<int32_t*>(out.data_ptr()), B, kc.size(2), HEAD, dt, s);
        });
    }
    return THPVariable_Wrap(out);
    CATCH
}

// (x, wq, scales, zeros | None, bias | None, resid | None, geglu, in, out, group) -> y
PyObject* linear_w4(PyObject*, PyObject* const* a, Py_ssize_t nargs) {
    TRY
    ARGS(10);
    const at::Tensor &x = tensor(a[0], "x"), &wq = tensor(a[1], "wq"), &sc = tensor(a[2], "scales");
    const at::Tensor *z = maybe(a[3], "zeros"), *bias = maybe(a[4], "bias"), *resid = maybe(a[5], "resid");
    const int dev = gpu_of(x, "HipLinear4"), dt = dtype_of(sc);
    TORCH_CHECK_TYPE(x.scalar_type() == sc.scalar_type() && on(sc, dev), "HipLinear4: input ", shape_of(x), ", scales ", shape_of(sc));
    const int geglu = PyObject_IsTrue(a[6]);
    const int64_t K = whole(a[7], "in"), N = whole(a[8], "out"), group = whole(a[9], "group");
    NEED(x.dim() > 0 && x.size(-1) == K, "HipLinear4: input ", x.sizes(), ", width ", K, " needed");
    NEED(!geglu || (!resid && !bias && N % 2 == 0), "HipLinear4: geglu takes an even number of columns, no bias and no residual");
    const int64_t tiles = (N + 15) / 16, kb = (K + 127) / 128, groups = group > 0 ? kb * (128 / group) : 0;
    NEED(on(wq, dev) && wq.scalar_type() == at::kByte && wq.numel() == tiles * kb * 1024 && wq.is_contiguous() && sc.numel() == tiles * groups * 16 && sc.is_contiguous() &&
         (!z || (on(*z, dev) && z->scalar_type() == at::kByte && z->numel() == sc.numel() && z->is_contiguous())) &&
         (!bias || (on(*bias, dev) && bias->scalar_type() == sc.scalar_type() && bias->numel() == N && bias->is_contiguous())), "HipLinear4: packed weights do not fit the layer");
    at::Tensor x2 = x;                                       // [rows][K], rows 16-byte aligned
    if (x.dim() != 2) x2 = x.reshape({-1, K});
    if (x2.stride(1) != 1 || x2.stride(0) % 8 || x2.stride(0) < 0 || x2.stride(0) > (1 << 23) || reinterpret_cast<uintptr_t>(x2.data_ptr()) % 16)
        x2 = x2.clone(at::MemoryFormat::Contiguous);
    auto shape = x.sizes().vec();
    const int64_t cols = geglu ? N / 2 : N, rows = x2.size(0);
    shape.back() = cols;
    const at::Tensor y = fresh(shape, x.scalar_type(), dev);
    at::Tensor r;
    if (resid) {
        NEED(resid->sizes() == y.sizes() && resid->scalar_type() == x.scalar_type() && on(*resid, dev), "HipLinear4: residual ", shape_of(*resid), " for ", shape_of(y));
        r = resid->contiguous();
    }
    if (rows) {
        NEED(rows <= INT32_MAX, "HipLinear4: ", rows, " rows");
        launch(dev, [&](void* s) {
            return valle_linear_w4(x2.data_ptr(), x2.stride(0), wq.data_ptr(), sc.data_ptr(), z ? static_cast<const uint8_t*>(z->data_ptr()) : nullptr,
                                   bias ? bias->data_ptr() : nullptr, resid ? r.data_ptr() : nullptr, y.data_ptr(), rows, N, K, group, cols,
                                   geglu ? VALLE_EPI_GEGLU : resid ? VALLE_EPI_RESID : VALLE_EPI_STORE, dt, s);
        });
    }
    return THPVariable_Wrap(y);
    CATCH
}

PyObject* set_error(PyObject*, PyObject* type) {
    Py_INCREF(type);
    g_error = type;
    Py_RETURN_NONE;
}

#define FAST(f) {#f, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(f)), METH_FASTCALL, nullptr}
PyMethodDef methods[] = {FAST(page_plan), FAST(rope_kv_paged), FAST(attn_tree), FAST(kv_commit), FAST(linear_w4), {"set_error", set_error, METH_O, nullptr}, {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_serving", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__serving(void) { return PyModule_Create(&module); }
