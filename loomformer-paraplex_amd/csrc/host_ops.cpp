// Host side of the paged cache's and the beam search's operators (module
// loom_amd._host): the argument checks, the outputs and workspaces, and the call
// of the C entry point, for the calls that a decode loop makes once per token
// and whose launches are a few microseconds long.  The functions take
// positional arguments; loom_amd/ops.py documents them and gives the defaults.
#include <Python.h>

#include <ATen/core/Tensor.h>
#include <ATen/ops/empty.h>
#include <c10/hip/HIPStream.h>
#include <hip/hip_runtime_api.h>
#include <torch/csrc/autograd/python_variable.h>

#include <algorithm>
#include <sstream>
#include <stdexcept>
#include <string>
#include <vector>

#include "../../include/loom_hip.h"

namespace {

template <typename... A>
[[noreturn]] void fail(const A&... a) {
    std::ostringstream s;
    (s << ... << a);
    throw std::runtime_error(s.str());
}
#define CHECK(cond, ...)             \
    do {                             \
        if (!(cond)) fail(__VA_ARGS__); \
    } while (0)

struct PyError {};                   // a Python error is already set

// ------------------------------------------------------------------ arguments

struct Args {
    const char* name;
    PyObject* const* a;
    Py_ssize_t n;
    Args(const char* name_, PyObject* const* a_, Py_ssize_t n_, Py_ssize_t want) : name(name_), a(a_), n(n_) {
        CHECK(n == want, name, ": ", want, " arguments, got ", n);
    }
    const at::Tensor& tensor(int i, const char* what) const {
        CHECK(THPVariable_Check(a[i]), name, ": ", what, " must be a tensor");
        const at::Tensor& t = THPVariable_Unpack(a[i]);
        CHECK(t.is_cuda(), name, ": all inputs must be CUDA tensors (", what, " is not)");
        return t;
    }
    bool none(int i) const { return a[i] == Py_None; }
    bool truth(int i) const {
        const int v = PyObject_IsTrue(a[i]);
        if (v < 0) throw PyError{};
        return v != 0;
    }
    int64_t integer(int i) const {
        const long long v = PyLong_AsLongLong(a[i]);
        if (v == -1 && PyErr_Occurred()) throw PyError{};
        return v;
    }
};

int dtype_code(const at::Tensor& t) {
    switch (t.scalar_type()) {
        case at::kFloat: return LOOM_F32;
        case at::kBFloat16: return LOOM_BF16;
        case at::kHalf: return LOOM_F16;
        default: return -1;
    }
}

// The tensors' device made current for the launches and workspace queries
struct OnDevice {
    int before = -1;
    explicit OnDevice(int dev) {
        int now = 0;
        CHECK(hipGetDevice(&now) == hipSuccess, "no current HIP device");
        if (now != dev) {
            CHECK(hipSetDevice(dev) == hipSuccess, "device ", dev, " cannot be made current");
            before = now;
        }
    }
    ~OnDevice() {
        if (before >= 0) (void)hipSetDevice(before);
    }
};

void* stream_of(int dev) { return (void*)c10::hip::getCurrentHIPStream((c10::DeviceIndex)dev).stream(); }

template <typename F>
void launch(F f) {
    int rc;
    Py_BEGIN_ALLOW_THREADS
    rc = f();
    Py_END_ALLOW_THREADS
    if (rc != LOOM_OK) throw std::runtime_error(loom_last_error());
}

const at::Tensor& i32(const Args& a, int i, const char* what, int64_t n, c10::Device dev) {
    const at::Tensor& t = a.tensor(i, what);
    CHECK(t.device() == dev && t.scalar_type() == at::kInt && t.dim() == 1 && t.size(0) == n && t.is_contiguous(),
          a.name, ": ", what, " must be a contiguous int32 tensor of ", n, " elements on ", dev);
    return t;
}

struct Table {
    int32_t* p;
    int64_t rows, ld, pages;
};

Table table_of(const Args& a, int i, c10::Device dev) {
    const at::Tensor& t = a.tensor(i, "table");
    CHECK(t.device() == dev && t.scalar_type() == at::kInt && t.dim() == 2 && (t.size(1) == 1 || t.stride(1) == 1),
          a.name, ": table must be an int32 [rows, max_pages] tensor of dense rows on ", dev);
    const int64_t w = t.size(1);
    return {(int32_t*)t.data_ptr(), t.size(0), t.size(0) > 1 ? t.stride(0) : std::max(w, t.stride(0)), w};
}

// The stride of a dimension of one entry says nothing: it is not compared, and
// `one` stands for it.
int64_t stride_of(const at::Tensor& t, int64_t d, int64_t one = 0) { return t.size(d) > 1 ? t.stride(d) : one; }

bool same_layout(const at::Tensor& a, const at::Tensor& b) {
    if (a.sizes() != b.sizes()) return false;
    for (int64_t d = 0; d < a.dim(); ++d)
        if (stride_of(a, d) != stride_of(b, d)) return false;
    return true;
}

// layer (0 without one), page, token and head strides
struct Pools {
    const at::Tensor &k, &v;
    int dtype;
    c10::Device dev;
    int64_t layer, page, tok, head;
};

Pools pools_of(const Args& a, int i, int64_t dim) {
    const at::Tensor &k = a.tensor(i, "k_pages"), &v = a.tensor(i + 1, "v_pages");
    CHECK(k.dim() == dim && v.dim() == dim && same_layout(k, v) && stride_of(k, dim - 1, 1) == 1, a.name,
          ": k_pages and v_pages must be [", dim == 5 ? "layers, " : "",
          "pages, kv_heads, page_size, head_dim] tensors of the same layout with dense heads");
    const int code = dtype_code(k);
    CHECK(code >= 0 && v.scalar_type() == k.scalar_type() && v.device() == k.device(), a.name,
          ": k_pages and v_pages must be float32, bfloat16 or float16 and have one dtype and one device");
    return {k, v, code, k.device(), dim == 5 ? stride_of(k, 0) : 0, stride_of(k, dim - 4), stride_of(k, dim - 2, k.size(dim - 1)),
            stride_of(k, dim - 3)};
}

at::Tensor bytes(int64_t n, c10::Device dev) {
    return at::empty({n}, at::TensorOptions().dtype(at::kByte).device(dev));
}

PyObject* list_of(std::initializer_list<const at::Tensor*> ts) {
    PyObject* l = PyList_New((Py_ssize_t)ts.size());
    if (l == nullptr) throw PyError{};
    Py_ssize_t i = 0;
    for (const at::Tensor* t : ts) {
        PyObject* o;
        if (t == nullptr || !t->defined()) {
            Py_INCREF(Py_None);
            o = Py_None;
        } else {
            o = THPVariable_Wrap(*t);
        }
        if (o == nullptr) {
            Py_DECREF(l);
            throw PyError{};
        }
        PyList_SET_ITEM(l, i++, o);
    }
    return l;
}

// ------------------------------------------------------------------ attention

PyObject* attention(const Args& a, bool step) {
    const Pools p = pools_of(a, 1, 4);
    const int64_t NP = p.k.size(0), KVH = p.k.size(1), PS = p.k.size(2), HD = p.k.size(3);
    const char* qname = step ? "qkv" : "q";
    at::Tensor q = a.tensor(0, qname);
    CHECK(q.device() == p.dev && q.scalar_type() == p.k.scalar_type(), a.name, ": ", qname,
          " must have the pools' dtype and device");
    int64_t QH;
    const at::Tensor *cos = nullptr, *sin = nullptr;
    if (step) {
        CHECK(q.dim() == 2 && HD > 0 && q.size(1) % HD == 0 && q.size(1) / HD > 2 * KVH, a.name,
              ": qkv must be [rows, (q_heads + 2 kv_heads) * head_dim]");
        QH = q.size(1) / HD - 2 * KVH;
        cos = &a.tensor(5, "cos");
        sin = &a.tensor(6, "sin");
        for (const at::Tensor* t : {cos, sin})
            CHECK(t->device() == p.dev && t->scalar_type() == at::kFloat && t->dim() == 2 && t->size(1) == HD &&
                      t->size(0) == cos->size(0) && t->is_contiguous(),
                  a.name, ": cos and sin must be contiguous float32 [positions, head_dim] tables");
    } else {
        CHECK(q.dim() == 3 && q.size(2) == HD, a.name, ": q must be [rows, q_heads, head_dim]");
        QH = q.size(1);
    }
    CHECK(KVH > 0 && QH > 0 && QH % KVH == 0, a.name, ": ", QH, " query heads over ", KVH, " kv heads");
    const Table t = table_of(a, 3, p.dev);
    const int64_t B = t.rows;
    CHECK(q.size(0) == B, a.name, ": ", q.size(0), " rows of ", qname, " for ", B, " rows of the table");
    const at::Tensor& lens = i32(a, 4, "lens", B, p.dev);
    const bool kctx = a.truth(step ? 7 : 5);

    // rows the kernels can load: dense and 16-byte aligned
    const int64_t width = q.size(1) * (step ? 1 : HD);
    const bool dense = step ? q.stride(1) == 1 : (q.stride(2) == 1 && (QH == 1 || q.stride(1) == HD));
    int64_t ld = B > 1 ? q.stride(0) : width;
    if (!dense || ld < width || (ld * q.element_size()) % 16 != 0 || (uintptr_t)q.data_ptr() % 16 != 0) {
        q = q.clone(at::MemoryFormat::Contiguous);
        ld = width;
    }
    OnDevice on(p.dev.index());
    const auto opt = p.k.options();
    at::Tensor c = at::empty({B, QH, HD}, opt), kx, qo;
    if (kctx) kx = at::empty({B, QH, HD}, opt);
    if (step) qo = at::empty({B, QH, HD}, opt);
    if (B == 0) return step ? list_of({&c, &kx, &qo}) : list_of({&c, &kx});
    const int64_t need = loom_paged_decode_workspace_bytes(B, t.pages * PS, QH, KVH, HD);
    at::Tensor ws;
    if (need > 0) ws = bytes(need, p.dev);
    float* w = need > 0 ? (float*)ws.data_ptr() : nullptr;
    void* st = stream_of(p.dev.index());
    void* kxp = kctx ? kx.data_ptr() : nullptr;
    const int32_t* lp = (const int32_t*)lens.data_ptr();
    launch([&] {
        if (step)
            return loom_paged_decode_step(p.dtype, q.data_ptr(), ld, p.k.data_ptr(), p.v.data_ptr(), p.page, p.tok,
                                          p.head, NP, PS, t.p, t.ld, t.pages, lp,
                                          (const float*)cos->data_ptr(), (const float*)sin->data_ptr(), cos->size(0),
                                          qo.data_ptr(), c.data_ptr(), kxp, QH * HD, w, need, B, QH, KVH, HD, st);
        return loom_paged_decode_attention(p.dtype, q.data_ptr(), ld, p.k.data_ptr(), p.v.data_ptr(), p.page, p.tok,
                                           p.head, NP, PS, t.p, t.ld, t.pages, lp, c.data_ptr(),
                                           kxp, QH * HD, w, need, B, QH, KVH, HD, st);
    });
    return step ? list_of({&c, &kx, &qo}) : list_of({&c, &kx});
}

// (qkv, k_pages, v_pages, table, lens, cos, sin, want_kctx)
PyObject* paged_decode_step(PyObject* const* x, Py_ssize_t n) {
    return attention(Args("paged_decode_step", x, n, 8), true);
}

// (q, k_pages, v_pages, table, lens, want_kctx)
PyObject* paged_decode_attention(PyObject* const* x, Py_ssize_t n) {
    return attention(Args("paged_decode_attention", x, n, 6), false);
}

// ------------------------------------------------------------------ pages

// (k_pages, v_pages, table, lens, refs, status, parent or None, n_new, advance)
PyObject* paged_update(PyObject* const* x, Py_ssize_t n) {
    const Args a("paged_update", x, n, 9);
    const Pools p = pools_of(a, 0, 5);
    const Table t = table_of(a, 2, p.dev);
    const at::Tensor &lens = i32(a, 3, "lens", t.rows, p.dev), &refs = i32(a, 4, "refs", p.k.size(1), p.dev),
                     &status = i32(a, 5, "status", 1, p.dev);
    const int32_t* parent = a.none(6) ? nullptr : (const int32_t*)i32(a, 6, "parent", t.rows, p.dev).data_ptr();
    const int64_t n_new = a.integer(7), advance = a.integer(8);
    if (t.rows == 0) Py_RETURN_NONE;
    OnDevice on(p.dev.index());
    const int64_t need = loom_paged_update_workspace_bytes(t.rows);
    const at::Tensor ws = bytes(need, p.dev);
    void* st = stream_of(p.dev.index());
    launch([&] {
        return loom_paged_update(p.dtype, p.k.data_ptr(), p.v.data_ptr(), p.k.size(0), p.layer, p.page, p.tok, p.head,
                                 p.k.size(1), p.k.size(3), p.k.size(2), p.k.size(4), t.p,
                                 t.ld, t.pages, (int32_t*)lens.data_ptr(), (int32_t*)refs.data_ptr(),
                                 (int32_t*)status.data_ptr(), parent, n_new, advance, ws.data_ptr(), need, t.rows, st);
    });
    Py_RETURN_NONE;
}

// (k_pages, v_pages, table, k_rows, v_rows, first, last)
PyObject* paged_write(PyObject* const* x, Py_ssize_t n) {
    const Args a("paged_write", x, n, 7);
    const Pools p = pools_of(a, 0, 5);
    const Table t = table_of(a, 2, p.dev);
    const at::Tensor &kr = a.tensor(3, "k_rows"), &vr = a.tensor(4, "v_rows");
    CHECK(kr.device() == p.dev && vr.device() == p.dev && kr.scalar_type() == p.k.scalar_type() &&
              vr.scalar_type() == p.k.scalar_type() && kr.dim() == 5 && vr.dim() == 5 && same_layout(kr, vr) &&
              kr.size(0) == p.k.size(0) && kr.size(1) == t.rows &&
              kr.size(2) == p.k.size(2) && kr.size(4) == p.k.size(4) && stride_of(kr, 4, 1) == 1,
          a.name, ": k_rows and v_rows must be [layers, rows, kv_heads, positions, head_dim] tensors of the pools' "
                  "dtype and one layout");
    const at::Tensor &first = i32(a, 5, "first", t.rows, p.dev), &last = i32(a, 6, "last", t.rows, p.dev);
    if (kr.numel() == 0) Py_RETURN_NONE;
    OnDevice on(p.dev.index());
    void* st = stream_of(p.dev.index());
    launch([&] {
        return loom_paged_write(p.dtype, p.k.data_ptr(), p.v.data_ptr(), p.k.size(0), p.layer, p.page, p.tok, p.head,
                                p.k.size(1), p.k.size(3), p.k.size(2), p.k.size(4), t.p,
                                t.ld, t.pages, kr.data_ptr(), vr.data_ptr(), stride_of(kr, 0), stride_of(kr, 1),
                                stride_of(kr, 2), stride_of(kr, 3, kr.size(4)), kr.size(3), (const int32_t*)first.data_ptr(),
                                (const int32_t*)last.data_ptr(), t.rows, st);
    });
    Py_RETURN_NONE;
}

// (k_pages, v_pages, table, refs, used)
PyObject* paged_compact(PyObject* const* x, Py_ssize_t n) {
    const Args a("paged_compact", x, n, 5);
    const Pools p = pools_of(a, 0, 5);
    const Table t = table_of(a, 2, p.dev);
    const at::Tensor &refs = i32(a, 3, "refs", p.k.size(1), p.dev), &used = i32(a, 4, "used", 1, p.dev);
    OnDevice on(p.dev.index());
    const int64_t need = loom_paged_compact_workspace_bytes(p.k.size(1));
    const at::Tensor ws = bytes(need, p.dev);
    void* st = stream_of(p.dev.index());
    launch([&] {
        return loom_paged_compact(p.dtype, p.k.data_ptr(), p.v.data_ptr(), p.k.size(0), p.layer, p.page, p.tok, p.head,
                                  p.k.size(1), p.k.size(3), p.k.size(2), p.k.size(4), t.p,
                                  t.ld, t.pages, (int32_t*)refs.data_ptr(), (int32_t*)used.data_ptr(), ws.data_ptr(),
                                  need, t.rows, st);
    });
    Py_RETURN_NONE;
}

// ------------------------------------------------------------------ beam search

// (logits, scores, n_out or None, finished or None, eos_id, pad_id)
PyObject* beam_select(PyObject* const* x, Py_ssize_t n) {
    const Args a("beam_select", x, n, 6);
    const at::Tensor& logits = a.tensor(0, "logits");
    const at::Tensor& scores = a.tensor(1, "scores");
    const c10::Device dev = logits.device();
    const int code = dtype_code(logits);
    CHECK(logits.dim() == 2 && code >= 0, a.name, ": logits must be a float32, bfloat16 or float16 [rows, V] tensor");
    CHECK(scores.device() == dev && scores.scalar_type() == at::kFloat && scores.dim() == 2 &&
              scores.numel() == logits.size(0),
          a.name, ": scores must be a float32 [groups, beams] tensor, a value for each row of logits");
    const int64_t S = scores.size(0), W = scores.size(1), V = logits.size(1);
    const int64_t K = a.none(2) ? W : a.integer(2);
    CHECK(K >= 1 && K <= 64 && S >= 1, a.name, ": n_out must be 1 to 64, got ", K, ", and there must be a group");
    const int64_t eos = a.integer(4), pad = a.integer(5);
    at::Tensor lg = logits;
    int64_t ld = S * W > 1 ? lg.stride(0) : V;
    if ((V > 1 && lg.stride(1) != 1) || ld < V) {
        lg = lg.clone(at::MemoryFormat::Contiguous);
        ld = V;
    }
    const at::Tensor sc = scores.contiguous();
    at::Tensor fin;
    if (!a.none(3)) {
        fin = a.tensor(3, "finished");
        CHECK(fin.device() == dev && fin.scalar_type() == at::kBool && fin.numel() == S * W, a.name,
              ": finished must be a bool tensor with a value for each row of logits");
        fin = fin.contiguous();
    }
    OnDevice on(dev.index());
    const auto opt = at::TensorOptions().device(dev);
    const at::Tensor os = at::empty({S, K}, opt.dtype(at::kFloat)), op = at::empty({S, K}, opt.dtype(at::kInt)),
                     ot = at::empty({S, K}, opt.dtype(at::kLong)), of = at::empty({S, K}, opt.dtype(at::kBool));
    const int64_t need = loom_beam_select_workspace_bytes(S, W, V, K);
    at::Tensor ws;
    if (need > 0) ws = bytes(need, dev);
    void* st = stream_of(dev.index());
    launch([&] {
        return loom_beam_select(code, lg.data_ptr(), ld, (const float*)sc.data_ptr(),
                                fin.defined() ? (const uint8_t*)fin.data_ptr() : nullptr, (float*)os.data_ptr(),
                                (int32_t*)op.data_ptr(), (int64_t*)ot.data_ptr(), (uint8_t*)of.data_ptr(), S, W, V, K,
                                eos, pad, need > 0 ? ws.data_ptr() : nullptr, need, st);
    });
    return list_of({&os, &op, &ot, &of});
}

// (tensors, parent, dims or None)
PyObject* reorder_rows(PyObject* const* x, Py_ssize_t n) {
    const Args a("reorder_rows", x, n, 3);
    const at::Tensor& parent = a.tensor(1, "parent");
    CHECK(parent.scalar_type() == at::kInt && parent.dim() == 1 && parent.is_contiguous(), a.name,
          ": parent must be a contiguous CUDA int32 tensor");
    const c10::Device dev = parent.device();
    const int64_t R = parent.size(0);
    struct Seq {
        PyObject* o = nullptr;
        ~Seq() { Py_XDECREF(o); }
    } ts, ds;
    ts.o = PySequence_Fast(x[0], "reorder_rows: tensors must be a sequence");
    if (ts.o == nullptr) throw PyError{};
    const Py_ssize_t count = PySequence_Fast_GET_SIZE(ts.o);
    if (!a.none(2)) {
        ds.o = PySequence_Fast(x[2], "reorder_rows: dims must be a sequence");
        if (ds.o == nullptr) throw PyError{};
        CHECK(PySequence_Fast_GET_SIZE(ds.o) == count, a.name, ": one dimension per tensor");
    }
    constexpr int kMax = 16;
    OnDevice on(dev.index());
    void* st = stream_of(dev.index());
    struct Seg {
        void* p;
        int64_t outer, step, row, inner;
    };
    std::vector<Seg> segs;
    segs.reserve((size_t)count);
    for (Py_ssize_t i = 0; i < count; ++i) {
        PyObject* to = PySequence_Fast_GET_ITEM(ts.o, i);
        CHECK(THPVariable_Check(to), a.name, ": tensors must hold tensors");
        const at::Tensor& t = THPVariable_Unpack(to);
        int64_t d = 0;
        if (ds.o != nullptr) {
            d = PyLong_AsLongLong(PySequence_Fast_GET_ITEM(ds.o, i));
            if (d == -1 && PyErr_Occurred()) throw PyError{};
        }
        CHECK(t.is_cuda() && t.device() == dev && d >= 0 && d < t.dim() && t.size(d) == R, a.name,
              ": every tensor must be on ", dev, " and have ", R, " rows in its row dimension");
        if (t.numel() == 0) continue;
        const int64_t es = (int64_t)t.element_size();
        int64_t inner = 1;
        for (int64_t k = t.dim() - 1; k > d; --k) {
            CHECK(t.size(k) == 1 || t.stride(k) == inner, a.name, ": the rows of a tensor must be dense");
            inner *= t.size(k);
        }
        int64_t outer = 1, step = 0;
        for (int64_t k = d - 1; k >= 0; --k) {
            if (t.size(k) == 1) continue;
            CHECK(outer == 1 || t.stride(k) == step * outer, a.name,
                  ": the dimensions before the row dimension must be one run of equal steps");
            if (outer == 1) step = t.stride(k);
            outer *= t.size(k);
        }
        const int64_t row = R > 1 ? t.stride(d) : inner;
        CHECK(row >= inner && (outer == 1 || step >= row * (R - 1) + inner ||
                               (row >= step * (outer - 1) + inner && step >= inner)),
              a.name, ": the rows of a tensor must not overlap");
        char* lo = (char*)t.data_ptr();
        char* hi = lo + (step * (outer - 1) + row * (R - 1) + inner) * es;
        const char* p = (const char*)parent.data_ptr();
        CHECK(hi <= p || lo >= p + 4 * R, a.name, ": parent must not lie in one of the tensors");
        for (const Seg& s : segs) CHECK(s.p != lo, a.name, ": a tensor is there twice");
        segs.push_back({lo, outer, step * es, row * es, inner * es});
    }
    for (size_t i = 0; i < segs.size(); i += kMax) {
        const int m = (int)std::min<size_t>(kMax, segs.size() - i);
        void* p[kMax];
        int64_t outer[kMax], step[kMax], row[kMax], inner[kMax];
        for (int j = 0; j < m; ++j) {
            const Seg& s = segs[i + j];
            p[j] = s.p;
            outer[j] = s.outer;
            step[j] = s.step;
            row[j] = s.row;
            inner[j] = s.inner;
        }
        launch([&] { return loom_reorder_rows(m, p, outer, step, row, inner, (const int32_t*)parent.data_ptr(), R, st); });
    }
    Py_RETURN_NONE;
}

// ------------------------------------------------------------------ the module

// No C++ exception leaves a function: each becomes a RuntimeError.
template <PyObject* (*F)(PyObject* const*, Py_ssize_t)>
PyObject* guarded(PyObject*, PyObject* const* x, Py_ssize_t n) {
    try {
        return F(x, n);
    } catch (const PyError&) {
        return nullptr;
    } catch (const c10::Error& e) {
        PyErr_SetString(PyExc_RuntimeError, e.what_without_backtrace());
    } catch (const std::exception& e) {
        PyErr_SetString(PyExc_RuntimeError, e.what());
    } catch (...) {
        PyErr_SetString(PyExc_RuntimeError, "loom_amd._host: unknown C++ exception");
    }
    return nullptr;
}

#define ENTRY(f) {#f, (PyCFunction)(void (*)(void))guarded<f>, METH_FASTCALL, nullptr}
PyMethodDef methods[] = {ENTRY(paged_decode_step), ENTRY(paged_decode_attention), ENTRY(paged_update),
                         ENTRY(paged_write),       ENTRY(paged_compact),          ENTRY(beam_select),
                         ENTRY(reorder_rows),      {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_host", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__host(void) { return PyModule_Create(&module); }
