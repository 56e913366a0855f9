// qdc_calls.cpp -- the host side of the cache's operators and of those on 4-bit weights: the
// checks of their tensors and the call of the entry point (include/qdc_hip_cache.h,
// include/qdc_hip_quant.h), as functions of a Python module.
//
// A step is many small calls, and their host side is what they cost.  The host's time for a
// call, its launch of 2.6 us and the output's allocation within it, with some fifteen tensors
// to look at and up to 46 arguments to convert, in Python / here: a token stored 12.1 / 4.9
// us, one attended to in one launch 10.8 / 4.6, its step of the recurrence 9.9 / 4.8.
// The functions take exactly the arguments that qdc_amd.cache_ops and qdc_amd.quant_ops pass
// them, by position; those document what they do and refuse.
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/utils/python_numbers.h>

#include <ATen/hip/EmptyTensor.h>
#include <ATen/ops/empty.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>

#include "qdc_hip_cache.h"
#include "qdc_hip_quant.h"

namespace {

typedef PyObject *const *Args;

PyObject *failed;  // called with (status, name) for a status that is not QDC_OK

const at::Tensor &tensor(PyObject *o, const char *name) {
    TORCH_CHECK_TYPE(THPVariable_Check(o), name, " must be a tensor");
    return THPVariable_Unpack(o);
}
int64_t integer(PyObject *o) { return THPUtils_unpackLong(o); }
float real(PyObject *o) {
    const double v = PyFloat_AsDouble(o);
    if (v == -1.0 && PyErr_Occurred()) throw python_error();
    return (float)v;
}
bool truth(PyObject *o) {
    const int v = PyObject_IsTrue(o);
    if (v < 0) throw python_error();
    return v == 1;
}
template <typename T> T *data(const at::Tensor &t) { return static_cast<T *>(t.data_ptr()); }

// What a call's tensors have in common: the device of the first one.
struct Call {
    c10::Device device;

    explicit Call(const at::Tensor &t) : device(t.device()) {
        TORCH_CHECK_VALUE(t.is_cuda(), "device tensors required (torch.device('cuda'))");
    }
    bool here(const at::Tensor &t) const { return t.device() == device; }
    // contiguous, of this type and device
    bool plain(const at::Tensor &t, at::ScalarType type) const {
        return t.scalar_type() == type && here(t) && t.is_contiguous();
    }

    // A contiguous int32 vector of n entries (-1: any number).
    int32_t *ints(PyObject *o, const char *name, int64_t n) const {
        const at::Tensor &t = tensor(o, name);
        const bool good = t.dim() == 1 && (n < 0 || t.size(0) == n) && plain(t, at::kInt);
        if (n < 0)
            TORCH_CHECK_VALUE(good, name,
                              " must be a contiguous int32 vector on the call's device");
        TORCH_CHECK_VALUE(good, name, " must be a contiguous int32 vector of ", n,
                          " entries on the call's device");
        return data<int32_t>(t);
    }
    int32_t *flag(PyObject *o) const {
        if (o == Py_None) return nullptr;
        const at::Tensor &t = tensor(o, "error_flag");
        TORCH_CHECK_VALUE(here(t) && t.scalar_type() == at::kInt && t.numel() >= 1,
                          "error_flag must be an int32 tensor on the call's device");
        return data<int32_t>(t);
    }
    const at::Tensor &table(PyObject *o) const {
        const at::Tensor &t = tensor(o, "table");
        TORCH_CHECK_VALUE(t.dim() == 2 && plain(t, at::kInt),
                          "table must be a contiguous int32 [rows, width] tensor on the call's "
                          "device");
        return t;
    }

    // fn(stream), an entry point's call, on the device and its current stream.
    template <typename F> void run(const char *name, F fn) const {
        const c10::DeviceGuard guard(device);
        const hipStream_t stream = c10::hip::getCurrentHIPStream(device.index()).stream();
        int32_t status;
        Py_BEGIN_ALLOW_THREADS
        status = fn(stream);
        Py_END_ALLOW_THREADS
        if (status == QDC_OK) return;
        THPObjectPtr none(PyObject_CallFunction(failed, "is", status, name));
        if (!none) throw python_error();
    }
    at::Tensor bytes(int64_t n) const {
        return at::empty({n}, at::TensorOptions(device).dtype(at::kByte));
    }
};

int32_t dtype_code(const at::Tensor &t) {
    if (t.scalar_type() == at::kFloat) return QDC_F32;
    TORCH_CHECK_VALUE(t.scalar_type() == at::kBFloat16, "unsupported dtype ", t.scalar_type(),
                      "; expected float32 or bfloat16");
    return QDC_BF16;
}

// A [n, heads, head_dim] view with contiguous rows; the strides of axes of one entry may be
// anything.
struct Rows {
    const at::Tensor &t;
    int64_t n, heads, dim, tok, head;

    Rows(const Call &call, PyObject *o, at::ScalarType type, const char *name)
        : t(tensor(o, name)) {
        TORCH_CHECK_VALUE(t.dim() == 3 && t.stride(2) == 1 && t.scalar_type() == type &&
                              call.here(t),
                          name, " must be [tokens, heads, head_dim] with contiguous rows, of "
                          "q's dtype and device");
        n = t.size(0);
        heads = t.size(1);
        dim = t.size(2);
        tok = n > 1 ? t.stride(0) : heads * dim;
        head = heads > 1 ? t.stride(1) : dim;
    }
};

// A layer's page tensors.
struct Pages {
    const at::Tensor &k, &v;

    Pages(const Call &call, PyObject *ko, PyObject *vo, at::ScalarType type)
        : k(tensor(ko, "k_pages")), v(tensor(vo, "v_pages")) {
        TORCH_CHECK_VALUE(k.dim() == 4 && v.sizes() == k.sizes() && call.plain(k, type) &&
                              call.plain(v, type),
                          "k_pages and v_pages must be contiguous [pages, kv_heads, page_size, "
                          "head_dim] tensors of q's dtype and device");
    }
};

struct Book {
    const at::Tensor &table;
    Call call;
    int32_t *lengths, *refs, *free;
    int64_t rows, width, pages, size;

    Book(PyObject *t, PyObject *l, PyObject *r, PyObject *f, PyObject *page_size)
        : table(tensor(t, "table")), call(table) {
        call.table(t);
        rows = table.size(0);
        width = table.size(1);
        lengths = call.ints(l, "lengths", rows);
        refs = call.ints(r, "refs", -1);
        pages = THPVariable_Unpack(r).size(0);
        free = call.ints(f, "free", 1 + pages);
        size = integer(page_size);
    }
};

// A contiguous [planes, items, ...] tensor; none: no planes.
struct Pool {
    char *at = nullptr;
    int64_t planes = 0, bytes = 0;  // bytes of an item

    Pool(const Call &call, PyObject *o, int64_t items) {
        if (o == Py_None) return;
        const at::Tensor &t = tensor(o, "pool");
        TORCH_CHECK_VALUE(t.dim() >= 3 && (items < 0 || t.size(1) == items) && call.here(t) &&
                              t.is_contiguous(),
                          "pool must be a contiguous [planes, items, ...] tensor on the call's "
                          "device, with an item for each page");
        at = data<char>(t);
        planes = t.size(0);
        const int64_t all = planes * t.size(1);
        bytes = t.numel() / (all > 0 ? all : 1) * t.element_size();
    }
};

PyObject *prepare_paged(Args a) {
    const at::Tensor &q0 = tensor(a[0], "q");
    const Call call(q0);
    const int32_t code = dtype_code(q0);
    const at::ScalarType type = q0.scalar_type();
    const Rows q(call, a[0], type, "q"), k(call, a[1], type, "k"), v(call, a[2], type, "v");
    TORCH_CHECK_VALUE(v.t.sizes() == k.t.sizes() && k.n == q.n && k.dim == q.dim,
                      "q must be [T, H, hd] and k, v [T, KV, hd]");
    const at::Tensor &q_norm = tensor(a[3], "q_norm"), &k_norm = tensor(a[4], "k_norm");
    for (const at::Tensor *w : {&q_norm, &k_norm})
        TORCH_CHECK_VALUE(w->numel() == q.dim && call.plain(*w, type),
                          "q_norm and k_norm must be contiguous vectors of ", q.dim,
                          " elements, of q's dtype and device");
    const int64_t rotary = integer(a[7]);
    const float *cos = nullptr, *sin = nullptr;
    int64_t table_len = 0;
    if (rotary) {
        TORCH_CHECK_VALUE(a[5] != Py_None && a[6] != Py_None,
                          "rotation needs the (cos, sin) tables of rope_tables");
        const at::Tensor &c = tensor(a[5], "cos"), &s = tensor(a[6], "sin");
        TORCH_CHECK_VALUE(c.dim() == 2 && c.size(1) == rotary / 2 && s.sizes() == c.sizes() &&
                              call.plain(c, at::kFloat) && call.plain(s, at::kFloat),
                          "cos and sin must be contiguous float32 [n_pos, rotary_dim//2] tables "
                          "of one shape on the call's device");
        cos = data<const float>(c);
        sin = data<const float>(s);
        table_len = c.size(0);
    }
    const float eps = real(a[8]);
    const int32_t *rows = call.ints(a[9], "rows", q.n);
    const int32_t *positions = call.ints(a[10], "positions", q.n);
    const at::Tensor &table = call.table(a[11]);
    const Pages pages(call, a[12], a[13], type);
    TORCH_CHECK_VALUE(pages.k.size(1) == k.heads && pages.k.size(3) == q.dim,
                      "k_pages and v_pages must hold k's heads");
    at::Tensor q_out;
    if (a[14] == Py_None) {
        q_out = at::empty({q.n, q.heads, q.dim}, q0.options());
    } else {
        q_out = tensor(a[14], "q_out");
        TORCH_CHECK_VALUE(q_out.sizes() == q0.sizes() && call.plain(q_out, type),
                          "q_out must be a contiguous tensor of q's shape, dtype and device");
    }
    void *k_out = nullptr;
    if (a[15] != Py_None) {
        const at::Tensor &t = tensor(a[15], "k_out");
        TORCH_CHECK_VALUE(t.sizes() == k.t.sizes() && call.plain(t, type),
                          "k_out must be a contiguous tensor of k's shape, dtype and device");
        k_out = t.data_ptr();
    }
    int32_t *flag = call.flag(a[16]);
    call.run("prepare_paged", [&](hipStream_t stream) {
        return qdc_prepare_paged(
            q_out.data_ptr(), k_out, pages.k.data_ptr(), pages.v.data_ptr(), q0.data_ptr(),
            k.t.data_ptr(), v.t.data_ptr(), q_norm.data_ptr(), k_norm.data_ptr(), cos, sin, rows,
            positions, data<const int32_t>(table), q.n, q.heads, k.heads, q.dim, rotary, table_len,
            table.size(0), table.size(1), pages.k.size(0), pages.k.size(2), q.tok, q.head, k.tok,
            k.head, v.tok, v.head, eps, code, flag, stream);
    });
    return THPVariable_Wrap(q_out);
}

// a[8]: the output's dtype code, -1 for q's
PyObject *paged_attention(Args a) {
    const at::Tensor &q0 = tensor(a[0], "q");
    const Call call(q0);
    const int32_t code = dtype_code(q0);
    const at::ScalarType type = q0.scalar_type();
    const Rows q(call, a[0], type, "q");
    const Pages pages(call, a[1], a[2], type);
    const int64_t kv = pages.k.size(1), page = pages.k.size(2);
    TORCH_CHECK_VALUE(pages.k.size(3) == q.dim && kv > 0 && q.heads % kv == 0,
                      "q's heads must be a multiple of those of k_pages, of one head_dim");
    const at::Tensor &table = call.table(a[3]);
    const int32_t *rows = call.ints(a[4], "rows", q.n);
    const int32_t *positions = call.ints(a[5], "positions", q.n);
    const float scale = real(a[6]);
    const void *gate = nullptr;
    int64_t gate_tok = 0, gate_head = q.dim;
    if (a[7] != Py_None) {
        const Rows g(call, a[7], type, "gate");
        TORCH_CHECK_VALUE(g.t.sizes() == q0.sizes(), "gate must be a view like q");
        gate = g.t.data_ptr();
        gate_tok = g.tok;
        gate_head = g.head;
    }
    int32_t out_code = (int32_t)integer(a[8]);
    if (out_code < 0) out_code = code;
    const int64_t width = q.heads * q.dim;
    const at::Tensor out =
        at::empty({q.n, out_code == QDC_BF16X2 ? 2 * width : width},
                  q0.options().dtype(out_code == QDC_F32 ? at::kFloat : at::kBFloat16));
    const int64_t need = qdc_paged_attention_workspace(q.n, q.heads, kv, q.dim, table.size(1),
                                                       page, code);
    const at::Tensor work = need > 0 ? call.bytes(need) : at::Tensor();
    int32_t *flag = call.flag(a[9]);
    call.run("paged_attention", [&](hipStream_t stream) {
        return qdc_paged_attention(
            out.data_ptr(), out_code, q0.data_ptr(), pages.k.data_ptr(), pages.v.data_ptr(), gate,
            data<const int32_t>(table), rows, positions, q.n, q.heads, kv, q.dim, table.size(0),
            table.size(1), pages.k.size(0), page, q.tok, q.head, gate_tok, gate_head, width, scale,
            code, need > 0 ? work.data_ptr() : nullptr, need, flag, stream);
    });
    return THPVariable_Wrap(out);
}

PyObject *extend_pages(Args a) {
    const Book b(a[0], a[1], a[2], a[3], a[4]);
    const int32_t *rows = b.call.ints(a[5], "rows", -1);
    const int64_t n = THPVariable_Unpack(a[5]).size(0);
    const int32_t *counts = a[6] == Py_None ? nullptr : b.call.ints(a[6], "counts", n);
    const at::Tensor positions =
        a[7] == Py_None ? at::empty({n}, b.table.options()) : tensor(a[7], "positions");
    int32_t *at = a[7] == Py_None ? data<int32_t>(positions) : b.call.ints(a[7], "positions", n);
    int32_t *flag = b.call.flag(a[8]);
    b.call.run("extend_pages", [&](hipStream_t stream) {
        return qdc_pages_extend(at, data<int32_t>(b.table), b.lengths, b.refs, b.free, rows, counts,
                                n, b.rows, b.width, b.pages, b.size, flag, stream);
    });
    return THPVariable_Wrap(positions);
}

PyObject *free_pages(Args a) {
    const Book b(a[0], a[1], a[2], a[3], a[4]);
    const int32_t *rows = b.call.ints(a[5], "rows", -1);
    const int64_t n = THPVariable_Unpack(a[5]).size(0);
    int32_t *flag = b.call.flag(a[6]);
    b.call.run("free_pages", [&](hipStream_t stream) {
        return qdc_pages_free(data<int32_t>(b.table), b.lengths, b.refs, b.free, rows, n, b.rows,
                              b.width, b.pages, b.size, flag, stream);
    });
    Py_RETURN_NONE;
}

PyObject *fork_pages(Args a) {
    const Book b(a[0], a[1], a[2], a[3], a[4]);
    const int32_t *parents = b.call.ints(a[5], "parents", -1);
    const int64_t n = THPVariable_Unpack(a[5]).size(0);
    const int32_t *children = b.call.ints(a[6], "children", n);
    const Pool pool(b.call, a[7], b.pages);
    int64_t heads = 0, token = 0;
    if (a[7] != Py_None) {
        const at::Tensor &t = THPVariable_Unpack(a[7]);
        TORCH_CHECK_VALUE(t.dim() == 5 && t.size(3) == b.size,
                          "pool must be [planes, pages, kv_heads, page_size, head_dim]");
        heads = t.size(2);
        token = t.size(4) * t.element_size();
    }
    const int64_t need = qdc_pages_fork_workspace(n, b.size, pool.planes, heads, token);
    const at::Tensor work = need > 0 ? b.call.bytes(need) : at::Tensor();
    int32_t *flag = b.call.flag(a[8]);
    b.call.run("fork_pages", [&](hipStream_t stream) {
        return qdc_pages_fork(data<int32_t>(b.table), b.lengths, b.refs, b.free, parents, children,
                              n, b.rows, b.width, b.pages, b.size, pool.at, pool.planes, heads,
                              token, need > 0 ? work.data_ptr() : nullptr, need, flag, stream);
    });
    Py_RETURN_NONE;
}

PyObject *compact_pages(Args a) {
    const Book b(a[0], a[1], a[2], a[3], a[4]);
    const Pool pool(b.call, a[5], b.pages);
    const int64_t need = qdc_pages_compact_workspace(b.pages);
    const at::Tensor work = b.call.bytes(need);
    b.call.run("compact_pages", [&](hipStream_t stream) {
        return qdc_pages_compact(data<int32_t>(b.table), b.refs, b.free, b.rows, b.width, b.pages,
                                 pool.at, pool.planes, pool.bytes, work.data_ptr(), need, stream);
    });
    Py_RETURN_NONE;
}

PyObject *copy_pages(Args a) {
    const at::Tensor &t = tensor(a[0], "pool");
    const Call call(t);
    const Pool pool(call, a[0], -1);
    const int32_t *src = call.ints(a[1], "src", -1);
    const int64_t n = THPVariable_Unpack(a[1]).size(0);
    const int32_t *dst = call.ints(a[2], "dst", n);
    int32_t *flag = call.flag(a[3]);
    call.run("copy_pages", [&](hipStream_t stream) {
        return qdc_copy_pages(pool.at, src, dst, n, pool.planes, t.size(1), pool.bytes, flag,
                              stream);
    });
    Py_RETURN_NONE;
}

// a[14]: whether the output is split
PyObject *delta_step(Args a) {
    const at::Tensor &proj = tensor(a[0], "proj");
    const Call call(proj);
    const int32_t code = dtype_code(proj);
    const at::ScalarType type = proj.scalar_type();
    const int64_t key_heads = integer(a[10]), key_dim = integer(a[11]);
    const int64_t value_heads = integer(a[12]), value_dim = integer(a[13]);
    const int64_t vw = value_heads * value_dim, channels = 2 * key_heads * key_dim + vw;
    TORCH_CHECK_VALUE(proj.dim() == 2 && proj.size(1) >= channels + vw + 2 * value_heads &&
                          proj.stride(1) == 1,
                      "proj must be [n, width] with contiguous rows of the q|k|v|z|a|b blocks");
    const int64_t n = proj.size(0), ld = n > 1 ? proj.stride(0) : proj.size(1);
    const at::Tensor &conv = tensor(a[1], "conv");
    TORCH_CHECK_VALUE(conv.dim() == 2 && conv.size(0) == channels && call.plain(conv, at::kFloat),
                      "conv must be a contiguous float32 [", channels,
                      ", taps] tensor (the q|k|v channels) on proj's device");
    const int64_t taps = conv.size(1);
    const at::Tensor &a_decay = tensor(a[2], "a_decay"), &dt_bias = tensor(a[3], "dt_bias");
    for (const at::Tensor *t : {&a_decay, &dt_bias})
        TORCH_CHECK_VALUE(t->numel() == value_heads && call.plain(*t, at::kFloat),
                          "a_decay and dt_bias must be contiguous float32 vectors of ",
                          value_heads, " elements on proj's device");
    const at::Tensor &norm = tensor(a[4], "norm");
    TORCH_CHECK_VALUE(norm.numel() == value_dim && call.plain(norm, type),
                      "norm must be a contiguous vector of ", value_dim,
                      " elements of proj's dtype and device");
    const float eps = real(a[5]);
    const at::Tensor &ring = tensor(a[6], "ring"), &state = tensor(a[7], "state");
    TORCH_CHECK_VALUE(state.dim() == 4 && state.size(1) == value_heads &&
                          state.size(2) == value_dim && state.size(3) == key_dim &&
                          call.plain(state, at::kFloat),
                      "state must be a contiguous float32 [cache rows, value_heads, value_dim, "
                      "key_dim] tensor on proj's device");
    const int64_t cache_rows = state.size(0);
    TORCH_CHECK_VALUE(ring.dim() == 3 && ring.size(0) == cache_rows && ring.size(1) == taps &&
                          ring.size(2) == channels && call.plain(ring, type),
                      "ring must be a contiguous [cache rows, ", taps, ", ", channels,
                      "] tensor of proj's dtype and device");
    const int32_t *rows = call.ints(a[8], "rows", n);
    const int32_t *positions = call.ints(a[9], "positions", n);
    const bool split = a[14] == Py_True;
    const at::Tensor out = at::empty({n, split ? 2 * vw : vw}, proj.options());
    int32_t *flag = call.flag(a[15]);
    call.run("delta_step", [&](hipStream_t stream) {
        return qdc_delta_step(out.data_ptr(), split ? QDC_BF16X2 : code, proj.data_ptr(), code, ld,
                              data<const float>(conv), taps, data<const float>(a_decay),
                              data<const float>(dt_bias), norm.data_ptr(), ring.data_ptr(),
                              data<float>(state), rows, positions, n, cache_rows, key_heads,
                              key_dim, value_heads, value_dim, eps, flag, stream);
    });
    return THPVariable_Wrap(out);
}

// A matrix with contiguous rows, ld elements apart.
struct Matrix {
    const at::Tensor &t;
    int64_t rows, width, ld;

    Matrix(const Call &call, PyObject *o, const char *name) : t(tensor(o, name)) {
        TORCH_CHECK_VALUE(t.dim() == 2 && call.here(t) && (t.size(1) < 2 || t.stride(1) == 1),
                          name, " must be a matrix with contiguous rows on the call's device");
        rows = t.size(0);
        width = t.size(1);
        ld = rows > 1 ? t.stride(0) : (width + 7) / 8 * 8;
    }
};

// Rows in 8 bits: values and the scales of their groups.
struct Rows8 {
    const at::Tensor &values, &scales;
    int64_t rows, width;

    Rows8(const Call &call, PyObject *v, PyObject *s)
        : values(tensor(v, "values")), scales(tensor(s, "scales")) {
        TORCH_CHECK_VALUE(values.dim() == 2 && call.plain(values, at::kChar) && scales.dim() == 2 &&
                              call.plain(scales, at::kFloat) &&
                              scales.size(0) == values.size(0) &&
                              scales.size(1) == (values.size(1) + 127) / 128,
                          "8-bit rows are contiguous int8 values [rows, width] and float32 scales "
                          "[rows, ceil(width / 128)] of one device");
        rows = values.size(0);
        width = values.size(1);
    }
};

// A weight in 4 bits: a[0..5] packed, scales, out, inner, group, gated.
struct Weight4 {
    const at::Tensor &packed, &scales;
    int64_t out, inner, group;
    bool gated;

    Weight4(const Call &call, Args a)
        : packed(tensor(a[0], "packed")), scales(tensor(a[1], "scales")), out(integer(a[2])),
          inner(integer(a[3])), group(integer(a[4])), gated(truth(a[5])) {
        TORCH_CHECK_VALUE(group == 32 || group == 64 || group == 128,
                          "group must be 32, 64 or 128");
        TORCH_CHECK_VALUE(out > 0 && inner > 0 && (!gated || out % 2 == 0),
                          "out and inner must be positive, a gated weight's out even");
        const int64_t nb = gated ? 2 * ((out / 2 + 15) / 16) : (out + 15) / 16;
        const int64_t kb = (inner + 127) / 128;
        TORCH_CHECK_VALUE(packed.dim() == 4 && packed.size(0) == nb && packed.size(1) == kb &&
                              packed.size(2) == 64 && packed.size(3) == 4 &&
                              call.plain(packed, at::kInt) && scales.dim() == 3 &&
                              scales.size(0) == nb && scales.size(1) == kb * (128 / group) &&
                              scales.size(2) == 16 && call.plain(scales, at::kBFloat16),
                          "a 4-bit weight is a contiguous int32 [", nb, ", ", kb,
                          ", 64, 4] tensor and contiguous bfloat16 scales [", nb, ", ",
                          kb * (128 / group), ", 16] on the call's device");
    }
};

// at::empty for the device, without its dispatch (0.3 us of a call's 4).
at::Tensor fresh(const Call &call, at::IntArrayRef size, at::ScalarType type) {
    return at::Tensor(at::detail::empty_cuda(size, type, call.device, std::nullopt));
}
at::Tensor q8_scales(const Call &call, int64_t rows, int64_t width) {
    return fresh(call, {rows, (width + 127) / 128}, at::kFloat);
}
PyObject *pair(const at::Tensor &a, const at::Tensor &b) {
    THPObjectPtr x(THPVariable_Wrap(a)), y(THPVariable_Wrap(b));
    PyObject *t = x && y ? PyTuple_Pack(2, x.get(), y.get()) : nullptr;
    if (!t) throw python_error();
    return t;
}
at::ScalarType type_of(int64_t code) { return code == QDC_F32 ? at::kFloat : at::kBFloat16; }

PyObject *pack_w4(Args a) {
    const Call call(tensor(a[0], "w"));
    const Matrix w(call, a[0], "w");
    const int32_t code = dtype_code(w.t);
    const int64_t group = integer(a[1]);
    const bool gated = truth(a[2]);
    TORCH_CHECK_VALUE(group == 32 || group == 64 || group == 128, "group must be 32, 64 or 128");
    TORCH_CHECK_VALUE(w.rows > 0 && w.width > 0 && w.width % 8 == 0 && (!gated || w.rows % 2 == 0),
                      "w must be [out, inner] with inner a multiple of 8, a gated one's out even");
    const int64_t nb = gated ? 2 * ((w.rows / 2 + 15) / 16) : (w.rows + 15) / 16;
    const int64_t kb = (w.width + 127) / 128;
    const at::Tensor packed = fresh(call, {nb, kb, 64, 4}, at::kInt);
    const at::Tensor scales = fresh(call, {nb, kb * (128 / group), 16}, at::kBFloat16);
    call.run("pack_w4", [&](hipStream_t stream) {
        return qdc_pack_w4(packed.data_ptr(), scales.data_ptr(), w.t.data_ptr(), w.rows, w.width,
                           w.ld, group, gated, code, stream);
    });
    return pair(packed, scales);
}

// a[6]: the output's dtype code
PyObject *unpack_w4(Args a) {
    const Call call(tensor(a[0], "packed"));
    const Weight4 w(call, a);
    const int32_t code = (int32_t)integer(a[6]);
    const at::Tensor out = fresh(call, {w.out, w.inner}, type_of(code));
    call.run("unpack_w4", [&](hipStream_t stream) {
        return qdc_unpack_w4(out.data_ptr(), w.packed.data_ptr(), w.scales.data_ptr(), w.out,
                             w.inner, w.group, w.gated, code, stream);
    });
    return THPVariable_Wrap(out);
}

PyObject *quantize_q8(Args a) {
    const Call call(tensor(a[0], "x"));
    const Matrix x(call, a[0], "x");
    const int32_t code = dtype_code(x.t);
    const at::Tensor values = fresh(call, {x.rows, x.width}, at::kChar);
    const at::Tensor scales = q8_scales(call, x.rows, x.width);
    call.run("quantize_q8", [&](hipStream_t stream) {
        return qdc_quantize_q8(values.data_ptr(), data<float>(scales), x.t.data_ptr(), x.rows,
                               x.width, x.ld, code, stream);
    });
    return pair(values, scales);
}

PyObject *dequantize_q8(Args a) {
    const Call call(tensor(a[0], "values"));
    const Rows8 q(call, a[0], a[1]);
    const int32_t code = (int32_t)integer(a[2]);
    const at::Tensor out = fresh(call, {q.rows, q.width}, type_of(code));
    call.run("dequantize_q8", [&](hipStream_t stream) {
        return qdc_dequantize_q8(out.data_ptr(), q.values.data_ptr(), data<const float>(q.scales),
                                 q.rows, q.width, code, stream);
    });
    return THPVariable_Wrap(out);
}

PyObject *residual_rms_q8(Args a) {
    const at::Tensor &x = tensor(a[0], "x");
    const Call call(x);
    TORCH_CHECK_VALUE(x.dim() == 2 && call.plain(x, at::kFloat),
                      "x must be a contiguous float32 matrix");
    const int64_t rows = x.size(0), width = x.size(1);
    const float *add = nullptr;
    if (a[1] != Py_None) {
        const at::Tensor &t = tensor(a[1], "add");
        TORCH_CHECK_VALUE(t.sizes() == x.sizes() && call.plain(t, at::kFloat),
                          "add must be a contiguous float32 tensor like x");
        add = data<const float>(t);
    }
    const at::Tensor &norm = tensor(a[2], "weight");
    const int32_t code = dtype_code(norm);
    TORCH_CHECK_VALUE(norm.numel() == width && call.here(norm) && norm.is_contiguous(),
                      "weight must be a contiguous vector of ", width, " elements on x's device");
    const float eps = real(a[3]);
    const int32_t *mask = nullptr;
    if (a[4] != Py_None) mask = call.ints(a[4], "token_mask", rows);
    const at::Tensor residual = add ? fresh(call, {rows, width}, at::kFloat) : x;
    const at::Tensor values = fresh(call, {rows, width}, at::kChar);
    const at::Tensor scales = q8_scales(call, rows, width);
    call.run("residual_rms_q8", [&](hipStream_t stream) {
        return qdc_residual_rmsnorm_q8(add ? data<float>(residual) : nullptr, values.data_ptr(),
                                       data<float>(scales), data<const float>(x), add,
                                       norm.data_ptr(), mask, rows, width, eps, code, stream);
    });
    THPObjectPtr r(THPVariable_Wrap(residual)), v(THPVariable_Wrap(values)),
        s(THPVariable_Wrap(scales));
    PyObject *t = r && v && s ? PyTuple_Pack(3, r.get(), v.get(), s.get()) : nullptr;
    if (!t) throw python_error();
    return t;
}

// a[0], a[1]: x, or the values and scales of 8-bit rows (a[1] not None); a[2..7]: the weight;
// a[8]: the output's dtype code, -1 for x's
PyObject *linear_w4(Args a) {
    const at::Tensor &x0 = tensor(a[0], "x");
    const Call call(x0);
    const Weight4 w(call, a + 2);
    int64_t rows, width, ld;
    int32_t code = QDC_Q8;
    const float *x_scales = nullptr;
    if (a[1] != Py_None) {
        const Rows8 x(call, a[0], a[1]);
        rows = x.rows;
        width = ld = x.width;
        x_scales = data<const float>(x.scales);
    } else {
        const Matrix x(call, a[0], "x");
        code = dtype_code(x0);
        rows = x.rows;
        width = x.width;
        ld = x.ld;
    }
    TORCH_CHECK_VALUE(width == w.inner, "x has rows of ", width, " values, the weight takes ",
                      w.inner);
    int32_t out_code = (int32_t)integer(a[8]);
    if (out_code < 0) out_code = code == QDC_Q8 ? QDC_BF16 : code;
    const int64_t cols = w.gated ? w.out / 2 : w.out;
    const at::Tensor y =
        fresh(call, {rows, cols}, out_code == QDC_Q8 ? at::kChar : type_of(out_code));
    const at::Tensor y_scales = out_code == QDC_Q8 ? q8_scales(call, rows, cols) : at::Tensor();
    const int64_t need = out_code == QDC_Q8 ? qdc_linear_w4_workspace(rows, w.out, w.inner, w.group,
                                                                      w.gated, out_code)
                                            : 0;
    const at::Tensor work = need > 0 ? fresh(call, {need}, at::kByte) : at::Tensor();
    call.run(w.gated ? "gated_w4" : "linear_w4", [&](hipStream_t stream) {
        return qdc_linear_w4(y.data_ptr(), out_code == QDC_Q8 ? data<float>(y_scales) : nullptr,
                             out_code, x0.data_ptr(), x_scales, code, w.packed.data_ptr(),
                             w.scales.data_ptr(), rows, w.out, w.inner, w.group, ld, w.gated,
                             need > 0 ? work.data_ptr() : nullptr, need > 0 ? need : 0, stream);
    });
    return out_code == QDC_Q8 ? pair(y, y_scales) : THPVariable_Wrap(y);
}

template <PyObject *(*F)(Args), Py_ssize_t N>
PyObject *function(PyObject *, Args args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    TORCH_CHECK_TYPE(n == N, "expected ", N, " arguments, got ", n);
    return F(args);
    END_HANDLE_TH_ERRORS
}

PyObject *on_failure(PyObject *, PyObject *f) {
    Py_INCREF(f);
    Py_XSETREF(failed, f);
    Py_RETURN_NONE;
}

#define QDC_FUNCTION(name, n)                                                            \
    {#name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(function<name, n>)), \
     METH_FASTCALL, nullptr}
PyMethodDef methods[] = {QDC_FUNCTION(prepare_paged, 17), QDC_FUNCTION(paged_attention, 10),
                         QDC_FUNCTION(extend_pages, 9), QDC_FUNCTION(free_pages, 7),
                         QDC_FUNCTION(fork_pages, 9), QDC_FUNCTION(compact_pages, 6),
                         QDC_FUNCTION(copy_pages, 4), QDC_FUNCTION(delta_step, 16),
                         QDC_FUNCTION(pack_w4, 3), QDC_FUNCTION(unpack_w4, 7),
                         QDC_FUNCTION(quantize_q8, 1), QDC_FUNCTION(dequantize_q8, 3),
                         QDC_FUNCTION(residual_rms_q8, 5), QDC_FUNCTION(linear_w4, 9),
                         {"on_failure", on_failure, METH_O, nullptr},
                         {nullptr, nullptr, 0, nullptr}};
#undef QDC_FUNCTION

PyModuleDef module = {PyModuleDef_HEAD_INIT, "qdc_calls", nullptr, -1, methods};

}  // namespace

// version, quant_version: of the headers whose entry points the functions call
PyMODINIT_FUNC PyInit_qdc_calls() {
    PyObject *m = PyModule_Create(&module);
    if (m && PyModule_AddStringConstant(m, "version", QDC_HIP_CACHE_VERSION) == 0 &&
        PyModule_AddStringConstant(m, "quant_version", QDC_HIP_QUANT_VERSION) == 0)
        return m;
    Py_XDECREF(m);
    return nullptr;
}
