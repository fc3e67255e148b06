// The host side of the serving loop's small calls (pages.py, beams.py, kvcache.py): argument checks, outputs and workspaces, and the
// call into the library (include/nemicli_qmv.h).  Their kernels take 2 to 25 us, and through ctypes and torch's Python functions the
// calls took 14 to 45 us on the host: 1.5 us an output, 0.5 us a checked argument, 1.5 us for ctypes.  A CPython module over
// libtorch, one function a call; every refusal is a RuntimeError, and nothing is launched before the checks.  Arguments are read under the
// interpreter's lock; allocations, copies and launches, which may wait for memory or for room in the stream, leave it to other threads.
#include <Python.h>

#include <algorithm>
#include <cmath>
#include <initializer_list>
#include <string>

#include <ATen/core/Tensor.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include "../../../include/nemicli_qmv.h"

namespace {

using at::Tensor;
using c10::ScalarType;

struct Refused {
    std::string text;
};
struct PythonError {};                    // already set

// (without iostreams: formatting a number through one crashed in a process that has torch's libraries)
std::string text(const char* s) { return s; }
std::string text(const std::string& s) { return s; }
std::string text(int64_t n) { return std::to_string(n); }
std::string text(int n) { return std::to_string(n); }
std::string text(double x) { return std::to_string(x); }
std::string text(ScalarType t) { return c10::toString(t); }
std::string text(const c10::Device& d) { return d.str(); }
template <class... A>
[[noreturn]] void refuse(const A&... parts) {
    throw Refused{(text(parts) + ...)};
}
std::string shape_of(const Tensor& t) {
    std::string s = "(";
    for (int64_t i = 0; i < t.dim(); ++i) s += (i ? ", " : "") + text(t.size(i));
    return s + ") " + text(t.scalar_type()) + " on " + text(t.device());
}
void check(int status, const char* what) {
    if (!status) return;
    std::string extra;
    if (status == QMV_ERR_LAUNCH) extra = " (cudaError " + std::to_string(qmv_last_cuda_error()) + ")";
    refuse(what, ": ", qmv_status_string(status), extra);
}

// ---- arguments
const Tensor& tensor(PyObject* o, const char* what) {
    if (!THPVariable_Check(o)) refuse(what, ": a tensor expected");
    return THPVariable_Unpack(o);
}
bool none(PyObject* o) { return o == Py_None; }
int64_t number(PyObject* o, const char* what) {
    const long long v = PyLong_AsLongLong(o);
    if (v == -1 && PyErr_Occurred()) {
        PyErr_Clear();
        refuse(what, ": a whole number expected");
    }
    return v;
}
int64_t number(PyObject* o, const char* what, int64_t lo, int64_t hi) {
    const int64_t v = number(o, what);
    if (v < lo || v > hi) refuse(what, ": ", v, " (", lo, " to ", hi, ")");
    return v;
}
// contiguous, of a type and device; sizes of -1 may be anything
void expect(const Tensor& t, const char* what, int device, ScalarType type, std::initializer_list<int64_t> sizes) {
    bool ok = t.scalar_type() == type && t.is_cuda() && t.get_device() == device && t.dim() == int64_t(sizes.size()) && t.is_contiguous();
    int64_t i = 0;
    if (ok)
        for (const int64_t n : sizes) ok &= n < 0 || t.size(i) == n, ++i;
    if (ok) return;
    std::string sizes_text;
    i = 0;
    for (const int64_t n : sizes) sizes_text += (i++ ? ", " : "") + (n < 0 ? text("any") : text(n));
    refuse(what, ": contiguous ", type, " (", sizes_text, ") on cuda:", device, " expected, got ", shape_of(t));
}
int* ints(const Tensor& t) { return static_cast<int*>(t.data_ptr()); }
long long* longs(const Tensor& t) { return static_cast<long long*>(t.data_ptr()); }

// ---- results
Tensor make(at::IntArrayRef sizes, ScalarType type, int device) {
    return at::detail::empty_cuda(sizes, type, c10::Device(c10::kCUDA, device), std::nullopt);
}
// The outputs of a call lie in one allocation, 16 bytes apart at least (an allocation takes 0.6 us, a part of one 0.1); the Python side's
// documentation says so, since each keeps all of it alive and has the next one's bytes behind its own.
struct Outputs {
    int device;
    int64_t bytes = 0;
    Tensor base;
    static int64_t room(at::IntArrayRef sizes, ScalarType type) {
        int64_t n = c10::elementSize(type);
        for (const int64_t s : sizes) n *= s;
        return (n + 15) / 16 * 16;
    }
    void plan(at::IntArrayRef sizes, ScalarType type) { bytes += room(sizes, type); }
    // the parts in the order in which they were planned
    Tensor take(at::IntArrayRef sizes, ScalarType type) {
        if (!base.defined()) base = make({bytes}, ScalarType::Byte, device), bytes = 0;
        Tensor t = at::detail::make_tensor<c10::TensorImpl>(c10::Storage(base.storage()), c10::DispatchKeySet(c10::DispatchKey::CUDA),
                                                            c10::scalarTypeToTypeMeta(type));
        t.unsafeGetTensorImpl()->set_sizes_contiguous(sizes);
        t.unsafeGetTensorImpl()->set_storage_offset(bytes / int64_t(c10::elementSize(type)));
        bytes += room(sizes, type);
        return t;
    }
};
PyObject* wrap(Tensor&& t) { return THPVariable_Wrap(std::move(t)); }
template <class... T>
PyObject* tuple(T&&... t) {
    PyObject* out = PyTuple_New(sizeof...(t));
    if (!out) throw PythonError{};
    Py_ssize_t i = 0;
    (PyTuple_SET_ITEM(out, i++, wrap(std::move(t))), ...);
    return out;
}
void* stream_of(int device) { return c10::cuda::getCurrentCUDAStream(device).stream(); }
// A call's work on the device: the interpreter's lock is free (no Python object is touched until the end of the scope; an exception leaves
// it with the lock taken again), and the device is the current one.
struct OnDevice {
    struct Unlocked {
        PyThreadState* state = PyEval_SaveThread();
        Unlocked() = default;
        Unlocked(const Unlocked&) = delete;
        Unlocked& operator=(const Unlocked&) = delete;
        ~Unlocked() { PyEval_RestoreThread(state); }
    } unlocked;
    c10::cuda::OptionalCUDAGuard guard;
    explicit OnDevice(int device) : guard(c10::Device(c10::kCUDA, device)) {}
};

// a function of a fixed number of arguments: C++ exceptions become Python's
template <int N, PyObject* (*F)(PyObject* const*)>
PyObject* call(PyObject*, PyObject* const* a, Py_ssize_t n) {
    try {
        if (n != N) refuse("internal: ", N, " arguments expected, got ", n);
        return F(a);
    } catch (const Refused& r) {
        PyErr_SetString(PyExc_RuntimeError, r.text.c_str());
    } catch (const PythonError&) {
    } catch (const c10::OutOfMemoryError& e) {
        PyObject* torch = PyImport_ImportModule("torch");         // torch.OutOfMemoryError, as torch's own functions raise it
        PyObject* kind = torch ? PyObject_GetAttrString(torch, "OutOfMemoryError") : nullptr;
        PyErr_Clear();
        PyErr_SetString(kind ? kind : PyExc_RuntimeError, e.what_without_backtrace());
        Py_XDECREF(kind);
        Py_XDECREF(torch);
    } catch (const c10::Error& e) {
        PyErr_SetString(PyExc_RuntimeError, e.what_without_backtrace());
    } catch (const std::exception& e) {
        PyErr_SetString(PyExc_RuntimeError, e.what());
    }
    return nullptr;
}

// ---- page tables ----------------------------------------------------------------------------------------------------

struct Tables {
    const Tensor &tables, &lens, &free, &counts;
    int device, n, width, page;
};
Tables tables_of(PyObject* const* a, const char* what) {          // lens, tables, free, counts, page
    const std::string w(what);
    Tables t{tensor(a[1], (w + " tables").c_str()), tensor(a[0], (w + " lens").c_str()), tensor(a[2], (w + " free").c_str()),
             tensor(a[3], (w + " counts").c_str()), -1, 0, 0, 0};
    if (!t.tables.is_cuda()) refuse(what, ": tables on ", t.tables.device(), "; the tables live on a CUDA device");
    t.device = t.tables.get_device();
    expect(t.tables, (w + " tables").c_str(), t.device, ScalarType::Int, {-1, -1});
    const int64_t n = t.tables.size(0), width = t.tables.size(1), page = number(a[4], (w + " page").c_str());
    expect(t.lens, (w + " lens").c_str(), t.device, ScalarType::Int, {n});
    expect(t.free, (w + " free").c_str(), t.device, ScalarType::Int, {-1});
    expect(t.counts, (w + " counts").c_str(), t.device, ScalarType::Int, {2});
    if (page < 16 || page > 1024 || (page & (page - 1)) || width == 0 || width > (1 << 30) / page || t.free.size(0) == 0 ||
        t.free.size(0) > 0x7FFFFFFF || n <= 0 || n > 65535)
        refuse(what, ": pages of 16 to 1024 tokens (a power of two), 1 to 65535 tables of up to 2^30 tokens, and a cache with a page expected, got pages of ",
               page, ", tables ", shape_of(t.tables), ", free ", shape_of(t.free));
    t.n = int(n), t.width = int(width), t.page = int(page);
    return t;
}

PyObject* plan(PyObject* const* a) {                              // lens, tables, free, counts, page, new, rows
    const Tables t = tables_of(a, "pages.plan");
    const Tensor& add = tensor(a[5], "pages.plan new");
    expect(add, "pages.plan new", t.device, ScalarType::Int, {t.n});
    const int64_t rows = number(a[6], "pages.plan rows", 0, 1 << 30);
    Tensor slots, positions, starts, lens, counts;
    {
        const OnDevice scope(t.device);
        Outputs o{t.device};
        o.plan({rows}, ScalarType::Long), o.plan({rows}, ScalarType::Long), o.plan({t.n + 1}, ScalarType::Int), o.plan({t.n}, ScalarType::Int), o.plan({2}, ScalarType::Int);
        slots = o.take({rows}, ScalarType::Long), positions = o.take({rows}, ScalarType::Long), starts = o.take({t.n + 1}, ScalarType::Int);
        lens = o.take({t.n}, ScalarType::Int), counts = o.take({2}, ScalarType::Int);
        check(qmv_page_plan(ints(t.lens), ints(add), ints(t.tables), t.n, t.width, t.page, ints(t.free), int(t.free.size(0)), ints(t.counts), rows,
                            longs(slots), longs(positions), ints(starts), ints(lens), ints(counts), stream_of(t.device)), "qmv_page_plan");
    }
    return tuple(std::move(slots), std::move(positions), std::move(starts), std::move(lens), std::move(counts));
}

PyObject* release(PyObject* const* a) {                           // lens, tables, free, counts, page, done
    const Tables t = tables_of(a, "pages.release");
    const Tensor& done = tensor(a[5], "pages.release done");
    expect(done, "pages.release done", t.device, ScalarType::Bool, {t.n});
    Tensor lens, counts;
    {
        const OnDevice scope(t.device);
        Outputs o{t.device};
        o.plan({t.n}, ScalarType::Int), o.plan({2}, ScalarType::Int);
        lens = o.take({t.n}, ScalarType::Int), counts = o.take({2}, ScalarType::Int);
        check(qmv_page_release(static_cast<const uint8_t*>(done.data_ptr()), ints(t.lens), ints(t.tables), t.n, t.width, t.page, ints(t.free),
                               int(t.free.size(0)), ints(t.counts), ints(lens), ints(counts), stream_of(t.device)), "qmv_page_release");
    }
    return tuple(std::move(lens), std::move(counts));
}

PyObject* reorder(PyObject* const* a) {                           // lens, tables, free, counts, page, parents, own
    const Tables t = tables_of(a, "pages.reorder");
    const Tensor& parents = tensor(a[5], "pages.reorder parents");
    expect(parents, "pages.reorder parents", t.device, ScalarType::Int, {-1, -1});
    const int64_t reqs = parents.size(0), beams = parents.size(1);
    if (beams < 1 || beams > 64 || reqs * beams != t.n) refuse("pages.reorder: parents ", shape_of(parents), " for ", t.n, " tables, up to 64 beams");
    const int* own = nullptr;
    if (!none(a[6])) {
        const Tensor& o = tensor(a[6], "pages.reorder own");
        expect(o, "pages.reorder own", t.device, ScalarType::Int, {reqs});
        own = ints(o);
    }
    const int64_t nbytes = qmv_page_reorder_workspace_bytes(int(reqs), int(beams), t.width);
    if (nbytes <= 0) refuse("pages.reorder: tables ", shape_of(t.tables), " of ", beams, " beams: up to 2^26 entries a request");
    Tensor tables, counts, lens, src, dst, used;
    {
        const OnDevice scope(t.device);
        Outputs o{t.device};
        o.plan({t.n, t.width}, ScalarType::Int), o.plan({2}, ScalarType::Int);
        for (int i = 0; i < 4; ++i) o.plan({t.n}, ScalarType::Int);
        tables = o.take({t.n, t.width}, ScalarType::Int), counts = o.take({2}, ScalarType::Int), lens = o.take({t.n}, ScalarType::Int);
        src = o.take({t.n}, ScalarType::Int), dst = o.take({t.n}, ScalarType::Int), used = o.take({t.n}, ScalarType::Int);
        const Tensor ws = make({nbytes}, ScalarType::Byte, t.device);
        check(qmv_page_reorder(ints(parents), ints(t.lens), ints(t.tables), own, int(reqs), int(beams), t.width, t.page, ints(t.free), int(t.free.size(0)),
                               ints(t.counts), ints(tables), ints(lens), ints(src), ints(dst), ints(used), ints(counts), ws.data_ptr(), nbytes,
                               stream_of(t.device)), "qmv_page_reorder");
    }
    return tuple(std::move(tables), std::move(lens), std::move(counts), std::move(src), std::move(dst), std::move(used));
}

// ---- beams ------------------------------------------------------------------------------------------------------------

int dtype_of(const Tensor& t) {
    return t.scalar_type() == ScalarType::Float ? QMV_OUT_F32 : t.scalar_type() == ScalarType::BFloat16 ? QMV_OUT_BF16
         : t.scalar_type() == ScalarType::Half ? QMV_OUT_F16 : -1;
}

void choose_best(Tensor logits, const Tensor& scores, int dtype, int n, const Tensor& out, const Tensor& parents, const Tensor& tokens) {
    const int64_t reqs = logits.size(0), k = logits.size(1), vocab = logits.size(2);
    int64_t by_req = logits.stride(0), by_beam = logits.stride(1);
    if ((logits.stride(2) != 1 && vocab > 1) || (k > 1 && by_beam < vocab) || (reqs > 1 && (by_req < vocab || (k > 1 && by_req != k * by_beam)))) {
        logits = logits.contiguous();
        by_beam = vocab, by_req = k * vocab;
    }
    const int64_t stride = k > 1 ? by_beam : reqs > 1 ? by_req : vocab;
    const int64_t nbytes = qmv_beam_workspace_bytes(int(reqs), int(k), int(vocab), n);
    const Tensor ws = make({nbytes}, ScalarType::Byte, logits.get_device());
    check(qmv_beam_select(logits.data_ptr(), dtype, stride, int(reqs), int(k), int(vocab), static_cast<const float*>(scores.data_ptr()), n,
                          static_cast<float*>(out.data_ptr()), ints(parents), ints(tokens), ws.data_ptr(), nbytes, stream_of(logits.get_device())),
          "qmv_beam_select");
}

PyObject* select(PyObject* const* a) {                            // logits, scores, n
    const Tensor &logits = tensor(a[0], "beams.select logits"), &scores = tensor(a[1], "beams.select scores");
    const int dtype = dtype_of(logits);
    if (logits.dim() != 3 || dtype < 0 || !logits.is_cuda())
        refuse("beams.select: logits (requests, beams, vocab) of float32, bfloat16 or float16 on a CUDA device expected, got ", shape_of(logits));
    const int device = logits.get_device();
    const int64_t reqs = logits.size(0), k = logits.size(1), vocab = logits.size(2);
    expect(scores, "beams.select scores", device, ScalarType::Float, {reqs, k});
    int64_t n = number(a[2], "beams.select n");
    if (n == 0) n = k;
    if (k < 1 || k > 64 || n < 1 || n > 64 || vocab < 1 || vocab > 1 << 30 || n > k * vocab || reqs * k > 65535)
        refuse("beams.select: ", reqs, " requests of ", k, " beams over ", vocab, " tokens, ", n, " best: up to 64 beams and candidates, 65535 beams in all");
    Tensor out, parents, tokens;
    {
        const OnDevice scope(device);
        Outputs o{device};
        o.plan({reqs, n}, ScalarType::Float), o.plan({reqs, n}, ScalarType::Int), o.plan({reqs, n}, ScalarType::Int);
        out = o.take({reqs, n}, ScalarType::Float), parents = o.take({reqs, n}, ScalarType::Int), tokens = o.take({reqs, n}, ScalarType::Int);
        if (reqs) choose_best(logits, scores, dtype, int(n), out, parents, tokens);
    }
    return tuple(std::move(out), std::move(parents), std::move(tokens));
}

// ---- the cache --------------------------------------------------------------------------------------------------------

struct Cache {
    const qmv_kv_cache* c;
    int device;
};
Cache cache_of(PyObject* const* a) {                              // address of the description, device
    return {reinterpret_cast<const qmv_kv_cache*>(number(a[0], "KVCache")), int(number(a[1], "KVCache device", 0, 1023))};
}
// (rows, heads, dim) of a type the kernels read
int tokens_of(const Tensor& t, const char* what, const Cache& c, int64_t heads = -1) {
    if (!t.is_cuda() || t.get_device() != c.device) refuse(what, ": tensor on ", t.device(), ", the cache on cuda:", c.device);
    const int dtype = dtype_of(t);
    if (t.dim() != 3 || t.size(2) != c.c->dim || dtype < 0 || (heads >= 0 && t.size(1) != heads) || t.size(1) == 0)
        refuse(what, ": (rows, ", heads >= 0 ? std::to_string(heads) : "heads", ", ", c.c->dim, ") of float32, bfloat16 or float16 expected, got ", shape_of(t));
    return dtype;
}
// as the kernels read it: the values of a row side by side, rows any multiple of 4 values apart, a start on four values
Tensor rows_of(const Tensor& t, int64_t& stride) {
    const int64_t row = t.size(1) * t.size(2);
    const uintptr_t four = 4 * t.element_size();
    const bool many = t.size(0) > 1;
    if (t.stride(2) == 1 && (t.size(1) == 1 || t.stride(1) == t.size(2)) && (!many || (t.stride(0) >= row && t.stride(0) % 4 == 0)) &&
        reinterpret_cast<uintptr_t>(t.data_ptr()) % four == 0) {
        stride = many ? t.stride(0) : row;
        return t;
    }
    stride = row;
    Tensor x = t.contiguous();
    return reinterpret_cast<uintptr_t>(x.data_ptr()) % four ? x.clone() : x;
}

void write_rows(const Cache& c, const Tensor& k_given, const Tensor& v_given, const Tensor& slots, const Tensor& q_given, const Tensor& out, int dtype,
                const float* cos, const float* sin, const long long* positions, int64_t n_pos, int rot, int paired, const uint8_t* axes, int n_axes) {
    int64_t ks, vs, qs = 0;
    const Tensor k = rows_of(k_given, ks), v = rows_of(v_given, vs), q = q_given.defined() ? rows_of(q_given, qs) : q_given;
    const void* qp = q.defined() ? q.data_ptr() : nullptr;
    void* op = q.defined() ? out.data_ptr() : nullptr;
    const int n_q = q.defined() ? int(q.size(1)) : 0;
    if (axes)
        check(qmv_kv_write_axes(c.c, k.data_ptr(), v.data_ptr(), dtype, ks, vs, longs(slots), k.size(0), cos, sin, positions, n_pos, rot, paired, axes, n_axes,
                                qp, qs, n_q, op, stream_of(c.device)), "qmv_kv_write_axes");
    else
        check(qmv_kv_write(c.c, k.data_ptr(), v.data_ptr(), dtype, ks, vs, longs(slots), k.size(0), cos, sin, positions, n_pos, rot, paired, qp, qs, n_q, op,
                           stream_of(c.device)), "qmv_kv_write");
}

PyObject* write(PyObject* const* a) {                             // cache (2), k, v, slots, q, cos, sin, positions, paired, axes
    const Cache c = cache_of(a);
    const Tensor &k = tensor(a[2], "KVCache.write k"), &v = tensor(a[3], "KVCache.write v"), &slots = tensor(a[4], "KVCache.write slots");
    const int dtype = tokens_of(k, "KVCache.write k", c, c.c->n_kv);
    const int64_t rows = k.size(0);
    if (tokens_of(v, "KVCache.write v", c, c.c->n_kv) != dtype || v.size(0) != rows) refuse("KVCache.write v: ", rows, " rows of ", k.scalar_type(), " expected");
    expect(slots, "KVCache.write slots", c.device, ScalarType::Long, {rows});
    const float *cos = nullptr, *sin = nullptr;
    const long long* positions = nullptr;
    int64_t n_pos = 0, rot = 0;
    const uint8_t* axes = nullptr;
    int n_axes = 0;
    if (!none(a[6])) {
        const Tensor &ct = tensor(a[6], "KVCache.write cos"), &st = tensor(a[7], "KVCache.write sin"), &pt = tensor(a[8], "KVCache.write positions");
        expect(ct, "KVCache.write cos", c.device, ScalarType::Float, {-1, -1});
        n_pos = ct.size(0), rot = 2 * ct.size(1);
        expect(st, "KVCache.write sin", c.device, ScalarType::Float, {n_pos, rot / 2});
        if (n_pos == 0 || rot % 8 || rot <= 0 || rot > c.c->dim)
            refuse("KVCache.write: tables (positions, rot / 2), rot a multiple of 8 up to ", c.c->dim, ", got ", shape_of(ct));
        if (none(a[10])) {
            expect(pt, "KVCache.write positions", c.device, ScalarType::Long, {rows});
        } else {
            expect(pt, "KVCache.write positions", c.device, ScalarType::Long, {-1, rows});
            const int64_t n = pt.size(0);
            if (!PyBytes_Check(a[10]) || PyBytes_GET_SIZE(a[10]) != rot / 2 || n < 1 || n > 4)
                refuse("KVCache.write: ", rot / 2, " axes and positions on 1 to 4 of them expected, got ", PyBytes_Check(a[10]) ? PyBytes_GET_SIZE(a[10]) : -1, " and ", n);
            axes = reinterpret_cast<const uint8_t*>(PyBytes_AS_STRING(a[10])), n_axes = int(n);
            for (int64_t f = 0; f < rot / 2; ++f)
                if (axes[f] >= n_axes) refuse("KVCache.write: axis ", int(axes[f]), " of ", n_axes);
        }
        cos = static_cast<const float*>(ct.data_ptr()), sin = static_cast<const float*>(st.data_ptr()), positions = longs(pt);
    } else if (!none(a[10])) {
        refuse("KVCache.write: axes without rope");
    }
    const int paired = PyObject_IsTrue(a[9]);
    if (paired < 0) throw PythonError{};
    Tensor q, out;
    if (!none(a[5])) {
        q = tensor(a[5], "KVCache.write q");
        if (tokens_of(q, "KVCache.write q", c) != dtype || q.size(0) != rows) refuse("KVCache.write q: ", rows, " rows of ", k.scalar_type(), " expected");
    }
    {
        const OnDevice scope(c.device);
        if (q.defined()) out = make(q.sizes(), q.scalar_type(), c.device);
        if (rows) write_rows(c, k, v, slots, q, out, dtype, cos, sin, positions, n_pos, int(rot), paired, axes, n_axes);
    }
    if (!out.defined()) Py_RETURN_NONE;
    return wrap(std::move(out));
}

PyObject* read(PyObject* const* a) {                              // cache (2), slots, dtype (QMV_OUT_*)
    const Cache c = cache_of(a);
    const Tensor& slots = tensor(a[2], "KVCache.read slots");
    expect(slots, "KVCache.read slots", c.device, ScalarType::Long, {-1});
    const int dtype = int(number(a[3], "KVCache.read dtype", 0, 2));
    const ScalarType type = dtype == QMV_OUT_F32 ? ScalarType::Float : dtype == QMV_OUT_BF16 ? ScalarType::BFloat16 : ScalarType::Half;
    const int64_t rows = slots.size(0);
    Tensor k, v;
    {
        const OnDevice scope(c.device);
        k = make({rows, c.c->n_kv, c.c->dim}, type, c.device), v = make({rows, c.c->n_kv, c.c->dim}, type, c.device);
        if (rows) check(qmv_kv_read(c.c, longs(slots), rows, k.data_ptr(), v.data_ptr(), dtype, stream_of(c.device)), "qmv_kv_read");
    }
    return tuple(std::move(k), std::move(v));
}

PyObject* copy(PyObject* const* a) {                              // cache (2), src, dst, used
    const Cache c = cache_of(a);
    const Tensor &src = tensor(a[2], "KVCache.copy src"), &dst = tensor(a[3], "KVCache.copy dst");
    const Tensor* used = none(a[4]) ? nullptr : &tensor(a[4], "KVCache.copy used");
    for (const Tensor* t : {&src, &dst, used})
        if (t && (t->scalar_type() != ScalarType::Int || !t->is_cuda() || t->get_device() != c.device || t->sizes() != src.sizes() || !t->is_contiguous()))
            refuse("KVCache.copy: src, dst and used contiguous int32 of one shape on cuda:", c.device, " expected, got ", shape_of(src), " and ", shape_of(*t));
    const int64_t n = src.numel();
    if (n > 0x7FFFFFFF) refuse("KVCache.copy: ", n, " copies");
    if (n) {
        const OnDevice scope(c.device);
        check(qmv_kv_copy(c.c, ints(src), ints(dst), used ? ints(*used) : nullptr, int(n), stream_of(c.device)), "qmv_kv_copy");
    }
    Py_RETURN_NONE;
}

struct Held {
    const Tensor &tables, &lens;
    const int* starts;
    int64_t n_seq, width;
};
Held held_of(PyObject* const* a, const Cache& c, const char* what) {          // tables, lens, starts
    const std::string w(what);
    Held h{tensor(a[0], (w + " tables").c_str()), tensor(a[1], (w + " lens").c_str()), nullptr, 0, 0};
    expect(h.tables, (w + " tables").c_str(), c.device, ScalarType::Int, {-1, -1});
    h.n_seq = h.tables.size(0), h.width = h.tables.size(1);
    expect(h.lens, (w + " lens").c_str(), c.device, ScalarType::Int, {h.n_seq});
    if (!none(a[2])) {
        const Tensor& s = tensor(a[2], (w + " starts").c_str());
        expect(s, (w + " starts").c_str(), c.device, ScalarType::Int, {h.n_seq + 1});
        h.starts = ints(s);
    }
    if (h.width > (1 << 30) / c.c->page || h.n_seq > 65535) refuse(what, ": up to 65535 tables of up to 2^30 tokens, got ", shape_of(h.tables));
    return h;
}
void* bounds_of(const Tensor& t, const char* what, const Cache& c) {
    expect(t, what, c.device, ScalarType::Half, {c.c->n_pages, c.c->n_kv, 2, c.c->dim});
    if (reinterpret_cast<uintptr_t>(t.data_ptr()) % 16) refuse(what, ": 16-byte aligned bounds expected");
    return t.data_ptr();
}

PyObject* summarise(PyObject* const* a) {                         // cache (2), tables, lens, starts, bounds, max_new (None: a table's)
    const Cache c = cache_of(a);
    void* bounds = bounds_of(tensor(a[5], "KVCache.summarise bounds"), "KVCache.summarise bounds", c);
    const Held h = held_of(a + 2, c, "KVCache.summarise");
    const int64_t cap = h.width * c.c->page, most = !h.starts ? 1 : none(a[6]) ? cap : number(a[6], "KVCache.summarise max_new", 0, INT64_MAX);
    if (h.n_seq && h.width && most) {
        const OnDevice scope(c.device);
        check(qmv_kv_bounds(c.c, ints(h.tables), int(h.width), ints(h.lens), h.starts, int(h.n_seq), int(std::min(most, cap)), bounds, stream_of(c.device)),
              "qmv_kv_bounds");
    }
    Py_RETURN_NONE;
}

PyObject* choose(PyObject* const* a) {                            // cache (2), tables, lens, starts, bounds, q, keep, first, last
    const Cache c = cache_of(a);
    const Tensor& given = tensor(a[6], "KVCache.choose q");
    const int dtype = tokens_of(given, "KVCache.choose q", c);
    const int64_t rows = given.size(0), heads = given.size(1);
    if (heads % c.c->n_kv || heads > 64LL * c.c->n_kv || heads > 65535) refuse("KVCache.choose: ", heads, " heads are not a multiple (at most 64) of ", c.c->n_kv, " key heads");
    void* bounds = bounds_of(tensor(a[5], "KVCache.choose bounds"), "KVCache.choose bounds", c);
    const Held h = held_of(a + 2, c, "KVCache.choose");
    if (!h.starts && rows < h.n_seq) refuse("KVCache.choose: ", rows, " query rows for ", h.n_seq, " sequences");
    const int64_t most = (1 << 30) / c.c->page, keep = number(a[7], "KVCache.choose keep", 1, most), first = number(a[8], "KVCache.choose first", 0, most),
                  last = number(a[9], "KVCache.choose last", 1, most);
    if (keep < first + last || rows > 65535) refuse("KVCache.choose: keep ", keep, " holds first ", first, " and last ", last, ", rows ", rows, " up to 65535");
    Tensor chosen, held;
    {
        const OnDevice scope(c.device);
        Outputs o{c.device};
        o.plan({rows, c.c->n_kv, keep}, ScalarType::Int), o.plan({rows}, ScalarType::Int);
        chosen = o.take({rows, c.c->n_kv, keep}, ScalarType::Int), held = o.take({rows}, ScalarType::Int);
        if (rows && (!h.n_seq || !h.width)) {
            chosen.fill_(-1), held.zero_();
        } else if (rows) {
            int64_t qs;
            const Tensor q = rows_of(given, qs);
            const int64_t nbytes = qmv_kv_choose_workspace_bytes(c.c, int(h.width), rows, int(keep));
            const Tensor ws = make({nbytes}, ScalarType::Byte, c.device);
            check(qmv_kv_choose(c.c, q.data_ptr(), dtype, qs, int(heads), bounds, ints(h.tables), int(h.width), ints(h.lens), h.starts, int(h.n_seq), rows,
                                int(keep), int(first), int(last), ints(chosen), ints(held), ws.data_ptr(), nbytes, stream_of(c.device)), "qmv_kv_choose");
        }
    }
    return tuple(std::move(chosen), std::move(held));
}

PyObject* attend_chosen(PyObject* const* a) {                     // cache (2), q, chosen, held, scale (None: dim ** -0.5), out
    const Cache c = cache_of(a);
    const Tensor &given = tensor(a[2], "KVCache.attend_chosen q"), &chosen = tensor(a[3], "KVCache.attend_chosen chosen"),
                 &held = tensor(a[4], "KVCache.attend_chosen held");
    const int dtype = tokens_of(given, "KVCache.attend_chosen q", c);
    const int64_t rows = given.size(0), heads = given.size(1);
    if (heads % c.c->n_kv || heads > 65535) refuse("KVCache.attend_chosen: ", heads, " heads are not a multiple of ", c.c->n_kv, " key heads");
    expect(chosen, "KVCache.attend_chosen chosen", c.device, ScalarType::Int, {rows, c.c->n_kv, -1});
    expect(held, "KVCache.attend_chosen held", c.device, ScalarType::Int, {rows});
    const int64_t keep = chosen.size(2);
    if (rows > 65535 || keep > (1 << 30) / c.c->page || (rows && keep == 0))
        refuse("KVCache.attend_chosen: up to 65535 rows of 1 to 2^30 / page pages, got ", shape_of(chosen));
    double scale = 1.0 / std::sqrt(double(c.c->dim));
    if (!none(a[5])) {
        scale = PyFloat_AsDouble(a[5]);
        if (scale == -1.0 && PyErr_Occurred()) {
            if (!PyErr_ExceptionMatches(PyExc_TypeError) && !PyErr_ExceptionMatches(PyExc_OverflowError)) throw PythonError{};
            PyErr_Clear();
            refuse("KVCache.attend_chosen: scale: a number within float32 expected");
        }
        if (!(std::abs(scale) < 3.4028235e38)) refuse("KVCache.attend_chosen: scale ", scale, " is not finite");
    }
    Tensor out;
    if (!none(a[6])) {
        out = tensor(a[6], "KVCache.attend_chosen out");
        if (out.sizes() != given.sizes() || out.scalar_type() != given.scalar_type() || out.device() != given.device() || !out.is_contiguous() ||
            reinterpret_cast<uintptr_t>(out.data_ptr()) % 16)
            refuse("KVCache.attend_chosen: out must be contiguous, 16-byte aligned and like q (", shape_of(given), "), got ", shape_of(out));
    }
    {
        const OnDevice scope(c.device);
        if (!out.defined()) out = make(given.sizes(), given.scalar_type(), c.device);
        if (rows) {
            int64_t qs;
            const Tensor q = rows_of(given, qs);
            const int64_t nbytes = qmv_kv_attend_chosen_workspace_bytes(c.c, int(heads), rows, dtype, int(keep));
            if (nbytes <= 0) refuse("KVCache.attend_chosen: ", heads, " heads, ", rows, " rows of ", keep, " pages not supported");
            const Tensor ws = make({nbytes}, ScalarType::Byte, c.device);
            check(qmv_kv_attend_chosen(c.c, q.data_ptr(), dtype, qs, int(heads), ints(chosen), int(keep), ints(held), rows, float(scale), out.data_ptr(),
                                       ws.data_ptr(), nbytes, stream_of(c.device)), "qmv_kv_attend_chosen");
        }
    }
    if (!none(a[6])) {
        Py_INCREF(a[6]);
        return a[6];
    }
    return wrap(std::move(out));
}

PyMethodDef methods[] = {
    {"plan", (PyCFunction)(void (*)())call<7, plan>, METH_FASTCALL, nullptr},
    {"release", (PyCFunction)(void (*)())call<6, release>, METH_FASTCALL, nullptr},
    {"reorder", (PyCFunction)(void (*)())call<7, reorder>, METH_FASTCALL, nullptr},
    {"select", (PyCFunction)(void (*)())call<3, select>, METH_FASTCALL, nullptr},
    {"write", (PyCFunction)(void (*)())call<11, write>, METH_FASTCALL, nullptr},
    {"read", (PyCFunction)(void (*)())call<4, read>, METH_FASTCALL, nullptr},
    {"copy", (PyCFunction)(void (*)())call<5, copy>, METH_FASTCALL, nullptr},
    {"summarise", (PyCFunction)(void (*)())call<7, summarise>, METH_FASTCALL, nullptr},
    {"choose", (PyCFunction)(void (*)())call<10, choose>, METH_FASTCALL, nullptr},
    {"attend_chosen", (PyCFunction)(void (*)())call<7, attend_chosen>, METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_qmv_host", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__qmv_host() { return PyModule_Create(&module); }
