// Host side of the operators of a step that verifies drafted tokens: checks of their operands, outputs and scratch from torch's allocator,
// one call of the CUDA launcher on the current stream.  Python's share of a call (checks and twenty arguments through ctypes)
// was 9 to 18 us, as long as or longer than the kernels of a small step; here it is 3.5 to 7.5.
//
// The launchers live in the libraries that kernels/loader.py compiles; the first call that wants one has it loaded.
#include <Python.h>

#include <ATen/ATen.h>
#include <ATen/cuda/CUDAContext.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <algorithm>
#include <initializer_list>
#include <string>

#include "../draft_args.h"

namespace {

PyObject* kernel_error = nullptr;       // exception types of kernels/loader.py
PyObject* kernel_unavailable = nullptr;
PyObject* load = nullptr;               // load(name): compiles and loads a launcher, and hands its address to set_launcher
PyObject* launches = nullptr;           // kernels/loader.py::LAUNCHES, a list of one number

struct Refused {};                      // the Python error is set

[[noreturn]] void refuse(const char* what, const std::string& why, PyObject* type = nullptr) {
    PyErr_SetString(type ? type : kernel_error, (std::string(what) + ": " + why).c_str());
    throw Refused();
}
std::string shape_text(at::IntArrayRef s) {
    std::string r = "[";
    for (size_t i = 0; i < s.size(); ++i) r += (i ? ", " : "") + std::to_string(s[i]);
    return r + "]";
}
std::string type_text(const at::Tensor& t) { return std::string(c10::toString(t.scalar_type())) + " " + shape_text(t.sizes()); }

const at::Tensor& tensor(const char* what, const char* name, PyObject* o) {
    if (!THPVariable_Check(o)) refuse(what, std::string(name) + " must be a tensor");
    return THPVariable_Unpack(o);
}
const at::Tensor* maybe(const char* what, const char* name, PyObject* o) { return o == Py_None ? nullptr : &tensor(what, name, o); }
long long integer(const char* what, const char* name, PyObject* o) {
    const long long v = PyLong_AsLongLong(o);
    if (v == -1 && PyErr_Occurred()) {
        PyErr_Clear();
        refuse(what, std::string(name) + " must be a whole number");
    }
    return v;
}

void ints(const char* what, const char* name, const at::Tensor& t, std::initializer_list<int64_t> shape) {
    if (t.scalar_type() != at::kInt || t.sizes() != at::IntArrayRef(shape) || !t.is_contiguous())
        refuse(what, std::string(name) + " must be a contiguous int32 tensor " + shape_text(at::IntArrayRef(shape)) + ", got " + type_text(t));
}
int* words(const at::Tensor& t) { return t.data_ptr<int>(); }
unsigned* bits(const at::Tensor& t) { return reinterpret_cast<unsigned*>(t.data_ptr<int>()); }
// The current device's stream, for operands that all live on that device.
cudaStream_t stream_of(const char* what, std::initializer_list<const at::Tensor*> ts) {
    for (const at::Tensor* t : ts)
        if (t && !t->is_cuda()) {
            if (!at::hasCUDA() || c10::cuda::device_count() == 0)
                refuse(what, "no CUDA device: this engine runs on sm_100a kernels only and has no CPU path", kernel_unavailable);
            refuse(what, "operands must live on the CUDA device");
        }
    const int dev = c10::cuda::current_device();
    for (const at::Tensor* t : ts)
        if (t && t->get_device() != dev)
            refuse(what, "operands must live on the current CUDA device (cuda:" + std::to_string(dev) + "), not on cuda:" + std::to_string(t->get_device()));
    return c10::cuda::getCurrentCUDAStream(dev).stream();
}
at::Tensor fresh(at::IntArrayRef shape, at::ScalarType type, const at::Tensor& like) {
    return at::detail::empty_cuda(shape, type, like.device(), std::nullopt);
}
// `count` elements of `base` from `offset` on, as a tensor of `shape` of its own
PyObject* part(const at::Tensor& base, int64_t offset, at::IntArrayRef shape) {
    auto impl = c10::make_intrusive<c10::TensorImpl>(c10::Storage(base.storage()), base.key_set(), base.dtype());
    impl->set_sizes_contiguous(shape);
    impl->set_storage_offset(offset);
    return THPVariable_Wrap(at::Tensor(std::move(impl)));
}
// a launcher has returned; `kernels` of ours were launched where that is no error
void launched(const char* what, int rc, int kernels) {
    if (rc == 0) {
        PyObject* sum = PyLong_FromLongLong(PyLong_AsLongLong(PyList_GetItem(launches, 0)) + kernels);
        if (!sum || PyList_SetItem(launches, 0, sum) < 0 || PyErr_Occurred()) throw Refused();
        return;
    }
    refuse(what, rc == -1   ? "bad argument (dtype or shape combination not accepted)"
                 : rc == -2 ? "size not supported by this kernel"
                 : rc == -3 ? "size beyond the kernel's stated maximum"
                            : "CUDA error " + std::to_string(rc));
}
int dtype_code(const char* what, const at::Tensor& t) {
    if (t.scalar_type() == at::kFloat) return 0;
    if (t.scalar_type() == at::kBFloat16) return 1;
    refuse(what, std::string("dtype ") + c10::toString(t.scalar_type()) + " is not taken by the kernels (float32, bfloat16)");
}

struct Pools { int64_t N, K, P, d; int code; };
Pools pools(const char* what, const at::Tensor& k, const at::Tensor& v) {
    if (k.dim() != 4 || v.sizes() != k.sizes() || v.scalar_type() != k.scalar_type())
        refuse(what, "keys and values must be pools of one shape and dtype, [pages, kv heads, page, d]");
    if (!k.is_contiguous() || !v.is_contiguous()) refuse(what, "the pools must be contiguous");
    const Pools p = {k.size(0), k.size(1), k.size(2), k.size(3), dtype_code(what, k)};
    if (!p.K || !p.P || !p.d || p.N * p.P > 0x7fffffff)
        refuse(what, "the pools' sizes " + shape_text(k.sizes()) + " are not taken (up to 2^31 - 1 cache slots, nothing empty)");
    return p;
}

int (*step_tables_fn)(const StArgs*, cudaStream_t) = nullptr;
int (*write_fn)(const CwArgs*, cudaStream_t) = nullptr;
int (*verify_fn)(const VdArgs*, cudaStream_t) = nullptr;
int (*chunks_f32_fn)(const ChCall*, int, cudaStream_t) = nullptr;
int (*chunks_mma_fn)(const ChCall*, int, cudaStream_t) = nullptr;
int (*chunks_tc_fn)(const ChCall*, cudaStream_t) = nullptr;

template <typename F> F* loaded(F*& fn, const char* name) {
    if (!fn) {
        PyObject* r = PyObject_CallFunction(load, "s", name);
        if (!r) throw Refused();
        Py_DECREF(r);
    }
    return fn;
}

template <typename F> PyObject* guarded(const char* name, Py_ssize_t got, Py_ssize_t wanted, F f) {
    if (got != wanted) {
        PyErr_Format(PyExc_TypeError, "%s takes %zd arguments, got %zd", name, wanted, got);
        return nullptr;
    }
    try {
        return f();
    } catch (const Refused&) {           // the error is set
        return nullptr;
    } catch (...) {                      // torch's own, as the exceptions that its operators raise (torch.OutOfMemoryError among them)
        torch::translate_exception_to_python(std::current_exception());
        return nullptr;
    }
}

PyObject* step_tables(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded("step_tables", n, 10, [&]() -> PyObject* {
        const char* w = "step_tables";
        const at::Tensor &cached = tensor(w, "cached", a[0]), &counts = tensor(w, "counts", a[1]), &held = tensor(w, "held", a[2]),
                         &tables = tensor(w, "tables", a[3]), &free_pages = tensor(w, "free_pages", a[4]),
                         &free_count = tensor(w, "free_count", a[5]), &err = tensor(w, "err", a[9]);
        const long long P = integer(w, "page_size", a[6]), num_pages = integer(w, "num_pages", a[7]), most = integer(w, "max_tokens", a[8]);
        if (tables.dim() != 2 || tables.size(1) == 0) refuse(w, "the tables must be [requests, pages]");
        const int64_t R = tables.size(0), W = tables.size(1), F = free_pages.numel();
        if (R < 1 || R > 4096) refuse(w, std::to_string(R) + " requests (1 to 4096 are taken)");
        if (P < 1 || P > 0x7fffffff || num_pages < 0 || num_pages > 0x7fffffff || num_pages * P > 0x7fffffff)
            refuse(w, std::to_string(num_pages) + " pages of " + std::to_string(P) + " tokens (1 to 2^31 - 1 cache slots are taken)");
        if (most < 0 || most > (1 << 30) || R * W > (1 << 30) || F > 0x7fffffff) refuse(w, "sizes beyond 2^30");
        ints(w, "cached", cached, {R});
        ints(w, "counts", counts, {R});
        ints(w, "held", held, {R});
        ints(w, "tables", tables, {R, W});
        ints(w, "free_pages", free_pages, {F});
        ints(w, "free_count", free_count, {1});
        ints(w, "err", err, {1});
        const cudaStream_t st = stream_of(w, {&cached, &counts, &held, &tables, &free_pages, &free_count, &err});
        // tables, held, free_count, q_start, q_len, positions, token_req, slots, one behind the other
        at::Tensor out = fresh({R * W + 3 * R + 1 + 3 * most}, at::kInt, tables);
        const StArgs args = {words(cached), words(counts), words(held), words(tables), words(free_pages),
                             words(free_count), words(out), bits(err), (int)R, (int)W, (int)F, (int)P, (int)num_pages, (int)most};
        launched(w, loaded(step_tables_fn, "aie_step_tables")(&args, st), 1);
        PyObject* t = PyTuple_New(8);
        if (!t) throw Refused();
        int64_t at_ = R * W;
        PyTuple_SET_ITEM(t, 0, part(out, 0, {R, W}));
        const int64_t sizes[7] = {R, 1, R, R, most, most, most};
        for (int i = 0; i < 7; ++i) {
            PyTuple_SET_ITEM(t, i + 1, part(out, at_, {sizes[i]}));
            at_ += sizes[i];
        }
        return t;
    });
}

PyObject* write_kv_slots(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded("write_kv_slots", n, 6, [&]() -> PyObject* {
        const char* w = "write_kv_slots";
        const at::Tensor &k = tensor(w, "k", a[0]), &v = tensor(w, "v", a[1]), &kp = tensor(w, "k_pages", a[2]), &vp = tensor(w, "v_pages", a[3]),
                         &slots = tensor(w, "slots", a[4]), &err = tensor(w, "err", a[5]);
        const Pools p = pools(w, kp, vp);
        if (k.dim() != 3 || k.size(1) != p.K || k.size(2) != p.d || v.sizes() != k.sizes() || v.scalar_type() != k.scalar_type())
            refuse(w, "keys " + type_text(k) + " and values " + type_text(v) + " must be [T, " + std::to_string(p.K) + ", " + std::to_string(p.d) + "], of one dtype");
        const int code = dtype_code(w, k);
        const int64_t T = k.size(0);
        if (T && p.d > 1 && (k.stride(2) != 1 || v.stride(2) != 1)) refuse(w, "the elements of a head must be contiguous");
        if (2 * p.K * p.d > 0x7fffffff || T > 0x7fffffff) refuse(w, "too many rows, or a token's rows are too long");
        ints(w, "slots", slots, {T});
        ints(w, "err", err, {1});
        const cudaStream_t st = stream_of(w, {&slots, &k, &v, &kp, &vp, &err});
        if (T) {
            const CwArgs args = {k.data_ptr(), v.data_ptr(), kp.data_ptr(), vp.data_ptr(), words(slots), bits(err),
                                 k.stride(0), k.stride(1), v.stride(0), v.stride(1), code, p.code, (int)T, (int)p.N, (int)p.P, (int)p.K, (int)p.d};
            launched(w, loaded(write_fn, "aie_write_kv_slots")(&args, st), 1);
        }
        Py_RETURN_NONE;
    });
}

PyObject* verify_drafts(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded("verify_drafts", n, 8, [&]() -> PyObject* {
        const char* w = "verify_drafts";
        const at::Tensor &target = tensor(w, "target_probs", a[0]), &start = tensor(w, "q_start", a[1]), &ids = tensor(w, "draft_tokens", a[2]);
        const at::Tensor *lens = maybe(w, "draft_len", a[3]), *guess = maybe(w, "draft_probs", a[4]);
        const at::Tensor &accept = tensor(w, "accept_draws", a[5]), &pick = tensor(w, "token_draws", a[6]), &err = tensor(w, "err", a[7]);
        if (target.dim() != 2 || ids.dim() != 2) refuse(w, "target_probs must be [T, V] and draft_tokens [R, N]");
        const int64_t T = target.size(0), V = target.size(1), R = ids.size(0), N = ids.size(1);
        if (V < 1 || V > (1 << 20)) refuse(w, "a vocabulary of " + std::to_string(V) + " (1 to 1048576 are taken)");
        if (T > 0x7fffffff || R * (N + 1) > 0x7fffffff) refuse(w, "too many rows");
        auto floats = [&](const char* name, const at::Tensor& t, std::initializer_list<int64_t> shape) {
            if (t.scalar_type() != at::kFloat || t.sizes() != at::IntArrayRef(shape))
                refuse(w, std::string(name) + " must be float32 " + shape_text(at::IntArrayRef(shape)) + ", got " + type_text(t));
        };
        floats("target_probs", target, {T, V});
        if (guess) floats("draft_probs", *guess, {R, N, V});
        floats("accept_draws", accept, {R, N});
        floats("token_draws", pick, {R});
        if (V > 1 && (target.stride(1) != 1 || (guess && guess->stride(2) != 1))) refuse(w, "the probabilities of a row must be contiguous");
        if (!accept.is_contiguous() || !pick.is_contiguous()) refuse(w, "draws must be contiguous");
        ints(w, "q_start", start, {R});
        ints(w, "draft_tokens", ids, {R, N});
        if (lens) ints(w, "draft_len", *lens, {R});
        ints(w, "err", err, {1});
        const cudaStream_t st = stream_of(w, {&start, &ids, lens, &err, &target, guess, &accept, &pick});
        at::Tensor tokens = fresh({R, N + 1}, at::kInt, ids), emitted = fresh({R}, at::kInt, ids);
        if (R) {
            const VdArgs args = {target.data_ptr<float>(), words(start), words(ids), lens ? words(*lens) : nullptr,
                                 guess ? guess->data_ptr<float>() : nullptr, accept.data_ptr<float>(), pick.data_ptr<float>(), words(tokens),
                                 words(emitted), bits(err), target.stride(0), guess ? guess->stride(0) : 0, guess ? guess->stride(1) : 0,
                                 (int)T, (int)V, (int)R, (int)N};
            launched(w, loaded(verify_fn, "aie_verify_drafts")(&args, st), 1);
        }
        PyObject* t = PyTuple_New(2);
        if (!t) throw Refused();
        PyTuple_SET_ITEM(t, 0, THPVariable_Wrap(std::move(tokens)));
        PyTuple_SET_ITEM(t, 1, THPVariable_Wrap(std::move(emitted)));
        return t;
    });
}

// The forms of the attention: FLOAT32 (and bfloat16 that the others do not take); MMA, items of 32 rows by the line; TCGEN05, items of 256 rows by the
// line; MMA + S, items of 32 rows, a cluster of S blocks for every request and key head.
enum { FLOAT32 = 0, MMA = 16, TCGEN05 = 1 };

// Which of them takes a call, by what the host knows: tokens, requests, and how many keys a request can have (the table's width; a
// window).  The least of the times that each would take, in us, fitted to 643 calls (1 to 64 requests of 1 to 200 tokens behind 40 to 20,000,
// four head layouts, tables as wide as the longest request: there the choice takes 1.2 % more than the best form of each call on average, 40 % where
// it is worst): a fixed part, one for every key tile of the busiest block, one for every part of an item that is joined.  Only these proportions
// count.  A wider table is taken for longer requests: with 512 pages of 16 one request of five tokens behind 1,000 goes by the line (10.1 us) and
// not by clusters (7.2), with 256 eight requests behind 500 to 2,000 do (20.4 and 18.7).
int chunk_form(int code, const Pools& p, int64_t R, int64_t W, int64_t T, int64_t G, int64_t window, int64_t sm_count) {
    if (code != 1 || (p.d != 64 && p.d != 128)) return FLOAT32;
    auto up = [](int64_t a, int64_t b) { return (a + b - 1) / b; };
    const int64_t items = R * p.K, rows = up(T * G, R), tile = p.d == 128 ? 64 : 128;
    int64_t keys = W * p.P;
    if (window > 0) keys = std::min(keys, window + up(T, R));
    const int64_t tiles = up(keys, tile);
    int form = MMA;
    const int64_t all = items * up(rows, 32), blocks = 2 * sm_count;
    double least = 6.5 + 1.5 * up(all * tiles, blocks) + (all < blocks ? 0.1 * std::min((double)tiles, (double)blocks / all) : 0.0);
    if (p.P % 8 == 0 && (128 % p.P == 0 || p.P % 128 == 0) && p.N * p.K * p.P / 8 < 0x7fffffff) {
        // a tile of more than 128 rows takes both streams of a block for every key tile, one of fewer rows takes one of them
        const int64_t rest = rows % 256, pairs = rows / 256 + (rest > 128), lone = rest > 0 && rest <= 128;
        const double t = 12.5 + (p.d == 128 ? 1.6 : 1.0) * up(items * (pairs + lone) * up(keys, 128), sm_count) * (2 * pairs + lone) / (pairs + lone);
        if (t < least) {
            least = t;
            form = TCGEN05;
        }
    }
    // clusters: every block there at once, a row tile or little more each, and few key tiles, since nothing evens out unequal lengths
    for (int S = 8; S >= 2 && rows <= 32; S /= 2) {
        const int64_t each = up(tiles, S);
        if (items * S > blocks || each > 8) continue;
        const double t = 5.0 + 0.9 * each;
        if (t < least) {
            least = t;
            form = MMA + S;
        }
    }
    return form;
}

PyObject* paged_attention_chunks(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded("paged_attention_chunks", n, 12, [&]() -> PyObject* {
        const char* w = "paged_attention_chunks";
        const at::Tensor &q = tensor(w, "q", a[0]), &kp = tensor(w, "k_pages", a[1]), &vp = tensor(w, "v_pages", a[2]),
                         &start = tensor(w, "q_start", a[3]), &len = tensor(w, "q_len", a[4]), &ctx = tensor(w, "ctx_len", a[5]),
                         &table = tensor(w, "block_table", a[6]), &err = tensor(w, "err", a[9]);
        const double scale = PyFloat_AsDouble(a[7]);
        if (scale == -1.0 && PyErr_Occurred()) {
            PyErr_Clear();
            refuse(w, "scale must be a number");
        }
        const long long window = integer(w, "window", a[8]);
        const at::Tensor* given = maybe(w, "out", a[10]);
        long long form = integer(w, "form", a[11]);
        const Pools p = pools(w, kp, vp);
        // (the launchers check the rest of what a form takes; the types of the operands they do not see)
        if (form > FLOAT32 && p.code != 1) refuse(w, "form " + std::to_string(form) + " takes bfloat16 pools only");
        if (q.dim() != 3 || q.size(2) != p.d || q.size(1) == 0 || q.size(1) % p.K || q.scalar_type() != kp.scalar_type())
            refuse(w, "queries " + type_text(q) + " must be [T, a multiple of " + std::to_string(p.K) + ", " + std::to_string(p.d) + "] in the pools' dtype");
        const int64_t T = q.size(0), H = q.size(1);
        if (p.d % 8 || p.d > 256) refuse(w, "head size " + std::to_string(p.d) + " must be a multiple of 8, at most 256");
        if (T * H > 0x7fffffff || p.N == 0) refuse(w, "too many rows of queries, or no pages");
        if (table.dim() != 2 || table.size(1) == 0) refuse(w, "the block table must be [requests, pages]");
        const int64_t R = table.size(0), W = table.size(1);
        if (R > 0x7fffffff || W * p.P > 0x7fffffff - 1024) refuse(w, "the table names more than 2^31 keys a request");
        if (window < 0 || window > 0x7fffffff) refuse(w, "a window is 0 (none) or a number of keys");
        const int64_t grid = 4 << p.code;                             // elements in 16 bytes
        if (T && (q.stride(2) != 1 || (q.stride(0) | q.stride(1)) % grid || (size_t)q.data_ptr() % 16))
            refuse(w, "every head's row of q must be contiguous and start on 16 bytes");
        if (((size_t)kp.data_ptr() | (size_t)vp.data_ptr()) % 16) refuse(w, "the pools must start on 16 bytes");
        if (given && (given->sizes() != q.sizes() || given->scalar_type() != q.scalar_type() || !given->is_contiguous() || (size_t)given->data_ptr() % 16))
            refuse(w, "out must be contiguous, of q's shape and dtype, and start on 16 bytes");
        ints(w, "q_start", start, {R});
        ints(w, "q_len", len, {R});
        ints(w, "ctx_len", ctx, {R});
        ints(w, "block_table", table, {R, W});
        ints(w, "err", err, {1});
        const cudaStream_t st = stream_of(w, {&start, &len, &ctx, &table, &err, &q, &kp, &vp, given});
        at::Tensor out = given ? *given : fresh(q.sizes(), q.scalar_type(), q);
        if (T && R) {
            const int64_t G = H / p.K;
            const int64_t sm_count = at::cuda::getCurrentDeviceProperties()->multiProcessorCount;
            if (form < 0) form = chunk_form(p.code, p, R, W, T, G, window, sm_count);
            const int64_t wide = form == FLOAT32 ? (p.d <= 64 ? 64 : p.d <= 128 ? 128 : 256) : p.d;
            const int64_t M = form == TCGEN05 ? 256 : 32;
            const int64_t blocks = form > MMA ? 0 : sm_count * (form == MMA ? 2 : 1), parts = 2 * blocks * M;
            // parts [parts][wide], their maxima and sums [parts][2], what is to be joined [blocks] int4
            at::Tensor scratch;
            if (blocks) scratch = fresh({parts * (wide + 2) + 4 * blocks}, at::kFloat, q);
            float* s = blocks ? scratch.data_ptr<float>() : nullptr;
            const ChCall call = {q.data_ptr(), kp.data_ptr(), vp.data_ptr(), out.data_ptr(), words(start), words(len), words(ctx),
                                 words(table), s, s ? s + parts * wide : nullptr, s ? reinterpret_cast<int4*>(s + parts * (wide + 2)) : nullptr, q.stride(0), q.stride(1), (int)R, (int)W, (int)T,
                                 (int)p.N, (int)p.P, (int)H, (int)p.K, (int)G, (int)p.d, (int)window, (float)(scale * 1.4426950408889634), bits(err), (int)blocks};
            launched(w, form == TCGEN05   ? loaded(chunks_tc_fn, "aie_attention_chunks_tc")(&call, st)
                        : form == FLOAT32 ? loaded(chunks_f32_fn, "aie_attention_chunks_f32")(&call, p.code, st)
                                          : loaded(chunks_mma_fn, "aie_attention_chunks_bf16")(&call, (int)form - MMA, st),
                     form > MMA ? 1 : 2);      // clusters join their parts themselves
        }
        return THPVariable_Wrap(std::move(out));
    });
}

PyObject* set_up(PyObject*, PyObject* args) {
    if (!PyArg_ParseTuple(args, "OOOO!", &kernel_error, &kernel_unavailable, &load, &PyList_Type, &launches)) return nullptr;
    Py_INCREF(kernel_error);
    Py_INCREF(kernel_unavailable);
    Py_INCREF(load);
    Py_INCREF(launches);
    Py_RETURN_NONE;
}
PyObject* set_launcher(PyObject*, PyObject* args) {
    const char* name;
    unsigned long long address;
    if (!PyArg_ParseTuple(args, "sK", &name, &address)) return nullptr;
    const std::string s = name;
#define SET(f, text) \
    if (s == text) f = reinterpret_cast<decltype(f)>(address)
    SET(step_tables_fn, "aie_step_tables");
    SET(write_fn, "aie_write_kv_slots");
    SET(verify_fn, "aie_verify_drafts");
    SET(chunks_f32_fn, "aie_attention_chunks_f32");
    SET(chunks_mma_fn, "aie_attention_chunks_bf16");
    SET(chunks_tc_fn, "aie_attention_chunks_tc");
#undef SET
    Py_RETURN_NONE;
}

PyMethodDef methods[] = {
    {"set_up", set_up, METH_VARARGS, "exception types (KernelError, KernelUnavailable), load(name), the list that counts launches"},
    {"set_launcher", set_launcher, METH_VARARGS, "name of a launcher, its address"},
    {"step_tables", (PyCFunction)(void (*)(void))step_tables, METH_FASTCALL, nullptr},
    {"write_kv_slots", (PyCFunction)(void (*)(void))write_kv_slots, METH_FASTCALL, nullptr},
    {"verify_drafts", (PyCFunction)(void (*)(void))verify_drafts, METH_FASTCALL, nullptr},
    {"paged_attention_chunks", (PyCFunction)(void (*)(void))paged_attention_chunks, METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_aie_draft_ops", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__aie_draft_ops() { return PyModule_Create(&module); }
