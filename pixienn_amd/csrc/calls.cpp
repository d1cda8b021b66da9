// Calls of the C ABI with torch tensors as they come from Python: checking a tensor, taking its address and converting the
// arguments costs a few hundred nanoseconds here, and five to eight microseconds through ctypes, which is what a small
// layer's kernel takes.  An entry point's argument types come from its declaration.  A call with anything but plain
// tensors, None and numbers is not made here: it answers None, and the caller goes through ctypes and its checks.
#include <torch/csrc/autograd/python_variable.h>

#include "pixienn_hip.h"

#include <algorithm>
#include <climits>
#include <exception>
#include <string_view>
#include <tuple>
#include <type_traits>
#include <utility>
#include <vector>

namespace {

// Thrown for an argument that is left to the caller.
struct NotHere {};

template<typename A>
A argument(PyObject* o)
{
    if constexpr (std::is_same_v<A, float*> || std::is_same_v<A, const float*>) {
        // a tensor the kernels take: fp32, contiguous, on a HIP device
        if (o == Py_None) return nullptr;
        if (!THPVariable_CheckExact(o)) throw NotHere{};
        const at::Tensor& t = THPVariable_Unpack(o);
        if (t.scalar_type() != at::kFloat || !t.is_cuda() || !t.is_contiguous()) throw NotHere{};
        return static_cast<float*>(t.data_ptr());
    } else if constexpr (std::is_pointer_v<A>) {
        if (o == Py_None) return nullptr;
        if (!PyLong_CheckExact(o)) throw NotHere{};
        void* p = PyLong_AsVoidPtr(o);
        if (PyErr_Occurred()) { PyErr_Clear(); throw NotHere{}; }
        return reinterpret_cast<A>(p);
    } else if constexpr (std::is_floating_point_v<A>) {
        if (!PyFloat_CheckExact(o)) throw NotHere{};
        return static_cast<A>(PyFloat_AS_DOUBLE(o));
    } else {
        static_assert(std::is_integral_v<A>, "a kind of argument of its own");
        if (!PyLong_CheckExact(o)) throw NotHere{};
        int overflow = 0;
        const long long v = PyLong_AsLongLongAndOverflow(o, &overflow);
        if (overflow || (std::is_same_v<A, int> && (v < INT_MIN || v > INT_MAX)) || (std::is_unsigned_v<A> && v < 0) ||
            (std::is_same_v<A, unsigned> && v > static_cast<long long>(UINT_MAX)))
            throw NotHere{};
        return static_cast<A>(v);
    }
}

template<typename F>
struct Entry;

// `self` holds the entry point's address in the loaded library.
template<typename... A>
struct Entry<int (*)(A...)> {
    using Function = int (*)(A...);

    template<size_t... I>
    static int call(Function f, PyObject* const* args, std::index_sequence<I...>)
    {
        const std::tuple<A...> values{ argument<A>(args[I])... };
        int rc;
        PyThreadState* const state = PyEval_SaveThread();
        rc = std::apply(f, values);
        PyEval_RestoreThread(state);
        return rc;
    }

    static PyObject* vectorcall(PyObject* self, PyObject* const* args, Py_ssize_t count)
    {
        if (count != static_cast<Py_ssize_t>(sizeof...(A))) Py_RETURN_NONE;
        const auto f = reinterpret_cast<Function>(PyLong_AsVoidPtr(self));
        try {
            return PyLong_FromLong(call(f, args, std::index_sequence_for<A...>{}));
        } catch (const NotHere&) {
        } catch (const std::exception&) {       // a tensor without storage, say: the caller's route reports it
        }
        Py_RETURN_NONE;
    }

    // which arguments are tensors
    static PyObject* tensors()
    {
        PyObject* t = PyTuple_New(sizeof...(A));
        Py_ssize_t i = 0;
        if (t) ((PyTuple_SET_ITEM(t, i++, PyBool_FromLong(std::is_same_v<A, float*> || std::is_same_v<A, const float*>))), ...);
        return t;
    }
};

struct Known {
    PyMethodDef def;
    PyObject* (*tensors)();
};

template<auto F>
Known known(const char* name)
{
    using E = Entry<decltype(F)>;
    return Known{ { name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(&E::vectorcall)), METH_FASTCALL, nullptr },
                  &E::tensors };
}

#define ENTRY(name) known<&name>(#name)

Known entries[] = {
    ENTRY(pxh_bn_train_act_forward), ENTRY(pxh_bn_train_act_shortcut_forward), ENTRY(pxh_bn_folded_act_forward),
    ENTRY(pxh_bn_folded_act_shortcut_forward), ENTRY(pxh_bn_folded_act_maxpool_forward), ENTRY(pxh_bias_act_forward),
    ENTRY(pxh_bn_act_backward), ENTRY(pxh_bn_act_backward_clipped), ENTRY(pxh_bias_act_backward),
    ENTRY(pxh_bias_act_backward_clipped), ENTRY(pxh_axpy), ENTRY(pxh_fill_f32), ENTRY(pxh_route_forward),
    ENTRY(pxh_route_backward), ENTRY(pxh_maxpool_forward), ENTRY(pxh_maxpool_backward), ENTRY(pxh_shortcut_backward_clipped),
    ENTRY(pxh_yolo_activate), ENTRY(pxh_yolo_detections_append), ENTRY(pxh_rescale_clip), ENTRY(pxh_adam_update),
    ENTRY(pxh_sgd_update), ENTRY(pxh_adamw_update_table),
};

// ---------------------------------------------------------------- layers of token models
// Their tensors have types and row strides, so the calls take the tensors of the Python function themselves and form the entry
// point's arguments.  What does not fit is left to the caller, which says what is wrong with it.

int type_of(const at::Tensor& t)
{
    switch (t.scalar_type()) {
    case at::kFloat: return PXH_F32;
    case at::kBFloat16: return PXH_BF16;
    case at::kHalf: return PXH_F16;
    case at::kFloat8_e4m3fn: return PXH_E4M3;
    default: throw NotHere{};
    }
}

const at::Tensor& tensor_of(PyObject* o)
{
    if (!THPVariable_CheckExact(o)) throw NotHere{};
    const at::Tensor& t = THPVariable_Unpack(o);
    if (!t.is_cuda()) throw NotHere{};
    return t;
}

// A tensor of rows: two dimensions, of which the last is packed, or any number of packed ones.
struct Rows {
    char* data = nullptr;
    long long rows = 0, width = 0, stride = 0;
    int type = 0;
    bool given = false;         // a tensor of no values has no address either, and is not a missing one

    Rows() = default;
    explicit Rows(PyObject* o)
    {
        if (o == Py_None) return;
        given = true;
        const at::Tensor& t = tensor_of(o);
        const auto dims = t.dim();
        if (dims == 0) throw NotHere{};
        type = type_of(t);
        width = t.size(dims - 1);
        if (dims == 2) {
            rows = t.size(0);
            if (t.stride(1) != 1 && width > 1) throw NotHere{};
            stride = rows > 1 ? t.stride(0) : std::max<long long>(t.stride(0), width);
        } else {
            if (!t.is_contiguous()) throw NotHere{};
            rows = width ? t.numel() / width : 0;
            stride = width;
        }
        data = static_cast<char*>(t.data_ptr());
        shape = t.sizes();
    }
    // of the same shape and, if asked, type
    const Rows& like(const Rows& o, int of_type) const
    {
        if (given && (shape != o.shape || type != of_type)) throw NotHere{};
        return *this;
    }

    at::IntArrayRef shape;
};

// A packed tensor of n values of a type, or None.
template<typename V>
V* packed(PyObject* o, long long n, at::ScalarType type)
{
    if (o == Py_None) return nullptr;
    const at::Tensor& t = tensor_of(o);
    if (t.scalar_type() != type || !t.is_contiguous() || t.numel() != n) throw NotHere{};
    return static_cast<V*>(t.data_ptr());
}

float* floats(PyObject* o, long long n) { return packed<float>(o, n, at::kFloat); }

struct Space {
    void* data = nullptr;
    size_t bytes = 0;
    explicit Space(PyObject* o)
    {
        if (o == Py_None) return;
        const at::Tensor& t = tensor_of(o);
        if (!t.is_contiguous()) throw NotHere{};
        data = t.data_ptr();
        bytes = static_cast<size_t>(t.numel()) * t.element_size();
    }
};

struct Targets {
    const void* data = nullptr;
    int wide = 0;
    Targets(PyObject* o, long long rows)
    {
        if (o == Py_None) return;
        const at::Tensor& t = tensor_of(o);
        wide = t.scalar_type() == at::kLong;
        if ((!wide && t.scalar_type() != at::kInt) || !t.is_contiguous() || t.numel() != rows) throw NotHere{};
        data = t.data_ptr();
    }
};

int fits(long long v)
{
    if (v > INT_MAX) throw NotHere{};
    return static_cast<int>(v);
}

// The row stride of a tensor that may be None.
long long stride_of(const Rows& r) { return r.given ? r.stride : 0; }

// f() with the interpreter free, its status as a number.
template<typename F>
PyObject* status(const F& f)
{
    int rc;
    PyThreadState* const state = PyEval_SaveThread();
    rc = f();
    PyEval_RestoreThread(state);
    return PyLong_FromLong(rc);
}

// body(args) where there are `count` arguments; None where it leaves the call.
template<size_t COUNT, typename F>
PyObject* guarded(PyObject* const* args, Py_ssize_t count, const F& body)
{
    if (count != static_cast<Py_ssize_t>(COUNT)) Py_RETURN_NONE;
    try {
        return body(args);
    } catch (const NotHere&) {
    } catch (const std::exception&) {
    }
    Py_RETURN_NONE;
}

// self: the entry point's address.  (x, y, weight, residual, sum, scales, rstd, eps, group, stream)
PyObject* rms_norm_forward(PyObject* self, PyObject* const* args, Py_ssize_t count)
{
    return guarded<10>(args, count, [&](PyObject* const* a) {
        const auto f = reinterpret_cast<decltype(&pxh_rms_norm_forward)>(PyLong_AsVoidPtr(self));
        const Rows x(a[0]), y(a[1]), residual(a[3]), sum(a[4]);
        const bool eight = y.type == PXH_E4M3;
        y.like(x, eight ? PXH_E4M3 : x.type);
        residual.like(x, x.type);
        sum.like(x, x.type);
        const int weight_type = type_of(tensor_of(a[2]));
        void* const weight = packed<void>(a[2], x.width, weight_type == PXH_F32 ? at::kFloat : weight_type == PXH_BF16 ? at::kBFloat16 : at::kHalf);
        const int group = argument<int>(a[8]);
        float* const scales = eight ? floats(a[5], x.rows * (group ? (x.width + 127) / 128 : 1)) : nullptr;
        float* const rstd = floats(a[6], x.rows);
        const float eps = argument<float>(a[7]);
        void* const stream = argument<void*>(a[9]);
        const int width = fits(x.width);
        return status([&] {
            return f(x.data, residual.data, sum.data, weight, y.data, scales, rstd, x.type, weight_type, y.type, x.rows, width, x.stride,
                     stride_of(residual), stride_of(sum), y.stride, group, eps, stream);
        });
    });
}

// (dy, h, weight, rstd, dx, dw, dsum, accumulate, workspace, stream)
PyObject* rms_norm_backward(PyObject* self, PyObject* const* args, Py_ssize_t count)
{
    return guarded<10>(args, count, [&](PyObject* const* a) {
        const auto f = reinterpret_cast<decltype(&pxh_rms_norm_backward)>(PyLong_AsVoidPtr(self));
        const Rows dy(a[0]), h(a[1]), dx(a[4]), dsum(a[6]);
        h.like(dy, dy.type);
        dx.like(dy, dy.type);
        dsum.like(dy, dy.type);
        const int weight_type = type_of(tensor_of(a[2]));
        void* const weight = packed<void>(a[2], dy.width, weight_type == PXH_F32 ? at::kFloat : weight_type == PXH_BF16 ? at::kBFloat16 : at::kHalf);
        float* const rstd = floats(a[3], dy.rows);
        float* const dw = floats(a[5], dy.width);
        const int accumulate = argument<int>(a[7]);
        const Space space(a[8]);
        void* const stream = argument<void*>(a[9]);
        const int width = fits(dy.width);
        return status([&] {
            return f(dy.data, h.data, weight, rstd, dsum.data, dx.data, dw, dy.type, weight_type, dy.rows, width, dy.stride, stride_of(h),
                     stride_of(dsum), stride_of(dx), accumulate, space.data, space.bytes, stream);
        });
    });
}

// (logits, targets, logp, entropy, lse, top_logp, top_ids, scale, workspace, stream)
PyObject* token_logprobs_forward(PyObject* self, PyObject* const* args, Py_ssize_t count)
{
    return guarded<10>(args, count, [&](PyObject* const* a) {
        const auto f = reinterpret_cast<decltype(&pxh_token_logprobs_forward)>(PyLong_AsVoidPtr(self));
        const Rows logits(a[0]);
        const Targets targets(a[1], logits.rows);
        float* const logp = floats(a[2], logits.rows);
        float* const entropy = floats(a[3], logits.rows);
        float* const lse = floats(a[4], logits.rows);
        int top = 0, *ids = nullptr;
        float* best = nullptr;
        if ((a[5] == Py_None) != (a[6] == Py_None)) throw NotHere{};
        if (a[6] != Py_None) {
            const at::Tensor& t = tensor_of(a[6]);
            if (t.dim() == 0) throw NotHere{};
            top = fits(t.size(t.dim() - 1));
            ids = packed<int>(a[6], logits.rows * top, at::kInt);
            best = floats(a[5], logits.rows * top);
        }
        const float scale = argument<float>(a[7]);
        const Space space(a[8]);
        void* const stream = argument<void*>(a[9]);
        const int vocab = fits(logits.width);
        return status([&] {
            return f(logits.data, targets.data, logp, entropy, lse, best, ids, logits.type, targets.wide, logits.rows, vocab, logits.stride, top,
                     scale, space.data, space.bytes, stream);
        });
    });
}

// (logits, targets, lse, d_logp, dlogits, entropy, d_entropy, scale, stream)
PyObject* token_logprobs_backward(PyObject* self, PyObject* const* args, Py_ssize_t count)
{
    return guarded<9>(args, count, [&](PyObject* const* a) {
        const auto f = reinterpret_cast<decltype(&pxh_token_logprobs_backward)>(PyLong_AsVoidPtr(self));
        const Rows logits(a[0]), d(a[4]);
        d.like(logits, logits.type);
        const Targets targets(a[1], logits.rows);
        const float* const lse = floats(a[2], logits.rows);
        const float* const d_logp = floats(a[3], logits.rows);
        const float* const entropy = floats(a[5], logits.rows);
        const float* const d_entropy = floats(a[6], logits.rows);
        const float scale = argument<float>(a[7]);
        void* const stream = argument<void*>(a[8]);
        const int vocab = fits(logits.width);
        return status([&] {
            return f(logits.data, targets.data, lse, entropy, d_logp, d_entropy, d.data, logits.type, targets.wide, logits.rows, vocab,
                     logits.stride, stride_of(d), scale, stream);
        });
    });
}

// (logits, targets, d_logp, dlogits, logp, entropy, lse, d_entropy, scale, stream)
PyObject* token_logprobs_forward_train(PyObject* self, PyObject* const* args, Py_ssize_t count)
{
    return guarded<10>(args, count, [&](PyObject* const* a) {
        const auto f = reinterpret_cast<decltype(&pxh_token_logprobs_forward_train)>(PyLong_AsVoidPtr(self));
        const Rows logits(a[0]), d(a[3]);
        d.like(logits, logits.type);
        const Targets targets(a[1], logits.rows);
        const float* const d_logp = floats(a[2], logits.rows);
        float* const logp = floats(a[4], logits.rows);
        float* const entropy = floats(a[5], logits.rows);
        float* const lse = floats(a[6], logits.rows);
        const float* const d_entropy = floats(a[7], logits.rows);
        const float scale = argument<float>(a[8]);
        void* const stream = argument<void*>(a[9]);
        const int vocab = fits(logits.width);
        return status([&] {
            return f(logits.data, targets.data, d_logp, d_entropy, d.data, logp, entropy, lse, logits.type, targets.wide, logits.rows, vocab,
                     logits.stride, stride_of(d), scale, stream);
        });
    });
}

// ---------------------------------------------------------------- calls that look at the tensors' device too
// The last arguments are the current device's index and its current stream: a tensor of another device is left to the caller.

struct Device {
    long long index;
    void* stream;

    const at::Tensor& tensor(PyObject* o) const
    {
        const at::Tensor& t = tensor_of(o);
        if (t.get_device() != index) throw NotHere{};
        return t;
    }
    Rows rows(PyObject* o) const
    {
        if (o != Py_None) tensor(o);
        return Rows(o);
    }
    // A packed tensor of n values, or None.
    template<typename V>
    V* packed(PyObject* o, long long n, at::ScalarType type) const
    {
        if (o != Py_None) tensor(o);
        return ::packed<V>(o, n, type);
    }
    float* floats(PyObject* o, long long n) const { return packed<float>(o, n, at::kFloat); }
    Space space(PyObject* o) const
    {
        if (o != Py_None) tensor(o);
        return Space(o);
    }
    // Weights of a norm and their type.
    void* weights(PyObject* o, long long n, int& type) const
    {
        const at::Tensor& t = tensor(o);
        type = type_of(t);
        if (type == PXH_E4M3) throw NotHere{};
        return packed<void>(o, n, t.scalar_type());
    }
    // Tokens that are there, of 32 or 64 bits.
    Targets tokens(PyObject* o, long long n) const
    {
        tensor(o);
        return Targets(o, n);
    }
};

// body(args, device, entry point) where there are COUNT arguments and the device's two; None where it leaves the call.
template<auto* F, size_t COUNT, typename B>
PyObject* on_device(PyObject* self, PyObject* const* args, Py_ssize_t count, const B& body)
{
    return guarded<COUNT + 2>(args, count, [&](PyObject* const* a) {
        const Device device{ argument<long long>(a[COUNT]), argument<void*>(a[COUNT + 1]) };
        return body(a, device, reinterpret_cast<decltype(F)>(PyLong_AsVoidPtr(self)));
    });
}

// (table, tokens, y, scale)
PyObject* embedding_forward(PyObject* self, PyObject* const* args, Py_ssize_t count)
{
    return on_device<&pxh_embedding_forward, 4>(self, args, count, [](PyObject* const* a, const Device& d, auto f) {
        const Rows table = d.rows(a[0]), y = d.rows(a[2]);
        if (!table.given || !y.given || y.width != table.width || y.type != table.type) throw NotHere{};
        const Targets tokens = d.tokens(a[1], y.rows);
        const float scale = argument<float>(a[3]);
        const int vocab = fits(table.rows), width = fits(table.width);
        return status([&] {
            return f(table.data, tokens.data, y.data, table.type, tokens.wide, y.rows, vocab, width, table.stride, y.stride, scale, d.stream);
        });
    });
}

// (dy, tokens, d, scale, accumulate, workspace)
PyObject* embedding_backward(PyObject* self, PyObject* const* args, Py_ssize_t count)
{
    return on_device<&pxh_embedding_backward, 6>(self, args, count, [](PyObject* const* a, const Device& d, auto f) {
        const Rows dy = d.rows(a[0]), table = d.rows(a[2]);
        if (!dy.given || !table.given || dy.width != table.width || (table.type != dy.type && table.type != PXH_F32)) throw NotHere{};
        const Targets tokens = d.tokens(a[1], dy.rows);
        const float scale = argument<float>(a[3]);
        const int accumulate = argument<int>(a[4]), vocab = fits(table.rows), width = fits(dy.width);
        const Space space = d.space(a[5]);
        return status([&] {
            return f(dy.data, tokens.data, table.data, dy.type, table.type, tokens.wide, dy.rows, vocab, width, dy.stride, table.stride, scale,
                     accumulate, space.data, space.bytes, d.stream);
        });
    });
}

// (x, y, weight, bias, residual, sum, mean, rstd, eps)
PyObject* layer_norm_forward(PyObject* self, PyObject* const* args, Py_ssize_t count)
{
    return on_device<&pxh_layer_norm_forward, 9>(self, args, count, [](PyObject* const* a, const Device& d, auto f) {
        const Rows x = d.rows(a[0]), y = d.rows(a[1]), residual = d.rows(a[4]), sum = d.rows(a[5]);
        if (!x.given || !y.given) throw NotHere{};
        y.like(x, x.type);
        residual.like(x, x.type);
        sum.like(x, x.type);
        int type, bias_type;
        void* const weight = d.weights(a[2], x.width, type);
        void* const bias = a[3] == Py_None ? nullptr : d.weights(a[3], x.width, bias_type);
        if (bias && bias_type != type) throw NotHere{};
        float* const mean = d.floats(a[6], x.rows);
        float* const rstd = d.floats(a[7], x.rows);
        const float eps = argument<float>(a[8]);
        const int width = fits(x.width);
        return status([&] {
            return f(x.data, residual.data, sum.data, weight, bias, y.data, mean, rstd, x.type, type, x.rows, width, x.stride, stride_of(residual),
                     stride_of(sum), y.stride, eps, d.stream);
        });
    });
}

// (dy, h, weight, mean, rstd, dx, dw, db, dsum, accumulate, workspace)
PyObject* layer_norm_backward(PyObject* self, PyObject* const* args, Py_ssize_t count)
{
    return on_device<&pxh_layer_norm_backward, 11>(self, args, count, [](PyObject* const* a, const Device& d, auto f) {
        const Rows dy = d.rows(a[0]), h = d.rows(a[1]), dx = d.rows(a[5]), dsum = d.rows(a[8]);
        if (!dy.given || !h.given || !dx.given) throw NotHere{};
        h.like(dy, dy.type);
        dx.like(dy, dy.type);
        dsum.like(dy, dy.type);
        int type;
        void* const weight = d.weights(a[2], dy.width, type);
        float* const mean = d.floats(a[3], dy.rows);
        float* const rstd = d.floats(a[4], dy.rows);
        float* const dw = d.floats(a[6], dy.width);
        float* const db = d.floats(a[7], dy.width);
        const int accumulate = argument<int>(a[9]), width = fits(dy.width);
        const Space space = d.space(a[10]);
        return status([&] {
            return f(dy.data, h.data, weight, mean, rstd, dsum.data, dx.data, dw, db, dy.type, type, dy.rows, width, dy.stride, h.stride,
                     stride_of(dsum), dx.stride, accumulate, space.data, space.bytes, d.stream);
        });
    });
}

// A number that may be None.
long long number_or(PyObject* o, long long none) { return o == Py_None ? none : argument<long long>(o); }

// The sequences that a call's tokens belong to, and their states.
struct Sequences {
    const int* starts = nullptr;
    int count = 0;

    Sequences(const Device& d, const Rows& tokens, PyObject* starts_, PyObject* sequences)
    {
        if (starts_ != Py_None) {
            const long long n = d.tensor(starts_).numel();
            if (n < 1) throw NotHere{};
            starts = d.packed<int>(starts_, n, at::kInt);
            count = fits(n - 1);
        } else {
            const long long n = number_or(sequences, tokens.shape.size() == 3 ? tokens.shape[0] : tokens.rows > 0);
            if (n < 0) throw NotHere{};
            count = fits(n);
        }
    }
};

struct States {
    const Device& d;
    long long count, width, slot_count = -1;
    const int* slots;

    States(const Device& device, PyObject* slots_, long long sequences, long long width_)
        : d(device), count(sequences), width(width_), slots(d.packed<int>(slots_, sequences, at::kInt)) {}
    float* of(PyObject* o)
    {
        if (o == Py_None) return nullptr;
        const at::Tensor& t = d.tensor(o);
        if (t.dim() != 2 || t.size(1) != width || (slot_count >= 0 && t.size(0) != slot_count)) throw NotHere{};
        slot_count = t.size(0);
        return d.floats(o, slot_count * width);
    }
    int places() const { return slot_count < 0 ? 0 : fits(slot_count); }
};

const Rows& needed(const Rows& r)
{
    if (!r.given) throw NotHere{};
    return r;
}

// (x, update, y, gate, starts, sequences, state, final, slots, saved, workspace)
PyObject* gated_scan_forward(PyObject* self, PyObject* const* args, Py_ssize_t count)
{
    return on_device<&pxh_gated_scan_forward, 11>(self, args, count, [](PyObject* const* a, const Device& d, auto f) {
        const Rows x = needed(d.rows(a[0])), u = needed(d.rows(a[1])), y = needed(d.rows(a[2])), gate = d.rows(a[3]);
        u.like(x, x.type);
        y.like(x, x.type);
        gate.like(x, x.type);
        const Sequences q(d, x, a[4], a[5]);
        States states(d, a[8], q.count, x.width);
        float* const state = states.of(a[6]);
        float* const final = states.of(a[7]);
        float* const saved = d.floats(a[9], (x.rows + PXH_SCAN_SAVED - 1) / PXH_SCAN_SAVED * x.width);
        const Space space = d.space(a[10]);
        const int width = fits(x.width), places = states.places();
        return status([&] {
            return f(x.data, u.data, gate.data, y.data, q.starts, state, final, states.slots, saved, x.type, x.rows, width, q.count, places,
                     x.stride, u.stride, stride_of(gate), y.stride, space.data, space.bytes, d.stream);
        });
    });
}

// (dy, x, update, saved, dx, dupdate, gate, dgate, starts, sequences, state, d_final, d_state, slots, workspace)
PyObject* gated_scan_backward(PyObject* self, PyObject* const* args, Py_ssize_t count)
{
    return on_device<&pxh_gated_scan_backward, 15>(self, args, count, [](PyObject* const* a, const Device& d, auto f) {
        const Rows dy = needed(d.rows(a[0])), x = needed(d.rows(a[1])), u = needed(d.rows(a[2])), dx = needed(d.rows(a[4])),
                   du = needed(d.rows(a[5])), gate = d.rows(a[6]), dgate = d.rows(a[7]);
        for (const Rows* r: { &x, &u, &dx, &du, &gate, &dgate }) r->like(dy, dy.type);
        const Sequences q(d, dy, a[8], a[9]);
        States states(d, a[13], q.count, dy.width);
        float* const state = states.of(a[10]);
        float* const d_final = states.of(a[11]);
        float* const d_state = states.of(a[12]);
        float* const saved = d.floats(a[3], (dy.rows + PXH_SCAN_SAVED - 1) / PXH_SCAN_SAVED * dy.width);
        const Space space = d.space(a[14]);
        const int width = fits(dy.width), places = states.places();
        return status([&] {
            return f(dy.data, x.data, u.data, gate.data, saved, dx.data, du.data, dgate.data, q.starts, state, d_final, d_state, states.slots, dy.type,
                     dy.rows, width, q.count, places, dy.stride, x.stride, u.stride, stride_of(gate), dx.stride, du.stride, stride_of(dgate),
                     space.data, space.bytes, d.stream);
        });
    });
}

// (x, update, y, state, gate, slots)
PyObject* gated_scan_step(PyObject* self, PyObject* const* args, Py_ssize_t count)
{
    return on_device<&pxh_gated_scan_step, 6>(self, args, count, [](PyObject* const* a, const Device& d, auto f) {
        const Rows x = needed(d.rows(a[0])), u = needed(d.rows(a[1])), y = needed(d.rows(a[2])), gate = d.rows(a[4]);
        u.like(x, x.type);
        y.like(x, x.type);
        gate.like(x, x.type);
        States states(d, a[5], x.rows, x.width);
        if (a[3] == Py_None) throw NotHere{};
        float* const state = states.of(a[3]);
        const int width = fits(x.width), places = states.places();
        return status([&] {
            return f(x.data, u.data, gate.data, y.data, state, states.slots, x.type, x.rows, width, places, x.stride, u.stride, stride_of(gate),
                     y.stride, d.stream);
        });
    });
}

// A packed tensor of two dimensions.
template<typename V>
V* table_of(const Device& d, PyObject* o, at::ScalarType type, long long& rows, long long& columns)
{
    const at::Tensor& t = d.tensor(o);
    if (t.dim() != 2 || (rows >= 0 && t.size(0) != rows) || (columns >= 0 && t.size(1) != columns)) throw NotHere{};
    rows = t.size(0);
    columns = t.size(1);
    return d.packed<V>(o, rows * columns, type);
}

// (logits, scores, out_scores, parents, tokens, ended, end_token, scale, workspace)
PyObject* beam_select(PyObject* self, PyObject* const* args, Py_ssize_t count)
{
    return on_device<&pxh_beam_select, 9>(self, args, count, [](PyObject* const* a, const Device& d, auto f) {
        const Rows logits = needed(d.rows(a[0]));
        long long batch = -1, beams = -1, best = -1;
        const float* const scores = table_of<float>(d, a[1], at::kFloat, batch, beams);
        float* const out = table_of<float>(d, a[2], at::kFloat, batch, best);
        int* const parents = table_of<int>(d, a[3], at::kInt, batch, best);
        int* const tokens = table_of<int>(d, a[4], at::kInt, batch, best);
        if (logits.rows != batch * beams) throw NotHere{};
        const unsigned char* ended = nullptr;
        if (a[5] != Py_None) {
            const at::ScalarType type = d.tensor(a[5]).scalar_type();
            if (type != at::kBool && type != at::kByte) throw NotHere{};
            ended = d.packed<unsigned char>(a[5], batch * beams, type);
        }
        const int end_token = argument<int>(a[6]), vocab = fits(logits.width);
        const float scale = argument<float>(a[7]);
        const Space space = d.space(a[8]);
        const int items = fits(batch), of_item = fits(beams), continuations = fits(best);
        return status([&] {
            return f(logits.data, scores, ended, out, parents, tokens, logits.type, items, of_item, vocab, logits.stride, continuations, end_token, scale,
                     space.data, space.bytes, d.stream);
        });
    });
}

// ([tensors], parents)
PyObject* beam_reorder(PyObject* self, PyObject* const* args, Py_ssize_t count)
{
    return on_device<&pxh_beam_reorder, 2>(self, args, count, [](PyObject* const* a, const Device& d, auto f) {
        if (!PyList_CheckExact(a[0])) throw NotHere{};
        long long batch = -1, beams = -1;
        const int* const parents = table_of<int>(d, a[1], at::kInt, batch, beams);
        const Py_ssize_t n = PyList_GET_SIZE(a[0]);
        std::vector<void*> data(n);
        std::vector<long long> bytes(n), strides(n);
        for (Py_ssize_t i = 0; i < n; ++i) {
            const at::Tensor& t = d.tensor(PyList_GET_ITEM(a[0], i));
            if (t.dim() == 0 || t.size(0) != batch * beams) throw NotHere{};
            const long long rows = t.size(0), size = static_cast<long long>(t.element_size());
            bytes[i] = rows ? t.numel() / rows * size : 0;
            if (t.is_contiguous()) strides[i] = bytes[i];
            else if (t.dim() == 2 && (t.stride(1) == 1 || t.size(1) == 1)) strides[i] = rows > 1 ? t.stride(0) * size : bytes[i];
            else throw NotHere{};
            data[i] = t.data_ptr();
        }
        const int tensors = fits(n), items = fits(batch), of_item = fits(beams);
        return status([&] { return f(tensors, data.data(), bytes.data(), strides.data(), parents, items, of_item, d.stream); });
    });
}

#define FUNCTION(name) \
    PyMethodDef { "pxh_" #name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(&name)), METH_FASTCALL, nullptr }

PyMethodDef functions[] = { FUNCTION(rms_norm_forward), FUNCTION(rms_norm_backward), FUNCTION(token_logprobs_forward),
                            FUNCTION(token_logprobs_backward), FUNCTION(token_logprobs_forward_train) };

PyMethodDef layers[] = { FUNCTION(embedding_forward), FUNCTION(embedding_backward), FUNCTION(layer_norm_forward), FUNCTION(layer_norm_backward),
                         FUNCTION(gated_scan_forward), FUNCTION(gated_scan_backward), FUNCTION(gated_scan_step),
                         FUNCTION(beam_select), FUNCTION(beam_reorder) };

// bind_function(name, address) -> the callable that takes a Python function's own arguments and the stream, or None
PyObject* bind_function(PyObject*, PyObject* args)
{
    const char* name;
    PyObject* address;
    if (!PyArg_ParseTuple(args, "sO!", &name, &PyLong_Type, &address)) return nullptr;
    for (PyMethodDef& def: functions)
        if (std::string_view(def.ml_name) == name) return PyCFunction_New(&def, address);
    for (PyMethodDef& def: layers)
        if (std::string_view(def.ml_name) == name) return PyCFunction_New(&def, address);
    Py_RETURN_NONE;
}

template<size_t N>
PyObject* names_of(const PyMethodDef (&defs)[N])
{
    PyObject* list = PyList_New(0);
    for (const PyMethodDef& def: defs) {
        PyObject* s = list ? PyUnicode_FromString(def.ml_name) : nullptr;
        if (!s || PyList_Append(list, s)) { Py_XDECREF(s); Py_XDECREF(list); return nullptr; }
        Py_DECREF(s);
    }
    return list;
}

// functions(), layers() -> their names
PyObject* function_names(PyObject*, PyObject*) { return names_of(functions); }
PyObject* layer_names(PyObject*, PyObject*) { return names_of(layers); }

// bind(name, address) -> (callable, which arguments are tensors), or None for an entry point that is not made here
PyObject* bind(PyObject*, PyObject* args)
{
    const char* name;
    PyObject* address;
    if (!PyArg_ParseTuple(args, "sO!", &name, &PyLong_Type, &address)) return nullptr;
    for (Known& k: entries) {
        if (std::string_view(k.def.ml_name) != name) continue;
        PyObject* f = PyCFunction_New(&k.def, address);
        PyObject* t = f ? k.tensors() : nullptr;
        if (!t) { Py_XDECREF(f); return nullptr; }
        return Py_BuildValue("(NN)", f, t);
    }
    Py_RETURN_NONE;
}

// names() -> the entry points that are made here
PyObject* names(PyObject*, PyObject*)
{
    PyObject* list = PyList_New(0);
    for (const Known& k: entries) {
        PyObject* s = list ? PyUnicode_FromString(k.def.ml_name) : nullptr;
        if (!s || PyList_Append(list, s)) { Py_XDECREF(s); Py_XDECREF(list); return nullptr; }
        Py_DECREF(s);
    }
    return list;
}

PyMethodDef methods[] = { { "bind", bind, METH_VARARGS, nullptr }, { "names", names, METH_NOARGS, nullptr },
                          { "bind_function", bind_function, METH_VARARGS, nullptr }, { "functions", function_names, METH_NOARGS, nullptr },
                          { "layers", layer_names, METH_NOARGS, nullptr },
                          { nullptr, nullptr, 0, nullptr } };
PyModuleDef module = { PyModuleDef_HEAD_INIT, "_calls", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr };

}  // namespace

PyMODINIT_FUNC PyInit__calls() { return PyModule_Create(&module); }
