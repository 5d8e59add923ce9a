// chainer_amd._host: the routines of sequence.h's kernels -- dropout, the causal convolution and the selective scan -- over the C ABI.
#include <vector>

#include "host.h"

namespace host {
namespace {

// The array itself, or a copy, with a dense last axis.
Ref DenseRows(Array* a) {
    const int last = a->d.ndim - 1;
    if (last < 0 || a->d.shape[last] <= 1 || a->d.strides[last] == ItemSize(a->d.dtype)) return NewRef(a);
    return CopyOf(a, a->d.dtype);
}

Array* Optional(PyObject* x, const char* what) { return Given(x) ? AsArray(x, what) : nullptr; }

Ref DenseRowsOrNone(Array* a) { return a != nullptr ? DenseRows(a) : Ref(); }
Ref ContiguousOrNone(Array* a) { return a != nullptr ? Contiguous(a) : Ref(); }
const hipcx_array* Descriptor(Array* a) { return a != nullptr ? &a->d : nullptr; }

// Empty arrays like the given ones, none for none.
Ref EmptyLikeOrNone(Array* a) { return a != nullptr ? EmptyLike(a, a->d.dtype) : Ref(); }

PyObject* Item(Ref* r) {
    if (*r) return r->release();
    Py_RETURN_NONE;
}

PyObject* Pack(std::initializer_list<Ref*> items) {
    PyObject* t = PyTuple_New(static_cast<Py_ssize_t>(items.size()));
    if (t == nullptr) throw PyError();
    Py_ssize_t i = 0;
    for (Ref* r : items) PyTuple_SET_ITEM(t, i++, Item(r));
    return t;
}

int Activation(PyObject* x) {
    if (!Given(x)) return HIPCX_ACTIVATION_NONE;
    if (PyUnicode_Check(x) && PyUnicode_CompareWithASCIIString(x, "silu") == 0) return HIPCX_ACTIVATION_SILU;
    PyErr_Format(g.exceptions[HIPCX_CHAINERX_ERROR], "unknown activation: %R (None or 'silu')", x);
    throw PyError();
}

int Truth(PyObject* x) {
    if (x == nullptr) return 0;
    const int v = PyObject_IsTrue(x);
    if (v < 0) throw PyError();
    return v;
}

void RequireAxes(const Array* a, int n, const char* what) {
    if (a->d.ndim != n) Raise(HIPCX_DIMENSION_ERROR, "%s must have %d axes, got %d", what, n, a->d.ndim);
}

// [batch, taps - 1, channels] for x and w.
Ref EmptyWindow(const Array* x, const Array* w) {
    const int64_t shape[3] = {x->d.shape[0], w->d.shape[1] > 0 ? w->d.shape[1] - 1 : 0, x->d.shape[2]};
    return Empty(3, shape, x->d.dtype);
}

}  // namespace

HOST_FN(Dropout) {
    HOST_TRY;
    HOST_ARGS("dropout", 3, "x", "ratio", "key", "site", "residual");
    Ref x = Contiguous(AsArray(arg[0], "x"));
    const double ratio = PyFloat_AsDouble(arg[1]);
    if (ratio == -1.0 && PyErr_Occurred()) throw PyError();
    Ref key = Contiguous(AsArray(arg[2], "key"));
    const int64_t site = Given(arg[3]) ? ToInt(arg[3]) : 0;
    Ref residual = ContiguousOrNone(Optional(arg[4], "residual"));
    Ref out = EmptyLike(x.arr(), x.arr()->d.dtype);
    void* stream = Stream();
    Call([&] { return hipcx_dropout(x.d(), ratio, key.d(), site, residual.d(), out.d(), stream); });
    return out.release();
    HOST_CATCH(nullptr);
}

HOST_FN(CausalConv) {
    HOST_TRY;
    HOST_ARGS("causal_conv", 2, "x", "w", "b", "state", "lengths", "activation", "out_state");
    Array *given = AsArray(arg[0], "x"), *filter = AsArray(arg[1], "w");
    RequireAxes(given, 3, "x");
    RequireAxes(filter, 2, "w");
    Ref x = DenseRows(given), w = Contiguous(filter), b = ContiguousOrNone(Optional(arg[2], "b")), state = DenseRowsOrNone(Optional(arg[3], "state"));
    Array* const lengths = Optional(arg[4], "lengths");
    const int activation = Activation(arg[5]);
    Ref new_state = Given(arg[6]) ? NewRef(AsArray(arg[6], "out_state")) : EmptyWindow(given, filter);
    Ref y = EmptyLike(given, given->d.dtype);
    void* stream = Stream();
    Call([&] { return hipcx_causal_conv(x.d(), w.d(), b.d(), state.d(), Descriptor(lengths), activation, y.d(), new_state.d(), stream); });
    return Pack({&y, &new_state});
    HOST_CATCH(nullptr);
}

// (gx, gw, gb or None, gstate or None)
HOST_FN(CausalConvGrad) {
    HOST_TRY;
    HOST_ARGS("causal_conv_grad", 4, "x", "w", "b", "gy", "state", "lengths", "activation", "gnew_state");
    Array *given = AsArray(arg[0], "x"), *filter = AsArray(arg[1], "w"), *bias = Optional(arg[2], "b"), *first = Optional(arg[4], "state");
    RequireAxes(given, 3, "x");
    RequireAxes(filter, 2, "w");
    Ref x = DenseRows(given), w = Contiguous(filter), b = ContiguousOrNone(bias), gy = DenseRows(AsArray(arg[3], "gy")), state = DenseRowsOrNone(first);
    Array* const lengths = Optional(arg[5], "lengths");
    const int activation = Activation(arg[6]);
    Ref gnew = DenseRowsOrNone(Optional(arg[7], "gnew_state"));
    Ref gx = EmptyLike(given, given->d.dtype), gw = EmptyLike(filter, filter->d.dtype), gb = EmptyLikeOrNone(bias), gstate = EmptyLikeOrNone(first);
    Workspace scratch(hipcx_causal_conv_grad_workspace_size(x.d(), w.d()));
    void* stream = Stream();
    Call([&] {
        return hipcx_causal_conv_grad(x.d(), w.d(), b.d(), state.d(), Descriptor(lengths), activation, gy.d(), gnew.d(), gx.d(), gw.d(), gb.d(), gstate.d(), scratch.ptr,
                                      scratch.bytes, stream);
    });
    return Pack({&gx, &gw, &gb, &gstate});
    HOST_CATCH(nullptr);
}

HOST_FN(SelectiveScan) {
    HOST_TRY;
    HOST_ARGS("selective_scan", 5, "u", "delta", "a", "b", "c", "d", "z", "delta_bias", "delta_softplus", "state", "lengths", "out_state");
    Array *given = AsArray(arg[0], "u"), *decay = AsArray(arg[2], "a");
    RequireAxes(given, 3, "u");
    RequireAxes(decay, 2, "a");
    Ref u = DenseRows(given), delta = DenseRows(AsArray(arg[1], "delta")), a = Contiguous(decay), b = DenseRows(AsArray(arg[3], "b")), c = DenseRows(AsArray(arg[4], "c"));
    Ref d = ContiguousOrNone(Optional(arg[5], "d")), z = DenseRowsOrNone(Optional(arg[6], "z")), bias = ContiguousOrNone(Optional(arg[7], "delta_bias"));
    const int softplus = Truth(arg[8]);
    Ref state = ContiguousOrNone(Optional(arg[9], "state"));
    Array* const lengths = Optional(arg[10], "lengths");
    const int64_t of_state[3] = {given->d.shape[0], given->d.shape[2], decay->d.shape[1]};
    Ref new_state = Given(arg[11]) ? NewRef(AsArray(arg[11], "out_state")) : Empty(3, of_state, HIPCX_FLOAT32);
    Ref y = EmptyLike(given, given->d.dtype);
    Workspace scratch(hipcx_selective_scan_workspace_size(u.d(), a.d()));
    void* stream = Stream();
    Call([&] {
        return hipcx_selective_scan(u.d(), delta.d(), a.d(), b.d(), c.d(), d.d(), z.d(), bias.d(), softplus, state.d(), Descriptor(lengths), y.d(), new_state.d(), scratch.ptr,
                                    scratch.bytes, stream);
    });
    return Pack({&y, &new_state});
    HOST_CATCH(nullptr);
}

// (gu, gdelta, ga, gb, gc, gd, gz, gdelta_bias, gstate); None for what is not given
HOST_FN(SelectiveScanGrad) {
    HOST_TRY;
    HOST_ARGS("selective_scan_grad", 6, "u", "delta", "a", "b", "c", "gy", "d", "z", "delta_bias", "delta_softplus", "state", "lengths", "gnew_state");
    Array *given = AsArray(arg[0], "u"), *step = AsArray(arg[1], "delta"), *decay = AsArray(arg[2], "a"), *in = AsArray(arg[3], "b"), *out = AsArray(arg[4], "c");
    Array *skip = Optional(arg[6], "d"), *gate = Optional(arg[7], "z"), *offset = Optional(arg[8], "delta_bias"), *first = Optional(arg[10], "state");
    RequireAxes(given, 3, "u");
    RequireAxes(decay, 2, "a");
    Ref u = DenseRows(given), delta = DenseRows(step), a = Contiguous(decay), b = DenseRows(in), c = DenseRows(out), gy = DenseRows(AsArray(arg[5], "gy"));
    Ref d = ContiguousOrNone(skip), z = DenseRowsOrNone(gate), bias = ContiguousOrNone(offset);
    const int softplus = Truth(arg[9]);
    Ref state = ContiguousOrNone(first);
    Array* const lengths = Optional(arg[11], "lengths");
    Ref gnew = ContiguousOrNone(Optional(arg[12], "gnew_state"));
    Ref gu = EmptyLikeOrNone(given), gdelta = EmptyLikeOrNone(step), ga = EmptyLikeOrNone(decay), gb = EmptyLikeOrNone(in), gc = EmptyLikeOrNone(out);
    Ref gd = EmptyLikeOrNone(skip), gz = EmptyLikeOrNone(gate), gbias = EmptyLikeOrNone(offset), gstate = EmptyLikeOrNone(first);
    Workspace scratch(hipcx_selective_scan_grad_workspace_size(u.d(), a.d(), b.d()));
    void* stream = Stream();
    Call([&] {
        return hipcx_selective_scan_grad(u.d(), delta.d(), a.d(), b.d(), c.d(), d.d(), z.d(), bias.d(), softplus, state.d(), Descriptor(lengths), gy.d(), gnew.d(), gu.d(),
                                         gdelta.d(), ga.d(), gb.d(), gc.d(), gd.d(), gz.d(), gbias.d(), gstate.d(), scratch.ptr, scratch.bytes, stream);
    });
    return Pack({&gu, &gdelta, &ga, &gb, &gc, &gd, &gz, &gbias, &gstate});
    HOST_CATCH(nullptr);
}

}  // namespace host
