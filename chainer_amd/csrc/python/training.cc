// chainer_amd._host: layer norm and AdamW over the C ABI.
#include <vector>

#include "host.h"

namespace host {
namespace {

Array* Optional(PyObject* x, const char* what) { return Given(x) ? AsArray(x, what) : nullptr; }
Ref ContiguousOrNone(Array* a) { return a != nullptr ? Contiguous(a) : Ref(); }

// The array itself, or a copy, with a dense last axis and rows that are equally far apart.
Ref EvenRows(Array* a) {
    const int last = a->d.ndim - 1, it = ItemSize(a->d.dtype);
    if (last < 0 || Size(a) == 0) return NewRef(a);
    bool even = a->d.shape[last] == 1 || a->d.strides[last] == it;
    int64_t expect = 0;
    bool seen = false;  // an inner axis (of a stride of 0, perhaps)
    for (int i = last - 1; i >= 0 && even; --i) {
        if (a->d.shape[i] == 1) continue;
        even = seen ? a->d.strides[i] == expect : a->d.strides[i] % it == 0;
        seen = true;
        expect = a->d.strides[i] * a->d.shape[i];
    }
    return even ? NewRef(a) : CopyOf(a, a->d.dtype);
}

double ToDouble(PyObject* x, double otherwise) {
    if (!Given(x)) return otherwise;
    const double v = PyFloat_AsDouble(x);
    if (v == -1.0 && PyErr_Occurred()) throw PyError();
    return v;
}

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

}  // namespace

// (y, mean, inv_std)
HOST_FN(LayerNorm) {
    HOST_TRY;
    HOST_ARGS("layer_norm", 1, "x", "gamma", "beta", "eps");
    Array* given = AsArray(arg[0], "x");
    Ref x = EvenRows(given), gamma = ContiguousOrNone(Optional(arg[1], "gamma")), beta = ContiguousOrNone(Optional(arg[2], "beta"));
    const double eps = ToDouble(arg[3], 2e-5);
    const int stats = given->d.dtype == HIPCX_FLOAT64 ? HIPCX_FLOAT64 : HIPCX_FLOAT32, axes = given->d.ndim > 0 ? given->d.ndim - 1 : 0;
    Ref y = EmptyLike(given, given->d.dtype), mean = Empty(axes, given->d.shape, stats), inv_std = Empty(axes, given->d.shape, stats);
    void* stream = Stream();
    Call([&] { return hipcx_layer_norm(x.d(), gamma.d(), beta.d(), eps, y.d(), mean.d(), inv_std.d(), stream); });
    return Pack({&y, &mean, &inv_std});
    HOST_CATCH(nullptr);
}

// (gx, ggamma or None, gbeta or None)
HOST_FN(LayerNormGrad) {
    HOST_TRY;
    HOST_ARGS("layer_norm_grad", 5, "x", "gamma", "gout", "mean", "inv_std", "beta_dtype");
    Array *given = AsArray(arg[0], "x"), *weights = Optional(arg[1], "gamma");
    Ref x = EvenRows(given), gamma = ContiguousOrNone(weights), gy = EvenRows(AsArray(arg[2], "gout"));
    Ref mean = Contiguous(AsArray(arg[3], "mean")), inv_std = Contiguous(AsArray(arg[4], "inv_std"));
    if (given->d.ndim < 1) Raise(HIPCX_DIMENSION_ERROR, "layer_norm: x needs an axis");
    const int64_t cols[1] = {given->d.shape[given->d.ndim - 1]};
    Ref gx = EmptyLike(given, given->d.dtype), ggamma = weights != nullptr ? EmptyLike(weights, weights->d.dtype) : Ref();
    Ref gbeta = Given(arg[5]) ? Empty(1, cols, DtypeCode(arg[5])) : Ref();
    Workspace scratch(ggamma || gbeta ? hipcx_layer_norm_grad_workspace_size(x.d()) : 0);
    void* stream = Stream();
    Call([&] {
        return hipcx_layer_norm_grad(x.d(), gamma.d(), gy.d(), mean.d(), inv_std.d(), gx.d(), ggamma.d(), gbeta.d(), scratch.ptr, scratch.bytes, stream);
    });
    return Pack({&gx, &ggamma, &gbeta});
    HOST_CATCH(nullptr);
}

// In place; `states`: (m, v, m_scale, v_scale, master) for every parameter.
HOST_FN(AdamWUpdate) {
    HOST_TRY;
    HOST_ARGS("adamw_update", 4, "params", "grads", "states", "t", "alpha", "beta1", "beta2", "eps", "eta", "weight_decay_rate", "seed");
    Ref lists[3];
    for (int i = 0; i < 3; ++i) {
        lists[i] = Ref(PySequence_List(arg[i]));
        if (!lists[i]) throw PyError();
    }
    const Py_ssize_t n = PyList_GET_SIZE(lists[0].get());
    if (PyList_GET_SIZE(lists[1].get()) != n || PyList_GET_SIZE(lists[2].get()) != n) Raise(HIPCX_DIMENSION_ERROR, "adamw_update: one gradient and one state per parameter are needed");
    std::vector<const hipcx_array*> arrays[7];  // params, grads, m, v, m_scale, v_scale, master
    std::vector<Ref> keep;
    keep.reserve(static_cast<size_t>(n) * 2);
    for (Py_ssize_t i = 0; i < n; ++i) {
        Array *p = AsArray(PyList_GET_ITEM(lists[0].get(), i), "parameter"), *g = AsArray(PyList_GET_ITEM(lists[1].get(), i), "gradient");
        if (Size(p) != Size(g)) Raise(HIPCX_DIMENSION_ERROR, "adamw_update: a gradient needs its parameter's size");
        Ref dense = Contiguous(g);
        keep.push_back(Reshape(dense.arr(), p->d.ndim, p->d.shape));
        arrays[0].push_back(&p->d);
        arrays[1].push_back(keep.back().d());
        Ref state(PySequence_Tuple(PyList_GET_ITEM(lists[2].get(), i)));
        if (!state) throw PyError();
        if (PyTuple_GET_SIZE(state.get()) != 5) Raise(HIPCX_CHAINERX_ERROR, "adamw_update: a state is (m, v, m_scale, v_scale, master)");
        static const char* const names[5] = {"m", "v", "m_scale", "v_scale", "master"};
        for (int k = 0; k < 5; ++k) {
            PyObject* const item = PyTuple_GET_ITEM(state.get(), k);
            Array* const a = k < 2 || Given(item) ? AsArray(item, names[k]) : nullptr;
            arrays[2 + k].push_back(a != nullptr ? &a->d : nullptr);
        }
        keep.push_back(std::move(state));
    }
    Array* const steps = IsArray(arg[3]) ? AsArray(arg[3], "t") : nullptr;
    const int64_t t = steps != nullptr ? 0 : ToInt(arg[3]);
    const double alpha = ToDouble(arg[4], 0.001), beta1 = ToDouble(arg[5], 0.9), beta2 = ToDouble(arg[6], 0.999), eps = ToDouble(arg[7], 1e-8), eta = ToDouble(arg[8], 1.0),
                 decay = ToDouble(arg[9], 0.0);
    const int64_t seed = Given(arg[10]) ? ToInt(arg[10]) : 0;
    void* stream = Stream();
    Call([&] {
        return hipcx_adamw_many(arrays[0].data(), arrays[1].data(), arrays[2].data(), arrays[3].data(), arrays[4].data(), arrays[5].data(), arrays[6].data(), static_cast<int>(n), t,
                                steps != nullptr ? &steps->d : nullptr, alpha, beta1, beta2, eps, eta, decay, seed, stream);
    });
    Py_RETURN_NONE;
    HOST_CATCH(nullptr);
}

}  // namespace host
