// Arrays [batch, time, ...] of the layers that run along time, padded batches of them, and the activations that they share.
#pragma once

#include <algorithm>

#include "common.h"

namespace hipcx {

// Rows of an array whose last axis is dense; strides in elements.
struct SequenceRows {
    void* data;  // null: the array is not given
    int64_t batch, row;
};

// Rows that a sequence of a padded batch has, in [0, all]; without an array of them all sequences are whole.
struct SequenceLengths {
    const void* data;
    int64_t stride;  // bytes
    int wide;        // int64
};

__device__ __forceinline__ int64_t LengthOf(const SequenceLengths& l, int64_t b, int64_t all) {
    if (l.data == nullptr) return all;
    const char* const at = static_cast<const char*>(l.data) + b * l.stride;
    const int64_t n = l.wide != 0 ? *reinterpret_cast<const int64_t*>(at) : *reinterpret_cast<const int32_t*>(at);
    return n < 0 ? 0 : n > all ? all : n;
}

constexpr float kLog2E = 1.44269504088896340736f;

// 1 / (1 + exp(-x)): 0 at -inf, 1 at inf, in two instructions of the transcendental unit.
__device__ __forceinline__ float LogisticOf(float x) { return __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(-kLog2E * x)); }

// A dense last axis, and whole elements from one row to the next.
inline SequenceRows RowsOf(const hipcx_array* a, const char* what) {
    if (a == nullptr) return {};
    const int64_t it = ItemSize(a->dtype);
    const int last = a->ndim - 1;
    HIPCX_REQUIRE(TotalSize(a) == 0 || a->shape[last] == 1 || a->strides[last] == it, HIPCX_DIMENSION_ERROR, std::string(what) + ": the last axis must be dense");
    for (int i = 0; i < last; ++i) HIPCX_REQUIRE(a->strides[i] % it == 0, HIPCX_DIMENSION_ERROR, std::string(what) + ": strides must be whole elements");
    return {a->data, a->strides[0] / it, a->ndim > 2 ? a->strides[1] / it : 0};
}

inline void RequireShape(const hipcx_array* a, std::initializer_list<int64_t> shape, int dtype, const std::string& what) {
    if (a == nullptr) return;
    ValidateArray(a, what.c_str());
    HIPCX_REQUIRE(a->dtype == dtype, HIPCX_DTYPE_ERROR, what + ": expected " + DtypeName(dtype) + ", got " + DtypeName(a->dtype));
    HIPCX_REQUIRE(a->ndim == static_cast<int>(shape.size()) && std::equal(shape.begin(), shape.end(), a->shape), HIPCX_DIMENSION_ERROR, what + ": unexpected shape " + ShapeStr(a));
}

inline void RequireDense(const hipcx_array* a, const std::string& what) {
    HIPCX_REQUIRE(a == nullptr || IsContiguous(a), HIPCX_DIMENSION_ERROR, what + ": must be C-contiguous");
}

inline SequenceLengths LengthsOf(const hipcx_array* a, int64_t batch, const std::string& what) {
    if (a == nullptr) return {};
    ValidateArray(a, "lengths");
    HIPCX_REQUIRE(a->dtype == HIPCX_INT32 || a->dtype == HIPCX_INT64, HIPCX_DTYPE_ERROR, what + ": lengths are int32 or int64, got " + DtypeName(a->dtype));
    HIPCX_REQUIRE(a->ndim == 1 && a->shape[0] == batch, HIPCX_DIMENSION_ERROR, what + ": one length for each sequence, got shape " + ShapeStr(a));
    return {a->data, a->strides[0], a->dtype == HIPCX_INT64};
}

}  // namespace hipcx
