// Dropout whose mask is drawn from a counter-based generator wherever it is needed and never stored.
#include <algorithm>
#include <cmath>

#include "common.h"
#include "philox.h"

namespace hipcx {
namespace {

struct DropoutArgs {
    const void* x;
    const void* residual;  // may be null
    void* out;
    const int64_t* key;  // {seed, step}
    int64_t n;           // elements
    int64_t first;       // the launch's first thread
    uint32_t site, threshold;
    double scale;
};

constexpr int kPerCounter = 8;  // elements that share a counter, 16 bits each

template <typename T>
struct __attribute__((packed, aligned(alignof(T)))) Eight {
    T v[kPerCounter];
};

// One rounding to T: the sum with the residual is a multiply-add in 32 bits or more.
template <typename T, bool RES>
__device__ __forceinline__ T Dropped(bool kept, T x, T residual, compute_t<T> scale) {
    using C = compute_t<T>;
    if constexpr (RES) return kept ? static_cast<T>(__builtin_elementwise_fma(static_cast<C>(x), scale, static_cast<C>(residual))) : residual;
    return kept ? static_cast<T>(static_cast<C>(x) * scale) : static_cast<T>(0);
}

// A counter to a thread.  Eight numbers of 16 bits from each, rather than four of 32: the generator's 20 wide products (5.6 cycles each) are 112 cycles of a wave's 256 or 512
// elements, at float16 two and a half times, with four numbers five times what its memory lets pass.  Bound by memory: 65536 x 2048 float16 and a residual 138 us, 5.8 TB/s
// (a copy of 256 MB: 4.9); 128 x 650 float32 2.4 us, a launch.
template <typename T, bool RES>
__global__ __launch_bounds__(256) void DropoutKernel(DropoutArgs p) {
    const int64_t group = p.first + static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x, at = group * kPerCounter;
    if (at >= p.n) return;
    const T* const x = static_cast<const T*>(p.x) + at;
    const T* const residual = RES ? static_cast<const T*>(p.residual) + at : nullptr;
    T* const out = static_cast<T*>(p.out) + at;
    const bool whole = at + kPerCounter <= p.n;
    Eight<T> xv{}, rv{};
    if (whole) {
        xv = *reinterpret_cast<const Eight<T>*>(x);
        if constexpr (RES) rv = *reinterpret_cast<const Eight<T>*>(residual);
    }
    const uint64_t seed = static_cast<uint64_t>(p.key[0]), step = static_cast<uint64_t>(p.key[1]);
    uint32_t c[4] = {static_cast<uint32_t>(group), p.site, static_cast<uint32_t>(step), static_cast<uint32_t>(step >> 32)};
    Philox(c, static_cast<uint32_t>(seed), static_cast<uint32_t>(seed >> 32));
    const auto kept = [&](int i) { return (i % 2 == 0 ? c[i / 2] & 0xffffu : c[i / 2] >> 16) >= p.threshold; };
    const auto scale = static_cast<compute_t<T>>(p.scale);
    if (whole) {
#pragma unroll
        for (int i = 0; i < kPerCounter; ++i) xv.v[i] = Dropped<T, RES>(kept(i), xv.v[i], rv.v[i], scale);
        *reinterpret_cast<Eight<T>*>(out) = xv;
    } else {
#pragma unroll
        for (int i = 0; i < kPerCounter; ++i) {
            if (at + i < p.n) out[i] = Dropped<T, RES>(kept(i), x[i], RES ? residual[i] : static_cast<T>(0), scale);
        }
    }
}

}  // namespace
}  // namespace hipcx

using namespace hipcx;

extern "C" int hipcx_dropout(const hipcx_array* x, double ratio, const hipcx_array* key, int64_t site, const hipcx_array* residual, const hipcx_array* out,
                             void* stream) {
    return Guard([&] {
        ValidateArray(x, "x");
        ValidateArray(key, "key");
        ValidateArray(out, "out");
        if (residual != nullptr) ValidateArray(residual, "residual");
        HIPCX_REQUIRE(IsFloatDtype(x->dtype), HIPCX_DTYPE_ERROR, std::string("dropout: floating point arrays only, got ") + DtypeName(x->dtype));
        HIPCX_REQUIRE(out->dtype == x->dtype && (residual == nullptr || residual->dtype == x->dtype), HIPCX_DTYPE_ERROR,
                      "dropout: x, residual and out must share a dtype");
        HIPCX_REQUIRE(key->dtype == HIPCX_INT64, HIPCX_DTYPE_ERROR, std::string("dropout: the key is an int64 array, got ") + DtypeName(key->dtype));
        HIPCX_REQUIRE(key->ndim == 1 && key->shape[0] == 2 && key->strides[0] == 8, HIPCX_DIMENSION_ERROR, "dropout: the key is a dense array of two elements, a seed and a step");
        HIPCX_REQUIRE(SameShape(x, out) && (residual == nullptr || SameShape(x, residual)), HIPCX_DIMENSION_ERROR, "dropout: x, residual and out must have one shape");
        HIPCX_REQUIRE(IsContiguous(x) && IsContiguous(out) && (residual == nullptr || IsContiguous(residual)), HIPCX_DIMENSION_ERROR, "dropout: arrays must be C-contiguous");
        HIPCX_REQUIRE(ratio >= 0 && ratio < 1, HIPCX_CHAINERX_ERROR, "dropout: the ratio must be at least 0 and less than 1");
        HIPCX_REQUIRE(site >= 0 && site < (int64_t{1} << 32), HIPCX_CHAINERX_ERROR, "dropout: the site must be at least 0 and less than 2^32");
        DropoutArgs p{};
        p.n = TotalSize(x);
        HIPCX_REQUIRE(p.n <= kPerCounter * (int64_t{1} << 32), HIPCX_NOT_IMPLEMENTED_ERROR, "dropout: more than 2^35 elements");
        if (p.n == 0) return;
        p.x = x->data, p.out = out->data, p.key = static_cast<const int64_t*>(key->data), p.site = static_cast<uint32_t>(site);
        if (residual != nullptr) p.residual = residual->data;
        // 16 bits an element: what is kept is scaled by the share that is kept, so that the expectation is x's for any ratio
        p.threshold = static_cast<uint32_t>(std::min(65535.0, std::floor(ratio * 65536 + 0.5)));
        p.scale = 65536.0 / (65536 - static_cast<int>(p.threshold));
        VisitFloatDtype(x->dtype, [&](auto tag) {
            using T = typename decltype(tag)::type;
            ForLaunches((p.n + kPerCounter - 1) / kPerCounter, [&](dim3 grid, int64_t first) {
                p.first = first;
                if (residual != nullptr) hipLaunchKernelGGL((DropoutKernel<T, true>), grid, dim3(256), 0, AsStream(stream), p);
                else hipLaunchKernelGGL((DropoutKernel<T, false>), grid, dim3(256), 0, AsStream(stream), p);
                CheckLaunch("dropout");
            });
        });
    });
}
