// A step of AdamW over many arrays at once, in place, with states in 32 bits or in 8 (chainer/optimizers/adam.py: AdamRule with weight_decay_rate):
//   m += (1 - beta1) (g - m),  v += (1 - beta2) (g^2 - v),  p -= a (m / (sqrt(v) + eps)) + d p
// with a = eta alpha sqrt(1 - beta2^t) / (1 - beta1^t) and d = eta weight_decay_rate; every operation is rounded to 32 bits.
//
// States in 8 bits: blocks of 256 elements share a scale, the power of two that no value of the block exceeds.  A code counts eighths of a power of two, down to 2^-14 of the
// scale for m (a sign, 4 bits of exponent) and 2^-30 for sqrt(v) (5 bits; a value that is not 0 is never stored as 0, as m is divided by it), and below that the lowest one's eighths.  Values are
// rounded to one of the two neighbours at random, in proportion: a step changes v by a thousandth, and rounded to the nearest of 8 bits it would never change at all.
// (sqrt(v) is what comes out right on average, so that v is larger by the variance of its roundings, some percent.)  The numbers come from
// a counter: 16 bits each for m and v of an element.
#include <algorithm>
#include <cmath>
#include <utility>
#include <vector>

#include "common.h"
#include "philox.h"

namespace hipcx {
namespace {

constexpr int kMaxArrays = 48;     // the descriptors travel as kernel arguments (4 KB at most)
constexpr int kStateBlock = 256;   // elements that share a scale
constexpr int kPerThread = 8;

struct AdamWArgs {
    void* p[kMaxArrays];
    const void* g[kMaxArrays];
    void* m[kMaxArrays];
    void* v[kMaxArrays];
    float* m_scale[kMaxArrays];
    float* v_scale[kMaxArrays];
    float* master[kMaxArrays];
    int64_t size[kMaxArrays];  // elements
    uint32_t block0[kMaxArrays];  // first workgroup
    uint32_t site[kMaxArrays];
    int n;
    float step, m_share, v_share, eps, decay;
    uint32_t key0, key1;
    int64_t t;
    const int64_t* t_array;  // null: t
    double alpha, beta1, beta2;
};

// beta^t by squarings, alike on the host and on the device.
__host__ __device__ inline double PowerOf(double beta, int64_t t) {
    double r = 1;
    for (; t > 0; t >>= 1, beta *= beta) {
        if (t & 1) r *= beta;
    }
    return r;
}

__host__ __device__ inline float StepSize(double alpha, double beta1, double beta2, int64_t t) {
    return static_cast<float>(alpha * sqrt(1 - PowerOf(beta2, t)) / (1 - PowerOf(beta1, t)));
}

template <typename T, int N>
struct __attribute__((packed, aligned(alignof(T)))) Run {
    T v[N];
};

__device__ __forceinline__ float PowerOfTwo(int e) { return __builtin_bit_cast(float, (e + 127) << 23); }

// What a code stands for, as a part of the scale; EXPONENTS powers of two.  Its bits are a float's: of the lowest eighths, which have no power, those of the next ones less their power.
template <int EXPONENTS>
__device__ __forceinline__ float PartOf(int code) {
    const bool low = code < 8;
    return __builtin_bit_cast(float, ((low ? code + 8 : code) << 20) + ((128 - EXPONENTS) << 23)) - (low ? PowerOfTwo(2 - EXPONENTS) : 0.f);
}

// A part of the scale, not negative, as a code: `random` of 16 bits and a half, as a part of a step, is added and what is beyond the code's bits cut off.
template <int EXPONENTS>
__device__ __forceinline__ int CodeOf(float part, uint32_t random) {
    int code = static_cast<int>((__builtin_bit_cast(uint32_t, part) + (random << 4) + 8) >> 20) - ((128 - EXPONENTS) << 3);
    if (part < PowerOfTwo(2 - EXPONENTS)) code = static_cast<int>(__builtin_fmaf(part, PowerOfTwo(EXPONENTS + 1), (static_cast<float>(random) + 0.5f) * 0x1p-16f));
    return min(code, 8 * EXPONENTS - 1);
}

// The power of two that `top`, in a float's bits, does not exceed, within 2^-100 and 2^100; not a number where top is not finite or larger.
__device__ __forceinline__ float ScaleOf(uint32_t top) {
    const int e = static_cast<int>((top + 0x7fffff) >> 23) - 127;
    return top <= __builtin_bit_cast(uint32_t, 0x1p100f) ? PowerOfTwo(max(e, -100)) : __builtin_nanf("");
}

template <int MOVE>
__device__ __forceinline__ uint32_t MaxMoved(uint32_t v) {
    return max(v, static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(v), MOVE, 0xf, 0xf, false)));
}
// The largest of 32 neighbours' values, which are not negative, by their bits: those of what is not a number are larger than all others.  Rotations among sixteen lanes, and the sixteen beside them.
__device__ __forceinline__ uint32_t TopOf32(uint32_t v) {
    v = MaxMoved<0x121>(MaxMoved<0x122>(MaxMoved<0x124>(MaxMoved<0x128>(v))));
    return max(v, static_cast<uint32_t>(__shfl_xor(static_cast<int>(v), 16)));
}

// A pass over memory.  A thread takes eight neighbours, 32 threads a block of states in 8 bits.  25.5 M float16 weights of 161 arrays with master copies: 163 us, 4.7 TB/s.  States in 8 bits are bound by
// the vector units, by a division and a root that round as IEEE 754 says and half a Philox counter to an element: 19.8 M weights 68 us, where their 198 MB would take 41.
template <typename P, typename G, bool EIGHT, bool MASTER>
__global__ __launch_bounds__(256) void AdamWKernel(AdamWArgs a) {
    constexpr int E = kPerThread;
    int lo = 0, hi = a.n;  // block0[lo] <= blockIdx.x < block0[hi]
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (blockIdx.x >= a.block0[mid]) lo = mid;
        else hi = mid;
    }
    const int64_t size = a.size[lo], group = static_cast<int64_t>(blockIdx.x - a.block0[lo]) * 256 + threadIdx.x, at = group * E;
    if (EIGHT ? at - threadIdx.x % 32 * E >= size : at >= size) return;  // a block's threads stay together
    using W = std::conditional_t<MASTER, float, P>;
    P* const p = static_cast<P*>(a.p[lo]) + at;
    const G* const g = static_cast<const G*>(a.g[lo]) + at;
    W* const w = MASTER ? reinterpret_cast<W*>(a.master[lo]) + at : reinterpret_cast<W*>(p);
    using S = std::conditional_t<EIGHT, uint8_t, float>;
    S *const m = static_cast<S*>(a.m[lo]) + at, *const v = static_cast<S*>(a.v[lo]) + at;
    const int here = static_cast<int>(size - at < 0 ? 0 : size - at < E ? size - at : E);
    Run<W, E> wv{};
    Run<G, E> gv{};
    Run<S, E> mv{}, vv{};
    if (here == E) {
        wv = *reinterpret_cast<const Run<W, E>*>(w);
        gv = *reinterpret_cast<const Run<G, E>*>(g);
        mv = *reinterpret_cast<const Run<S, E>*>(m);
        vv = *reinterpret_cast<const Run<S, E>*>(v);
    } else {
#pragma unroll
        for (int e = 0; e < E; ++e) {
            if (e < here) wv.v[e] = w[e], gv.v[e] = g[e], mv.v[e] = m[e], vv.v[e] = v[e];
        }
    }
    const int64_t block = at / kStateBlock;
    float m_scale = 0, v_scale = 0;
    if constexpr (EIGHT) m_scale = a.m_scale[lo][block], v_scale = a.v_scale[lo][block];
    int64_t t = a.t;
    float step = a.step;
    if (a.t_array != nullptr) {
        t = *a.t_array;
        step = StepSize(a.alpha, a.beta1, a.beta2, t);
    }
    float new_m[E], root[E], new_v[E], new_w[E];
    uint32_t m_top = 0, root_top = 0;
#pragma unroll
    for (int e = 0; e < E; ++e) {
        float old_m, old_v;
        if constexpr (EIGHT) {
            const int code = mv.v[e];
            const float part = PartOf<16>(code & 127) * m_scale, r = PartOf<32>(vv.v[e]) * v_scale;
            old_m = code & 128 ? -part : part;
            old_v = r * r;
        } else {
            old_m = mv.v[e], old_v = vv.v[e];
        }
        const float grad = static_cast<float>(gv.v[e]), weight = static_cast<float>(wv.v[e]);
        new_m[e] = old_m + a.m_share * (grad - old_m);
        new_v[e] = old_v + a.v_share * (grad * grad - old_v);
        root[e] = sqrtf(new_v[e]);
        new_w[e] = weight - (step * (new_m[e] / (root[e] + a.eps)) + a.decay * weight);
        if constexpr (EIGHT) {
            m_top = max(m_top, __builtin_bit_cast(uint32_t, fabsf(new_m[e])));
            root_top = max(root_top, __builtin_bit_cast(uint32_t, root[e]));
        }
    }
    if constexpr (EIGHT) {
        m_scale = ScaleOf(TopOf32(m_top)), v_scale = ScaleOf(TopOf32(root_top));
        const float m_part = 1 / m_scale, v_part = 1 / v_scale;  // powers of two
        if (threadIdx.x % 32 == 0) a.m_scale[lo][block] = m_scale, a.v_scale[lo][block] = v_scale;
#pragma unroll
        for (int c = 0; c < E / 4; ++c) {
            uint32_t word[4] = {static_cast<uint32_t>(group * (E / 4) + c), a.site[lo], static_cast<uint32_t>(t), static_cast<uint32_t>(static_cast<uint64_t>(t) >> 32)};
            Philox(word, a.key0, a.key1);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int e = c * 4 + i;
                const int code = CodeOf<16>(fabsf(new_m[e]) * m_part, word[i] & 0xffff);
                mv.v[e] = static_cast<S>(code | (__builtin_bit_cast(uint32_t, new_m[e]) >> 31 << 7));
                const int root_code = CodeOf<32>(root[e] * v_part, word[i] >> 16);
                vv.v[e] = static_cast<S>(root[e] > 0 ? max(root_code, 1) : root_code);
            }
        }
    } else {
#pragma unroll
        for (int e = 0; e < E; ++e) mv.v[e] = new_m[e], vv.v[e] = new_v[e];
    }
    Run<P, E> pv;
#pragma unroll
    for (int e = 0; e < E; ++e) pv.v[e] = static_cast<P>(new_w[e]);
    if (here == E) {
        *reinterpret_cast<Run<P, E>*>(p) = pv;
        *reinterpret_cast<Run<S, E>*>(m) = mv;
        *reinterpret_cast<Run<S, E>*>(v) = vv;
        if constexpr (MASTER) {
#pragma unroll
            for (int e = 0; e < E; ++e) wv.v[e] = new_w[e];
            *reinterpret_cast<Run<W, E>*>(w) = wv;
        }
    } else {
#pragma unroll
        for (int e = 0; e < E; ++e) {
            if (e >= here) continue;
            p[e] = pv.v[e], m[e] = mv.v[e], v[e] = vv.v[e];
            if constexpr (MASTER) w[e] = new_w[e];
        }
    }
}

// The arrays of one combination of types.
template <typename P, typename G, bool EIGHT, bool MASTER>
struct AdamWLaunch {
    static constexpr int64_t kEach = 256 * kPerThread;
    AdamWArgs a;
    int64_t blocks = 0;
    hipStream_t stream;

    AdamWLaunch(const AdamWArgs& all, hipStream_t s) : a(all), stream(s) {}
    void Flush() {
        if (a.n == 0) return;
        hipLaunchKernelGGL((AdamWKernel<P, G, EIGHT, MASTER>), dim3(static_cast<unsigned>(blocks)), dim3(256), 0, stream, a);
        CheckLaunch("adamw");
        a.n = 0;
        blocks = 0;
    }
    void Add(const hipcx_array* p, const hipcx_array* g, const hipcx_array* m, const hipcx_array* v, const hipcx_array* m_scale, const hipcx_array* v_scale,
             const hipcx_array* master, uint32_t site) {
        const int64_t size = TotalSize(p), more = (size + kEach - 1) / kEach;
        if (a.n == kMaxArrays || blocks + more > kBlocksPerLaunch) Flush();
        const int i = a.n++;
        a.p[i] = p->data, a.g[i] = g->data, a.m[i] = m->data, a.v[i] = v->data, a.size[i] = size, a.site[i] = site, a.block0[i] = static_cast<uint32_t>(blocks);
        a.m_scale[i] = EIGHT ? static_cast<float*>(m_scale->data) : nullptr, a.v_scale[i] = EIGHT ? static_cast<float*>(v_scale->data) : nullptr;
        a.master[i] = MASTER ? static_cast<float*>(master->data) : nullptr;
        blocks += more;
    }
};

template <typename P, typename G, bool MASTER>
struct AdamWLaunches {
    AdamWLaunch<P, G, false, MASTER> wide;
    AdamWLaunch<P, G, true, MASTER> eight;
    AdamWLaunches(const AdamWArgs& all, hipStream_t s) : wide(all, s), eight(all, s) {}
};

constexpr int64_t kMostElements = int64_t{1} << 33;  // a counter has 32 bits for four elements' words, and a launch takes any array whole

// What is written, and what is read, by address.
struct Extent {
    const char *from, *to;
    bool written;
};

}  // namespace
}  // namespace hipcx

using namespace hipcx;

extern "C" int hipcx_adamw_many(const hipcx_array* const* params, const hipcx_array* const* grads, const hipcx_array* const* ms, const hipcx_array* const* vs,
                                const hipcx_array* const* m_scales, const hipcx_array* const* v_scales, const hipcx_array* const* masters, int n, int64_t t,
                                const hipcx_array* t_array, double alpha, double beta1, double beta2, double eps, double eta, double weight_decay_rate, int64_t seed,
                                void* stream) {
    return Guard([&] {
        HIPCX_REQUIRE(n >= 0 && (n == 0 || (params != nullptr && grads != nullptr && ms != nullptr && vs != nullptr && m_scales != nullptr && v_scales != nullptr && masters != nullptr)),
                      HIPCX_CHAINERX_ERROR, "adamw: null arrays");
        HIPCX_REQUIRE(beta1 >= 0 && beta1 < 1 && beta2 >= 0 && beta2 < 1, HIPCX_CHAINERX_ERROR, "adamw: beta1 and beta2 must be at least 0 and less than 1");
        HIPCX_REQUIRE(eps >= 0 && eps < HUGE_VAL, HIPCX_CHAINERX_ERROR, "adamw: eps must be finite and not negative");
        HIPCX_REQUIRE(std::isfinite(alpha) && std::isfinite(eta) && std::isfinite(weight_decay_rate), HIPCX_CHAINERX_ERROR, "adamw: alpha, eta and weight_decay_rate must be finite");
        std::vector<Extent> extents;
        extents.reserve(static_cast<size_t>(n) * 7 + 1);
        if (t_array != nullptr) {
            ValidateArray(t_array, "t");
            HIPCX_REQUIRE(t_array->dtype == HIPCX_INT64, HIPCX_DTYPE_ERROR, std::string("adamw: t is an int64 array, got ") + DtypeName(t_array->dtype));
            HIPCX_REQUIRE(TotalSize(t_array) == 1, HIPCX_DIMENSION_ERROR, "adamw: t is an array of one element, got shape " + ShapeStr(t_array));
            extents.push_back({static_cast<const char*>(t_array->data), static_cast<const char*>(t_array->data) + sizeof(int64_t), false});
        } else {
            HIPCX_REQUIRE(t >= 1, HIPCX_CHAINERX_ERROR, "adamw: t counts steps from 1");
        }
        for (int i = 0; i < n; ++i) {
            const hipcx_array *p = params[i], *g = grads[i], *m = ms[i], *v = vs[i], *m_scale = m_scales[i], *v_scale = v_scales[i], *master = masters[i];
            const auto require = [&](const hipcx_array* a, const char* what, std::initializer_list<int> dtypes, bool written) {
                ValidateArray(a, what);
                HIPCX_REQUIRE(std::find(dtypes.begin(), dtypes.end(), a->dtype) != dtypes.end(), HIPCX_DTYPE_ERROR,
                              std::string("adamw: ") + what + " has dtype " + DtypeName(a->dtype) + ", expected " + DtypeName(*dtypes.begin()));
                HIPCX_REQUIRE(IsContiguous(a), HIPCX_DIMENSION_ERROR, std::string("adamw: ") + what + " must be C-contiguous");
                const int64_t bytes = TotalSize(a) * ItemSize(a->dtype);
                if (bytes > 0) extents.push_back({static_cast<const char*>(a->data), static_cast<const char*>(a->data) + bytes, written});
            };
            require(p, "a parameter", {HIPCX_FLOAT32, HIPCX_FLOAT16}, true);
            const int64_t size = TotalSize(p);
            HIPCX_REQUIRE(size <= kMostElements, HIPCX_NOT_IMPLEMENTED_ERROR, "adamw: more than 2^33 elements in an array");
            require(g, "a gradient", {p->dtype, HIPCX_FLOAT32}, false);
            require(m, "m", {HIPCX_FLOAT32, HIPCX_UINT8}, true);
            require(v, "v", {m->dtype}, true);
            for (const hipcx_array* a : {g, m, v}) {
                HIPCX_REQUIRE(SameShape(a, p), HIPCX_DIMENSION_ERROR, "adamw: a parameter, its gradient and its states must have one shape, got " + ShapeStr(p) + " and " + ShapeStr(a));
            }
            if (m->dtype == HIPCX_UINT8) {
                require(m_scale, "m_scale", {HIPCX_FLOAT32}, true);
                require(v_scale, "v_scale", {HIPCX_FLOAT32}, true);
                for (const hipcx_array* a : {m_scale, v_scale}) {
                    HIPCX_REQUIRE(a->ndim == 1 && a->shape[0] == (size + kStateBlock - 1) / kStateBlock, HIPCX_DIMENSION_ERROR,
                                  "adamw: states in 8 bits have a scale for every 256 elements, got shape " + ShapeStr(a));
                }
            } else {
                HIPCX_REQUIRE(m_scale == nullptr && v_scale == nullptr, HIPCX_CHAINERX_ERROR, "adamw: scales belong to states in 8 bits");
            }
            if (master != nullptr) {
                HIPCX_REQUIRE(p->dtype == HIPCX_FLOAT16, HIPCX_DTYPE_ERROR, "adamw: a master copy belongs to a float16 parameter");
                require(master, "a master copy", {HIPCX_FLOAT32}, true);
                HIPCX_REQUIRE(SameShape(master, p), HIPCX_DIMENSION_ERROR, "adamw: a master copy must have its parameter's shape, got " + ShapeStr(master));
            }
        }
        // nothing that is written may lie in another array of the call
        std::sort(extents.begin(), extents.end(), [](const Extent& a, const Extent& b) { return a.from < b.from; });
        Extent reach{}, written_reach{};  // of what begins before: the farthest end, and the farthest of what is written
        for (const Extent& e : extents) {
            HIPCX_REQUIRE(!(e.from < written_reach.to || (e.written && e.from < reach.to)), HIPCX_CHAINERX_ERROR,
                          "adamw: arrays that are updated share memory with each other, with gradients or with t");
            if (e.to > reach.to) reach = e;
            if (e.written && e.to > written_reach.to) written_reach = e;
        }
        AdamWArgs all{};
        all.eps = static_cast<float>(eps), all.m_share = static_cast<float>(1 - beta1), all.v_share = static_cast<float>(1 - beta2);
        all.decay = static_cast<float>(eta * weight_decay_rate), all.alpha = eta * alpha, all.beta1 = beta1, all.beta2 = beta2, all.t = t;
        all.key0 = static_cast<uint32_t>(seed), all.key1 = static_cast<uint32_t>(static_cast<uint64_t>(seed) >> 32);
        if (t_array != nullptr) all.t_array = static_cast<const int64_t*>(t_array->data);
        else all.step = StepSize(all.alpha, beta1, beta2, t);
        const hipStream_t s = AsStream(stream);
        AdamWLaunches<float, float, false> floats(all, s);
        AdamWLaunches<half_t, half_t, false> halves(all, s);
        AdamWLaunches<half_t, float, false> mixed(all, s);
        AdamWLaunches<half_t, half_t, true> halves_master(all, s);
        AdamWLaunches<half_t, float, true> mixed_master(all, s);
        for (int i = 0; i < n; ++i) {
            if (TotalSize(params[i]) == 0) continue;
            const auto add = [&](auto& launches) {
                if (ms[i]->dtype == HIPCX_UINT8) launches.eight.Add(params[i], grads[i], ms[i], vs[i], m_scales[i], v_scales[i], masters[i], static_cast<uint32_t>(i));
                else launches.wide.Add(params[i], grads[i], ms[i], vs[i], m_scales[i], v_scales[i], masters[i], static_cast<uint32_t>(i));
            };
            const bool half_grad = grads[i]->dtype == HIPCX_FLOAT16;
            if (params[i]->dtype == HIPCX_FLOAT32) add(floats);
            else if (masters[i] != nullptr) half_grad ? add(halves_master) : add(mixed_master);
            else half_grad ? add(halves) : add(mixed);
        }
        const auto flush = [](auto& launches) { launches.wide.Flush(), launches.eight.Flush(); };
        flush(floats), flush(halves), flush(mixed), flush(halves_master), flush(mixed_master);
    });
}
