// The selective scan: whole sequences, and one row of each.
#include "selective_scan.h"

namespace hipcx {
namespace {

// A workgroup's part of the sequence: 64 channels, a chunk of rows.  Rows go by in tiles of 16, whose b and c lie in LDS; a lane reads u, delta and z of every fourth row
// of its channel, prepares dt, dt u and the gate once, and hands them to the quad's other lanes.
template <typename T, int NPL>
__global__ __launch_bounds__(256) void SelectiveScanKernel(ScanArgs p) {
    constexpr int NP = 4 * NPL, kEach = (kScanTile * NP + 255) / 256;
    __shared__ float bs[2][kScanTile][NP], cs[2][kScanTile][NP];
    const ScanPlace at(p, blockIdx.x, p.chunks);
    const int64_t len = LengthOf(p.lengths, at.b, p.length);
    const int64_t t0 = static_cast<int64_t>(at.chunk) * p.chunk_rows, end = std::min(t0 + p.chunk_rows, p.length), last = std::min(end, len);
    const int n0 = at.q * NPL;
    float a[NPL], h[NPL];
    LoadStates<NPL>(p.a + static_cast<int64_t>(at.channel) * p.states, n0, p.states, a);
#pragma unroll
    for (int i = 0; i < NPL; ++i) a[i] *= kLog2E, h[i] = 0.f;
    const int64_t of_state = (at.b * p.channels + at.channel) * p.states;
    if (p.state != nullptr) LoadStates<NPL>(p.state + of_state, n0, p.states, h);
    const float bias = p.bias != nullptr ? p.bias[at.channel] : 0.f, d = p.d != nullptr ? p.d[at.channel] : 0.f;
    const T* const b = static_cast<const T*>(p.b.data) + at.b * p.b.batch + at.group * p.b.group;
    const T* const c = static_cast<const T*>(p.c.data) + at.b * p.c.batch + at.group * p.c.group;

    float ub[4], db[4], zb[4], bb[kEach], cb[kEach];  // of the next tile
    const auto fetch = [&](int64_t t) {
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            const int64_t row = t + 4 * g + at.q;
            ub[g] = db[g] = zb[g] = 0.f;
            if (row < last) {
                ub[g] = ScanRead<T>(p.u, at.b, row, at.channel);
                db[g] = ScanRead<T>(p.delta, at.b, row, at.channel);
                if (p.z.data != nullptr) zb[g] = ScanRead<T>(p.z, at.b, row, at.channel);
            }
        }
#pragma unroll
        for (int i = 0; i < kEach; ++i) {
            const int e = i * 256 + static_cast<int>(threadIdx.x), r = e / NP, n = e % NP;
            bb[i] = cb[i] = 0.f;
            if (r < kScanTile && n < p.states && t + r < last) {
                bb[i] = static_cast<float>(b[(t + r) * p.b.row + n]);
                cb[i] = static_cast<float>(c[(t + r) * p.c.row + n]);
            }
        }
    };
    fetch(t0);
    int buffer = 0;
    for (int64_t t = t0; t < last; t += kScanTile, buffer ^= 1) {
#pragma unroll
        for (int i = 0; i < kEach; ++i) {
            const int e = i * 256 + static_cast<int>(threadIdx.x);
            if (e < kScanTile * NP) bs[buffer][e / NP][e % NP] = bb[i], cs[buffer][e / NP][e % NP] = cb[i];
        }
        __syncthreads();
        float u[4], dt[4], z[4];
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            const bool counts = t + 4 * g + at.q < last;
            u[g] = ub[g], z[g] = zb[g];
            const float raw = db[g] + bias;
            dt[g] = counts ? (p.softplus != 0 ? SoftplusOf(raw) : raw) : 0.f;
        }
        fetch(t + kScanTile);
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            const float x = dt[g] * u[g];
            float sums[4];
            const auto step = [&](auto lane) {
                constexpr int S = decltype(lane)::value;
                const float dts = OfQuadLane<S>(dt[g]), xs = OfQuadLane<S>(x);
                float sum = 0.f;
#pragma unroll
                for (int i = 0; i < NPL; ++i) {
                    const float e = __builtin_amdgcn_exp2f(dts * a[i]);
                    h[i] = __builtin_fmaf(xs, bs[buffer][4 * g + S][n0 + i], e * h[i]);
                    sum = __builtin_fmaf(cs[buffer][4 * g + S][n0 + i], h[i], sum);
                }
                sums[S] = sum;
            };
            step(std::integral_constant<int, 0>{});
            step(std::integral_constant<int, 1>{});
            step(std::integral_constant<int, 2>{});
            step(std::integral_constant<int, 3>{});
            float y = __builtin_fmaf(d, u[g], QuadTransposedSum(sums, at.q));
            if (p.z.data != nullptr) y *= z[g] * LogisticOf(z[g]);
            const int64_t row = t + 4 * g + at.q;
            if (at.inside && row < last) static_cast<T*>(p.y.data)[at.b * p.y.batch + row * p.y.row + at.channel] = static_cast<T>(y);
        }
    }
    if (!at.inside) return;
    for (int64_t row = std::max(t0, len) + at.q; row < end; row += 4) static_cast<T*>(p.y.data)[at.b * p.y.batch + row * p.y.row + at.channel] = static_cast<T>(0);
    if (at.chunk == p.chunks - 1) StoreStates<NPL>(p.new_state + of_state, n0, p.states, h);
}

}  // namespace

ScanArgs DescribeScan(const std::string& what, const hipcx_array* u, const hipcx_array* delta, const hipcx_array* a, const hipcx_array* b, const hipcx_array* c,
                      const hipcx_array* d, const hipcx_array* z, const hipcx_array* delta_bias, int delta_softplus, const hipcx_array* state,
                      const hipcx_array* lengths) {
    ValidateArray(u, "u");
    ValidateArray(a, "a");
    ValidateArray(b, "b");
    HIPCX_REQUIRE(delta != nullptr && c != nullptr, HIPCX_CHAINERX_ERROR, what + ": delta and c are needed");
    HIPCX_REQUIRE(u->dtype == HIPCX_FLOAT16 || u->dtype == HIPCX_FLOAT32, HIPCX_DTYPE_ERROR, what + ": float16 and float32 only, got " + DtypeName(u->dtype));
    HIPCX_REQUIRE(u->ndim == 3, HIPCX_DIMENSION_ERROR, what + ": u must be [batch, time, channels], got " + ShapeStr(u));
    HIPCX_REQUIRE(a->ndim == 2 && a->shape[0] == u->shape[2], HIPCX_DIMENSION_ERROR, what + ": a must be [channels, states], got " + ShapeStr(a));
    const int64_t batch = u->shape[0], length = u->shape[1], channels = u->shape[2], states = a->shape[1];
    HIPCX_REQUIRE(states >= 1 && states <= 64, HIPCX_NOT_IMPLEMENTED_ERROR, what + ": 1 to 64 states, got " + std::to_string(states));
    HIPCX_REQUIRE(channels < (int64_t{1} << 24), HIPCX_NOT_IMPLEMENTED_ERROR, what + ": 2^24 channels or more");
    HIPCX_REQUIRE(b->ndim == 3 || b->ndim == 4, HIPCX_DIMENSION_ERROR, what + ": b must be [batch, time, states] or [batch, time, groups, states], got " + ShapeStr(b));
    HIPCX_REQUIRE(length < (int64_t{1} << 30), HIPCX_NOT_IMPLEMENTED_ERROR, what + ": 2^30 rows or more");
    const int64_t groups = b->ndim == 4 ? b->shape[2] : 1;
    HIPCX_REQUIRE(groups >= 1 && channels % groups == 0, HIPCX_DIMENSION_ERROR, what + ": the groups of b must divide the channels");
    for (const hipcx_array* s : {b, c}) {
        if (b->ndim == 4) RequireShape(s, {batch, length, groups, states}, u->dtype, what + ": b and c");
        else RequireShape(s, {batch, length, states}, u->dtype, what + ": b and c");
    }
    RequireShape(delta, {batch, length, channels}, u->dtype, what + ": delta");
    RequireShape(z, {batch, length, channels}, u->dtype, what + ": z");
    RequireShape(a, {channels, states}, HIPCX_FLOAT32, what + ": a");
    RequireShape(d, {channels}, HIPCX_FLOAT32, what + ": d");
    RequireShape(delta_bias, {channels}, HIPCX_FLOAT32, what + ": delta_bias");
    RequireShape(state, {batch, channels, states}, HIPCX_FLOAT32, what + ": state");
    for (const hipcx_array* s : {a, d, delta_bias, state}) RequireDense(s, what + ": a, d, delta_bias and state");
    ScanArgs p{};
    p.u = RowsOf(u, "u"), p.delta = RowsOf(delta, "delta"), p.z = RowsOf(z, "z");
    const auto shared = [&](const hipcx_array* s, const char* name) {
        const SequenceRows r = RowsOf(s, name);
        return ScanShared{r.data, r.batch, r.row, s->ndim == 4 ? s->strides[2] / ItemSize(s->dtype) : 0};
    };
    p.b = shared(b, "b"), p.c = shared(c, "c");
    const auto floats = [](const hipcx_array* s) { return s != nullptr ? static_cast<const float*>(s->data) : nullptr; };
    p.a = floats(a), p.d = floats(d), p.bias = floats(delta_bias), p.state = floats(state);
    p.lengths = LengthsOf(lengths, batch, what);
    p.batch = batch, p.length = length, p.softplus = delta_softplus;
    p.channels = static_cast<int>(channels), p.states = static_cast<int>(states), p.group_channels = static_cast<int>(channels / groups);
    p.group_blocks = DivUp(p.group_channels, kScanChannels);
    p.blocks = static_cast<int>(groups) * p.group_blocks;
    return p;
}

}  // namespace hipcx

using namespace hipcx;

extern "C" {

size_t hipcx_selective_scan_workspace_size(const hipcx_array* u, const hipcx_array* a) {
    (void)u, (void)a;
    return 0;
}

int hipcx_selective_scan(const hipcx_array* u, const hipcx_array* delta, const hipcx_array* a, const hipcx_array* b, const hipcx_array* c, const hipcx_array* d,
                         const hipcx_array* z, const hipcx_array* delta_bias, int delta_softplus, const hipcx_array* state, const hipcx_array* lengths,
                         const hipcx_array* y, const hipcx_array* new_state, void* workspace, size_t workspace_bytes, void* stream) {
    return Guard([&] {
        const std::string what = "selective_scan";
        ScanArgs p = DescribeScan(what, u, delta, a, b, c, d, z, delta_bias, delta_softplus, state, lengths);
        HIPCX_REQUIRE(y != nullptr && new_state != nullptr, HIPCX_CHAINERX_ERROR, what + ": y and new_state are needed");
        RequireShape(y, {p.batch, p.length, p.channels}, u->dtype, what + ": y");
        RequireShape(new_state, {p.batch, p.channels, p.states}, HIPCX_FLOAT32, what + ": new_state");
        RequireDense(new_state, what + ": new_state");
        p.y = RowsOf(y, "y"), p.new_state = static_cast<float*>(new_state->data);
        if (p.batch == 0 || p.channels == 0) return;
        const size_t need = hipcx_selective_scan_workspace_size(u, a);
        HIPCX_REQUIRE(workspace_bytes >= need && (need == 0 || workspace != nullptr), HIPCX_CHAINERX_ERROR, what + ": the workspace is too small");
        p.chunks = 1, p.chunk_rows = static_cast<int>(DivUp(p.length, kScanTile)) * kScanTile;
        const int64_t blocks = p.batch * p.chunks * p.blocks;
        HIPCX_REQUIRE(blocks <= kBlocksPerLaunch, HIPCX_NOT_IMPLEMENTED_ERROR, what + ": too many elements");
        VisitScan(u->dtype, p.states, [&](auto tag, auto share) {
            using T = typename decltype(tag)::type;
            hipLaunchKernelGGL((SelectiveScanKernel<T, decltype(share)::value>), dim3(static_cast<unsigned>(blocks)), dim3(256), 0, AsStream(stream), p);
            CheckLaunch("selective_scan");
        });
    });
}

}  // extern "C"
