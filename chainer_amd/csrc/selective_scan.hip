// The selective scan: whole sequences, and one row of each.
#include "selective_scan.h"

#include <cmath>

namespace hipcx {
namespace {

// The state that a chunk starts from, which is behind `n` others.  A chunk's decay may leave float32's range where no row's does: nothing times infinity, and infinity times 0, are NaN then,
// which the rows one by one do not make.  So whoever ends at infinity or NaN, where what made it stays, goes through the chunks once more, by the decay's root twice; a state of 0, and one of
// infinity that decays, stay what they are.
template <int NPL>
__device__ __forceinline__ void StartOfChunk(float (&s)[NPL], const float (&a)[NPL], const float* state, const float* adds, const float* steps, int n, int64_t per_chunk, int64_t channels,
                                             int n0, int states) {
    LoadStates<NPL>(state, n0, states, s);
    ThroughChunks<NPL>(s, a, adds, steps, n, 1, per_chunk, channels, n0, states);
    bool finite = true;
#pragma unroll
    for (int i = 0; i < NPL; ++i) finite = finite && __builtin_fabsf(s[i]) <= FLT_MAX;
    if (finite) return;
    LoadStates<NPL>(state, n0, states, s);
#pragma unroll 1
    for (int j = 0; j < n; ++j) {
        float add[NPL];
        LoadStates<NPL>(adds + j * per_chunk, n0, states, add);
        const float dt = steps[j * channels];
#pragma unroll
        for (int i = 0; i < NPL; ++i) {
            const float exponent = dt * a[i], root = __builtin_amdgcn_exp2f(0.5f * exponent);
            const bool stays = s[i] == 0.f || (__builtin_fabsf(s[i]) > FLT_MAX && __builtin_fabsf(exponent) <= FLT_MAX);
            s[i] = (stays ? s[i] : s[i] * root * root) + add[i];
        }
    }
}

// Waves to a SIMD that the registers leave room for without spills in the rows.  9 to 16 states take 97 registers, which is four waves; held to 96, for a fifth, the rows take longer, so
// that only launches of more than four workgroups to a compute unit are.  us with four (FEW) and five, 16 states, float16: one sequence of 16384 rows and 2048 channels 282, 276,
// 4 x 2048 x 1024 83.4, 81.1; 16 x 2048 x 2048 397, 425, 32 x 2048 x 2048 632, 646.
template <typename T, int NPL, bool FEW>
constexpr int kScanWaves = NPL == 1 ? (sizeof(T) == 4 ? 7 : 6) : NPL <= 4 ? (FEW ? 4 : 5) : NPL == 8 ? 4 : 3;

// A workgroup's part of the sequence: 64 channels, a chunk of rows.  Chunks that come after others need the state there, and a state goes through a chunk linearly:
// h -> exp(a * sum of dt) h + what the chunk makes of zeros.  So ENDS runs the chunks but the last from zeros, without outputs, and the second launch runs all of them
// from the states that it puts together on the way.  Rows go by in tiles of 16, whose b and c lie in LDS; a lane reads u, delta and z of every fourth row
// of its channel, prepares dt, dt u and the gate once, and hands them to the quad's other lanes.
// Bound by the vector units.  A state costs a row an exponential (8 cycles of a wave) and four instructions of 4 cycles: 82 us for 16384 rows of 2048 channels and 16 states,
// whose memory traffic takes 46 at 5.8 TB/s.  Beside a row's 20 instructions on states there are 17, for softplus, the gate, the sum over the quad, loads and
// LDS.  32 sequences of 2048 rows and channels, float16: 630 us, 185 cycles a row of 16 channels.  One sequence of 16384 rows: 275, of which two fifths from zeros; 76 % of the issue slots
// are taken there, 80 % with outputs.  Four lanes to a channel: one would leave a quarter of the waves, and what they share is done once either way.
// REPEATS: fewer than 4 * NPL states, some of them twice.  Zeros in the room that is left, b = c = 0, become NaN where dt u is infinite, and with them sums that the states make infinite; to
// leave them out of the sums takes a selection a state and row, and registers (48 states, 20 x 35 rows of 650 channels: 19.3 -> 21.6 us), while whole lanes of states are read at once.
template <typename T, int NPL, bool ENDS, bool REPEATS, bool FEW>
__global__ __launch_bounds__(256, (kScanWaves<T, NPL, FEW>)) void SelectiveScanKernel(ScanArgs p) {
    constexpr int NP = 4 * NPL;
    __shared__ float bs[2][kScanTile][NP], cs[ENDS ? 1 : 2][ENDS ? 1 : kScanTile][NP];
    const ScanPlace at(p, blockIdx.x, ENDS ? p.chunks - 1 : p.chunks);
    const int64_t len = LengthOf(p.lengths, at.b, p.length);
    const int64_t t0 = static_cast<int64_t>(at.chunk) * p.chunk_rows, end = std::min(t0 + p.chunk_rows, p.length), last = std::min(end, len);
    const int place = at.q * NPL, n0 = REPEATS ? FirstOfLane<NPL>(at.q, p.states) : place;  // the lane's states in LDS, and in memory
    float a[NPL], h[NPL];
    LoadExponents<NPL>(p.a + static_cast<int64_t>(at.channel) * p.states, n0, p.states, a);
#pragma unroll
    for (int i = 0; i < NPL; ++i) h[i] = 0.f;
    const int64_t of_state = (at.b * p.channels + at.channel) * p.states, per_chunk = static_cast<int64_t>(p.channels) * p.states;
    float* const ends = p.ends + (at.b * p.chunks * p.channels + at.channel) * p.states;
    const float* const steps = p.steps + at.b * (p.chunks - 1) * p.channels + at.channel;
    if (ENDS || p.chunks == 1) {
        if (p.state != nullptr) LoadStates<NPL>(p.state + of_state, n0, p.states, h);
        if (ENDS) {  // the other launch writes new_state, which may be state, and so does not read it
            if (at.chunk == 0 && at.inside) StoreStates<NPL>(ends, n0, p.states, h);
#pragma unroll
            for (int i = 0; i < NPL; ++i) h[i] = 0.f;
        }
    } else {
        StartOfChunk<NPL>(h, a, ends, ends + per_chunk, steps, at.chunk, per_chunk, p.channels, n0, p.states);
    }
    float all_steps = 0.f;
    const float bias = p.bias != nullptr ? p.bias[at.channel] : 0.f, d = p.d != nullptr ? p.d[at.channel] : 0.f;
    TileRows<T, kScanTile> us(p.u, at, t0), ds(p.delta, at, t0), zs(p.z, at, t0), ys(p.y, at, t0);
    TileShared<T, NPL, kScanTile, ENDS ? 1 : 2, REPEATS> shared(p, at, t0);
    const bool gated = !ENDS && p.z.data != nullptr, skips = p.d != nullptr;  // (0 times an infinite u would be NaN)
    const auto fetch = [&](int rows, auto whole) __attribute__((always_inline)) {
        constexpr bool kWhole = decltype(whole)::value;
        us.template Fetch<kWhole>(at.q, rows);
        ds.template Fetch<kWhole>(at.q, rows);
        if (gated) zs.template Fetch<kWhole>(at.q, rows);
        shared.template Fetch<kWhole>(rows);
        us.Move(1), ds.Move(1), zs.Move(1), shared.Move(1);
    };
    // `rows` of the tile at t, all 16 of them or fewer
    const auto run = [&](int64_t t, int buffer, const float (&u)[4], const float (&gate)[4], const float (&dt)[4], auto whole) __attribute__((always_inline)) {
        constexpr bool kWhole = decltype(whole)::value;
        float y[4];
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
                    h[i] = __builtin_fmaf(xs, bs[buffer][4 * g + S][place + i], e * h[i]);
                    if constexpr (!ENDS) sum = __builtin_fmaf(cs[buffer][4 * g + S][place + i], h[i], sum);
                }
                sums[S] = sum;
            };
            step(std::integral_constant<int, 0>{});
            step(std::integral_constant<int, 1>{});
            step(std::integral_constant<int, 2>{});
            step(std::integral_constant<int, 3>{});
            if constexpr (!ENDS) {
                y[g] = __builtin_fmaf(d, skips ? u[g] : 0.f, QuadTransposedSum(sums, at.q)) * gate[g];
            }
        }
        if constexpr (!ENDS) {
            if (at.inside) {
#pragma unroll
                for (int g = 0; g < 4; ++g) {
                    if (kWhole || t + 4 * g + at.q < last) ys[g] = static_cast<T>(y[g]);
                }
            }
        }
    };
    const auto fetch_tile = [&](int64_t t) {
        if (t + kScanTile <= last) fetch(kScanTile, std::true_type{});
        else if (t < last) fetch(static_cast<int>(last - t), std::false_type{});
    };
    fetch_tile(t0);
    int buffer = 0;
    for (int64_t t = t0; t < last; t += kScanTile, buffer ^= 1) {
        shared.template Stage<0>(bs[buffer]);
        if constexpr (!ENDS) shared.template Stage<1>(cs[buffer]);
        __syncthreads();
        float u[4], dt[4], gate[4];
#pragma unroll
        for (int g = 0; g < 4; ++g) u[g] = us.Held(g), dt[g] = ds.Held(g) + bias, gate[g] = 1.f;
        if (p.softplus != 0) {
#pragma unroll
            for (int g = 0; g < 4; ++g) dt[g] = SoftplusOf(dt[g]);
        }
        if (gated) {
#pragma unroll
            for (int g = 0; g < 4; ++g) gate[g] = zs.Held(g) * LogisticOf(zs.Held(g));
        }
        fetch_tile(t + kScanTile);
        if (t + kScanTile <= last) {
            run(t, buffer, u, gate, dt, std::true_type{});
        } else {
#pragma unroll
            for (int g = 0; g < 4; ++g) dt[g] = t + 4 * g + at.q < last ? dt[g] : 0.f;
            run(t, buffer, u, gate, dt, std::false_type{});
        }
        ys.Move(1);
        if constexpr (ENDS) all_steps += (dt[0] + dt[1]) + (dt[2] + dt[3]);
    }
    if (!at.inside) return;
    if constexpr (ENDS) {
        StoreStates<NPL>(ends + (at.chunk + 1) * per_chunk, n0, p.states, h);
        all_steps += QuadSwap1(all_steps);
        all_steps += QuadSwap2(all_steps);
        if (at.q == 0) p.steps[(at.b * (p.chunks - 1) + at.chunk) * p.channels + at.channel] = all_steps;
        return;
    }
    for (int64_t row = std::max(t0, len) + at.q; row < end; row += 4) static_cast<T*>(p.y.data)[at.b * p.y.batch + row * p.y.row + at.channel] = static_cast<T>(0);
    if (at.chunk == p.chunks - 1) StoreStates<NPL>(p.new_state + of_state, n0, p.states, h);
}

// One row of each of V sequences: what a token costs is its states, read and written once: 128 x 4096 channels of 16 states in 17 us, 4.1 TB/s, and 256 in 27.5, 5.2.  The kernel
// above, whose threads start with tiles and LDS, takes 43 us for the first.  Four threads to a channel, each with a quarter of the states.
template <typename T, int NPL, int V>
__global__ __launch_bounds__(256) void ScanTokenKernel(ScanArgs p, int64_t first) {
    const int64_t index = first + static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x, line = index >> 2, b0 = line / p.channels * V;
    if (b0 >= p.batch) return;  // whole quads
    const int channel = static_cast<int>(line % p.channels), group = channel / p.group_channels, n0 = (static_cast<int>(threadIdx.x) & 3) * NPL;
    float h[V][NPL], a[NPL], bs[V][NPL], cs[V][NPL], u[V], raw[V], z[V];
    bool counts[V];
    LoadExponents<NPL>(p.a + static_cast<int64_t>(channel) * p.states, n0, p.states, a);
    const float bias = p.bias != nullptr ? p.bias[channel] : 0.f, d = p.d != nullptr ? p.d[channel] : 0.f;
#pragma unroll
    for (int v = 0; v < V; ++v) {
        const int64_t b = b0 + v < p.batch ? b0 + v : p.batch - 1;  // once more, for nothing, rather than a branch between the loads
        counts[v] = LengthOf(p.lengths, b, 1) != 0;
#pragma unroll
        for (int i = 0; i < NPL; ++i) h[v][i] = 0.f;
        if (p.state != nullptr) LoadStates<NPL>(p.state + (b * p.channels + channel) * p.states, n0, p.states, h[v]);
        const T* const from_b = static_cast<const T*>(p.b.data) + b * p.b.batch + group * p.b.group;
        const T* const from_c = static_cast<const T*>(p.c.data) + b * p.c.batch + group * p.c.group;
#pragma unroll
        for (int i = 0; i < NPL; ++i) {
            const int n = n0 + i < p.states ? n0 + i : p.states - 1;  // (a state that is not there is multiplied by what is, and left alone)
            bs[v][i] = static_cast<float>(from_b[n]), cs[v][i] = static_cast<float>(from_c[n]);
        }
        u[v] = static_cast<float>(static_cast<const T*>(p.u.data)[b * p.u.batch + channel]);
        raw[v] = static_cast<float>(static_cast<const T*>(p.delta.data)[b * p.delta.batch + channel]) + bias;
        z[v] = p.z.data != nullptr ? static_cast<float>(static_cast<const T*>(p.z.data)[b * p.z.batch + channel]) : 0.f;
    }
#pragma unroll
    for (int v = 0; v < V; ++v) {
        if (b0 + v >= p.batch) break;
        const float dt = p.softplus != 0 ? SoftplusOf(raw[v]) : raw[v], x = dt * u[v];
        float sum = 0.f;
#pragma unroll
        for (int i = 0; i < NPL; ++i) {
            const float next = __builtin_fmaf(x, bs[v][i], __builtin_amdgcn_exp2f(dt * a[i]) * h[v][i]);
            h[v][i] = counts[v] ? next : h[v][i];
            sum = n0 + i < p.states ? __builtin_fmaf(cs[v][i], next, sum) : sum;
        }
        sum += QuadSwap1(sum);
        sum += QuadSwap2(sum);
        const int64_t b = b0 + v;
        if (n0 == 0) {
            float y = __builtin_fmaf(d, p.d != nullptr ? u[v] : 0.f, sum);  // (0 times an infinite u would be NaN)
            if (p.z.data != nullptr) y *= z[v] * LogisticOf(z[v]);
            static_cast<T*>(p.y.data)[b * p.y.batch + channel] = static_cast<T>(counts[v] ? y : 0.f);
        }
        StoreStates<NPL>(p.new_state + (b * p.channels + channel) * p.states, n0, p.states, h[v]);
    }
}

}  // namespace

// us, forward, 16384 rows of 512 channels in 64, 128, 256 chunks: 102, 101, 147; of 64 channels in 64, 128, 256: 77, 67, 85; 4096 rows of 64 channels in 32, 64, 128: 42, 36, 46: a
// chunk goes through those before it, so that as many chunks as a chunk has rows are the best, less what a tile's 16 rows round off.  2048 rows, 2048 channels: 16 sequences (two
// workgroups to a compute unit) whole 404, in four chunks 469; 8 sequences whole 462, in 8 chunks 248; 4 sequences for 4, 8, 12 workgroups to a compute unit 142, 134, 141.
void CutScan(ScanArgs* p, int enough, int each, int least) {
    const int64_t tiles = DivUp(p->length, kScanTile), lines = p->batch * DivUp(p->channels, kScanChannels);
    int64_t chunks = 1;
    if (lines > 0 && lines < int64_t{NumCUs()} * enough) {
        chunks = std::min({int64_t{NumCUs()} * each / lines, tiles / least, static_cast<int64_t>(std::sqrt(static_cast<double>(p->length)))});
        chunks = std::max<int64_t>(chunks, 1);
    }
    const int64_t to_chunk = std::max<int64_t>(1, (tiles + chunks - 1) / chunks);
    p->chunk_rows = static_cast<int>(to_chunk) * kScanTile;
    p->chunks = static_cast<int>(std::max<int64_t>(1, (tiles + to_chunk - 1) / to_chunk));
}

namespace {

struct ScanWorkspace {
    int64_t ends, steps;  // floats
    explicit ScanWorkspace(const ScanArgs& p) : ends(0), steps(0) {
        if (p.chunks == 1) return;
        ends = p.batch * p.chunks * p.channels * p.states, steps = p.batch * (p.chunks - 1) * p.channels;
    }
    size_t Bytes() const { return static_cast<size_t>(ends + steps) * sizeof(float); }
};

}  // namespace

SequenceRows ScanRowsOf(const hipcx_array* a, const std::string& what) {
    SequenceRows r = RowsOf(a, what.c_str());
    if (a != nullptr && a->shape[1] <= 1) r.row = 0;
    HIPCX_REQUIRE(std::abs(r.row) < kMaxScanRow, HIPCX_NOT_IMPLEMENTED_ERROR, what + ": rows 2^26 elements apart or more");
    return r;
}

bool ScanSizesOf(const hipcx_array* u, const hipcx_array* a, ScanArgs* p) {
    if (u == nullptr || a == nullptr || u->ndim != 3 || a->ndim != 2 || a->shape[0] != u->shape[2]) return false;
    const int64_t batch = u->shape[0], length = u->shape[1], channels = u->shape[2], states = a->shape[1];
    if (batch < 0 || length < 0 || length >= kMaxScanLength || channels < 0 || channels >= kMaxScanChannels || states < 1 || states > kMaxScanStates) return false;
    p->batch = batch, p->length = length, p->channels = static_cast<int>(channels), p->states = static_cast<int>(states);
    return true;
}

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
    HIPCX_REQUIRE(states >= 1 && states <= kMaxScanStates, HIPCX_NOT_IMPLEMENTED_ERROR, what + ": 1 to 64 states, got " + std::to_string(states));
    HIPCX_REQUIRE(channels < kMaxScanChannels, HIPCX_NOT_IMPLEMENTED_ERROR, what + ": 2^24 channels or more");
    HIPCX_REQUIRE(b->ndim == 3 || b->ndim == 4, HIPCX_DIMENSION_ERROR, what + ": b must be [batch, time, states] or [batch, time, groups, states], got " + ShapeStr(b));
    HIPCX_REQUIRE(length < kMaxScanLength, HIPCX_NOT_IMPLEMENTED_ERROR, what + ": 2^30 rows or more");
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
    p.u = ScanRowsOf(u, what + ": u"), p.delta = ScanRowsOf(delta, what + ": delta"), p.z = ScanRowsOf(z, what + ": z");
    const auto shared = [&](const hipcx_array* s, const char* name) {
        const SequenceRows r = ScanRowsOf(s, what + name);
        return ScanShared{r.data, r.batch, r.row, s->ndim == 4 ? s->strides[2] / ItemSize(s->dtype) : 0};
    };
    p.b = shared(b, ": b"), p.c = shared(c, ": c");
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
    ScanArgs p{};
    if (!ScanSizesOf(u, a, &p)) return 0;
    CutScan(&p, 2, 8, 2);
    return ScanWorkspace(p).Bytes();
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
        p.y = ScanRowsOf(y, what + ": y"), p.new_state = static_cast<float*>(new_state->data);
        if (p.batch == 0 || p.channels == 0) return;
        CutScan(&p, 2, 8, 2);
        const ScanWorkspace w(p);
        HIPCX_REQUIRE(workspace_bytes >= w.Bytes() && (w.Bytes() == 0 || workspace != nullptr), HIPCX_CHAINERX_ERROR, what + ": the workspace is too small");
        p.ends = static_cast<float*>(workspace), p.steps = p.ends + w.ends;
        const int64_t blocks = p.batch * p.chunks * p.blocks;
        HIPCX_REQUIRE(p.length == 1 || blocks <= kBlocksPerLaunch, HIPCX_NOT_IMPLEMENTED_ERROR, what + ": too many elements");
        VisitScan(u->dtype, p.states, [&](auto tag, auto share) {
            using T = typename decltype(tag)::type;
            constexpr int NPL = decltype(share)::value;
            if (p.length == 1) {
                // Two sequences to a thread where that leaves a compute unit 16 waves.  us a call, with the host's part, of one, two and four: 128 x 4096 channels of 16
                // states, float16, 21.0, 19.0, 19.0; 256 x 4096 31.9, 30.0, 32.9; 128 x 4096 of 64 states 83, 79, 99.
                const bool two = p.batch / 2 * p.channels * 4 >= int64_t{NumCUs()} * 1024;
                ForLaunches((two ? (p.batch + 1) / 2 : p.batch) * p.channels * 4, [&](dim3 grid, int64_t first) {
                    if (two) hipLaunchKernelGGL((ScanTokenKernel<T, NPL, 2>), grid, dim3(256), 0, AsStream(stream), p, first);
                    else hipLaunchKernelGGL((ScanTokenKernel<T, NPL, 1>), grid, dim3(256), 0, AsStream(stream), p, first);
                    CheckLaunch("selective_scan");
                });
                return;
            }
            if (p.chunks > 1) {
                hipLaunchKernelGGL((SelectiveScanKernel<T, NPL, true, false, false>), dim3(static_cast<unsigned>(blocks - p.batch * p.blocks)), dim3(256), 0, AsStream(stream), p);
                CheckLaunch("selective_scan");
            }
            const auto launch = [&](auto repeats, auto few) {
                constexpr bool kRepeats = decltype(repeats)::value, kFew = decltype(few)::value;
                hipLaunchKernelGGL((SelectiveScanKernel<T, NPL, false, kRepeats, kFew>), dim3(static_cast<unsigned>(blocks)), dim3(256), 0, AsStream(stream), p);
            };
            const auto with_states = [&](auto few) { p.states == 4 * NPL ? launch(std::false_type{}, few) : launch(std::true_type{}, few); };
            if (NPL == 4 && blocks <= int64_t{NumCUs()} * 4) with_states(std::bool_constant<NPL == 4>{});
            else with_states(std::false_type{});
            CheckLaunch("selective_scan");
        });
    });
}

}  // extern "C"
