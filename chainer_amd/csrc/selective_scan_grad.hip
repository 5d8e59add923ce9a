// Gradients of the selective scan.  With g0 = gy silu(z) and q[t] the gradient of h[t]:
//   q[t] = g0[t] c[t] + exp(dt[t+1] a) q[t+1], x[t] = q[t] exp(dt[t] a) h[t-1]
//   gc[t] = sum over channels of g0 h[t],  gb[t] = sum over channels of q[t] dt u,  gu = d g0 + dt (q . b),  gdt = x . a + u (q . b),  ga = sum over t of dt x
#include "selective_scan.h"

namespace hipcx {
namespace {

struct ScanGradArgs {
    ScanArgs s;
    SequenceRows gy, gu, gdelta, gz;
    const float* gnew;  // gradient of the new state, or null
    float* gstate;      // or null
    float* states;      // [batch][tiles][channels][4 * NPL]: where each tile starts, of a chunk that starts from zeros
    float* passed;      // [batch][tiles][channels]: dt summed over the chunk's rows before the tile
    float* shared_parts;   // [batch][length][blocks][2][states]: gb and gc by workgroups along the channels
    float* channel_parts;  // [batch * chunks][channels][states + 2]: ga, gd, gbias
    float* starts;         // [batch][chunks][channels][states]: what a chunk's outputs give the state before it (of s.ends: where a chunk ends that starts from zeros)
    int tiles;             // of a sequence
};

// Rows whose states a lane keeps in registers on the way back: 64 states.  Those of 33 to 64 states take 256 registers and some 110 of the accumulators', with 3 to 6 spilled there, and leave one
// wave to a SIMD: 1.09 ms for 4 x 2048 rows of 2048 channels and 64 states, 2.7 times as long as 32.
template <int NPL>
constexpr int kGradTile = NPL <= 2 ? 16 : NPL == 4 ? 8 : 4;

__device__ __forceinline__ float AddRowRotations(float v) {  // over the four quads of 16 lanes
    v += __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, v), 0x128, 0xf, 0xf, true));
    return v + __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, v), 0x124, 0xf, 0xf, true));
}

template <typename V>
__device__ __forceinline__ float SumOf(const V& pair) {  // (a cast of an element in place reads the first one)
    const unsigned first = pair[0], second = pair[1];
    return __builtin_bit_cast(float, first) + __builtin_bit_cast(float, second);
}

// Sums over the wave's 16 channels of 4 * NPL values to a lane.  Two exchanges of half the registers leave every 16 lanes a quarter of the values, summed over the
// four rows of lanes: lanes 16 r .. 16 r + 15 hold values r * NPL .. r * NPL + NPL - 1.
template <int NPL>
__device__ __forceinline__ void SumOverChannels(const float (&v)[4 * NPL], float (&out)[NPL]) {
    float half[2 * NPL];
#pragma unroll
    for (int j = 0; j < 2 * NPL; ++j) {
        const auto r = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(unsigned, v[j]), __builtin_bit_cast(unsigned, v[j + 2 * NPL]), false, false);
        half[j] = SumOf(r);
    }
#pragma unroll
    for (int j = 0; j < NPL; ++j) {
        const auto r = __builtin_amdgcn_permlane16_swap(__builtin_bit_cast(unsigned, half[j]), __builtin_bit_cast(unsigned, half[j + NPL]), false, false);
        out[j] = AddRowRotations(SumOf(r));
    }
}

// dt, and dt u, of the rows that a lane has fetched; zeros behind the sequence's end.
template <typename T, int ROWS>
__device__ __forceinline__ void ScanSteps(const ScanArgs& p, const TileRows<T, ROWS>& us, const TileRows<T, ROWS>& ds, int q, int rows, float bias, float (&dt)[ROWS / 4],
                                          float (&x)[ROWS / 4]) {
#pragma unroll
    for (int g = 0; g < ROWS / 4; ++g) dt[g] = ds.Held(g) + bias;
    if (p.softplus != 0) {
#pragma unroll
        for (int g = 0; g < ROWS / 4; ++g) dt[g] = SoftplusOf(dt[g]);
    }
#pragma unroll
    for (int g = 0; g < ROWS / 4; ++g) {
        dt[g] = 4 * g + q < rows ? dt[g] : 0.f;
        x[g] = dt[g] * us.Held(g);
    }
}

// Chunks by themselves, from zeros: the states that their tiles start from, where they end, and what a chunk's outputs give the state before it -- the sum over its rows
// of g0 c times the decay since the chunk began, which runs forwards too.  CHUNKS: there is more than one, else the last two are not needed.
// Tiles' states as they come out of zeros, so that they are there before the state that the chunk starts from is known: the next launch adds exp(a * sum of dt) times it, an
// exponential a tile instead of a run through the rows (444 -> 425 us in all).  Stored in every tile without a condition: in a branch they cost a third of the waves (152 registers for
// 97, 137 us for 115 at 4 x 2048 rows of 2048 channels).  Bound by the vector units: seven instructions and an exponential a state, 44 instructions a row, 77 % of the issue slots.
template <typename T, int NPL, bool CHUNKS>
__device__ __forceinline__ void MakeTileStates(const ScanGradArgs& pg, const ScanPlace& at) {
    const ScanArgs& p = pg.s;
    constexpr int NP = 4 * NPL, kTile = kGradTile<NPL>;
    __shared__ float bs[2][kScanTile][NP], cs[CHUNKS ? 2 : 1][CHUNKS ? kScanTile : 1][NP];
    const int64_t len = LengthOf(p.lengths, at.b, p.length);
    const int64_t t0 = static_cast<int64_t>(at.chunk) * p.chunk_rows, last = std::min(std::min(t0 + p.chunk_rows, p.length), len);
    const int n0 = at.q * NPL;
    const int64_t per_tile = static_cast<int64_t>(p.channels) * NP;
    float a[NPL], h[NPL], start[NPL], decay[NPL];
    LoadExponents<NPL>(p.a + static_cast<int64_t>(at.channel) * p.states, n0, p.states, a);
#pragma unroll
    for (int i = 0; i < NPL; ++i) h[i] = start[i] = 0.f, decay[i] = 1.f;
    const float bias = p.bias != nullptr ? p.bias[at.channel] : 0.f;
    const bool gated = CHUNKS && p.z.data != nullptr;
    const int64_t first_tile = (at.b * pg.tiles + t0 / kTile) * p.channels + at.channel;
    float *states = pg.states + first_tile * NP + n0, *passed = pg.passed + first_tile;
    TileRows<T, kScanTile> us(p.u, at, t0), ds(p.delta, at, t0), zs(p.z, at, t0), gs(pg.gy, at, t0);
    TileShared<T, NPL, kScanTile, CHUNKS ? 2 : 1> shared(p, at, t0);
    const auto fetch_rows = [&](int rows, auto whole) __attribute__((always_inline)) {
        constexpr bool kWhole = decltype(whole)::value;
        us.template Fetch<kWhole>(at.q, rows);
        ds.template Fetch<kWhole>(at.q, rows);
        if constexpr (CHUNKS) gs.template Fetch<kWhole>(at.q, rows);
        if (gated) zs.template Fetch<kWhole>(at.q, rows);
        shared.template Fetch<kWhole>(rows);
        us.Move(1), ds.Move(1), zs.Move(1), gs.Move(1), shared.Move(1);
    };
    const auto fetch = [&](int64_t t) {
        if (t + kScanTile <= last) fetch_rows(kScanTile, std::true_type{});
        else if (t < last) fetch_rows(static_cast<int>(last - t), std::false_type{});
    };
    fetch(t0);
    float all_steps = 0.f;
    int buffer = 0;
    for (int64_t t = t0; t < last; t += kScanTile, buffer ^= 1) {
        shared.template Stage<0>(bs[buffer]);
        if constexpr (CHUNKS) shared.template Stage<1>(cs[buffer]);
        __syncthreads();
        float dt[4], x[4], g0[4];
        ScanSteps(p, us, ds, at.q, static_cast<int>(std::min<int64_t>(last - t, kScanTile)), bias, dt, x);
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            g0[g] = CHUNKS ? gs.Held(g) : 0.f;
            if (gated) g0[g] *= zs.Held(g) * LogisticOf(zs.Held(g));
        }
        fetch(t + kScanTile);
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            if (4 * g % kTile == 0) {  // unconditionally: a branch costs half the waves; lanes that stand for no channel write what the channel's own do
                LaneStates<NPL> tile_start;
#pragma unroll
                for (int i = 0; i < NPL; ++i) tile_start.v[i] = h[i];
                *reinterpret_cast<LaneStates<NPL>*>(states) = tile_start;
                *passed = all_steps;
                states += per_tile, passed += p.channels;
            }
            float four = dt[g] + QuadSwap1(dt[g]);
            four += QuadSwap2(four);
            all_steps += four;
            const auto step = [&](auto lane) __attribute__((always_inline)) {
                constexpr int S = decltype(lane)::value;
                const float dts = OfQuadLane<S>(dt[g]), xs = OfQuadLane<S>(x[g]), gys = OfQuadLane<S>(g0[g]);
#pragma unroll
                for (int i = 0; i < NPL; ++i) {
                    const float e = __builtin_amdgcn_exp2f(dts * a[i]);
                    h[i] = __builtin_fmaf(xs, bs[buffer][4 * g + S][n0 + i], e * h[i]);
                    if constexpr (CHUNKS) {
                        decay[i] *= e;
                        start[i] = __builtin_fmaf(gys * cs[buffer][4 * g + S][n0 + i], decay[i], start[i]);
                    }
                }
            };
            step(std::integral_constant<int, 0>{});
            step(std::integral_constant<int, 1>{});
            step(std::integral_constant<int, 2>{});
            step(std::integral_constant<int, 3>{});
        }
    }
    if (!CHUNKS || !at.inside) return;
    const int64_t line = (at.b * p.chunks + at.chunk) * p.channels + at.channel;
    StoreStates<NPL>(p.ends + line * p.states, n0, p.states, h);
    StoreStates<NPL>(pg.starts + line * p.states, n0, p.states, start);
    if (at.q == 0) p.steps[line] = all_steps;
}

template <typename T, int NPL, bool CHUNKS>
__global__ __launch_bounds__(256) void ScanGradStatesKernel(ScanGradArgs pg) {
    MakeTileStates<T, NPL, CHUNKS>(pg, ScanPlace(pg.s, blockIdx.x, pg.s.chunks));
}

// A chunk from its last tile to its first: the tile's states again, in registers, from those that it starts from, and the gradients.  STATES: sequences are whole, and their tiles'
// states are made here too.
// Bound by the vector units: 13 instructions and an exponential a state, the sums over channels (of two numbers a state and row; 18 % of the issue slots), 104 a row, 73 % of the issue slots at
// two waves to a SIMD.  4 x 2048 rows of 2048 channels of 16 states, float16: 271 us; 32 sequences 2040.  Tiles of 8 rows: 16 keep twice the states and decays, which
// leaves one wave (588 us in all for 462), and held to three waves by fewer registers it spills (1140).  One barrier a tile, with LDS for two.
template <typename T, int NPL, bool STATES>
__global__ __launch_bounds__(256) void SelectiveScanGradKernel(ScanGradArgs pg) {
    const ScanArgs& p = pg.s;
    constexpr int NP = 4 * NPL, kTile = kGradTile<NPL>, kGroups = kTile / 4;
    __shared__ float bs[2][kTile][NP], cs[2][kTile][NP], sums[2][4][kTile][2][NP];
    const ScanPlace at(p, blockIdx.x, p.chunks);
    if constexpr (STATES) MakeTileStates<T, NPL, false>(pg, at);  // every thread reads what it has written itself
    const int64_t len = LengthOf(p.lengths, at.b, p.length);
    const int64_t t0 = static_cast<int64_t>(at.chunk) * p.chunk_rows, end = std::min(t0 + p.chunk_rows, p.length), last = std::min(end, len);
    const int n0 = at.q * NPL, lane = static_cast<int>(threadIdx.x) & 63, wave = static_cast<int>(threadIdx.x) >> 6;
    const int64_t of_state = (at.b * p.channels + at.channel) * p.states, per_chunk = static_cast<int64_t>(p.channels) * p.states;
    float a[NPL], q[NPL], ga[NPL], first[NPL];  // first: the state that the chunk starts from
    LoadExponents<NPL>(p.a + static_cast<int64_t>(at.channel) * p.states, n0, p.states, a);
#pragma unroll
    for (int i = 0; i < NPL; ++i) q[i] = ga[i] = first[i] = 0.f;
    const float bias = p.bias != nullptr ? p.bias[at.channel] : 0.f, d = p.d != nullptr ? p.d[at.channel] : 0.f;
    const int64_t first_line = at.b * p.chunks * p.channels + at.channel;  // of the first chunk
    if (at.inside) {  // a lane that stands for no channel keeps zeros: it adds nothing to the sums over channels
        if (p.state != nullptr) LoadStates<NPL>(p.state + of_state, n0, p.states, first);
        ThroughChunks<NPL>(first, a, p.ends + first_line * p.states, p.steps + first_line, at.chunk, 1, per_chunk, p.channels, n0, p.states);
        if (pg.gnew != nullptr) LoadStates<NPL>(pg.gnew + of_state, n0, p.states, q);
        const int64_t last_line = first_line + static_cast<int64_t>(p.chunks - 1) * p.channels;
        ThroughChunks<NPL>(q, a, pg.starts + last_line * p.states, p.steps + last_line, p.chunks - 1 - at.chunk, -1, per_chunk, p.channels, n0, p.states);
    }
    const float* const states = pg.states + (at.b * pg.tiles * p.channels + at.channel) * NP + n0;
    const float* const passed = pg.passed + at.b * pg.tiles * p.channels + at.channel;
    const unsigned of_channels = blockIdx.x % static_cast<unsigned>(p.blocks);
    float gd = 0.f, gbias = 0.f;
    const bool gated = p.z.data != nullptr;
    const int64_t tiles = last > t0 ? (last - t0 + kTile - 1) / kTile : 0, top = t0 + (tiles - 1) * kTile;
    TileRows<T, kTile> us(p.u, at, top), ds(p.delta, at, top), zs(p.z, at, top), gys(pg.gy, at, top), gus(pg.gu, at, top), gds(pg.gdelta, at, top), gzs(pg.gz, at, top);
    TileShared<T, NPL, kTile, 2> shared(p, at, top);
    float next[NPL] = {}, next_passed = 0.f;  // where the fetched tile starts
    const auto fetch_rows = [&](int rows, auto whole) __attribute__((always_inline)) {
        constexpr bool kWhole = decltype(whole)::value;
        us.template Fetch<kWhole>(at.q, rows);
        ds.template Fetch<kWhole>(at.q, rows);
        gys.template Fetch<kWhole>(at.q, rows);
        if (gated) zs.template Fetch<kWhole>(at.q, rows);
    };
    const auto fetch = [&](int64_t t) __attribute__((always_inline)) {
        if (at.inside) {
            if (t + kTile <= last) fetch_rows(kTile, std::true_type{});
            else fetch_rows(static_cast<int>(last - t), std::false_type{});
            const LaneStates<NPL> start = *reinterpret_cast<const LaneStates<NPL>*>(states + t / kTile * p.channels * NP);
#pragma unroll
            for (int i = 0; i < NPL; ++i) next[i] = start.v[i];
            next_passed = passed[t / kTile * p.channels];
        }
        shared.template Fetch<false>(static_cast<int>(std::min<int64_t>(last - t, kTile)));
        us.Move(-1), ds.Move(-1), zs.Move(-1), gys.Move(-1), shared.Move(-1);
    };
    int buffer = 0;
    if (tiles > 0) {
        fetch(top);
        shared.template Stage<0>(bs[0]);
        shared.template Stage<1>(cs[0]);
        __syncthreads();
    }
    for (int64_t t = top; t >= t0; t -= kTile, buffer ^= 1) {
        const int rows = static_cast<int>(std::min<int64_t>(last - t, kTile)), own_rows = at.inside ? rows : 0;
        float u[kGroups], dt[kGroups], x[kGroups], g0[kGroups], slope[kGroups];
        ScanSteps(p, us, ds, at.q, own_rows, bias, dt, x);
        float h[kTile + 1][NPL], e[kTile][NPL], gz[kGroups], gu[kGroups], gdelta[kGroups];
        float of_y[kGroups];  // gz is the sum over states times this
#pragma unroll
        for (int g = 0; g < kGroups; ++g) u[g] = us.Held(g), g0[g] = gys.Held(g), slope[g] = 1.f, of_y[g] = 0.f;
        if (p.softplus != 0) {
#pragma unroll
            for (int g = 0; g < kGroups; ++g) slope[g] = LogisticOf(ds.Held(g) + bias);
        }
        if (gated) {
#pragma unroll
            for (int g = 0; g < kGroups; ++g) {
                const float z = zs.Held(g), l = LogisticOf(z);
                of_y[g] = g0[g] * l * __builtin_fmaf(z, 1.f - l, 1.f);
                g0[g] *= z * l;
            }
        }
#pragma unroll
        for (int i = 0; i < NPL; ++i) h[0][i] = __builtin_fmaf(__builtin_amdgcn_exp2f(next_passed * a[i]), first[i], next[i]);
        if (t > t0) fetch(t - kTile);
#pragma unroll
        for (int g = 0; g < kGroups; ++g) {
            float y[4];
            const auto step = [&](auto which) __attribute__((always_inline)) {
                constexpr int S = decltype(which)::value;
                const int r = 4 * g + S;
                const float dts = OfQuadLane<S>(dt[g]), xs = OfQuadLane<S>(x[g]);
                y[S] = 0.f;
#pragma unroll
                for (int i = 0; i < NPL; ++i) {
                    e[r][i] = __builtin_amdgcn_exp2f(dts * a[i]);
                    h[r + 1][i] = __builtin_fmaf(xs, bs[buffer][r][n0 + i], e[r][i] * h[r][i]);
                    y[S] = __builtin_fmaf(cs[buffer][r][n0 + i], h[r + 1][i], y[S]);
                }
            };
            step(std::integral_constant<int, 0>{});
            step(std::integral_constant<int, 1>{});
            step(std::integral_constant<int, 2>{});
            step(std::integral_constant<int, 3>{});
            gz[g] = of_y[g] * __builtin_fmaf(d, u[g], QuadTransposedSum(y, at.q));
        }
#pragma unroll
        for (int g = kGroups - 1; g >= 0; --g) {
            float qb[4], xa[4], of_b[4 * NPL], of_c[4 * NPL];
            const auto step = [&](auto which) __attribute__((always_inline)) {
                constexpr int S = decltype(which)::value;
                const int r = 4 * g + S;
                const float dts = OfQuadLane<S>(dt[g]), xs = OfQuadLane<S>(x[g]), gs = OfQuadLane<S>(g0[g]);
                qb[S] = xa[S] = 0.f;
#pragma unroll
                for (int i = 0; i < NPL; ++i) {
                    q[i] = __builtin_fmaf(gs, cs[buffer][r][n0 + i], q[i]);
                    of_c[S * NPL + i] = gs * h[r + 1][i];
                    of_b[S * NPL + i] = q[i] * xs;
                    qb[S] = __builtin_fmaf(q[i], bs[buffer][r][n0 + i], qb[S]);
                    q[i] *= e[r][i];
                    const float xi = q[i] * h[r][i];
                    ga[i] = __builtin_fmaf(dts, xi, ga[i]);
                    xa[S] = __builtin_fmaf(xi, a[i], xa[S]);
                }
            };
            step(std::integral_constant<int, 3>{});
            step(std::integral_constant<int, 2>{});
            step(std::integral_constant<int, 1>{});
            step(std::integral_constant<int, 0>{});
            const float qb_sum = QuadTransposedSum(qb, at.q), xa_sum = QuadTransposedSum(xa, at.q) * (1.f / kLog2E);
            gdelta[g] = __builtin_fmaf(u[g], qb_sum, xa_sum) * slope[g];
            gu[g] = __builtin_fmaf(d, g0[g], dt[g] * qb_sum);
            gbias += 4 * g + at.q < own_rows ? gdelta[g] : 0.f;
            gd = __builtin_fmaf(g0[g], u[g], gd);
            float sum_b[NPL], sum_c[NPL];
            SumOverChannels<NPL>(of_b, sum_b);
            SumOverChannels<NPL>(of_c, sum_c);
#pragma unroll
            for (int i = 0; i < NPL; ++i) sums[buffer][wave][4 * g + (lane >> 4)][(lane >> 2) & 1][n0 + i] = (lane & 4) == 0 ? sum_b[i] : sum_c[i];
        }
#pragma unroll
        for (int g = 0; g < kGroups; ++g) {  // (the stores together: branches between the groups would keep the compiler from mixing them)
            if (4 * g + at.q < own_rows) {
                gus[g] = static_cast<T>(gu[g]), gds[g] = static_cast<T>(gdelta[g]);
                if (gated) gzs[g] = static_cast<T>(gz[g]);
            }
        }
        gus.Move(-1), gds.Move(-1), gzs.Move(-1);
        if (t > t0) {
            shared.template Stage<0>(bs[buffer ^ 1]);
            shared.template Stage<1>(cs[buffer ^ 1]);
        }
        __syncthreads();  // of the other buffers, what was read before the last one of these
        for (int i = threadIdx.x; i < kTile * 2 * NP; i += 256) {
            const int r = i / (2 * NP), of = i / NP % 2, n = i % NP;
            if (n < p.states && r < rows) {
                const float s = (sums[buffer][0][r][of][n] + sums[buffer][1][r][of][n]) + (sums[buffer][2][r][of][n] + sums[buffer][3][r][of][n]);
                pg.shared_parts[(((at.b * p.length + t + r) * p.blocks + of_channels) * 2 + of) * p.states + n] = s;
            }
        }
    }
    gd += QuadSwap1(gd), gbias += QuadSwap1(gbias);
    gd += QuadSwap2(gd), gbias += QuadSwap2(gbias);
    if (!at.inside) return;
    for (int64_t row = std::max(t0, len) + at.q; row < end; row += 4) {
        for (const SequenceRows* r : {&pg.gu, &pg.gdelta, &pg.gz}) {
            if (r->data != nullptr) static_cast<T*>(r->data)[at.b * r->batch + row * r->row + at.channel] = static_cast<T>(0);
        }
    }
    if (pg.gstate != nullptr && at.chunk == 0) StoreStates<NPL>(pg.gstate + of_state, n0, p.states, q);
    float* const parts = pg.channel_parts + (first_line + static_cast<int64_t>(at.chunk) * p.channels) * (p.states + 2);
    StoreStates<NPL>(parts, n0, p.states, ga);
    if (at.q == 0) parts[p.states] = gd, parts[p.states + 1] = gbias;
}

struct ScanSumArgs {
    const float *shared, *channel;  // parts of gb and gc, of ga, gd and gbias
    SequenceLengths lengths;
    int64_t batch, length, shared_blocks, channel_parts, channels;
    int groups, group_blocks, states;
    void *gb, *gc;
    float *ga, *gd, *gbias;  // gd and gbias: or null
    int64_t first;           // the launch's first workgroup
};

// Both kinds of partial sums in one launch.  gb and gc: the workgroups along a group's channels, as many rows to a workgroup as it has threads for, an element to a thread.  Behind them ga, gd and
// gbias: the sequences and chunks, four threads to a column.
template <typename T>
__global__ __launch_bounds__(256) void ScanSumKernel(ScanSumArgs p) {
    __shared__ float sums[256];
    const int64_t block = p.first + blockIdx.x;
    float s = 0.f;
    if (block < p.shared_blocks) {
        const int width = 2 * p.states, rows = 256 / width, row = static_cast<int>(threadIdx.x) / width, within = static_cast<int>(threadIdx.x) - row * width;
        const int64_t at = block * rows + row;  // a sequence's row, a group
        if (row >= rows || at >= p.batch * p.length * p.groups) return;
        bool counts = true;
        if (p.lengths.data != nullptr) {
            const int64_t line = at / p.groups;
            counts = line % p.length < LengthOf(p.lengths, line / p.length, p.length);
        }
        if (counts) {
            const float* const from = p.shared + at * p.group_blocks * width + within;
#pragma unroll 8
            for (int i = 0; i < p.group_blocks; ++i) s += from[static_cast<int64_t>(i) * width];
        }
        const bool of_b = within < p.states;
        static_cast<T*>(of_b ? p.gb : p.gc)[at * p.states + (of_b ? within : within - p.states)] = static_cast<T>(s);
        return;
    }
    const int64_t width = p.channels * (p.states + 2), at = (block - p.shared_blocks) * 64 + (threadIdx.x & 63);
    if (at < width) {
#pragma unroll 4
        for (int64_t i = threadIdx.x >> 6; i < p.channel_parts; i += 4) s += p.channel[i * width + at];
    }
    sums[threadIdx.x] = s;
    __syncthreads();
    if (threadIdx.x >= 64 || at >= width) return;
    const float all = (sums[threadIdx.x] + sums[threadIdx.x + 64]) + (sums[threadIdx.x + 128] + sums[threadIdx.x + 192]);
    const int64_t channel = at / (p.states + 2);
    const int n = static_cast<int>(at % (p.states + 2));
    if (n < p.states) p.ga[channel * p.states + n] = all;
    else if (n == p.states && p.gd != nullptr) p.gd[channel] = all;
    else if (n > p.states && p.gbias != nullptr) p.gbias[channel] = all;
}

int GradTileOf(int states) { return states <= 8 ? 16 : states <= 16 ? 8 : 4; }

int PaddedStates(int states) { return states <= 4 ? 4 : states <= 8 ? 8 : states <= 16 ? 16 : states <= 32 ? 32 : 64; }

// Of a sequence, in whole tiles of the run that makes their states.
int64_t GradTiles(const ScanArgs& p) { return (p.length + kScanTile - 1) / kScanTile * (kScanTile / GradTileOf(p.states)); }

struct GradWorkspace {
    int64_t states, passed, shared, channels, ends, steps;  // floats
    explicit GradWorkspace(const ScanArgs& p)
        : states(p.batch * GradTiles(p) * p.channels * PaddedStates(p.states)), passed(states / PaddedStates(p.states)), shared(p.batch * p.length * p.blocks * 2 * p.states),
          channels(p.batch * p.chunks * p.channels * (p.states + 2)), ends(0), steps(0) {
        if (p.chunks > 1) ends = p.batch * p.chunks * p.channels * p.states, steps = p.batch * p.chunks * p.channels;
    }
    size_t Bytes() const { return static_cast<size_t>(states + passed + shared + channels + 2 * ends + steps) * sizeof(float); }
};

void CutScanGrad(ScanArgs* p) { CutScan(p, 2, 4, 2); }

}  // namespace
}  // namespace hipcx

using namespace hipcx;

extern "C" {

size_t hipcx_selective_scan_grad_workspace_size(const hipcx_array* u, const hipcx_array* a, const hipcx_array* b) {
    ScanArgs p{};
    if (!ScanSizesOf(u, a, &p) || b == nullptr || (b->ndim != 3 && b->ndim != 4)) return 0;
    const int64_t groups = b->ndim == 4 ? b->shape[2] : 1;
    if (b->shape[0] != p.batch || b->shape[1] != p.length || b->shape[b->ndim - 1] != p.states || groups < 1 || p.channels % groups != 0) return 0;
    if (p.batch == 0 || p.channels == 0) return 0;
    p.blocks = static_cast<int>(groups) * DivUp(p.channels / groups, kScanChannels);
    CutScanGrad(&p);
    return GradWorkspace(p).Bytes();
}

int hipcx_selective_scan_grad(const hipcx_array* u, const hipcx_array* delta, const hipcx_array* a, const hipcx_array* b, const hipcx_array* c, const hipcx_array* d,
                              const hipcx_array* z, const hipcx_array* delta_bias, int delta_softplus, const hipcx_array* state, const hipcx_array* lengths,
                              const hipcx_array* gy, const hipcx_array* gnew_state, const hipcx_array* gu, const hipcx_array* gdelta, const hipcx_array* ga,
                              const hipcx_array* gb, const hipcx_array* gc, const hipcx_array* gd, const hipcx_array* gz, const hipcx_array* gdelta_bias,
                              const hipcx_array* gstate, void* workspace, size_t workspace_bytes, void* stream) {
    return Guard([&] {
        const std::string what = "selective_scan_grad";
        ScanGradArgs p{};
        p.s = DescribeScan(what, u, delta, a, b, c, d, z, delta_bias, delta_softplus, state, lengths);
        const ScanArgs& s = p.s;
        for (const hipcx_array* x : {gy, gu, gdelta, ga, gb, gc}) HIPCX_REQUIRE(x != nullptr, HIPCX_CHAINERX_ERROR, what + ": gy, gu, gdelta, ga, gb and gc are needed");
        HIPCX_REQUIRE((z != nullptr) == (gz != nullptr), HIPCX_CHAINERX_ERROR, what + ": gz goes with z");
        for (const hipcx_array* x : {gy, gu, gdelta, gz}) RequireShape(x, {s.batch, s.length, s.channels}, u->dtype, what + ": gy, gu, gdelta and gz");
        for (const hipcx_array* x : {gb, gc}) {
            if (b->ndim == 4) RequireShape(x, {s.batch, s.length, b->shape[2], s.states}, u->dtype, what + ": gb and gc");
            else RequireShape(x, {s.batch, s.length, s.states}, u->dtype, what + ": gb and gc");
        }
        RequireShape(ga, {s.channels, s.states}, HIPCX_FLOAT32, what + ": ga");
        for (const hipcx_array* x : {gd, gdelta_bias}) RequireShape(x, {s.channels}, HIPCX_FLOAT32, what + ": gd and gdelta_bias");
        for (const hipcx_array* x : {gnew_state, gstate}) RequireShape(x, {s.batch, s.channels, s.states}, HIPCX_FLOAT32, what + ": gnew_state and gstate");
        for (const hipcx_array* x : {ga, gb, gc, gd, gdelta_bias, gnew_state, gstate}) RequireDense(x, what + ": ga, gb, gc, gd, gdelta_bias, gnew_state and gstate");
        p.gy = ScanRowsOf(gy, what + ": gy"), p.gu = ScanRowsOf(gu, what + ": gu"), p.gdelta = ScanRowsOf(gdelta, what + ": gdelta"), p.gz = ScanRowsOf(gz, what + ": gz");
        const auto floats = [](const hipcx_array* x) { return x != nullptr ? static_cast<float*>(x->data) : nullptr; };
        p.gnew = floats(gnew_state), p.gstate = floats(gstate);
        CutScanGrad(&p.s);
        const GradWorkspace w(s);
        const size_t need = w.Bytes();
        HIPCX_REQUIRE(workspace_bytes >= need && (need == 0 || workspace != nullptr), HIPCX_CHAINERX_ERROR, what + ": the workspace is too small");
        p.states = static_cast<float*>(workspace), p.passed = p.states + w.states, p.shared_parts = p.passed + w.passed, p.channel_parts = p.shared_parts + w.shared;
        p.s.ends = p.channel_parts + w.channels, p.starts = p.s.ends + w.ends, p.s.steps = p.starts + w.ends;
        p.tiles = static_cast<int>(GradTiles(s));
        const int64_t blocks = s.batch * s.chunks * s.blocks;
        HIPCX_REQUIRE(blocks <= kBlocksPerLaunch, HIPCX_NOT_IMPLEMENTED_ERROR, what + ": too many elements");
        VisitScan(u->dtype, s.states, [&](auto tag, auto share) {
            using T = typename decltype(tag)::type;
            constexpr int NPL = decltype(share)::value;
            if (blocks != 0) {
                const dim3 grid(static_cast<unsigned>(blocks));
                // Few whole sequences: a launch less counts for more than the tiles' states at the other kernel's waves.  us, two launches and one: 4 x 16 rows of 64 channels 51.5, 48.7,
                // 20 x 35 of 650 51.8, 50.0; 128 x 35 of 650 and 8 states 97.7, 100.7, 32 x 2048 of 2048 3276, 3465.
                if (s.chunks == 1 && blocks <= NumCUs()) {
                    hipLaunchKernelGGL((SelectiveScanGradKernel<T, NPL, true>), grid, dim3(256), 0, AsStream(stream), p);
                } else {
                    if (s.chunks > 1) hipLaunchKernelGGL((ScanGradStatesKernel<T, NPL, true>), grid, dim3(256), 0, AsStream(stream), p);
                    else hipLaunchKernelGGL((ScanGradStatesKernel<T, NPL, false>), grid, dim3(256), 0, AsStream(stream), p);
                    CheckLaunch(what.c_str());
                    hipLaunchKernelGGL((SelectiveScanGradKernel<T, NPL, false>), grid, dim3(256), 0, AsStream(stream), p);
                }
                CheckLaunch(what.c_str());
            }
            ScanSumArgs q{};
            q.shared = p.shared_parts, q.channel = p.channel_parts, q.lengths = s.lengths;
            q.batch = s.batch, q.length = s.length, q.channel_parts = s.batch * s.chunks, q.channels = s.channels;
            q.groups = b->ndim == 4 ? static_cast<int>(b->shape[2]) : 1, q.group_blocks = s.group_blocks, q.states = s.states;
            q.gb = gb->data, q.gc = gc->data, q.ga = floats(ga), q.gd = floats(gd), q.gbias = floats(gdelta_bias);
            const int64_t rows = 256 / (2 * s.states);
            q.shared_blocks = (s.batch * s.length * q.groups + rows - 1) / rows;
            const int64_t sum_blocks = q.shared_blocks + (static_cast<int64_t>(s.channels) * (s.states + 2) + 63) / 64;
            for (; q.first < sum_blocks; q.first += kBlocksPerLaunch) {
                hipLaunchKernelGGL(ScanSumKernel<T>, dim3(static_cast<unsigned>(std::min(sum_blocks - q.first, kBlocksPerLaunch))), dim3(256), 0, AsStream(stream), q);
                CheckLaunch(what.c_str());
            }
        });
    });
}

}  // extern "C"
