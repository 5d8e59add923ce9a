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
    float* states;      // [batch][tiles][channels][states]: where each tile starts
    float* shared_parts;   // [batch][length][blocks][2][states]: gb and gc by workgroups along the channels
    float* channel_parts;  // [batch * chunks][channels][states + 2]: ga, gd, gbias
    int tiles;             // of a sequence
};

// Rows whose states a lane keeps in registers on the way back: 64 states.
template <int NPL>
constexpr int kGradTile = NPL <= 4 ? 16 : 64 / NPL;

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

// The states that each tile starts from: the forward recurrence, without its outputs.
template <typename T, int NPL>
__global__ __launch_bounds__(256) void ScanStatesKernel(ScanGradArgs pg) {
    const ScanArgs& p = pg.s;
    constexpr int NP = 4 * NPL, kEach = (kScanTile * NP + 255) / 256, kTile = kGradTile<NPL>;
    __shared__ float bs[2][kScanTile][NP];
    const ScanPlace at(p, blockIdx.x, 1);
    const int64_t len = LengthOf(p.lengths, at.b, p.length);
    const int n0 = at.q * NPL;
    float a[NPL], h[NPL];
    LoadStates<NPL>(p.a + static_cast<int64_t>(at.channel) * p.states, n0, p.states, a);
#pragma unroll
    for (int i = 0; i < NPL; ++i) a[i] *= kLog2E, h[i] = 0.f;
    if (p.state != nullptr) LoadStates<NPL>(p.state + (at.b * p.channels + at.channel) * p.states, n0, p.states, h);
    const float bias = p.bias != nullptr ? p.bias[at.channel] : 0.f;
    const T* const b = static_cast<const T*>(p.b.data) + at.b * p.b.batch + at.group * p.b.group;
    int buffer = 0;
    for (int64_t t = 0; t < len; t += kScanTile, buffer ^= 1) {
#pragma unroll
        for (int i = 0; i < kEach; ++i) {
            const int e = i * 256 + static_cast<int>(threadIdx.x), r = e / NP, n = e % NP;
            if (e < kScanTile * NP) bs[buffer][r][n] = n < p.states && t + r < len ? static_cast<float>(b[(t + r) * p.b.row + n]) : 0.f;
        }
        __syncthreads();
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            const int64_t row = t + 4 * g + at.q;
            float dt = 0.f, x = 0.f;
            if (row < len) {
                const float raw = ScanRead<T>(p.delta, at.b, row, at.channel) + bias;
                dt = p.softplus != 0 ? SoftplusOf(raw) : raw;
                x = dt * ScanRead<T>(p.u, at.b, row, at.channel);
            }
            if (4 * g % kTile == 0 && t + 4 * g < len && at.inside) {
                float* const to = pg.states + ((at.b * pg.tiles + (t + 4 * g) / kTile) * p.channels + at.channel) * p.states;
                StoreStates<NPL>(to, n0, p.states, h);
            }
            const auto step = [&](auto lane) {
                constexpr int S = decltype(lane)::value;
                const float dts = OfQuadLane<S>(dt), xs = OfQuadLane<S>(x);
#pragma unroll
                for (int i = 0; i < NPL; ++i) h[i] = __builtin_fmaf(xs, bs[buffer][4 * g + S][n0 + i], __builtin_amdgcn_exp2f(dts * a[i]) * h[i]);
            };
            step(std::integral_constant<int, 0>{});
            step(std::integral_constant<int, 1>{});
            step(std::integral_constant<int, 2>{});
            step(std::integral_constant<int, 3>{});
        }
    }
}

template <typename T, int NPL>
__global__ __launch_bounds__(256) void SelectiveScanGradKernel(ScanGradArgs pg) {
    const ScanArgs& p = pg.s;
    constexpr int NP = 4 * NPL, kTile = kGradTile<NPL>, kGroups = kTile / 4;
    __shared__ float bs[kTile][NP], cs[kTile][NP], sums[4][kTile][2][NP];
    const ScanPlace at(p, blockIdx.x, 1);
    const int64_t len = LengthOf(p.lengths, at.b, p.length);
    const int n0 = at.q * NPL, lane = static_cast<int>(threadIdx.x) & 63, wave = static_cast<int>(threadIdx.x) >> 6;
    const int64_t of_state = (at.b * p.channels + at.channel) * p.states;
    float a[NPL], q[NPL], ga[NPL];
    LoadStates<NPL>(p.a + static_cast<int64_t>(at.channel) * p.states, n0, p.states, a);
#pragma unroll
    for (int i = 0; i < NPL; ++i) a[i] *= kLog2E, q[i] = ga[i] = 0.f;
    if (pg.gnew != nullptr && at.inside) LoadStates<NPL>(pg.gnew + of_state, n0, p.states, q);
    const float bias = p.bias != nullptr ? p.bias[at.channel] : 0.f, d = p.d != nullptr ? p.d[at.channel] : 0.f;
    const T* const b = static_cast<const T*>(p.b.data) + at.b * p.b.batch + at.group * p.b.group;
    const T* const c = static_cast<const T*>(p.c.data) + at.b * p.c.batch + at.group * p.c.group;
    const unsigned of_channels = blockIdx.x % static_cast<unsigned>(p.blocks);
    float gd = 0.f, gbias = 0.f;
    for (int64_t tile = (len + kTile - 1) / kTile - 1; tile >= 0; --tile) {
        const int64_t t = tile * kTile;
        for (int e = threadIdx.x; e < kTile * NP; e += 256) {
            const int r = e / NP, n = e % NP;
            const bool is = n < p.states && t + r < len;
            bs[r][n] = is ? static_cast<float>(b[(t + r) * p.b.row + n]) : 0.f;
            cs[r][n] = is ? static_cast<float>(c[(t + r) * p.c.row + n]) : 0.f;
        }
        float u[kGroups], dt[kGroups], x[kGroups], g0[kGroups], gy[kGroups], slope[kGroups], z[kGroups];
#pragma unroll
        for (int g = 0; g < kGroups; ++g) {
            const int64_t row = t + 4 * g + at.q;
            u[g] = dt[g] = x[g] = g0[g] = gy[g] = z[g] = 0.f, slope[g] = 1.f;
            if (row < len && at.inside) {  // a lane that stands for no channel keeps zeros: it adds nothing to the sums over channels
                const float raw = ScanRead<T>(p.delta, at.b, row, at.channel) + bias;
                u[g] = ScanRead<T>(p.u, at.b, row, at.channel);
                dt[g] = p.softplus != 0 ? SoftplusOf(raw) : raw;
                if (p.softplus != 0) slope[g] = LogisticOf(raw);
                x[g] = dt[g] * u[g];
                g0[g] = gy[g] = ScanRead<T>(pg.gy, at.b, row, at.channel);
                if (p.z.data != nullptr) {
                    z[g] = ScanRead<T>(p.z, at.b, row, at.channel);
                    g0[g] *= z[g] * LogisticOf(z[g]);
                }
            }
        }
        float h[kTile + 1][NPL], e[kTile][NPL];
#pragma unroll
        for (int i = 0; i < NPL; ++i) h[0][i] = 0.f;
        if (at.inside) LoadStates<NPL>(pg.states + ((at.b * pg.tiles + tile) * p.channels + at.channel) * p.states, n0, p.states, h[0]);
        __syncthreads();
#pragma unroll
        for (int g = 0; g < kGroups; ++g) {
            float y[4];
            const auto step = [&](auto which) {
                constexpr int S = decltype(which)::value;
                const int r = 4 * g + S;
                const float dts = OfQuadLane<S>(dt[g]), xs = OfQuadLane<S>(x[g]);
                y[S] = 0.f;
#pragma unroll
                for (int i = 0; i < NPL; ++i) {
                    e[r][i] = __builtin_amdgcn_exp2f(dts * a[i]);
                    h[r + 1][i] = __builtin_fmaf(xs, bs[r][n0 + i], e[r][i] * h[r][i]);
                    y[S] = __builtin_fmaf(cs[r][n0 + i], h[r + 1][i], y[S]);
                }
            };
            step(std::integral_constant<int, 0>{});
            step(std::integral_constant<int, 1>{});
            step(std::integral_constant<int, 2>{});
            step(std::integral_constant<int, 3>{});
            if (p.z.data != nullptr) {
                const float y0 = __builtin_fmaf(d, u[g], QuadTransposedSum(y, at.q)), l = LogisticOf(z[g]);
                const int64_t row = t + 4 * g + at.q;
                if (at.inside && row < len) {
                    static_cast<T*>(pg.gz.data)[at.b * pg.gz.batch + row * pg.gz.row + at.channel] = static_cast<T>(gy[g] * y0 * l * __builtin_fmaf(z[g], 1.f - l, 1.f));
                }
            }
        }
#pragma unroll
        for (int g = kGroups - 1; g >= 0; --g) {
            float qb[4], xa[4], of_b[4 * NPL], of_c[4 * NPL];
            const auto step = [&](auto which) {
                constexpr int S = decltype(which)::value;
                const int r = 4 * g + S;
                const float dts = OfQuadLane<S>(dt[g]), xs = OfQuadLane<S>(x[g]), gs = OfQuadLane<S>(g0[g]);
                qb[S] = xa[S] = 0.f;
#pragma unroll
                for (int i = 0; i < NPL; ++i) {
                    q[i] = __builtin_fmaf(gs, cs[r][n0 + i], q[i]);
                    of_c[S * NPL + i] = gs * h[r + 1][i];
                    of_b[S * NPL + i] = q[i] * xs;
                    qb[S] = __builtin_fmaf(q[i], bs[r][n0 + i], qb[S]);
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
            const float gdelta = __builtin_fmaf(u[g], qb_sum, xa_sum) * slope[g];
            const int64_t row = t + 4 * g + at.q;
            if (row < len) {
                gbias += gdelta;
                gd = __builtin_fmaf(g0[g], u[g], gd);
                if (at.inside) {
                    static_cast<T*>(pg.gu.data)[at.b * pg.gu.batch + row * pg.gu.row + at.channel] = static_cast<T>(__builtin_fmaf(d, g0[g], dt[g] * qb_sum));
                    static_cast<T*>(pg.gdelta.data)[at.b * pg.gdelta.batch + row * pg.gdelta.row + at.channel] = static_cast<T>(gdelta);
                }
            }
            float sum_b[NPL], sum_c[NPL];
            SumOverChannels<NPL>(of_b, sum_b);
            SumOverChannels<NPL>(of_c, sum_c);
            if (((lane >> 2) & 3) == 0) {
#pragma unroll
                for (int i = 0; i < NPL; ++i) sums[wave][4 * g + (lane >> 4)][0][n0 + i] = sum_b[i], sums[wave][4 * g + (lane >> 4)][1][n0 + i] = sum_c[i];
            }
        }
        __syncthreads();
        for (int i = threadIdx.x; i < kTile * 2 * NP; i += 256) {
            const int r = i / (2 * NP), of = i / NP % 2, n = i % NP;
            if (n < p.states && t + r < len) {
                const float s = (sums[0][r][of][n] + sums[1][r][of][n]) + (sums[2][r][of][n] + sums[3][r][of][n]);
                pg.shared_parts[(((at.b * p.length + t + r) * p.blocks + of_channels) * 2 + of) * p.states + n] = s;
            }
        }
    }
    gd += QuadSwap1(gd), gbias += QuadSwap1(gbias);
    gd += QuadSwap2(gd), gbias += QuadSwap2(gbias);
    if (!at.inside) return;
    for (int64_t row = len + at.q; row < p.length; row += 4) {
        for (const SequenceRows* r : {&pg.gu, &pg.gdelta, &pg.gz}) {
            if (r->data != nullptr) static_cast<T*>(r->data)[at.b * r->batch + row * r->row + at.channel] = static_cast<T>(0);
        }
    }
    if (pg.gstate != nullptr) StoreStates<NPL>(pg.gstate + of_state, n0, p.states, q);
    float* const parts = pg.channel_parts + (at.b * p.channels + at.channel) * (p.states + 2);
    StoreStates<NPL>(parts, n0, p.states, ga);
    if (at.q == 0) parts[p.states] = gd, parts[p.states + 1] = gbias;
}

// gb and gc: the workgroups along a group's channels added up, an element to a thread.
template <typename T>
__global__ __launch_bounds__(256) void ScanSharedSumKernel(const float* parts, SequenceLengths lengths, int64_t batch, int64_t length, int groups, int group_blocks, int states,
                                                          T* gb, T* gc, int64_t first) {
    const int64_t index = first + static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
    const int n = static_cast<int>(index % states);
    const int64_t rest = index / states;
    const int of = static_cast<int>(rest % 2), group = static_cast<int>(rest / 2 % groups);
    const int64_t line = rest / 2 / groups;
    if (line >= batch * length) return;
    float s = 0.f;
    if (line % length < LengthOf(lengths, line / length, length)) {
        const float* const from = parts + (((line * groups + group) * group_blocks) * 2 + of) * states + n;
        for (int i = 0; i < group_blocks; ++i) s += from[static_cast<int64_t>(i) * 2 * states];
    }
    (of == 0 ? gb : gc)[(line * groups + group) * states + n] = static_cast<T>(s);
}

// ga, gd and gbias: the sequences and chunks added up, four threads to a column.
__global__ __launch_bounds__(256) void ScanChannelSumKernel(const float* parts, int64_t n_parts, int64_t channels, int states, float* ga, float* gd, float* gbias) {
    __shared__ float sums[256];
    const int64_t width = channels * (states + 2), at = static_cast<int64_t>(blockIdx.x) * 64 + (threadIdx.x & 63);
    float s = 0.f;
    if (at < width) {
        for (int64_t i = threadIdx.x >> 6; i < n_parts; i += 4) s += parts[i * width + at];
    }
    sums[threadIdx.x] = s;
    __syncthreads();
    if (threadIdx.x >= 64 || at >= width) return;
    const float all = (sums[threadIdx.x] + sums[threadIdx.x + 64]) + (sums[threadIdx.x + 128] + sums[threadIdx.x + 192]);
    const int64_t channel = at / (states + 2);
    const int n = static_cast<int>(at % (states + 2));
    if (n < states) ga[channel * states + n] = all;
    else if (n == states && gd != nullptr) gd[channel] = all;
    else if (n > states && gbias != nullptr) gbias[channel] = all;
}

int GradTileOf(int states) { return states <= 16 ? 16 : states <= 32 ? 8 : 4; }

struct GradWorkspace {
    int64_t states, shared, channels;  // floats
    GradWorkspace(const ScanArgs& p)
        : states(p.batch * ((p.length + GradTileOf(p.states) - 1) / GradTileOf(p.states)) * p.channels * p.states),
          shared(p.batch * p.length * p.blocks * 2 * p.states), channels(p.batch * p.channels * (p.states + 2)) {}
    size_t Bytes() const { return static_cast<size_t>(states + shared + channels) * sizeof(float); }
};

}  // namespace
}  // namespace hipcx

using namespace hipcx;

extern "C" {

size_t hipcx_selective_scan_grad_workspace_size(const hipcx_array* u, const hipcx_array* a, const hipcx_array* b) {
    if (u == nullptr || a == nullptr || b == nullptr || u->ndim != 3 || a->ndim != 2 || (b->ndim != 3 && b->ndim != 4)) return 0;
    ScanArgs p{};
    const int64_t groups = b->ndim == 4 ? b->shape[2] : 1;
    if (groups < 1 || u->shape[0] <= 0 || u->shape[2] <= 0 || u->shape[2] % groups != 0) return 0;
    p.batch = u->shape[0], p.length = u->shape[1], p.channels = static_cast<int>(u->shape[2]), p.states = static_cast<int>(a->shape[1]);
    p.blocks = static_cast<int>(groups) * DivUp(u->shape[2] / groups, kScanChannels);
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
        p.gy = RowsOf(gy, "gy"), p.gu = RowsOf(gu, "gu"), p.gdelta = RowsOf(gdelta, "gdelta"), p.gz = RowsOf(gz, "gz");
        const auto floats = [](const hipcx_array* x) { return x != nullptr ? static_cast<float*>(x->data) : nullptr; };
        p.gnew = floats(gnew_state), p.gstate = floats(gstate);
        const GradWorkspace w(s);
        const size_t need = w.Bytes();
        HIPCX_REQUIRE(workspace_bytes >= need && (need == 0 || workspace != nullptr), HIPCX_CHAINERX_ERROR, what + ": the workspace is too small");
        p.states = static_cast<float*>(workspace), p.shared_parts = p.states + w.states, p.channel_parts = p.shared_parts + w.shared;
        p.tiles = DivUp(s.length, GradTileOf(s.states));
        const int64_t blocks = s.batch * s.blocks;
        HIPCX_REQUIRE(blocks <= kBlocksPerLaunch, HIPCX_NOT_IMPLEMENTED_ERROR, what + ": too many elements");
        VisitScan(u->dtype, s.states, [&](auto tag, auto share) {
            using T = typename decltype(tag)::type;
            constexpr int NPL = decltype(share)::value;
            if (blocks != 0) {
                hipLaunchKernelGGL((ScanStatesKernel<T, NPL>), dim3(static_cast<unsigned>(blocks)), dim3(256), 0, AsStream(stream), p);
                CheckLaunch(what.c_str());
                hipLaunchKernelGGL((SelectiveScanGradKernel<T, NPL>), dim3(static_cast<unsigned>(blocks)), dim3(256), 0, AsStream(stream), p);
                CheckLaunch(what.c_str());
            }
            const int groups = b->ndim == 4 ? static_cast<int>(b->shape[2]) : 1;
            ForLaunches(s.batch * s.length * groups * 2 * s.states, [&](dim3 grid, int64_t first) {
                hipLaunchKernelGGL(ScanSharedSumKernel<T>, grid, dim3(256), 0, AsStream(stream), p.shared_parts, s.lengths, s.batch, s.length, groups, s.group_blocks,
                                   s.states, static_cast<T*>(gb->data), static_cast<T*>(gc->data), first);
                CheckLaunch(what.c_str());
            });
        });
        const int64_t columns = static_cast<int64_t>(s.channels) * (s.states + 2);
        if (columns == 0) return;
        hipLaunchKernelGGL(ScanChannelSumKernel, dim3(static_cast<unsigned>((columns + 63) / 64)), dim3(256), 0, AsStream(stream), p.channel_parts, s.batch, s.channels, s.states,
                           floats(ga), floats(gd), floats(gdelta_bias));
        CheckLaunch(what.c_str());
    });
}

}  // extern "C"
