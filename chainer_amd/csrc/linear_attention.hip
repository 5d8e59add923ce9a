// Linear attention: chunks of rows as matrix products, single rows as they come.
#include <cstdlib>

#include "igemm.h"
#include "linear_attention.h"

namespace hipcx {
namespace {

struct AttendTag {};

__device__ __forceinline__ float Finite(float v) { return v - v; }  // 0, or not a number

// Tiles of 64 rows, one after another.  With G the decays summed up from the tile's first row and S the state before it,
//   P[t][s] = exp(G[t] - G[s]) q[t] k[s] for s <= t,  y = P v + exp(G) q S,  S <- exp(G[63]) S + (exp(G[63] - G) k)^T v.
// A workgroup of four waves has 64 columns of v: a wave multiplies 32 rows by 32 columns of y, and has half of the keys and 32 columns of S in its accumulators (a copy is in LDS, for the products with q).
// P stays in registers: as k q^T its column t is a lane, whose rows s are the reduction of the product v^T P.
// Products run on the float pipe (v_mfma_f32_32x32x2_f32).
template <int KD, bool OUT>
__global__ __launch_bounds__(256) void AttendKernel(AttendArgs p) {
    using T = float;
    constexpr int KP = KD + 4, VB = kAttendColumns, C = kAttendTile, NS = KD / 64;
    extern __shared__ __align__(16) char lds[];
    float* const ks = reinterpret_cast<float*>(lds);      // [C][KP]
    float* const vs = ks + C * KP;                        // [C][VB]
    float* const ss = vs + C * VB;                        // [KD][VB]
    float* const red = ss + KD * VB;                      // [4][VB]
    AttendDecays* const dec = reinterpret_cast<AttendDecays*>(red + 4 * VB);
    int* const odd = reinterpret_cast<int*>(dec + 1);     // v has infinities or what is not a number

    int id = AttendNumber(p);
    if (id < 0) return;
    const int block = id % p.blocks;
    id /= p.blocks;
    const int bh = id % static_cast<int>(p.batch * p.heads);
    const int segment_turn = id / static_cast<int>(p.batch * p.heads);
    int which = 0;
    while (which + 1 < p.runs && block >= p.run[which + 1].first) ++which;
    const AttendRun& run = p.run[which];
    const int segment = run.back ? p.segments - 1 - segment_turn : segment_turn;
    const int64_t b = bh / p.heads;
    const int h = bh % p.heads;
    const int64_t length = LengthOf(p.lengths, b, p.length);
    const AttendSpan span(p, length, segment);
    const int64_t rows = span.end - span.first;
    const int col0 = (block - run.first) * VB, cols = min(VB, run.values - col0);

    const int tid = threadIdx.x, lane = tid % 64, wave = tid / 64, l32 = lane % 32, half = lane / 32;
    const int tw = wave / 2, dw = wave % 2;
    const T* const kp = static_cast<const T*>(run.k.data) + b * run.k.batch + (h / run.k.share) * run.k.head;
    const T* const vp = static_cast<const T*>(run.v.data) + b * run.v.batch + (h / run.v.share) * run.v.head + col0;
    const T* const qp = OUT ? static_cast<const T*>(run.q.data) + b * run.q.batch + (h / run.q.share) * run.q.head : nullptr;
    const T* const dp = OUT && run.dots != nullptr ? static_cast<const T*>(run.dot.data) + b * run.dot.batch + (h / run.dot.share) * run.dot.head + col0 : nullptr;
    const int64_t y0 = OUT ? b * run.y.batch + h * run.y.head + col0 : 0;
    float* const dots = OUT && run.dots != nullptr ? run.dots + (static_cast<int64_t>(bh) * run.blocks + block - run.first) * p.length : nullptr;

    // element r of a state's accumulator n: row i, column j of the workgroup's
    const auto state_row = [&](int n, int r) { return KD / 2 * tw + 32 * n + 8 * (r / 4) + 4 * half + r % 4; };
    const int state_col = 32 * dw + l32;
    attend16_t s[NS];
#pragma unroll
    for (int n = 0; n < NS; ++n) {
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            const int i = state_row(n, r);
            s[n][r] = OUT && run.start.data != nullptr && i < run.keys && state_col < cols
                          ? run.start.data[bh * run.start.head + segment * run.start.segment + i * run.start.i + (col0 + state_col) * run.start.j]
                          : 0.f;
        }
    }
    const auto keep_state = [&] {
#pragma unroll
        for (int n = 0; n < NS; ++n) {
#pragma unroll
            for (int r = 0; r < 16; ++r) ss[state_row(n, r) * VB + state_col] = s[n][r];
        }
    };
    if (OUT) keep_state();
    double passed = 0;  // log decay of the tiles so far

    for (int64_t r0 = 0; r0 < rows; r0 += C) {
        const int here = static_cast<int>(rows - r0 < C ? rows - r0 : C);
        if (tid == 0) *odd = 0;
        __syncthreads();
        for (int at = tid; at < C * KD / 4; at += 256) {
            const int row = at / (KD / 4), i = at % (KD / 4) * 4;
            attend4_t v{0, 0, 0, 0};
            if (row < here) {
                const AttendPiece<T, 4> piece = AttendLoad<T, 4>(kp + AttendRowOf(span, run.back, r0 + row) * run.k.row, i, run.keys);
#pragma unroll
                for (int e = 0; e < 4; ++e) v[e] = static_cast<float>(piece.v[e]);
            }
            *reinterpret_cast<attend4_t*>(ks + row * KP + i) = v;
        }
        for (int at = tid; at < C * VB / 4; at += 256) {
            const int row = at / (VB / 4), j = at % (VB / 4) * 4;
            attend4_t v{0, 0, 0, 0};
            if (row < here) {
                const AttendPiece<T, 4> piece = AttendLoad<T, 4>(vp + AttendRowOf(span, run.back, r0 + row) * run.v.row, j, cols);
#pragma unroll
                for (int e = 0; e < 4; ++e) v[e] = static_cast<float>(piece.v[e]);
                if (OUT && Finite(v[0]) + Finite(v[1]) + Finite(v[2]) + Finite(v[3]) != 0) *odd = 1;
            }
            *reinterpret_cast<attend4_t*>(vs + row * VB + j) = v;
        }
        if (wave == 0) SumDecays(dec, lane < here ? AttendStep(p, run, span, b, h, length, r0 + lane) : 0, here, run.kv_scale);
        attend4_t q[OUT ? KD / 8 : 1];
        const int t = 32 * tw + l32;  // this lane's row
        if constexpr (OUT) {
#pragma unroll
            for (int m = 0; m < KD / 8; ++m) {
                q[m] = attend4_t{0, 0, 0, 0};
                if (t < here) {
                    const AttendPiece<T, 4> piece = AttendLoad<T, 4>(qp + AttendRowOf(span, run.back, r0 + t) * run.q.row, 8 * m + 4 * half, run.keys);
#pragma unroll
                    for (int e = 0; e < 4; ++e) q[m][e] = static_cast<float>(piece.v[e]);
                }
            }
        }
        __syncthreads();
        passed += dec->sum;
        if (OUT && *odd != 0) {
            // An infinity of a later row, times P's zeros, would reach earlier ones: row by row instead, on the copy in LDS.
            const int j = lane;
            for (int r = 0; r < here; ++r) {
                const int64_t row = AttendRowOf(span, run.back, r0 + r);
                const float step = dec->step[r], v = vs[r * VB + j] * run.kv_scale;
                float y = 0;
                for (int i = wave * (KD / 4); i < (wave + 1) * (KD / 4); ++i) {
                    const float now = ss[i * VB + j] * step + ks[r * KP + i] * v;
                    ss[i * VB + j] = now;
                    if (i < run.keys) y += static_cast<float>(qp[row * run.q.row + i]) * now;
                }
                red[wave * VB + j] = y;
                __syncthreads();
                if (wave == 0) {
                    y = (red[j] + red[VB + j] + red[2 * VB + j] + red[3 * VB + j]) * run.out_scale;
                    if (j < cols) {
                        if (run.wide) static_cast<float*>(run.y.data)[y0 + row * run.y.row + j] = y;
                        else static_cast<T*>(run.y.data)[y0 + row * run.y.row + j] = static_cast<T>(y);
                    }
                    if (dots != nullptr) {
                        float dot = j < cols ? y * static_cast<float>(dp[row * run.dot.row + j]) : 0.f;
#pragma unroll
                        for (int o = 1; o < 64; o <<= 1) dot += __shfl_xor(dot, o);
                        if (lane == 0) dots[row] = dot;
                    }
                }
                __syncthreads();
            }
#pragma unroll
            for (int n = 0; n < NS; ++n) {
#pragma unroll
                for (int r = 0; r < 16; ++r) s[n][r] = ss[state_row(n, r) * VB + state_col];
            }
            continue;
        }
        if constexpr (OUT) {
            const float high = dec->high[t], low = dec->low[t];
            attend16_t y{};
#pragma unroll
            for (int m = 0; m < KD / 8; ++m) {
#pragma unroll
                for (int e = 0; e < 4; ++e) y = __builtin_amdgcn_mfma_f32_32x32x2f32(ss[(8 * m + 4 * half + e) * VB + state_col], q[m][e], y, 0, 0, 0);
            }
            const float from_start = __builtin_amdgcn_exp2f(high + low);
#pragma unroll
            for (int r = 0; r < 16; ++r) y[r] *= from_start;
            for (int sb = 0; sb <= tw; ++sb) {  // rows up to this wave's
                attend16_t a{};
#pragma unroll
                for (int m = 0; m < KD / 8; ++m) {
                    const attend4_t k = *reinterpret_cast<const attend4_t*>(ks + (32 * sb + l32) * KP + 8 * m + 4 * half);
#pragma unroll
                    for (int e = 0; e < 4; ++e) a = __builtin_amdgcn_mfma_f32_32x32x2f32(k[e], q[m][e], a, 0, 0, 0);
                }
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    const int at = 32 * sb + 8 * (r / 4) + 4 * half + r % 4;
                    const float weight = __builtin_amdgcn_exp2f((high - dec->high[at]) + (low - dec->low[at])) * run.kv_scale;
                    a[r] = at <= t ? a[r] * weight : 0.f;
                }
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    const int at = 32 * sb + 8 * (r / 4) + 4 * half + r % 4;
                    y = __builtin_amdgcn_mfma_f32_32x32x2f32(vs[at * VB + state_col], a[r], y, 0, 0, 0);
                }
            }
            const int64_t row = AttendRowOf(span, run.back, r0 + t);
            float dot = 0;
            if (t < here) {
#pragma unroll
                for (int g = 0; g < 4; ++g) {
                    const int j = 32 * dw + 8 * g + 4 * half;
                    AttendPiece<float, 4> v;
#pragma unroll
                    for (int e = 0; e < 4; ++e) v.v[e] = y[4 * g + e] * run.out_scale;
                    if (dots != nullptr) {
                        const AttendPiece<T, 4> with = AttendLoad<T, 4>(dp + row * run.dot.row, j, cols);
#pragma unroll
                        for (int e = 0; e < 4; ++e) dot += j + e < cols ? v.v[e] * static_cast<float>(with.v[e]) : 0.f;
                    }
                    const int64_t to = y0 + row * run.y.row + j;
                    if (j + 4 <= cols) {
                        if (run.wide) {
                            *reinterpret_cast<AttendPiece<float, 4>*>(static_cast<float*>(run.y.data) + to) = v;
                        } else {
                            AttendPiece<T, 4> o;
#pragma unroll
                            for (int e = 0; e < 4; ++e) o.v[e] = static_cast<T>(v.v[e]);
                            *reinterpret_cast<AttendPiece<T, 4>*>(static_cast<T*>(run.y.data) + to) = o;
                        }
                    } else {
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            if (j + e >= cols) continue;
                            if (run.wide) static_cast<float*>(run.y.data)[to + e] = v.v[e];
                            else static_cast<T*>(run.y.data)[to + e] = static_cast<T>(v.v[e]);
                        }
                    }
                }
            }
            if (dots != nullptr) {  // the two halves of the columns meet in LDS
                dot += __shfl_xor(dot, 32);
                if (half == 0 && dw == 1) red[t] = dot;
            }
            __syncthreads();  // the copy of the state has been read
            if (dots != nullptr && half == 0 && dw == 0 && t < here) dots[row] = dot + red[t];
        }
        const float all = dec->all;
#pragma unroll
        for (int n = 0; n < NS; ++n) {
#pragma unroll
            for (int r = 0; r < 16; ++r) s[n][r] *= all;
        }
#pragma unroll 4
        for (int m = 0; m < C / 2; ++m) {
            const int at = 2 * m + half;
            const float v = vs[at * VB + state_col] * dec->end[at];
#pragma unroll
            for (int n = 0; n < NS; ++n) s[n] = __builtin_amdgcn_mfma_f32_32x32x2f32(ks[at * KP + KD / 2 * tw + 32 * n + l32], v, s[n], 0, 0, 0);
        }
        if (OUT) keep_state();
    }

    if constexpr (!OUT) {
        float* const to = run.last.data + bh * run.last.head + segment * run.last.segment;
#pragma unroll
        for (int n = 0; n < NS; ++n) {
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const int i = state_row(n, r);
                if (i < run.keys && state_col < cols) to[i * run.last.i + (col0 + state_col) * run.last.j] = s[n][r];
            }
        }
        if (tid == 0 && block == run.first) run.decays[static_cast<int64_t>(bh) * p.segments + segment] = __builtin_amdgcn_exp2f(static_cast<float>(passed));
        return;
    }
    // rows behind the sequence's end
    for (int64_t row = (span.end > span.first ? span.end : span.first) + wave; row < span.whole; row += 4) {
        if (lane >= cols) continue;
        const int64_t to = y0 + row * run.y.row + lane;
        if (run.wide) static_cast<float*>(run.y.data)[to] = 0.f;
        else static_cast<T*>(run.y.data)[to] = static_cast<T>(0);
    }
    if (run.ends != nullptr) {
        // <state behind the segment, its gradient there>; one wave after another adds its part up in the same order always
        float dot = 0;
        if (run.other.data != nullptr) {
#pragma unroll
            for (int n = 0; n < NS; ++n) {
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    const int i = state_row(n, r);
                    if (i < run.keys && state_col < cols)
                        dot += s[n][r] * run.other.data[bh * run.other.head + segment * run.other.segment + i * run.other.i + (col0 + state_col) * run.other.j];
                }
            }
        }
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) dot += __shfl_xor(dot, o);
        __syncthreads();
        if (lane == 0) red[wave] = dot;
        __syncthreads();
        if (tid == 0) {
            const float behind = span.end < length ? __builtin_amdgcn_exp2f(static_cast<float>(AttendDecay(p, b, h, span.end))) : 1.f;
            run.ends[(static_cast<int64_t>(bh) * p.segments + segment) * run.blocks + block - run.first] = (red[0] + red[1] + red[2] + red[3]) * behind;
        }
    }
    if (run.last.data != nullptr && segment_turn == p.segments - 1) {
        const float more = run.decay_last && length > 0 ? __builtin_amdgcn_exp2f(static_cast<float>(AttendDecay(p, b, h, 0))) : 1.f;
        float* const to = run.last.data + bh * run.last.head;
#pragma unroll
        for (int n = 0; n < NS; ++n) {
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const int i = state_row(n, r);
                if (i < run.keys && state_col < cols) to[i * run.last.i + (col0 + state_col) * run.last.j] = s[n][r] * more;
            }
        }
    }
}

__global__ __launch_bounds__(256) void AttendStartsKernel(AttendStates at, AttendStates initial, const float* decays, int keys, int values, int segments, int back) {
    const int bh = blockIdx.y, e = blockIdx.x * 256 + threadIdx.x;
    if (e >= keys * values) return;
    const int i = e / values, j = e % values;
    float* const to = at.data + bh * at.head + i * at.i + j * at.j;
    float now = initial.data != nullptr ? initial.data[bh * initial.head + i * initial.i + j * initial.j] : 0.f;
    for (int n = 0; n < segments; ++n) {
        const int segment = back ? segments - 1 - n : n;
        float* const here = to + segment * at.segment;
        const float more = n + 1 < segments ? *here : 0.f;
        *here = now;
        if (n + 1 < segments) now = __builtin_elementwise_fma(now, decays[static_cast<int64_t>(bh) * segments + segment], more);
    }
}

// Few rows, one after another: a workgroup has 64 columns of the state in its registers, four of them and every sixteenth row to a thread.  Bound by the state, read and written once.
template <typename T, int KD>
__global__ __launch_bounds__(256) void AttendTokensKernel(AttendArgs p) {
    constexpr int VB = kAttendColumns, N = KD / 16;
    __shared__ __align__(16) float red[16][VB];
    const AttendRun& run = p.run[0];
    int id = static_cast<int>(blockIdx.x);
    const int block = id % run.blocks, bh = id / run.blocks;
    const int64_t b = bh / p.heads;
    const int h = bh % p.heads;
    const int64_t length = LengthOf(p.lengths, b, p.length);
    const int col0 = block * VB, cols = min(VB, run.values - col0);
    const int tid = threadIdx.x, j = tid % 16 * 4, i0 = tid / 16;
    const T* const kp = static_cast<const T*>(run.k.data) + b * run.k.batch + (h / run.k.share) * run.k.head;
    const T* const vp = static_cast<const T*>(run.v.data) + b * run.v.batch + h * run.v.head + col0;
    const T* const qp = static_cast<const T*>(run.q.data) + b * run.q.batch + (h / run.q.share) * run.q.head;
    const float* const from = run.start.data != nullptr ? run.start.data + bh * run.start.head + col0 : nullptr;
    attend4_t s[N];
#pragma unroll
    for (int n = 0; n < N; ++n) {
        const int i = i0 + 16 * n;
        s[n] = attend4_t{0, 0, 0, 0};
        if (from != nullptr && i < run.keys) {
            const AttendPiece<float, 4> piece = AttendLoad<float, 4>(from + i * run.start.i, j, cols);
#pragma unroll
            for (int e = 0; e < 4; ++e) s[n][e] = piece.v[e];
        }
    }
    for (int64_t t = 0; t < p.length; ++t) {
        T* const to = static_cast<T*>(run.y.data) + b * run.y.batch + t * run.y.row + h * run.y.head + col0;
        if (t >= length) {
            if (tid < cols) to[tid] = static_cast<T>(0);
            continue;
        }
        const float step = __builtin_amdgcn_exp2f(static_cast<float>(AttendDecay(p, b, h, t)));
        const AttendPiece<T, 4> vv = AttendLoad<T, 4>(vp + t * run.v.row, j, cols);
        attend4_t v, y{0, 0, 0, 0};
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = static_cast<float>(vv.v[e]);
#pragma unroll
        for (int n = 0; n < N; ++n) {
            const int i = i0 + 16 * n;
            const float k = i < run.keys ? static_cast<float>(kp[t * run.k.row + i]) : 0.f, q = i < run.keys ? static_cast<float>(qp[t * run.q.row + i]) : 0.f;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                s[n][e] = __builtin_elementwise_fma(k, v[e], s[n][e] * step);
                if (i < run.keys) y[e] = __builtin_elementwise_fma(q, s[n][e], y[e]);
            }
        }
        __syncthreads();  // the last row's sums have been read
        *reinterpret_cast<attend4_t*>(&red[i0][j]) = y;
        __syncthreads();
        if (tid < cols) {
            float sum = 0;
#pragma unroll
            for (int g = 0; g < 16; ++g) sum += red[g][tid];
            to[tid] = static_cast<T>(sum * run.out_scale);
        }
    }
    float* const last = run.last.data + bh * run.last.head + col0;
#pragma unroll
    for (int n = 0; n < N; ++n) {
        const int i = i0 + 16 * n;
        if (i >= run.keys) continue;
        AttendPiece<float, 4> piece;
#pragma unroll
        for (int e = 0; e < 4; ++e) piece.v[e] = s[n][e];
        if (j + 4 <= cols) {
            *reinterpret_cast<AttendPiece<float, 4>*>(last + i * run.last.i + j) = piece;
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                if (j + e < cols) last[i * run.last.i + j + e] = piece.v[e];
            }
        }
    }
}

template <int KD>
constexpr int AttendLds() {
    return (kAttendTile * (KD + 4) + kAttendTile * kAttendColumns + KD * kAttendColumns + 4 * kAttendColumns) * 4 + static_cast<int>(sizeof(AttendDecays)) + 16;
}

template <typename F>
void VisitKeys(int keys, F&& f) {
    if (keys <= 64) f(std::integral_constant<int, 64>{});
    else if (keys <= 128) f(std::integral_constant<int, 128>{});
    else f(std::integral_constant<int, 256>{});
}

template <typename F>
void VisitAttendType(int dtype, F&& f) {
    if (dtype == HIPCX_FLOAT16) f(Tag<half_t>{});
    else f(Tag<float>{});
}

}  // namespace

void LaunchAttend(const AttendArgs& args, int dtype, bool states_alone, hipStream_t stream) {
    AttendArgs p = args;
    int keys = 0;
    for (int i = 0; i < p.runs; ++i) keys = std::max(keys, p.run[i].keys);
    const int64_t turns = states_alone ? p.segments - 1 : p.segments, groups = p.batch * p.heads * turns, blocks = (groups + 7) / 8 * 8 * p.blocks;
    HIPCX_REQUIRE(blocks <= kBlocksPerLaunch, HIPCX_NOT_IMPLEMENTED_ERROR, "linear_attention: too many elements");
    if (blocks == 0) return;
    p.groups = static_cast<int>(groups);
    if (dtype == HIPCX_FLOAT16) return LaunchAttendHalf(p, keys, blocks, states_alone, stream);
    VisitKeys(keys, [&](auto kd) {
        constexpr int KD = decltype(kd)::value, kLds = AttendLds<KD>();
        const dim3 grid(static_cast<unsigned>(blocks));
        if (states_alone) {
            EnsureDynamicLds<AttendTag>(reinterpret_cast<const void*>(AttendKernel<KD, false>), kLds);
            hipLaunchKernelGGL((AttendKernel<KD, false>), grid, dim3(256), kLds, stream, p);
        } else {
            EnsureDynamicLds<AttendTag>(reinterpret_cast<const void*>(AttendKernel<KD, true>), kLds);
            hipLaunchKernelGGL((AttendKernel<KD, true>), grid, dim3(256), kLds, stream, p);
        }
        CheckLaunch("linear_attention");
    });
}

void LaunchAttendStarts(const AttendArgs& p, int which, const AttendStates& initial, hipStream_t stream) {
    const AttendRun& run = p.run[which];
    for (int64_t first = 0; first < p.batch * p.heads; first += 65535) {  // (a grid's second axis)
        AttendStates at = run.last, from = initial;
        at.data += first * at.head;
        if (from.data != nullptr) from.data += first * from.head;
        const dim3 grid(static_cast<unsigned>(DivUp(run.keys * run.values, 256)), static_cast<unsigned>(std::min<int64_t>(65535, p.batch * p.heads - first)));
        hipLaunchKernelGGL(AttendStartsKernel, grid, dim3(256), 0, stream, at, from, run.decays + first * p.segments, run.keys, run.values, p.segments, run.back);
        CheckLaunch("linear_attention");
    }
}

namespace {

constexpr int64_t kMaxAttendRow = int64_t{1} << 24;  // elements from one row to the next: a tile's offsets have 32 bits

// Rows [batch, time, heads, elements]; a stride along an axis of one says nothing.
AttendRows AttendRowsOf(const hipcx_array* a, int heads, const std::string& what) {
    const int64_t it = ItemSize(a->dtype);
    HIPCX_REQUIRE(TotalSize(a) == 0 || a->shape[3] == 1 || a->strides[3] == it, HIPCX_DIMENSION_ERROR, what + ": the last axis must be dense");
    for (int i = 0; i < 3; ++i) HIPCX_REQUIRE(a->strides[i] % it == 0 || a->shape[i] <= 1, HIPCX_DIMENSION_ERROR, what + ": strides must be whole elements");
    const auto stride = [&](int i) { return a->shape[i] > 1 ? a->strides[i] / it : 0; };
    HIPCX_REQUIRE(std::abs(stride(1)) < kMaxAttendRow, HIPCX_NOT_IMPLEMENTED_ERROR, what + ": rows 2^24 elements apart or more");
    return {a->data, stride(0), stride(1), stride(2), heads / static_cast<int>(std::max<int64_t>(1, a->shape[2]))};
}

}  // namespace

bool AttendSizesOf(const hipcx_array* q, const hipcx_array* v, AttendCall* c) {
    if (q == nullptr || v == nullptr || q->ndim != 4 || v->ndim != 4 || q->shape[0] != v->shape[0] || q->shape[1] != v->shape[1]) return false;
    const int64_t kh = q->shape[2], h = v->shape[2];
    if (q->shape[0] < 0 || q->shape[1] < 0 || q->shape[1] >= (int64_t{1} << 30) || kh < 1 || h < 1 || h >= (1 << 20) || h % kh != 0) return false;
    if (q->shape[3] < 1 || q->shape[3] > kMaxAttend || v->shape[3] < 1 || v->shape[3] > kMaxAttend || q->shape[0] > kBlocksPerLaunch / h) return false;
    c->p.batch = q->shape[0], c->p.length = q->shape[1], c->p.heads = static_cast<int>(h);
    c->keys = static_cast<int>(q->shape[3]), c->values = static_cast<int>(v->shape[3]), c->key_heads = static_cast<int>(kh);
    return true;
}

AttendCall DescribeAttend(const std::string& what, const hipcx_array* q, const hipcx_array* k, const hipcx_array* v, const hipcx_array* log_decay, double scale,
                          const hipcx_array* state, const hipcx_array* lengths) {
    ValidateArray(q, "q");
    ValidateArray(k, "k");
    ValidateArray(v, "v");
    HIPCX_REQUIRE(q->dtype == HIPCX_FLOAT16 || q->dtype == HIPCX_FLOAT32, HIPCX_DTYPE_ERROR, what + ": float16 and float32 only, got " + DtypeName(q->dtype));
    HIPCX_REQUIRE(q->ndim == 4 && v->ndim == 4, HIPCX_DIMENSION_ERROR, what + ": q, k and v must be [batch, time, heads, elements], got " + ShapeStr(q) + " and " + ShapeStr(v));
    AttendCall c;
    RequireShape(k, {q->shape[0], q->shape[1], q->shape[2], q->shape[3]}, q->dtype, what + ": k");
    RequireShape(v, {q->shape[0], q->shape[1], v->shape[2], v->shape[3]}, q->dtype, what + ": v");
    HIPCX_REQUIRE(q->shape[2] >= 1 && v->shape[2] >= 1 && v->shape[2] % q->shape[2] == 0, HIPCX_DIMENSION_ERROR, what + ": the heads of q and k must divide those of v");
    HIPCX_REQUIRE(q->shape[3] >= 1 && q->shape[3] <= kMaxAttend && v->shape[3] >= 1 && v->shape[3] <= kMaxAttend, HIPCX_NOT_IMPLEMENTED_ERROR,
                  what + ": heads of 1 to 256 elements, got " + std::to_string(q->shape[3]) + " and " + std::to_string(v->shape[3]));
    HIPCX_REQUIRE(q->shape[1] < (int64_t{1} << 30), HIPCX_NOT_IMPLEMENTED_ERROR, what + ": 2^30 rows or more");
    HIPCX_REQUIRE(AttendSizesOf(q, v, &c), HIPCX_NOT_IMPLEMENTED_ERROR, what + ": too many heads");
    HIPCX_REQUIRE(std::isfinite(static_cast<float>(scale)), HIPCX_CHAINERX_ERROR, what + ": the scale must be finite in float32");
    const int64_t batch = c.p.batch, length = c.p.length, heads = c.p.heads;
    if (log_decay != nullptr) {
        ValidateArray(log_decay, "log_decay");
        if (log_decay->ndim == 1) RequireShape(log_decay, {heads}, HIPCX_FLOAT32, what + ": log_decay");
        else RequireShape(log_decay, {batch, length, heads}, HIPCX_FLOAT32, what + ": log_decay");
        for (int i = 0; i < log_decay->ndim; ++i) HIPCX_REQUIRE(log_decay->strides[i] % 4 == 0 || log_decay->shape[i] <= 1, HIPCX_DIMENSION_ERROR, what + ": strides must be whole elements");
        const auto stride = [&](int i) { return log_decay->shape[i] > 1 ? log_decay->strides[i] / 4 : 0; };
        c.p.decay = static_cast<const float*>(log_decay->data);
        c.p.decay_head = stride(log_decay->ndim - 1);
        if (log_decay->ndim == 3) c.p.decay_batch = stride(0), c.p.decay_row = stride(1);
    }
    RequireShape(state, {batch, heads, c.keys, c.values}, HIPCX_FLOAT32, what + ": state");
    RequireDense(state, what + ": state");
    c.state = state != nullptr ? static_cast<const float*>(state->data) : nullptr;
    c.q = AttendRowsOf(q, c.p.heads, what + ": q"), c.k = AttendRowsOf(k, c.p.heads, what + ": k"), c.v = AttendRowsOf(v, c.p.heads, what + ": v");
    c.p.lengths = LengthsOf(lengths, batch, what);
    return c;
}

AttendRows DescribeAttendRows(const hipcx_array* a, const AttendCall& c, int64_t heads, int64_t width, int dtype, const std::string& what) {
    ValidateArray(a, what.c_str());
    RequireShape(a, {c.p.batch, c.p.length, heads, width}, dtype, what);
    return AttendRowsOf(a, c.p.heads, what);
}

namespace {

// Up to so many rows go one after another.
constexpr int kAttendTokens = 8;

void CutForward(AttendCall* c) {
    if (c->p.length <= kAttendTokens) c->p.segments = 1, c->p.segment_rows = kAttendTile;
    else CutAttend(&c->p, AttendBlocks(c->values));
}

size_t ForwardWorkspace(const AttendCall& c) {
    if (c.p.segments < 2) return 0;
    return static_cast<size_t>(c.p.batch * c.p.heads * c.p.segments * (static_cast<int64_t>(c.keys) * c.values + 1) * 4);
}

}  // namespace
}  // namespace hipcx

using namespace hipcx;

extern "C" {

size_t hipcx_linear_attention_workspace_size(const hipcx_array* q, const hipcx_array* v) {
    AttendCall c;
    if (!AttendSizesOf(q, v, &c)) return 0;
    CutForward(&c);
    return ForwardWorkspace(c);
}

int hipcx_linear_attention(const hipcx_array* q, const hipcx_array* k, const hipcx_array* v, const hipcx_array* log_decay, double scale, const hipcx_array* state,
                           const hipcx_array* lengths, const hipcx_array* y, const hipcx_array* new_state, void* workspace, size_t workspace_bytes, void* stream) {
    return Guard([&] {
        const std::string what = "linear_attention";
        AttendCall c = DescribeAttend(what, q, k, v, log_decay, scale, state, lengths);
        HIPCX_REQUIRE(y != nullptr && new_state != nullptr, HIPCX_CHAINERX_ERROR, what + ": y and new_state are needed");
        AttendArgs& p = c.p;
        const AttendRows to = DescribeAttendRows(y, c, p.heads, c.values, q->dtype, what + ": y");
        RequireShape(new_state, {p.batch, p.heads, c.keys, c.values}, HIPCX_FLOAT32, what + ": new_state");
        RequireDense(new_state, what + ": new_state");
        if (p.batch == 0) return;
        CutForward(&c);
        HIPCX_REQUIRE(workspace_bytes >= ForwardWorkspace(c) && (ForwardWorkspace(c) == 0 || workspace != nullptr), HIPCX_CHAINERX_ERROR, what + ": the workspace is too small");
        AttendRun& run = p.run[0];
        run.q = c.q, run.k = c.k, run.v = c.v, run.y = to;
        run.kv_scale = 1, run.out_scale = static_cast<float>(scale);
        run.keys = c.keys, run.values = c.values, run.blocks = AttendBlocks(c.values);
        p.runs = 1, p.blocks = run.blocks;
        const AttendStates given = AttendStatesOf(c.state, c.keys, c.values, false), last = AttendStatesOf(static_cast<const float*>(new_state->data), c.keys, c.values, false);
        run.start = given, run.last = last;
        if (p.length <= kAttendTokens) {
            VisitAttendType(q->dtype, [&](auto tag) {
                using T = typename decltype(tag)::type;
                VisitKeys(c.keys, [&](auto kd) {
                    const int64_t blocks = p.blocks * p.batch * p.heads;
                    HIPCX_REQUIRE(blocks <= kBlocksPerLaunch, HIPCX_NOT_IMPLEMENTED_ERROR, what + ": too many elements");
                    hipLaunchKernelGGL((AttendTokensKernel<T, decltype(kd)::value>), dim3(static_cast<unsigned>(blocks)), dim3(256), 0, AsStream(stream), p);
                    CheckLaunch("linear_attention");
                });
            });
            return;
        }
        if (p.segments > 1) {
            const AttendStates starts = AttendSegments(static_cast<float*>(workspace), p, c.keys, c.values);
            run.last = starts, run.decays = starts.data + p.batch * p.heads * starts.head;
            LaunchAttend(p, q->dtype, true, AsStream(stream));
            LaunchAttendStarts(p, 0, given, AsStream(stream));
            run.start = starts, run.last = last;
        }
        LaunchAttend(p, q->dtype, false, AsStream(stream));
    });
}

}  // extern "C"
