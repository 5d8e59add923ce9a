// Linear attention: chunks of rows as matrix products, single rows as they come.
#include <cstdlib>

#include "igemm.h"
#include "linear_attention.h"

namespace hipcx {
namespace {

// Tiles of 64 rows, one after another.  With G the decays summed up from the tile's first row and S the state before it,
//   P[t][s] = exp(G[t] - G[s]) q[t] k[s] for s <= t,  y = P v + exp(G) q S,  S <- exp(G[63]) S + (exp(G[63] - G) k)^T v.
// A workgroup of four waves has 64 columns of v: a wave has sixteen rows of y, and sixteen columns of S in its accumulators (a copy is in LDS, turned, for the products with q).
// P stays in registers: as k q^T its column t is a lane, whose rows s are the reduction of the product v^T P.
// Products run on the float pipe (v_mfma_f32_16x16x4_f32), with the reduction's elements in an order that gives a lane four neighbours.  Bound by a tile's chain: at 64 keys and values the wave of the
// last rows multiplies for 8.2 thousand cycles of a tile's 16, and two workgroups share a compute unit.  20 padded prompts of up to 777 rows, 13 heads of 50 x 50: 61 us, the states of their three
// segments before it 30; rows of 32 to a wave, and loads that waited for one another, took 222 in one segment.  At 128 keys and values 24 x 478 rows of 11 heads with gradients run at 72 TFLOP/s.
// GRAD: what the passes of the gradients have beyond the forward one.
template <int KD, bool OUT>
struct AttendLds {
    static_assert(kAttendTile == kAttendColumns, "the rows of k and the columns of the state share a place");
    static constexpr int kPitch = KD + 4, kValuePitch = kAttendColumns + 4;  // floats; four rows on is sixteen banks on
    // At 128 keys the copy of the state and the rows of k, as many, take turns in one place, so that two workgroups fit into a compute unit: for two more barriers a tile, 24 x 478 rows of 11 heads
    // with gradients 898 -> 723 us.  64 keys fit twice as they are; with turns three times, which is no quicker for the barriers
    // (20 padded prompts of 777 rows: 94 us, with turns 109); 256 fit once.
    static constexpr bool kTurns = KD == 128;
    static constexpr int kValues = kAttendTile * kPitch, kStates = kTurns ? 0 : kValues + kAttendTile * kValuePitch;
    static constexpr int kSums = (kTurns ? kValues + kAttendTile * kValuePitch : kStates + (OUT ? kAttendColumns * kPitch : 0));
    static constexpr int kDecays = kSums + 4 * kAttendColumns;
    static constexpr int kBytes = kDecays * 4 + 2 * static_cast<int>(sizeof(AttendDecays)) + 16;
    static_assert(AttendResident(false, KD) * kBytes <= kLdsOfUnit, "as many workgroups as the time axis is cut for");
};

__device__ __forceinline__ attend4_t Mfma4(float a, float b, attend4_t c) { return __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, c, 0, 0, 0); }

template <int KD, bool OUT, int WIDTHS, bool GRAD>
__global__ __launch_bounds__(256, AttendResident(false, KD)) void AttendKernel(AttendArgs p) {
    using Lds = AttendLds<KD, OUT>;
    constexpr int VB = kAttendColumns, C = kAttendTile, NS = KD / 16, KP = Lds::kPitch, VP = Lds::kValuePitch, DB = VB / 16;
    extern __shared__ __align__(16) float lds[];
    float *const ks = lds, *const vs = lds + Lds::kValues, *const ss = lds + Lds::kStates, *const sums = lds + Lds::kSums;  // rows, rows, columns of the state
    AttendDecays* const decays = reinterpret_cast<AttendDecays*>(lds + Lds::kDecays);
    int* const odd = reinterpret_cast<int*>(decays + 2);  // v has infinities or what is not a number

    int id = AttendNumber(p);
    if (id < 0) return;
    const int block = id % p.blocks;
    id /= p.blocks;
    const int bh = id % static_cast<int>(p.batch * p.heads);
    const int segment_turn = id / static_cast<int>(p.batch * p.heads);
    int which = 0;
    if (GRAD) {
        while (which + 1 < p.runs && block >= p.run[which + 1].first) ++which;
    }
    const AttendRun& run = p.run[GRAD ? which : 0];
    const bool back = GRAD && run.back != 0, with_dots = GRAD && OUT && run.dots != nullptr;
    const float kv_scale = GRAD ? run.kv_scale : 1.f;
    const int segment = back ? p.segments - 1 - segment_turn : segment_turn;
    const int64_t b = bh / p.heads;
    const int h = bh % p.heads;
    const int64_t length = LengthOf(p.lengths, b, p.length);
    const AttendSpan span(p, length, segment);
    const int64_t rows = span.end - span.first;
    int keys = run.keys;
    const int col0 = (block - run.first) * VB, cols = min(VB, run.values - col0);
    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid / 64);
    int lane = tid % 64;
    float* const dots = with_dots ? run.dots + (static_cast<int64_t>(bh) * run.blocks + block - run.first) * p.length : nullptr;

    const auto state_row = [&](int n, int r) { return 16 * n + lane / 16 * 4 + r; };
    const auto state_col = [&] { return 16 * wave + lane % 16; };
    attend4_t s[NS]{};
    // Elements that are not there are read as the last ones, so that all loads go out at once; the compiler would have each wait for its condition.
    const auto states_at = [&](const AttendStates& of, attend4_t (&to)[NS]) {
        const float* const from = of.data + bh * of.head + segment * of.segment + (col0 + min(state_col(), cols - 1)) * of.j;
        if (of.i == 1 && keys % 4 == 0) {  // (a transpose: a lane's four are neighbours)
#pragma unroll
            for (int n = 0; n < NS; ++n) {
                const AttendPiece<float, 4> four = *reinterpret_cast<const AttendPiece<float, 4>*>(from + min(state_row(n, 0), keys - 4));
                to[n] = __builtin_bit_cast(attend4_t, four);
            }
        } else {
#pragma unroll
            for (int n = 0; n < NS; ++n) {
#pragma unroll
                for (int r = 0; r < 4; ++r) to[n][r] = from[min(state_row(n, r), keys - 1) * of.i];
            }
        }
#pragma unroll
        for (int n = 0; n < NS; ++n) {
            asm volatile("" : "+v"(to[n]));
#pragma unroll
            for (int r = 0; r < 4; ++r) to[n][r] = state_row(n, r) < keys && state_col() < cols ? to[n][r] : 0.f;
        }
    };
    const auto keep_state = [&] {
#pragma unroll
        for (int n = 0; n < NS; ++n) *reinterpret_cast<attend4_t*>(ss + state_col() * KP + state_row(n, 0)) = s[n];
    };

    // A tile's rows on their way: pieces of four elements.  Rows that are not there are the last one again (their weights are zeros; behind the last tile every row is, since a branch round the loads
    // would have those of the tile before, too, waited for where the two ways meet); elements that are not there become zeros.  Rows lie less than 2^24 elements apart, so that a tile's are within
    // 32 bits of its first.
    constexpr int KR = 1024 / KD, NK = C / KR, NV = C / 16;  // rows of k that are read at once, and times
    const int key_row = tid / (KD / 4), key_col = tid % (KD / 4) * 4, value_row = tid / 16, value_col = tid % 16 * 4;
    const auto own_row = [&] { return 16 * wave + lane % 16; };  // of a tile
    const int way = back ? -1 : 1;
    const int64_t row0 = back ? span.end - 1 : span.first;
    const float* kp = static_cast<const float*>(run.k.data) + b * run.k.batch + (h / run.k.share) * run.k.head + row0 * run.k.row;
    const float* vp = static_cast<const float*>(run.v.data) + b * run.v.batch + (h / run.v.share) * run.v.head + row0 * run.v.row + col0;
    const float* qp = OUT ? static_cast<const float*>(run.q.data) + b * run.q.batch + (h / run.q.share) * run.q.head + row0 * run.q.row : nullptr;
    const int k_row = way * static_cast<int>(run.k.row), v_row = way * static_cast<int>(run.v.row), q_row = OUT ? way * static_cast<int>(run.q.row) : 0;
    float* yp = OUT ? static_cast<float*>(run.y.data) + b * run.y.batch + h * run.y.head + row0 * run.y.row + col0 : nullptr;
    const int y_row = OUT ? way * static_cast<int>(run.y.row) : 0;
    const float* dp = with_dots ? static_cast<const float*>(run.dot.data) + b * run.dot.batch + (h / run.dot.share) * run.dot.head + row0 * run.dot.row + col0 : nullptr;
    const int d_row = with_dots ? way * static_cast<int>(run.dot.row) : 0;
    const float* gp = p.decay != nullptr ? p.decay + b * p.decay_batch + h * p.decay_head : nullptr;
    const int64_t g_rows = AttendNoDecay(span.end, length, back);
    AttendPiece<float, 4> k_next[NK], v_next[NV], q_next[OUT ? NS : 1];
    const auto placed = [&](const AttendPiece<float, 4>& piece, int col, int end) {
        const AttendPiece<float, 4> there = AttendPlace<WIDTHS>(piece, col, end);
        return attend4_t{there.v[0], there.v[1], there.v[2], there.v[3]};
    };
    const auto load = [&](int64_t r0) {  // k and v; at the tile's first row
        const int last = static_cast<int>(rows - r0 < C ? rows - r0 : C) - 1;
#pragma unroll
        for (int n = 0; n < NK; ++n) k_next[n] = AttendFetch<WIDTHS, 4>(kp + min(key_row + n * KR, last) * k_row, key_col, keys);
#pragma unroll
        for (int n = 0; n < NV; ++n) v_next[n] = AttendFetch<WIDTHS, 4>(vp + min(value_row + n * 16, last) * v_row, value_col, cols);
        kp += static_cast<int64_t>(k_row) * C, vp += static_cast<int64_t>(v_row) * C;
    };
    const auto load_q = [&](int64_t r0) {
        if constexpr (OUT) {
            const float* const at = qp + min(own_row(), static_cast<int>(rows - r0 < C ? rows - r0 : C) - 1) * q_row;
#pragma unroll
            for (int m = 0; m < NS; ++m) q_next[m] = AttendFetch<WIDTHS, 4>(at, 16 * m + lane / 16 * 4, keys);
            qp += static_cast<int64_t>(q_row) * C;
        }
    };
    // Log decays, by one wave, a lane to a row: summed up a tile ahead, on their way two tiles ahead, so that nothing waits for what was asked for in the same tile.
    float g_now = 0, g_next = 0;
    const auto decay_at = [&](int64_t r) { return gp[AttendDecayRow(span.first, span.end, length, back, r) * p.decay_row]; };
    const auto load_decays = [&](int64_t r0) {  // of a row that is there; sum_decays takes those that count
        if (gp != nullptr) g_next = decay_at(r0 + lane);
    };
    const auto sum_decays = [&](int64_t r0, AttendDecays* to) {
        const int here = static_cast<int>(rows - r0 < C ? rows - r0 : C);
        SumDecays(to, gp != nullptr && lane < here && r0 + lane >= g_rows ? LogOfDecay(g_now) : 0, here, kv_scale);
    };
    if (tid == 0) odd[0] = odd[1] = 0;
    if (rows > 0) {
        if (wave == 0) {
            load_decays(0);
            g_now = g_next;
            load_decays(C);
        }
        load(0);
        load_q(0);
        if (wave == 0) sum_decays(0, decays);
    }
    if (OUT) {
        if (run.start.data != nullptr) states_at(run.start, s);
        keep_state();
    }
    double passed = 0;  // log decay of the tiles so far
    int turn = 0;
    int64_t r0 = 0;
    __syncthreads();  // the flags
    for (; r0 < rows; r0 += C, turn ^= 1) {
        asm volatile("" : "+v"(lane));  // (what follows from these is found again in every tile, and takes no registers over the loop)
        asm volatile("" : "+s"(keys));
        const int quarter = lane / 16;
        const AttendDecays* const dec = decays + turn;
        const int here = static_cast<int>(rows - r0 < C ? rows - r0 : C);
        const bool live = OUT && 16 * wave < here;  // this wave has rows
        const bool more = r0 + C < rows;
        // (the last tile's rows of v have been read by all)
        float finite = 0;  // or not a number
#pragma unroll
        for (int n = 0; n < NV; ++n) {
            const attend4_t v = placed(v_next[n], value_col, cols);
            *reinterpret_cast<attend4_t*>(vs + (value_row + n * 16) * VP + value_col) = v;
#pragma unroll
            for (int e = 0; e < 4; ++e) finite = __builtin_fmaf(v[e], 0.f, finite);
        }
        if (OUT && !(finite == 0)) odd[turn] = 1;
        const auto place_k = [&] {
#pragma unroll
            for (int n = 0; n < NK; ++n) *reinterpret_cast<attend4_t*>(ks + (key_row + n * KR) * KP + key_col) = placed(k_next[n], key_col, keys);
            __syncthreads();
        };
        constexpr bool kTurns = OUT && Lds::kTurns;
        if (!kTurns) place_k();
        attend4_t q[OUT ? NS : 1], y[DB]{};
        float high = 0, low = 0;
        if (live) {
            // this wave's sixteen rows by all columns, in blocks of 16 x 16
            high = dec->high[own_row()], low = dec->low[own_row()];
#pragma unroll
            for (int m = 0; m < NS; ++m) q[OUT ? m : 0] = placed(q_next[OUT ? m : 0], 16 * m + 4 * quarter, keys);
            const float* const at = ss + lane % 16 * KP + 4 * quarter;
            attend4_t part[2][DB];
            const auto read = [&](int m, attend4_t (&to)[DB]) {
#pragma unroll
                for (int d = 0; d < DB; ++d) to[d] = *reinterpret_cast<const attend4_t*>(at + 16 * d * KP + 16 * m);
            };
            read(0, part[0]);
#pragma unroll
            for (int m = 0; m < NS; ++m) {  // reads of the next step under the products of this one; nothing for sixteen keys that are not there
                if (16 * m >= keys) break;
                if (m + 1 < NS) read(m + 1, part[m % 2 ^ 1]);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
#pragma unroll
                    for (int d = 0; d < DB; ++d) y[d] = Mfma4(part[m % 2][d][e], q[OUT ? m : 0][e], y[d]);
                }
                __builtin_amdgcn_sched_barrier(0);
            }
            const float from_start = __builtin_amdgcn_exp2f(high + low);
#pragma unroll
            for (int d = 0; d < DB; ++d) y[d] *= from_start;
        }
        if (kTurns) {
            __syncthreads();  // the copy of the state has been read
            place_k();
        }
        passed += dec->sum;
        // An infinity of a later row, times P's zeros, would reach earlier ones: the rest goes row by row.
        if (OUT && odd[turn] != 0) break;
        g_now = g_next;
        load(r0 + C);
        if (wave == 0) load_decays(r0 + 2 * C);  // (behind the others: what waits for them must not wait for this one)
        if (live) {
            attend4_t a[4]{};
            {
                const float* const at = ks + lane % 16 * KP + 4 * quarter;
                attend4_t part[2][4];
                const auto read = [&](int m, attend4_t (&to)[4]) {
#pragma unroll
                    for (int sb = 0; sb < 4; ++sb) to[sb] = *reinterpret_cast<const attend4_t*>(at + 16 * min(sb, wave) * KP + 16 * m);
                };
                read(0, part[0]);
#pragma unroll
                for (int m = 0; m < NS; ++m) {
                    if (16 * m >= keys) break;
                    if (m + 1 < NS) read(m + 1, part[m % 2 ^ 1]);
#pragma unroll
                    for (int sb = 0; sb < 4; ++sb) {
                        if (sb > wave) continue;
#pragma unroll
                        for (int e = 0; e < 4; ++e) a[sb] = Mfma4(part[m % 2][sb][e], q[m][e], a[sb]);
                    }
                    __builtin_amdgcn_sched_barrier(0);
                }
            }
            load_q(r0 + C);
#pragma unroll
            for (int sb = 0; sb < 4; ++sb) {
                if (sb > wave) continue;
                const int first = 16 * sb + 4 * quarter;
                const attend4_t highs = *reinterpret_cast<const attend4_t*>(dec->high + first), lows = *reinterpret_cast<const attend4_t*>(dec->low + first);
                float v[DB][4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
#pragma unroll
                    for (int d = 0; d < DB; ++d) v[d][e] = vs[(first + e) * VP + 16 * d + lane % 16];
                }
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float weighted = a[sb][e] * (__builtin_amdgcn_exp2f((high - highs[e]) + (low - lows[e])) * kv_scale);
                    a[sb][e] = first + e <= own_row() ? weighted : 0.f;
                }
#pragma unroll
                for (int e = 0; e < 4; ++e) {
#pragma unroll
                    for (int d = 0; d < DB; ++d) y[d] = Mfma4(v[d][e], a[sb][e], y[d]);
                }
            }
            float* const to = yp + static_cast<int64_t>(own_row()) * y_row;
            const bool there = r0 + own_row() < rows;
            float dot = 0;
#pragma unroll
            for (int d = 0; d < DB; ++d) {
                const int j = 16 * d + 4 * quarter;
                AttendPiece<float, 4> out;
#pragma unroll
                for (int e = 0; e < 4; ++e) out.v[e] = y[d][e] * run.out_scale;
                if (!there) continue;
                if (with_dots) {
                    const float* const row = dp + static_cast<int64_t>(own_row()) * d_row;
                    const AttendPiece<float, 4> with = AttendPlace<WIDTHS>(AttendFetch<WIDTHS, 4>(row, j, cols), j, cols);
#pragma unroll
                    for (int e = 0; e < 4; ++e) dot += j + e < cols ? out.v[e] * with.v[e] : 0.f;
                }
                if (WIDTHS == kAttendWhole ? j < cols : j + 4 <= cols) {
                    *reinterpret_cast<AttendPiece<float, 4>*>(to + j) = out;
                } else if (WIDTHS != kAttendWhole) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        if (j + e < cols) to[j + e] = out.v[e];
                    }
                }
            }
            if (with_dots) {
                dot += __shfl_xor(dot, 16);
                dot += __shfl_xor(dot, 32);
                if (quarter == 0 && there) dots[row0 + way * (r0 + own_row())] = dot;
                dp += static_cast<int64_t>(d_row) * C;
            }
            yp += static_cast<int64_t>(y_row) * C;
        }
        if (wave == 0 && more) sum_decays(r0 + C, decays + (turn ^ 1));
        if (tid == 0) odd[turn ^ 1] = 0;
        __builtin_amdgcn_sched_barrier(0);
        {
            // this wave's columns of v times their rows' weights
            const float all = dec->all;
#pragma unroll
            for (int n = 0; n < NS; ++n) s[n] *= all;
            const float *const from = vs + 4 * quarter * VP + state_col(), *const at = ks + 4 * quarter * KP + lane % 16;
            constexpr int N = 4;  // accumulators between the reads
#pragma unroll
            for (int sb = 0; sb < 4; ++sb) {
                if (16 * sb >= here) break;
                const attend4_t end = *reinterpret_cast<const attend4_t*>(dec->end + 16 * sb + 4 * quarter);
                float v[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) v[e] = from[(16 * sb + e) * VP] * end[e];
#pragma unroll
                for (int n0 = 0; n0 < NS; n0 += N) {
                    if (16 * n0 >= keys) break;
                    float k[4][N];
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
#pragma unroll
                        for (int n = 0; n < N; ++n) k[e][n] = at[(16 * sb + e) * KP + 16 * (n0 + n)];
                    }
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
#pragma unroll
                        for (int n = 0; n < N; ++n) s[n0 + n] = Mfma4(k[e][n], v[e], s[n0 + n]);
                    }
                }
            }
        }
        __syncthreads();  // the rows of k and v have been read
        if (OUT) keep_state();
        if (kTurns) __syncthreads();
    }

    if (OUT && r0 < rows) {
        // row by row, on the copy
        __syncthreads();
        keep_state();
        __syncthreads();
        const int j = lane;
        for (; r0 < rows; ++r0) {
            const int64_t row = row0 + way * r0;
            const float* const k = static_cast<const float*>(run.k.data) + b * run.k.batch + (h / run.k.share) * run.k.head + row * run.k.row;
            const float* const x = static_cast<const float*>(run.q.data) + b * run.q.batch + (h / run.q.share) * run.q.head + row * run.q.row;
            const float* const of_v = static_cast<const float*>(run.v.data) + b * run.v.batch + (h / run.v.share) * run.v.head + row * run.v.row + col0;
            const float step = gp != nullptr && r0 >= g_rows ? __builtin_amdgcn_exp2f(static_cast<float>(LogOfDecay(decay_at(r0)))) : 1.f, v = j < cols ? of_v[j] * kv_scale : 0.f;
            float y = 0;
            for (int i = wave * (KD / 4); i < (wave + 1) * (KD / 4) && i < keys; ++i) {
                const float now = ss[j * KP + i] * step + k[i] * v;
                ss[j * KP + i] = now;
                y += x[i] * now;
            }
            sums[wave * VB + j] = y;
            __syncthreads();
            if (wave == 0) {
                y = (sums[j] + sums[VB + j] + sums[2 * VB + j] + sums[3 * VB + j]) * run.out_scale;
                if (j < cols) static_cast<float*>(run.y.data)[b * run.y.batch + h * run.y.head + row * run.y.row + col0 + j] = y;
                if (with_dots) {
                    float dot = 0;
                    if (j < cols) dot = y * (static_cast<const float*>(run.dot.data) + b * run.dot.batch + (h / run.dot.share) * run.dot.head + row * run.dot.row + col0)[j];
#pragma unroll
                    for (int o = 1; o < 64; o <<= 1) dot += __shfl_xor(dot, o);
                    if (lane == 0) dots[row] = dot;
                }
            }
            __syncthreads();
        }
#pragma unroll
        for (int n = 0; n < NS; ++n) s[n] = *reinterpret_cast<const attend4_t*>(ss + state_col() * KP + state_row(n, 0));
    }
    if constexpr (!OUT) {
        float* const to = run.last.data + bh * run.last.head + segment * run.last.segment;
#pragma unroll
        for (int n = 0; n < NS; ++n) {
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int i = state_row(n, r);
                if (i < keys && state_col() < cols) to[i * run.last.i + (col0 + state_col()) * run.last.j] = s[n][r];
            }
        }
        if (tid == 0 && block == run.first) run.decays[static_cast<int64_t>(bh) * p.segments + segment] = __builtin_amdgcn_exp2f(static_cast<float>(passed));
        return;
    }
    // rows behind the sequence's end
    for (int64_t row = (span.end > span.first ? span.end : span.first) + wave; row < span.whole; row += 4) {
        if (lane < cols) static_cast<float*>(run.y.data)[b * run.y.batch + h * run.y.head + row * run.y.row + col0 + lane] = 0.f;
    }
    if (GRAD && run.ends != nullptr) {
        // <state behind the segment, its gradient there>, the waves' parts added up in the same order always
        float dot = 0;
        if (run.other.data != nullptr) {
            attend4_t other[NS];
            states_at(run.other, other);
#pragma unroll
            for (int n = 0; n < NS; ++n) {
#pragma unroll
                for (int r = 0; r < 4; ++r) dot += state_row(n, r) < keys && state_col() < cols ? s[n][r] * other[n][r] : 0.f;
            }
        }
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) dot += __shfl_xor(dot, o);
        __syncthreads();
        if (lane == 0) sums[wave] = dot;
        __syncthreads();
        if (tid == 0) {
            const float behind = span.end < length ? __builtin_amdgcn_exp2f(static_cast<float>(AttendDecay(p, b, h, span.end))) : 1.f;
            run.ends[(static_cast<int64_t>(bh) * p.segments + segment) * run.blocks + block - run.first] = (sums[0] + sums[1] + sums[2] + sums[3]) * behind;
        }
    }
    if (run.last.data != nullptr && segment_turn == p.segments - 1) {
        const float more = GRAD && run.decay_last && length > 0 ? __builtin_amdgcn_exp2f(static_cast<float>(AttendDecay(p, b, h, 0))) : 1.f;
        float* const to = run.last.data + bh * run.last.head;
#pragma unroll
        for (int n = 0; n < NS; ++n) {
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int i = state_row(n, r);
                if (i < keys && state_col() < cols) to[i * run.last.i + (col0 + state_col()) * run.last.j] = s[n][r] * more;
            }
        }
    }
}

// An element of a state to a thread.  Bound by memory and its latency, once the segments' loads go out together.
__global__ __launch_bounds__(256) void AttendStartsKernel(AttendStates at, AttendStates initial, const float* decays, int keys, int values, int segments, int back) {
    const int bh = blockIdx.y, e = blockIdx.x * 256 + threadIdx.x;
    if (e >= keys * values) return;
    const int i = e / values, j = e % values;
    float* const to = at.data + bh * at.head + i * at.i + j * at.j;
    float now = initial.data != nullptr ? initial.data[bh * initial.head + i * initial.i + j * initial.j] : 0.f;
    const float* const decay = decays + static_cast<int64_t>(bh) * segments;
    constexpr int N = 8;  // segments whose loads go out together
    for (int n = 0; n < segments; n += N) {
        float more[N], keep[N];
#pragma unroll
        for (int k = 0; k < N; ++k) {  // (the last one's own share and decay have no place to go, and those behind it are it again)
            const int turn = min(n + k, segments - 2), segment = back ? segments - 1 - turn : turn;
            more[k] = to[segment * at.segment], keep[k] = decay[segment];
        }
#pragma unroll
        for (int k = 0; k < N; ++k) {
            if (n + k >= segments) continue;
            to[(back ? segments - 1 - n - k : n + k) * at.segment] = now;
            now = __builtin_elementwise_fma(now, keep[k], more[k]);
        }
    }
}

// Few rows, one after another: a workgroup has 64 columns of the state in its registers, four of them and every sixteenth row to a thread.  Bound by the state, read and written once: one row of 128
// sequences, 16 heads of 128 x 128 in float16, takes 44.6 us, 6.0 TB/s (with loads behind branches 58).  Up to eight rows it is quicker than a tile, which multiplies for sixteen at least.
// Rows of the state that are not there are read as the last one; their q and k are zeros.
template <typename T, int KD, int WIDTHS>
__global__ __launch_bounds__(256) void AttendTokensKernel(AttendArgs p) {
    constexpr int VB = kAttendColumns, N = KD / 16;
    __shared__ __align__(16) float red[16][VB];
    const AttendRun& run = p.run[0];
    int id = static_cast<int>(blockIdx.x);
    const int block = id % run.blocks, bh = id / run.blocks;
    const int64_t b = bh / p.heads;
    const int h = bh % p.heads;
    const int64_t length = LengthOf(p.lengths, b, p.length);
    const int col0 = block * VB, cols = min(VB, run.values - col0), keys = run.keys;
    const int tid = threadIdx.x, j = tid % 16 * 4, i0 = tid / 16;
    const T* const kp = static_cast<const T*>(run.k.data) + b * run.k.batch + (h / run.k.share) * run.k.head;
    const T* const vp = static_cast<const T*>(run.v.data) + b * run.v.batch + h * run.v.head + col0;
    const T* const qp = static_cast<const T*>(run.q.data) + b * run.q.batch + (h / run.q.share) * run.q.head;
    AttendPiece<float, 4> first[N];
    if (run.start.data != nullptr) {
        const float* const from = run.start.data + bh * run.start.head + col0;
#pragma unroll
        for (int n = 0; n < N; ++n) first[n] = AttendFetch<WIDTHS, 4>(from + min(i0 + 16 * n, keys - 1) * run.start.i, j, cols);
    }
    T k[N], q[N];
    AttendPiece<T, 4> v;
    float decay = 0;
    const auto load = [&](int64_t t) {  // a row that is there
        v = AttendFetch<WIDTHS, 4>(vp + t * run.v.row, j, cols);
#pragma unroll
        for (int n = 0; n < N; ++n) k[n] = kp[t * run.k.row + min(i0 + 16 * n, keys - 1)], q[n] = qp[t * run.q.row + min(i0 + 16 * n, keys - 1)];
        if (p.decay != nullptr) decay = p.decay[b * p.decay_batch + t * p.decay_row + h * p.decay_head];
    };
    if (length > 0) load(0);
    attend4_t s[N];
#pragma unroll
    for (int n = 0; n < N; ++n) {
        s[n] = attend4_t{0, 0, 0, 0};
        if (run.start.data == nullptr) continue;
        const AttendPiece<float, 4> piece = AttendPlace<WIDTHS>(first[n], j, cols);
#pragma unroll
        for (int e = 0; e < 4; ++e) s[n][e] = piece.v[e];
    }
    for (int64_t t = 0; t < p.length; ++t) {
        T* const to = static_cast<T*>(run.y.data) + b * run.y.batch + t * run.y.row + h * run.y.head + col0;
        if (t >= length) {
            if (tid < cols) to[tid] = static_cast<T>(0);
            continue;
        }
        const float step = __builtin_amdgcn_exp2f(static_cast<float>(LogOfDecay(decay)));
        const AttendPiece<T, 4> vv = AttendPlace<WIDTHS>(v, j, cols);
        attend4_t y{0, 0, 0, 0};
#pragma unroll
        for (int n = 0; n < N; ++n) {
            const bool there = i0 + 16 * n < keys;
            const float ki = there ? static_cast<float>(k[n]) : 0.f, qi = static_cast<float>(q[n]);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                s[n][e] = __builtin_elementwise_fma(ki, static_cast<float>(vv.v[e]), s[n][e] * step);
                y[e] = there ? __builtin_elementwise_fma(qi, s[n][e], y[e]) : y[e];
            }
        }
        if (t + 1 < length) load(t + 1);
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
        if (i >= keys) continue;
        AttendPiece<float, 4> piece;
#pragma unroll
        for (int e = 0; e < 4; ++e) piece.v[e] = s[n][e];
        if (j + 4 <= cols) {
            *reinterpret_cast<AttendPiece<float, 4>*>(last + i * run.last.i + j) = piece;
        } else if (WIDTHS != kAttendWhole) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                if (j + e < cols) last[i * run.last.i + j + e] = piece.v[e];
            }
        }
    }
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
    const AttendWidths widths = AttendWidthsOf(p, 4);
    VisitKeys(keys, [&](auto kd) {
        const auto kernel = [&](auto out, auto rows, auto grad) {
            constexpr int KD = decltype(kd)::value, kLds = AttendLds<KD, decltype(out)::value>::kBytes;
            void (*const k)(AttendArgs) = AttendKernel<KD, decltype(out)::value, decltype(rows)::value, decltype(grad)::value>;
            struct Tag {};  // a type of its own for every instantiation of this lambda
            EnsureDynamicLds<Tag>(reinterpret_cast<const void*>(k), kLds);
            hipLaunchKernelGGL(k, dim3(static_cast<unsigned>(blocks)), dim3(256), kLds, stream, p);
            CheckLaunch("linear_attention");
        };
        VisitWidths(widths, p.runs > 1, [&](auto rows, auto grad) { states_alone ? kernel(std::false_type{}, rows, grad) : kernel(std::true_type{}, rows, grad); });
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
    if (q == nullptr || v == nullptr || (q->dtype != HIPCX_FLOAT16 && q->dtype != HIPCX_FLOAT32) || q->ndim != 4 || v->ndim != 4 || q->shape[0] != v->shape[0] || q->shape[1] != v->shape[1]) return false;
    const int64_t kh = q->shape[2], h = v->shape[2];
    if (q->shape[0] < 0 || q->shape[1] < 0 || q->shape[1] >= (int64_t{1} << 30) || kh < 1 || h < 1 || h >= (1 << 20) || h % kh != 0) return false;
    if (q->shape[3] < 1 || q->shape[3] > kMaxAttend || v->shape[3] < 1 || v->shape[3] > kMaxAttend || q->shape[0] > kBlocksPerLaunch / h) return false;
    c->p.batch = q->shape[0], c->p.length = q->shape[1], c->p.heads = static_cast<int>(h);
    c->keys = static_cast<int>(q->shape[3]), c->values = static_cast<int>(v->shape[3]), c->key_heads = static_cast<int>(kh), c->dtype = q->dtype;
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

void CutForward(AttendCall* c, bool padded) {
    if (c->p.length <= kAttendTokens) c->p.segments = 1, c->p.segment_rows = kAttendTile;
    else CutAttend(&c->p, padded, AttendBlocks(c->values), AttendBlocks(c->values), AttendResident(c->dtype == HIPCX_FLOAT16, c->keys), static_cast<int64_t>(c->keys) * c->values);
}

size_t ForwardWorkspace(const AttendCall& c) {
    if (c.p.segments < 2) return 0;
    return static_cast<size_t>(c.p.batch * c.p.heads * c.p.segments * (static_cast<int64_t>(c.keys) * c.values + 1) * 4);
}

}  // namespace
}  // namespace hipcx

using namespace hipcx;

extern "C" {

size_t hipcx_linear_attention_workspace_size(const hipcx_array* q, const hipcx_array* v, const hipcx_array* lengths) {
    AttendCall c;
    if (!AttendSizesOf(q, v, &c)) return 0;
    CutForward(&c, lengths != nullptr);
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
        CutForward(&c, lengths != nullptr);
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
                    constexpr int KD = decltype(kd)::value;
                    void (*const kernel)(AttendArgs) = c.values < 4 ? AttendTokensKernel<T, KD, kAttendNarrow> : c.values % 4 == 0 ? AttendTokensKernel<T, KD, kAttendWhole> : AttendTokensKernel<T, KD, kAttendPart>;
                    hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(blocks)), dim3(256), 0, AsStream(stream), p);
                    CheckLaunch("linear_attention");
                });
            });
            return;
        }
        if (p.segments > 1) {
            HIPCX_REQUIRE(reinterpret_cast<uintptr_t>(workspace) % 16 == 0, HIPCX_CHAINERX_ERROR, "workspace must be 16-byte aligned");
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
