// Linear attention of float16: the passes of linear_attention.h on the float16 matrix pipe, with nothing that was computed in fewer than 22 bits.
#include "igemm.h"
#include "linear_attention.h"

namespace hipcx {
namespace {

struct AttendHalfTag {};

typedef short attend_short4_t __attribute__((ext_vector_type(4)));
typedef _Float16 attend_half4_t __attribute__((ext_vector_type(4)));
typedef _Float16 attend_half8_t __attribute__((ext_vector_type(8)));

// Four rows of a lane's column, of a block of 4 rows x 16 columns that sixteen lanes read together (lane l: row l / 4, columns 4 (l % 4) and on).
__device__ __forceinline__ attend_half4_t ReadTurned(const char* at) {
    return __builtin_bit_cast(attend_half4_t, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) attend_short4_t*)at));
}
__device__ __forceinline__ attend_half8_t Join(attend_half4_t a, attend_half4_t b) { return attend_half8_t{a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]}; }

// The power of two that brings `most`, the largest of some values, to at least 2^14 and below 2^15; and the one that brings them back.
struct Scale {
    float in, out;
    __device__ __forceinline__ explicit Scale(float most) {
        const int e = max((__builtin_bit_cast(int, most) >> 23) - 141, -112);
        in = __builtin_bit_cast(float, (127 - e) << 23);
        out = __builtin_bit_cast(float, (127 + e) << 23);
    }
};

// Eight values of at most 2^15 as the sum of two float16: 22 bits of those from 2^-14 on.
__device__ __forceinline__ void Split(const float (&v)[8], attend_half8_t* high, attend_half8_t* low) {
    attend_half8_t h, l;
#pragma unroll
    for (int e = 0; e < 8; e += 2) {
        const auto hi = __builtin_amdgcn_cvt_pkrtz(v[e], v[e + 1]);
        const auto lo = __builtin_amdgcn_cvt_pkrtz(__builtin_fmaf(static_cast<float>(hi[0]), -1.f, v[e]), __builtin_fmaf(static_cast<float>(hi[1]), -1.f, v[e + 1]));
        h[e] = hi[0], h[e + 1] = hi[1], l[e] = lo[0], l[e + 1] = lo[1];
    }
    *high = h, *low = l;
}
__device__ __forceinline__ void Split(const float (&v)[4], attend_half4_t* high, attend_half4_t* low) {
    attend_half4_t h, l;
#pragma unroll
    for (int e = 0; e < 4; e += 2) {
        const auto hi = __builtin_amdgcn_cvt_pkrtz(v[e], v[e + 1]);
        const auto lo = __builtin_amdgcn_cvt_pkrtz(__builtin_fmaf(static_cast<float>(hi[0]), -1.f, v[e]), __builtin_fmaf(static_cast<float>(hi[1]), -1.f, v[e + 1]));
        h[e] = hi[0], h[e + 1] = hi[1], l[e] = lo[0], l[e + 1] = lo[1];
    }
    *high = h, *low = l;
}

__device__ __forceinline__ attend16_t Mfma(attend_half8_t a, attend_half8_t b, attend16_t c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }

// LDS of a workgroup, in bytes.  Rows' pitches keep the banks apart: of k, read by rows (32 of them, 16 bytes each) and in blocks of 4 x 16, 80 bytes more than a multiple of 128; of v, read in
// such blocks alone, 64 more; of the state's copies, read by rows, 16 more.
template <int KD>
struct AttendHalfLds {
    static constexpr int kKeyPitch = KD * 2 + 80, kValuePitch = kAttendColumns * 2 + 64, kStatePitch = KD * 2 + 16;
    static constexpr int kValues = kAttendTile * kKeyPitch, kStates = kValues + kAttendTile * kValuePitch, kLow = kStates + kAttendColumns * kStatePitch,
                         kScales = kLow + kAttendColumns * kStatePitch, kSums = kScales + 2 * kAttendColumns * 4, kDecays = kSums + 4 * kAttendColumns * 4,
                         kOdd = kDecays + 2 * static_cast<int>(sizeof(AttendDecays)), kBytes = kOdd + 16;
    static_assert(kValues % 16 == 0 && kStates % 16 == 0 && kDecays % 16 == 0 && sizeof(AttendDecays) % 16 == 0, "aligned parts");
};

// As AttendKernel (linear_attention.hip): a wave multiplies 32 rows by 32 columns of y, and has half of the keys and 32 columns of the state in its accumulators.
//   P^T = K Q^T (rows s, a lane to a row t) from float16 as they come; times the weights, brought to float16's range by a power of two for each t, in two parts;
//   y^T = V^T P^T + S^T Q^T, S in two parts of float16 in LDS, with a power of two for each column and half of the keys;
//   S <- exp(G[63]) S + K^T (exp(G[63] - G) V), V's products in two parts, with a power of two for each column.
// A reduction over rows s takes them in the order in which accumulators have them, eight to a lane: 4 h + j and 8 + 4 h + j of sixteen, for both operands.
template <int KD, bool OUT>
__global__ __launch_bounds__(256, KD == 256 ? 1 : 2) void AttendHalfKernel(AttendArgs p) {
    using T = half_t;
    using Lds = AttendHalfLds<KD>;
    constexpr int VB = kAttendColumns, C = kAttendTile, NS = KD / 64, NK = KD / 32, NV = VB / 32, NQ = KD / 16;
    extern __shared__ __align__(16) char lds[];
    char *const ks = lds, *const vs = lds + Lds::kValues, *const high_copy = lds + Lds::kStates, *const low_copy = lds + Lds::kLow;
    float* const scales = reinterpret_cast<float*>(lds + Lds::kScales);  // [2][VB]
    float* const sums = reinterpret_cast<float*>(lds + Lds::kSums);      // [4][VB]
    AttendDecays* const decays = reinterpret_cast<AttendDecays*>(lds + Lds::kDecays);
    int* const odd = reinterpret_cast<int*>(lds + Lds::kOdd);            // v has infinities or what is not a number

    int id = static_cast<int>(blockIdx.x);
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
    const int keys = run.keys, col0 = (block - run.first) * VB, cols = min(VB, run.values - col0);

    const int tid = threadIdx.x, lane = tid % 64, wave = tid / 64, l32 = lane % 32, half = lane / 32;
    const int tw = wave / 2, dw = wave % 2;
    const T* const kp = static_cast<const T*>(run.k.data) + b * run.k.batch + (h / run.k.share) * run.k.head;
    const T* const vp = static_cast<const T*>(run.v.data) + b * run.v.batch + (h / run.v.share) * run.v.head + col0;
    const T* const qp = OUT ? static_cast<const T*>(run.q.data) + b * run.q.batch + (h / run.q.share) * run.q.head : nullptr;
    const T* const dp = OUT && run.dots != nullptr ? static_cast<const T*>(run.dot.data) + b * run.dot.batch + (h / run.dot.share) * run.dot.head + col0 : nullptr;
    const int64_t y0 = OUT ? b * run.y.batch + h * run.y.head + col0 : 0;
    const int parts = 2 * run.blocks;
    float* const dots = OUT && run.dots != nullptr ? run.dots + static_cast<int64_t>(bh) * p.length * parts + (block - run.first) * 2 : nullptr;

    const auto state_row = [&](int n, int r) { return KD / 2 * tw + 32 * n + 8 * (r / 4) + 4 * half + r % 4; };
    const int state_col = 32 * dw + l32;
    attend16_t s[NS];
#pragma unroll
    for (int n = 0; n < NS; ++n) {
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            const int i = state_row(n, r);
            s[n][r] = OUT && run.start.data != nullptr && i < keys && state_col < cols
                          ? run.start.data[bh * run.start.head + segment * run.start.segment + i * run.start.i + (col0 + state_col) * run.start.j]
                          : 0.f;
        }
    }
    const auto keep_state = [&] {
        float most = 0;
#pragma unroll
        for (int n = 0; n < NS; ++n) {
#pragma unroll
            for (int r = 0; r < 16; ++r) most = fmaxf(most, fabsf(s[n][r]));
        }
        most = fmaxf(most, __shfl_xor(most, 32));
        const Scale scale(most);
        if (half == 0) scales[tw * VB + state_col] = scale.out;
#pragma unroll
        for (int n = 0; n < NS; ++n) {
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const float v[4] = {s[n][4 * g] * scale.in, s[n][4 * g + 1] * scale.in, s[n][4 * g + 2] * scale.in, s[n][4 * g + 3] * scale.in};
                attend_half4_t hi, lo;
                Split(v, &hi, &lo);
                const int at = state_col * Lds::kStatePitch + state_row(n, 4 * g) * 2;
                *reinterpret_cast<attend_half4_t*>(high_copy + at) = hi;
                *reinterpret_cast<attend_half4_t*>(low_copy + at) = lo;
            }
        }
    };
    if (OUT) keep_state();

    // A tile's rows on their way: pieces of eight elements of k and of v, and this lane's row of q.  Rows that are not there are the last one again; columns that are not there are zeros that
    // stay in LDS.
    const int key_row = tid / (KD / 8), key_col = tid % (KD / 8) * 8, value_row = tid / (VB / 8), value_col = tid % (VB / 8) * 8;
    const bool even = keys % 8 == 0 && cols % 8 == 0;
    const int t = 32 * tw + l32;  // this lane's row of a tile
    attend_half8_t k_next[NK], v_next[NV], q_next[OUT ? NQ : 1];
    double g_next = 0;
    const auto load = [&](int64_t r0) {
        const auto at = [&](int64_t r) { return AttendRowOf(span, run.back, r0 + r < rows ? r0 + r : rows - 1); };
        if (even) {
#pragma unroll
            for (int n = 0; n < NK; ++n) {
                const AttendPiece<T, 8> piece = *reinterpret_cast<const AttendPiece<T, 8>*>(kp + at(key_row + n * (2048 / KD)) * run.k.row + (key_col < keys ? key_col : 0));
#pragma unroll
                for (int e = 0; e < 8; ++e) k_next[n][e] = piece.v[e];
            }
#pragma unroll
            for (int n = 0; n < NV; ++n) {
                const AttendPiece<T, 8> piece = *reinterpret_cast<const AttendPiece<T, 8>*>(vp + at(value_row + n * 32) * run.v.row + (value_col < cols ? value_col : 0));
#pragma unroll
                for (int e = 0; e < 8; ++e) v_next[n][e] = piece.v[e];
            }
            if constexpr (OUT) {
                const T* const q = qp + at(t) * run.q.row;
#pragma unroll
                for (int m = 0; m < NQ; ++m) {
                    const int i = 16 * m + 8 * half;
                    const AttendPiece<T, 8> piece = *reinterpret_cast<const AttendPiece<T, 8>*>(q + (i < keys ? i : 0));
#pragma unroll
                    for (int e = 0; e < 8; ++e) q_next[m][e] = piece.v[e];
                }
            }
        } else {
#pragma unroll
            for (int n = 0; n < NK; ++n) {
                const AttendPiece<T, 8> piece = AttendLoad<T, 8>(kp + at(key_row + n * (2048 / KD)) * run.k.row, key_col, keys);
#pragma unroll
                for (int e = 0; e < 8; ++e) k_next[n][e] = piece.v[e];
            }
#pragma unroll
            for (int n = 0; n < NV; ++n) {
                const AttendPiece<T, 8> piece = AttendLoad<T, 8>(vp + at(value_row + n * 32) * run.v.row, value_col, cols);
#pragma unroll
                for (int e = 0; e < 8; ++e) v_next[n][e] = piece.v[e];
            }
            if constexpr (OUT) {
                const T* const q = qp + at(t) * run.q.row;
#pragma unroll
                for (int m = 0; m < NQ; ++m) {
                    const AttendPiece<T, 8> piece = AttendLoad<T, 8>(q, 16 * m + 8 * half, keys);
#pragma unroll
                    for (int e = 0; e < 8; ++e) q_next[m][e] = piece.v[e];
                }
            }
        }
        g_next = r0 + lane < rows ? AttendStep(p, run, span, b, h, length, r0 + lane) : 0;
    };
    const auto sum_next = [&](int64_t r0, AttendDecays* to) { SumDecays(to, g_next, static_cast<int>(rows - r0 < C ? rows - r0 : C), run.kv_scale); };
    if (even) {
#pragma unroll
        for (int n = 0; n < NK; ++n) {
            if (key_col >= keys) *reinterpret_cast<attend_half8_t*>(ks + (key_row + n * (2048 / KD)) * Lds::kKeyPitch + key_col * 2) = attend_half8_t{};
        }
#pragma unroll
        for (int n = 0; n < NV; ++n) {
            if (value_col >= cols) *reinterpret_cast<attend_half8_t*>(vs + (value_row + n * 32) * Lds::kValuePitch + value_col * 2) = attend_half8_t{};
        }
    }
    if (tid == 0) odd[0] = odd[1] = 0;
    if (rows > 0) {
        load(0);
        if (wave == 0) sum_next(0, decays);
    }
    double passed = 0;  // log decay of the tiles so far
    // where a lane reads blocks of 4 x 16: rows 4 half and on, columns of its 32
    const int turned_row = 4 * half + lane % 16 / 4, turned_col = (lane / 16 % 2 * 16 + lane % 4 * 4) * 2;

    int turn = 0;
    __syncthreads();  // the flags
    for (int64_t r0 = 0; r0 < rows; r0 += C, turn ^= 1) {
        const int here = static_cast<int>(rows - r0 < C ? rows - r0 : C);
        const AttendDecays* const dec = decays + turn;
        attend_half8_t q[OUT ? NQ : 1];
        // (the last tile's rows of k and v have been read by all)
#pragma unroll
        for (int n = 0; n < NK; ++n) {
            if (!even || key_col < keys) *reinterpret_cast<attend_half8_t*>(ks + (key_row + n * (2048 / KD)) * Lds::kKeyPitch + key_col * 2) = k_next[n];
        }
        attend_half8_t finite{};
#pragma unroll
        for (int n = 0; n < NV; ++n) {
            if (!even || value_col < cols) *reinterpret_cast<attend_half8_t*>(vs + (value_row + n * 32) * Lds::kValuePitch + value_col * 2) = v_next[n];
            finite += v_next[n] - v_next[n];
        }
        if constexpr (OUT) {
            const T all = finite[0] + finite[1] + finite[2] + finite[3] + finite[4] + finite[5] + finite[6] + finite[7];
            if (all != 0) odd[turn] = 1;
#pragma unroll
            for (int m = 0; m < NQ; ++m) q[m] = q_next[m];
        }
        __syncthreads();
        passed += dec->sum;
        const bool more = r0 + C < rows;
        if (more) load(r0 + C);
        if (OUT && odd[turn] != 0) {
            // An infinity of a later row, times P's zeros, would reach earlier ones: row by row instead, on a copy of the state in 32 bits in the place of the others.
            float* const ss = reinterpret_cast<float*>(high_copy);  // [KD][VB]
#pragma unroll
            for (int n = 0; n < NS; ++n) {
#pragma unroll
                for (int r = 0; r < 16; ++r) ss[state_row(n, r) * VB + state_col] = s[n][r];
            }
            if (wave == 0 && more) sum_next(r0 + C, decays + (turn ^ 1));
            if (tid == 0) odd[turn ^ 1] = 0;
            __syncthreads();
            const int j = lane;
            for (int r = 0; r < here; ++r) {
                const int64_t row = AttendRowOf(span, run.back, r0 + r);
                const float step = dec->step[r], v = static_cast<float>(*reinterpret_cast<const T*>(vs + r * Lds::kValuePitch + j * 2)) * run.kv_scale;
                float y = 0;
                for (int i = wave * (KD / 4); i < (wave + 1) * (KD / 4); ++i) {
                    const float now = ss[i * VB + j] * step + static_cast<float>(*reinterpret_cast<const T*>(ks + r * Lds::kKeyPitch + i * 2)) * v;
                    ss[i * VB + j] = now;
                    if (i < keys) y += static_cast<float>(qp[row * run.q.row + i]) * now;
                }
                sums[wave * VB + j] = y;
                __syncthreads();
                if (wave == 0) {
                    y = (sums[j] + sums[VB + j] + sums[2 * VB + j] + sums[3 * VB + j]) * run.out_scale;
                    if (j < cols) {
                        if (run.wide) static_cast<float*>(run.y.data)[y0 + row * run.y.row + j] = y;
                        else static_cast<T*>(run.y.data)[y0 + row * run.y.row + j] = static_cast<T>(y);
                    }
                    if (dots != nullptr) {
                        float dot = j < cols ? y * static_cast<float>(dp[row * run.dot.row + j]) : 0.f;
#pragma unroll
                        for (int o = 1; o < 32; o <<= 1) dot += __shfl_xor(dot, o);
                        if (l32 == 0) dots[row * parts + half] = dot;
                    }
                }
                __syncthreads();
            }
#pragma unroll
            for (int n = 0; n < NS; ++n) {
#pragma unroll
                for (int r = 0; r < 16; ++r) s[n][r] = ss[state_row(n, r) * VB + state_col];
            }
            __syncthreads();
            keep_state();
            continue;
        }
        // this wave's columns of v, for the products with P and with k: rows 16 u + ... of step u
        attend_half8_t v[C / 16];
#pragma unroll
        for (int u = 0; u < C / 16; ++u) {
            const char* const at = vs + (16 * u + turned_row) * Lds::kValuePitch + dw * 64 + turned_col;
            v[u] = Join(ReadTurned(at), ReadTurned(at + 8 * Lds::kValuePitch));
        }
        if constexpr (OUT) {
            attend16_t a[2]{}, of_state[2]{};
#pragma unroll
            for (int sb = 0; sb < 2; ++sb) {
                if (sb > tw) continue;
                const char* const at = ks + (32 * sb + l32) * Lds::kKeyPitch + 16 * half;
#pragma unroll
                for (int m = 0; m < NQ; ++m) a[sb] = Mfma(*reinterpret_cast<const attend_half8_t*>(at + 32 * m), q[m], a[sb]);
            }
            {
                const int at = state_col * Lds::kStatePitch + 16 * half;
#pragma unroll
                for (int m = 0; m < NQ; ++m) {
                    attend16_t& to = of_state[m / (NQ / 2)];
                    to = Mfma(*reinterpret_cast<const attend_half8_t*>(low_copy + at + 32 * m), q[m], to);
                    to = Mfma(*reinterpret_cast<const attend_half8_t*>(high_copy + at + 32 * m), q[m], to);
                }
            }
            if (wave == 3 && more) sum_next(r0 + C, decays + (turn ^ 1));
            if (tid == 0) odd[turn ^ 1] = 0;
            const float high = dec->high[t], low = dec->low[t];
            float most = 0;
#pragma unroll
            for (int sb = 0; sb < 2; ++sb) {
                if (sb > tw) continue;
#pragma unroll
                for (int g = 0; g < 4; ++g) {
                    const int first = 32 * sb + 8 * g + 4 * half;
                    const attend4_t highs = *reinterpret_cast<const attend4_t*>(dec->high + first), lows = *reinterpret_cast<const attend4_t*>(dec->low + first);
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const float weighted = a[sb][4 * g + e] * __builtin_amdgcn_exp2f((high - highs[e]) + (low - lows[e]));
                        a[sb][4 * g + e] = first + e <= t ? weighted : 0.f;
                        most = fmaxf(most, fabsf(a[sb][4 * g + e]));
                    }
                }
            }
            const Scale scale(fmaxf(most, __shfl_xor(most, 32)));
            attend16_t of_rows{};
#pragma unroll
            for (int sb = 0; sb < 2; ++sb) {
                if (sb > tw) continue;
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    float w[8];
#pragma unroll
                    for (int e = 0; e < 8; ++e) w[e] = a[sb][8 * u + e] * scale.in;
                    attend_half8_t hi, lo;
                    Split(w, &hi, &lo);
                    of_rows = Mfma(v[2 * sb + u], lo, of_rows);
                    of_rows = Mfma(v[2 * sb + u], hi, of_rows);
                }
            }
            const float from_start = __builtin_amdgcn_exp2f(high + low) * run.out_scale, from_rows = scale.out * run.kv_scale * run.out_scale;
            const int64_t row = AttendRowOf(span, run.back, r0 + t);
            float dot = 0;
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const int j = 32 * dw + 8 * g + 4 * half;
                const attend4_t first = *reinterpret_cast<const attend4_t*>(scales + j), second = *reinterpret_cast<const attend4_t*>(scales + VB + j);
                AttendPiece<float, 4> y;
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    y.v[e] = __builtin_fmaf(__builtin_fmaf(of_state[0][4 * g + e], first[e], of_state[1][4 * g + e] * second[e]), from_start, of_rows[4 * g + e] * from_rows);
                if (t >= here) continue;
                if (dots != nullptr) {
                    const AttendPiece<T, 4> with = AttendLoad<T, 4>(dp + row * run.dot.row, j, cols);
#pragma unroll
                    for (int e = 0; e < 4; ++e) dot += j + e < cols ? y.v[e] * static_cast<float>(with.v[e]) : 0.f;
                }
                const int64_t to = y0 + row * run.y.row + j;
                if (j + 4 <= cols) {
                    if (run.wide) {
                        *reinterpret_cast<AttendPiece<float, 4>*>(static_cast<float*>(run.y.data) + to) = y;
                    } else {
                        AttendPiece<T, 4> o;
#pragma unroll
                        for (int e = 0; e < 4; ++e) o.v[e] = static_cast<T>(y.v[e]);
                        *reinterpret_cast<AttendPiece<T, 4>*>(static_cast<T*>(run.y.data) + to) = o;
                    }
                } else {
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        if (j + e >= cols) continue;
                        if (run.wide) static_cast<float*>(run.y.data)[to + e] = y.v[e];
                        else static_cast<T*>(run.y.data)[to + e] = static_cast<T>(y.v[e]);
                    }
                }
            }
            if (dots != nullptr) {
                dot += __shfl_xor(dot, 32);
                if (half == 0 && t < here) dots[row * parts + dw] = dot;
            }
        } else {
            if (wave == 3 && more) sum_next(r0 + C, decays + (turn ^ 1));
        }
        // v times its rows' weights, in two parts
        float w[C / 16][8], most = 0;
#pragma unroll
        for (int u = 0; u < C / 16; ++u) {
#pragma unroll
            for (int g = 0; g < 2; ++g) {
                const attend4_t end = *reinterpret_cast<const attend4_t*>(dec->end + 16 * u + 8 * g + 4 * half);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    w[u][4 * g + e] = static_cast<float>(v[u][4 * g + e]) * end[e];
                    most = fmaxf(most, fabsf(w[u][4 * g + e]));
                }
            }
        }
        const Scale scale(fmaxf(most, __shfl_xor(most, 32)));
        attend16_t add[NS]{};
#pragma unroll
        for (int u = 0; u < C / 16; ++u) {
#pragma unroll
            for (int e = 0; e < 8; ++e) w[u][e] *= scale.in;
            attend_half8_t hi, lo;
            Split(w[u], &hi, &lo);
#pragma unroll
            for (int n = 0; n < NS; ++n) {
                const char* const at = ks + (16 * u + turned_row) * Lds::kKeyPitch + (KD / 2 * tw + 32 * n) * 2 + turned_col;
                const attend_half8_t k = Join(ReadTurned(at), ReadTurned(at + 8 * Lds::kKeyPitch));
                add[n] = Mfma(k, lo, add[n]);
                add[n] = Mfma(k, hi, add[n]);
            }
        }
        const float all = dec->all;
#pragma unroll
        for (int n = 0; n < NS; ++n) {
#pragma unroll
            for (int r = 0; r < 16; ++r) s[n][r] = __builtin_fmaf(s[n][r], all, add[n][r] * scale.out);
        }
        __syncthreads();  // the copies of the state, and the rows of k and v, have been read
        if (OUT) keep_state();
    }

    if constexpr (!OUT) {
        float* const to = run.last.data + bh * run.last.head + segment * run.last.segment;
#pragma unroll
        for (int n = 0; n < NS; ++n) {
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const int i = state_row(n, r);
                if (i < keys && state_col < cols) to[i * run.last.i + (col0 + state_col) * run.last.j] = s[n][r];
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
        // <state behind the segment, its gradient there>, the waves' parts added up in the same order always
        float dot = 0;
        if (run.other.data != nullptr) {
#pragma unroll
            for (int n = 0; n < NS; ++n) {
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    const int i = state_row(n, r);
                    if (i < keys && state_col < cols)
                        dot += s[n][r] * run.other.data[bh * run.other.head + segment * run.other.segment + i * run.other.i + (col0 + state_col) * run.other.j];
                }
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
        const float more = run.decay_last && length > 0 ? __builtin_amdgcn_exp2f(static_cast<float>(AttendDecay(p, b, h, 0))) : 1.f;
        float* const to = run.last.data + bh * run.last.head;
#pragma unroll
        for (int n = 0; n < NS; ++n) {
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const int i = state_row(n, r);
                if (i < keys && state_col < cols) to[i * run.last.i + (col0 + state_col) * run.last.j] = s[n][r] * more;
            }
        }
    }
}

}  // namespace

void LaunchAttendHalf(const AttendArgs& p, int keys, bool states_alone, hipStream_t stream) {
    const int64_t blocks = p.blocks * p.batch * p.heads * (states_alone ? p.segments - 1 : p.segments);
    const auto launch = [&](auto kd) {
        constexpr int KD = decltype(kd)::value, kLds = AttendHalfLds<KD>::kBytes;
        const dim3 grid(static_cast<unsigned>(blocks));
        if (states_alone) {
            EnsureDynamicLds<AttendHalfTag>(reinterpret_cast<const void*>(AttendHalfKernel<KD, false>), kLds);
            hipLaunchKernelGGL((AttendHalfKernel<KD, false>), grid, dim3(256), kLds, stream, p);
        } else {
            EnsureDynamicLds<AttendHalfTag>(reinterpret_cast<const void*>(AttendHalfKernel<KD, true>), kLds);
            hipLaunchKernelGGL((AttendHalfKernel<KD, true>), grid, dim3(256), kLds, stream, p);
        }
        CheckLaunch("linear_attention");
    };
    if (keys <= 64) launch(std::integral_constant<int, 64>{});
    else if (keys <= 128) launch(std::integral_constant<int, 128>{});
    else launch(std::integral_constant<int, 256>{});
}

}  // namespace hipcx
