// Linear attention of float16: the passes of linear_attention.h on the float16 matrix pipe, with nothing that was computed in fewer than 23 bits.
#include "igemm.h"
#include "linear_attention.h"

namespace hipcx {
namespace {

typedef short attend_short4_t __attribute__((ext_vector_type(4)));
typedef _Float16 attend_half2_t __attribute__((ext_vector_type(2)));
typedef _Float16 attend_half4_t __attribute__((ext_vector_type(4)));
typedef _Float16 attend_half8_t __attribute__((ext_vector_type(8)));

// Four rows of a lane's column, of a block of 4 rows x 16 columns that sixteen lanes read together (lane l: row l / 4, columns 4 (l % 4) and on).
__device__ __forceinline__ attend_half4_t ReadTurned(const char* at) {
    return __builtin_bit_cast(attend_half4_t, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) attend_short4_t*)at));
}
__device__ __forceinline__ attend_half8_t Join(attend_half4_t a, attend_half4_t b) { return attend_half8_t{a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]}; }

// The larger of a lane's value and that of the lane 32 or 16 away: two registers exchange halves, or rows of 16 lanes.  (As assembly, with the waits that the vector units' results need: of the
// builtin's two results the compiler takes the first for both.)
__device__ __forceinline__ float MaxOver32(float v) {
    float w = v;
    asm("s_nop 1\n\tv_permlane32_swap_b32 %0, %1\n\ts_nop 1" : "+v"(v), "+v"(w));
    return fmaxf(v, w);
}
__device__ __forceinline__ float MaxOver16(float v) {
    float w = v;
    asm("s_nop 1\n\tv_permlane16_swap_b32 %0, %1\n\ts_nop 1" : "+v"(v), "+v"(w));
    return fmaxf(v, w);
}

// The power of two that brings `most`, the largest of some values, to at least 2^14 and below 2^15; and the one that brings them back.
struct Scale {
    float in, out;
    __device__ __forceinline__ explicit Scale(float most) {
        const int e = max((__builtin_bit_cast(int, most) >> 23) - 141, -112);
        in = __builtin_bit_cast(float, (127 - e) << 23);
        out = __builtin_bit_cast(float, (127 + e) << 23);
    }
};

__device__ __forceinline__ int ExponentOf(float v) { return (__builtin_bit_cast(int, v) >> 23) - 127; }  // of v >= 0
__device__ __forceinline__ float Power(int e) { return __builtin_bit_cast(float, (127 + e) << 23); }       // of -126 to 127

// Values of at most 2^15 as the sum of two float16, each rounded to nearest: 23 bits and a sign of those from 2^-2 on, 2^-25 of the others.  (Cut off instead, as quickly, they kept 21 bits and
// all errors had one sign.)  `minus`: -1, which the compiler is not to know, so that the difference is one instruction that takes a float16 as it is.
template <int N>
__device__ __forceinline__ void Split(const float (&v)[N], float minus, _Float16 __attribute__((ext_vector_type(N)))* high, _Float16 __attribute__((ext_vector_type(N)))* low) {
    typedef float float2_t __attribute__((ext_vector_type(2)));
#pragma unroll
    for (int e = 0; e < N; e += 2) {
        const attend_half2_t hi = __builtin_convertvector((float2_t{v[e], v[e + 1]}), attend_half2_t);
        const float2_t rest{__builtin_fmaf(static_cast<float>(hi[0]), minus, v[e]), __builtin_fmaf(static_cast<float>(hi[1]), minus, v[e + 1])};
        const attend_half2_t lo = __builtin_convertvector(rest, attend_half2_t);
        (*high)[e] = hi[0], (*high)[e + 1] = hi[1], (*low)[e] = lo[0], (*low)[e + 1] = lo[1];
    }
}

__device__ __forceinline__ attend4_t Mfma(attend_half8_t a, attend_half8_t b, attend4_t c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }

// The value of lane L of a row of 16 lanes.
template <int L>
__device__ __forceinline__ double OfLaneInRow(double v) {
    const uint64_t b = __builtin_bit_cast(uint64_t, v);
    const uint32_t lo = __builtin_amdgcn_mov_dpp(static_cast<int>(b), 0x150 + L, 0xf, 0xf, true), hi = __builtin_amdgcn_mov_dpp(static_cast<int>(b >> 32), 0x150 + L, 0xf, 0xf, true);
    return __builtin_bit_cast(double, static_cast<uint64_t>(hi) << 32 | lo);
}

// Factors of P's rows s, 0 for rows whose v is zeros: they have no part in the power of two of the others.
struct AttendHalfDecays : AttendDecays {
    alignas(16) float near[kAttendTile];  // from a row to the last of its sixteen, as a factor
    alignas(16) float own[kAttendTile];   // `low`, or infinity, which takes exp2(high - high[s] + low - own[s]) to 0
};
typedef uint32_t attend_uint4_t __attribute__((ext_vector_type(4)));
// Whether a piece is zeros.
__device__ __forceinline__ bool IsZeros(AttendPiece<half_t, 8> piece) {
    const attend_uint4_t d = __builtin_bit_cast(attend_uint4_t, piece);
    return ((d[0] | d[1] | d[2] | d[3]) & 0x7fff7fffu) == 0;
}
// Whether one of some pieces may be: its first two elements, taken for a float, are one below 2^-126 then.  An instruction to two pieces (the compiler would make what is not a number quiet first).
template <int N>
__device__ __forceinline__ float LeastOf(const AttendPiece<half_t, 8> (&pieces)[N], float least) {
#pragma unroll
    for (int n = 0; n < N; n += 2) {
        const uint32_t a = __builtin_bit_cast(attend_uint4_t, pieces[n])[0], b = __builtin_bit_cast(attend_uint4_t, pieces[n + 1 < N ? n + 1 : n])[0];
        asm("v_min3_f32 %0, |%0|, |%1|, |%2|" : "+v"(least) : "v"(a), "v"(b));
    }
    return least;
}

// LDS of a workgroup, in bytes.  Rows' pitches keep the banks apart.  Clocks of a wave's instruction (eight waves at work), at 128 keys: k and the state's copies read by rows, sixteen rows of 64
// bytes each, 4.0 with 32 or 96 bytes more than a multiple of 256, 7.9 with 16, 6.6 with 80; v in blocks of 4 x 16, sixteen rows, 2.6 with 32 more than 128, 4.0 with 64; the state's copies
// written, 8.0 with 32, 5.0 with 16.
template <int KD, bool OUT>
struct AttendHalfLds {
    static constexpr int kKeyPitch = KD * 2 + 96, kValuePitch = kAttendColumns * 2 + 32, kStatePitch = KD * 2 + 32;
    static constexpr int kValues = kAttendTile * kKeyPitch, kStates = kValues + kAttendTile * kValuePitch,
                         kLow = kStates + (OUT ? kAttendColumns * kStatePitch : 0), kScales = kLow + (OUT ? kAttendColumns * kStatePitch : 0), kSums = kScales + kAttendColumns * 4, kDecays = kSums + 4 * kAttendColumns * 4,
                         kOdd = kDecays + 2 * static_cast<int>(sizeof(AttendHalfDecays)), kBytes = kOdd + 16;
    static_assert(AttendResident(true, KD) * kBytes <= kLdsOfUnit, "as many workgroups as the time axis is cut for");
    static_assert(kValues % 16 == 0 && kStates % 16 == 0 && kDecays % 16 == 0 && sizeof(AttendHalfDecays) % 16 == 0, "aligned parts");
};

// As AttendKernel (linear_attention.hip): a wave has sixteen rows of y with all 64 columns, and sixteen columns of the state with all keys in its accumulators.
//   y^T = S^T Q^T, S in two parts of float16 in LDS;
//   P^T = K Q^T (rows s, a lane to a row t) from float16 as they come; times the weights, brought to float16's range by a power of two for each t, in two parts; y^T += V^T P^T;
//   S <- exp(G[63]) S + K^T (exp(G[63] - G) V), V's products in two parts.
// S and what is added to it are counted in a power of two for each column (`unit`), which changes when the largest element of the column or of what is added (V's products) leaves 2^4 to 2^15 of
// it, so that parts of float16 keep 23 bits, or 2^-29 of that largest element; a row of P in one of its own, so that they keep 23 bits or 2^-39 of its largest.  Rows of k that are zeros have no part
// in the largest of what is added, nor rows of v that are zeros in P's, whatever a mask has left on the other side (told by an
// instruction to two pieces and the flag of infinities: 0.5 % of the prompt of 16384 rows; of gradients at 50 and 256 keys 3 and 2 %).
// A reduction over 32 rows s takes them in the order in which accumulators have them, eight to a lane, for both operands: 4 q + j and 16 + 4 q + j for quarter q of a wave.
// (32 rows by 32 columns of y to a wave have every block of P computed by two waves; half of the keys by 32 columns of S every product with V.)
// Bound by a tile's chain at two workgroups to a compute unit: of its cycles the vector units work in 45 %, LDS in 40, the matrix pipes in 17.  One sequence of 16384 rows, 16 heads of 128 x 128: 100 us
// and 42 for the states of its 16 segments; on the float pipe 1.1 ms.  Gradients of 4 x 2048 rows, 16 heads of 128 x 128, three passes: 227 us.
// GRAD: what the passes of the gradients have beyond the forward one.
template <int KD, bool OUT, int WIDTHS, bool GRAD>
__global__ __launch_bounds__(256, AttendResident(true, KD)) void AttendHalfKernel(AttendArgs p) {
    using T = half_t;
    constexpr bool EVEN = WIDTHS == kAttendWhole;
    using Lds = AttendHalfLds<KD, OUT>;
    constexpr int VB = kAttendColumns, C = kAttendTile, NS = KD / 16, NK = KD / 32, NV = VB / 32, NQ = KD / 32, DB = VB / 16;
    extern __shared__ __align__(16) char lds[];
    char *const ks = lds, *const vs = lds + Lds::kValues, *const high_copy = lds + Lds::kStates, *const low_copy = lds + Lds::kLow;
    float* const scales = reinterpret_cast<float*>(lds + Lds::kScales);  // [2][VB]
    float* const sums = reinterpret_cast<float*>(lds + Lds::kSums);      // [4][VB]
    AttendHalfDecays* const decays = reinterpret_cast<AttendHalfDecays*>(lds + Lds::kDecays);
    int* const odd = reinterpret_cast<int*>(lds + Lds::kOdd);            // [2][2]: v has infinities or what is not a number; a row may be zeros

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
    const bool back = GRAD && run.back != 0, wide = GRAD && run.wide != 0, with_dots = GRAD && OUT && run.dots != nullptr;
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
    // What follows from the lane is found again in every tile: kept over the loop, it would take the registers of what is multiplied.
    const auto dots = [&] { return run.dots + (static_cast<int64_t>(bh) * run.blocks + block - run.first) * p.length; };

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
    float minus = -1;
    asm volatile("" : "+s"(minus));
    int unit = 0;    // the state is s times 2^unit
    float most = 0;  // the largest |s| of the column
    const auto find_most = [&] {
        most = 0;
#pragma unroll
        for (int n = 0; n < NS; ++n) {
#pragma unroll
            for (int r = 0; r < 4; ++r) most = fmaxf(most, fabsf(s[n][r]));
        }
        most = MaxOver32(MaxOver16(most));
        const bool over = most >= 0x1p15f && most < HUGE_VALF;
        if (__any(over)) {
            const int up = over ? min(ExponentOf(most) - 13, 114 - unit) : 0;
            unit += up;
            most *= Power(-up);
#pragma unroll
            for (int n = 0; n < NS; ++n) s[n] *= Power(-up);
        }
    };
    const auto keep_state = [&] {
        if (lane / 16 == 0) scales[state_col()] = Power(unit);
#pragma unroll
        for (int n = 0; n < NS; ++n) {
            const float v[4] = {s[n][0], s[n][1], s[n][2], s[n][3]};
            attend_half4_t hi, lo;
            Split<4>(v, minus, &hi, &lo);
            const int at = state_col() * Lds::kStatePitch + state_row(n, 0) * 2;
            *reinterpret_cast<attend_half4_t*>(high_copy + at) = hi;
            *reinterpret_cast<attend_half4_t*>(low_copy + at) = lo;
        }
    };
    if (OUT) {
        if (run.start.data != nullptr) states_at(run.start, s);
        find_most();
        if (most > 0 && most < 0x1p4f) {
            const int down = max(ExponentOf(most) - 13, -112);
            unit = down;
            most *= Power(-down);
#pragma unroll
            for (int n = 0; n < NS; ++n) s[n] *= Power(-down);
        }
        keep_state();
    }

    // A tile's rows on their way: pieces of eight elements of k and of v.  Rows that are not there are the last one again; columns that are not there are zeros that stay in LDS.  Rows lie less
    // than 2^24 elements apart, so that a tile's are within 32 bits of its first.
    const int key_row = tid / (KD / 8), key_col = tid % (KD / 8) * 8, value_row = tid / (VB / 8), value_col = tid % (VB / 8) * 8;
    const auto own_row = [&] { return 16 * wave + lane % 16; };  // of a tile
    const int way = back ? -1 : 1;
    const int64_t row0 = back ? span.end - 1 : span.first;
    const T* kp = static_cast<const T*>(run.k.data) + b * run.k.batch + (h / run.k.share) * run.k.head + row0 * run.k.row;
    const T* vp = static_cast<const T*>(run.v.data) + b * run.v.batch + (h / run.v.share) * run.v.head + row0 * run.v.row + col0;
    const T* qp = OUT ? static_cast<const T*>(run.q.data) + b * run.q.batch + (h / run.q.share) * run.q.head + row0 * run.q.row : nullptr;
    const int k_row = way * static_cast<int>(run.k.row), v_row = way * static_cast<int>(run.v.row), q_row = OUT ? way * static_cast<int>(run.q.row) : 0;
    // of y and the rows that its products are wanted with, too
    char* yp = OUT ? static_cast<char*>(run.y.data) + (b * run.y.batch + h * run.y.head + row0 * run.y.row + col0) * (wide ? 4 : 2) : nullptr;
    const int y_row = OUT ? way * static_cast<int>(run.y.row) * (wide ? 4 : 2) : 0;
    const T* dp = with_dots ? static_cast<const T*>(run.dot.data) + b * run.dot.batch + (h / run.dot.share) * run.dot.head + row0 * run.dot.row + col0 : nullptr;
    const int d_row = with_dots ? way * static_cast<int>(run.dot.row) : 0;
    const float* gp = p.decay != nullptr ? p.decay + b * p.decay_batch + h * p.decay_head : nullptr;
    const int64_t g_rows = AttendNoDecay(span.end, length, back);
    AttendPiece<T, 8> k_next[NK], v_next[NV], q_next[OUT ? NQ : 1];
    const auto placed = [&](const AttendPiece<T, 8>& piece, int col, int end) {  // (where all pieces are whole, zeros behind the columns stay in LDS and in the state)
        return __builtin_bit_cast(attend_half8_t, EVEN ? piece : AttendPlace<WIDTHS>(piece, col, end));
    };
    // (Behind the last tile every row is the last one: a branch round the loads would have those of the tile before, too, waited for where the two ways meet.)
    const auto load = [&](int64_t r0) {  // k and v; at the tile's first row
        const int last = static_cast<int>(rows - r0 < C ? rows - r0 : C) - 1;
#pragma unroll
        for (int n = 0; n < NK; ++n) k_next[n] = AttendFetch<WIDTHS, 8>(kp + min(key_row + n * (2048 / KD), last) * k_row, key_col, keys);
#pragma unroll
        for (int n = 0; n < NV; ++n) v_next[n] = AttendFetch<WIDTHS, 8>(vp + min(value_row + n * 32, last) * v_row, value_col, cols);
        kp += static_cast<int64_t>(k_row) * C, vp += static_cast<int64_t>(v_row) * C;
    };
    const auto load_q = [&](int64_t r0) {
        if constexpr (OUT) {
            const T* const at = qp + min(own_row(), static_cast<int>(rows - r0 < C ? rows - r0 : C) - 1) * q_row;
#pragma unroll
            for (int m = 0; m < NQ; ++m) q_next[m] = AttendFetch<WIDTHS, 8>(at, 32 * m + lane / 16 * 8, keys);
            qp += static_cast<int64_t>(q_row) * C;
        }
    };
    // Log decays, by one wave, a lane to a row: summed up a tile ahead, on their way two tiles ahead, so that nothing waits for what was asked for in the same tile.
    float g_now = 0, g_next = 0;
    const auto decay_at = [&](int64_t r) { return gp[AttendDecayRow(span.first, span.end, length, back, r) * p.decay_row]; };
    const auto load_decays = [&](int64_t r0) {  // of a row that is there; sum_decays takes those that count
        if (gp != nullptr) g_next = decay_at(r0 + lane);
    };
    const auto sum_decays = [&](int64_t r0, AttendHalfDecays* to) {
        const int here = static_cast<int>(rows - r0 < C ? rows - r0 : C);
        const double sum = SumDecays(to, gp != nullptr && lane < here && r0 + lane >= g_rows ? LogOfDecay(g_now) : 0, here, kv_scale);
        if (OUT) {
            to->near[lane] = __builtin_amdgcn_exp2f(static_cast<float>(OfLaneInRow<15>(sum) - sum));
            to->own[lane] = static_cast<float>(sum - static_cast<float>(sum));
        }
    };
    if (EVEN) {
#pragma unroll
        for (int n = 0; n < NK; ++n) {
            if (key_col >= keys) *reinterpret_cast<attend_half8_t*>(ks + (key_row + n * (2048 / KD)) * Lds::kKeyPitch + key_col * 2) = attend_half8_t{};
        }
#pragma unroll
        for (int n = 0; n < NV; ++n) {
            if (value_col >= cols) *reinterpret_cast<attend_half8_t*>(vs + (value_row + n * 32) * Lds::kValuePitch + value_col * 2) = attend_half8_t{};
        }
    }
    if (tid == 0) odd[0] = odd[1] = odd[2] = odd[3] = 0;
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
    double passed = 0;  // log decay of the tiles so far
    int turn = 0;
    int64_t r0 = 0;
    __syncthreads();  // the flags
    for (; r0 < rows; r0 += C, turn ^= 1) {
        asm volatile("" : "+v"(lane));
        asm volatile("" : "+s"(keys));
        AttendHalfDecays* const dec = decays + turn;
        // (the last tile's rows of k and v have been read by all)
#pragma unroll
        for (int n = 0; n < NK; ++n) {
            if (!EVEN || key_col < keys) *reinterpret_cast<attend_half8_t*>(ks + (key_row + n * (2048 / KD)) * Lds::kKeyPitch + key_col * 2) = placed(k_next[n], key_col, keys);
        }
        attend_half2_t finite{};  // 0, or not a number
#pragma unroll
        for (int n = 0; n < NV; ++n) {
            const attend_half8_t v = placed(v_next[n], value_col, cols);
            if (!EVEN || value_col < cols) *reinterpret_cast<attend_half8_t*>(vs + (value_row + n * 32) * Lds::kValuePitch + value_col * 2) = v;
#pragma unroll
            for (int e = 0; e < 8; e += 2) finite = __builtin_elementwise_fma(attend_half2_t{v[e], v[e + 1]}, attend_half2_t{}, finite);
        }
        // Rows of zeros: what they are multiplied with, which a mask may have left as it was, is not to decide the power of two that the others are counted in.
        const auto leave_out_zeros = [&] {
            int thread = tid;
            asm volatile("" : "+v"(thread));
            const auto zeros = [&](const AttendPiece<T, 8>& piece, int lanes) {  // of `lanes` neighbours, whose pieces are a row
                return (__ballot(!IsZeros(piece)) >> (thread % 64 & -lanes) & (~uint64_t{0} >> (64 - lanes))) == 0;
            };
#pragma unroll
            for (int n = 0; n < NK; ++n) {
                if (zeros(k_next[n], KD / 8)) dec->end[thread / (KD / 8) + n * (2048 / KD)] = 0;
            }
#pragma unroll
            for (int n = 0; n < (OUT ? NV : 0); ++n) {
                const int row = thread / (VB / 8) + n * 32;
                if (zeros(v_next[n], VB / 8)) dec->near[row] = 0, dec->own[row] = HUGE_VALF;
            }
        };
        float least = LeastOf(k_next, 1.f);
        if (OUT) least = LeastOf(v_next, least);
        const bool bad = OUT && !(finite[0] + finite[1] == 0), empty = !(least >= 0x1p-126f);
        if (OUT) {
            if (bad || empty) odd[2 * turn + (bad ? 0 : 1)] = 1;
        } else if (__builtin_expect(__any(empty), 0)) {
            leave_out_zeros();
        }
        __syncthreads();
        passed += dec->sum;
        if (OUT) {
            const int any_bad = __builtin_amdgcn_readfirstlane(odd[2 * turn]), any_empty = __builtin_amdgcn_readfirstlane(odd[2 * turn + 1]);
            if (__builtin_expect((any_bad | any_empty) != 0, 0)) {
                // An infinity of a later row, times P's zeros, would reach earlier ones: the rest goes row by row.
                if (any_bad != 0) break;
                leave_out_zeros();
                __syncthreads();
            }
        }
        const bool more = r0 + C < rows;
        g_now = g_next;
        load(r0 + C);
        if (wave == 0) load_decays(r0 + 2 * C);  // (behind the others: what waits for them must not wait for this one)
        // This wave's columns of v times their rows' weights, in two parts of the unit that the state will have, and the state in that unit: in pieces, which go between the products with the state.
        const int block = lane / 16 * 4 + lane % 16 / 4, piece = lane % 4 * 8;
        attend_half8_t of_v[2], hi[2], lo[2];
        attend4_t end[2][2];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const char* const from = vs + (block + 32 * u) * Lds::kValuePitch + 32 * wave + piece;
            of_v[u] = Join(ReadTurned(from), ReadTurned(from + 16 * Lds::kValuePitch));
#pragma unroll
            for (int g = 0; g < 2; ++g) end[u][g] = *reinterpret_cast<const attend4_t*>(dec->end + 32 * u + 16 * g + lane / 16 * 4);
        }
        float w[2][8], largest_v = 0, keep = 1, in = 1;
        const float all = dec->all;
        constexpr int kPieces = 7;
        const auto prepare = [&](int at) {
            if (at < 2) {
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    w[at][e] = __builtin_fmaf(static_cast<float>(of_v[at][e]), end[at][e / 4][e % 4], 0.f);
                    largest_v = fmaxf(largest_v, fabsf(w[at][e]));
                }
            } else if (at == 2) {
                // (in exponents: what is added may be further from the unit than a float reaches)
                const float decayed = most * all, added = MaxOver32(MaxOver16(largest_v));
                const int size = max(decayed < HUGE_VALF ? ExponentOf(decayed) : -127, added > 0 ? ExponentOf(added) - unit : -127);
                int up = 0;
                if (size >= 15 || (size < 4 && size > -127)) up = min(max(max(size - 13, -112 - unit), -112), 114 - unit);
                unit += up;
                keep = all * Power(max(-up, -126)), in = Power(-unit);
            } else if (at < 5) {
#pragma unroll
                for (int n = (at - 3) * (NS / 2); n < (at - 2) * (NS / 2); ++n) s[n] *= keep;
            } else {
#pragma unroll
                for (int e = 0; e < 8; ++e) w[at - 5][e] *= in;
                Split<8>(w[at - 5], minus, &hi[at - 5], &lo[at - 5]);
            }
        };
        const int here = static_cast<int>(rows - r0 < C ? rows - r0 : C);
        if (!OUT || 16 * wave >= here) {
#pragma unroll
            for (int i = 0; i < kPieces; ++i) prepare(i);
        } else if constexpr (OUT) {
            // this wave's sixteen rows by all columns, in blocks of 16 x 16
            const int quarter = lane / 16;
            const float high = dec->high[own_row()], low = dec->low[own_row()];
            attend_half8_t q[NQ];
#pragma unroll
            for (int m = 0; m < NQ; ++m) q[m] = placed(q_next[m], 32 * m + 8 * quarter, keys);
            attend4_t y[DB];
            {
                attend4_t of_state[DB]{};
                const int at = lane % 16 * Lds::kStatePitch + 16 * quarter;
                attend_half8_t part[2][DB];
                const auto read = [&](int step, attend_half8_t (&to)[DB]) {  // step 2 m: the low parts, 2 m + 1: the high ones
                    const char* const from = (step % 2 == 0 ? low_copy : high_copy) + at + 64 * (step / 2);
#pragma unroll
                    for (int d = 0; d < DB; ++d) to[d] = *reinterpret_cast<const attend_half8_t*>(from + 16 * d * Lds::kStatePitch);
                };
                read(0, part[0]);
#pragma unroll
                for (int step = 0; step < 2 * NQ; ++step) {  // reads of the next step under the products of this one
                    if (step + 1 < 2 * NQ) read(step + 1, part[step % 2 ^ 1]);
#pragma unroll
                    for (int d = 0; d < DB; ++d) of_state[d] = Mfma(part[step % 2][d], q[step / 2], of_state[d]);
#pragma unroll
                    for (int i = 0; i < kPieces; ++i) {
                        if (i * (2 * NQ) / kPieces == step) prepare(i);
                    }
                    __builtin_amdgcn_sched_barrier(0);
                }
                const float from_start = __builtin_amdgcn_exp2f(high + low) * run.out_scale;
#pragma unroll
                for (int d = 0; d < DB; ++d) {
                    const attend4_t units = *reinterpret_cast<const attend4_t*>(scales + 16 * d + 4 * quarter);
#pragma unroll
                    for (int e = 0; e < 4; ++e) y[d][e] = of_state[d][e] * units[e] * from_start;
                }
            }
            __builtin_amdgcn_sched_barrier(0);  // (the products with the state need as many registers as those with k)
            attend4_t a[4]{};
            {
                const char* const at = ks + lane % 16 * Lds::kKeyPitch + 16 * quarter;
                attend_half8_t part[2][NQ];
                const auto read = [&](int sb, attend_half8_t (&to)[NQ]) {
#pragma unroll
                    for (int m = 0; m < NQ; ++m) to[m] = *reinterpret_cast<const attend_half8_t*>(at + 16 * sb * Lds::kKeyPitch + 64 * m);
                };
                read(0, part[0]);
#pragma unroll
                for (int sb = 0; sb < 4; ++sb) {
                    if (sb > wave) continue;
                    if (sb < 3) read(sb + 1, part[sb % 2 ^ 1]);  // (of the last one, of no use)
#pragma unroll
                    for (int m = 0; m < NQ; ++m) a[sb] = Mfma(part[sb % 2][m], q[m], a[sb]);
                    __builtin_amdgcn_sched_barrier(0);
                }
            }
            if (wave == 0 && more) sum_decays(r0 + C, decays + (turn ^ 1));
            if (tid == 0) odd[2 * (turn ^ 1)] = odd[2 * (turn ^ 1) + 1] = 0;
            // weights: of the sixteen rows that this one is among, exp(G[t] - G[s]); of earlier ones, whose last is l, exp(G[l] - G[s]) here and exp(G[t] - G[l]) with the power of two
            float largest = 0, since[4];
#pragma unroll
            for (int sb = 0; sb < 4; ++sb) {
                if (sb > wave) continue;
                const int first = 16 * sb + 4 * quarter;
                if (sb == wave) {
                    const attend4_t highs = *reinterpret_cast<const attend4_t*>(dec->high + first), owns = *reinterpret_cast<const attend4_t*>(dec->own + first);
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const float weighted = a[sb][e] * __builtin_amdgcn_exp2f((high - highs[e]) + (low - owns[e]));
                        a[sb][e] = 4 * quarter + e <= lane % 16 ? weighted : 0.f;
                    }
                    since[sb] = 1;
                } else {
                    const attend4_t near = *reinterpret_cast<const attend4_t*>(dec->near + first);
#pragma unroll
                    for (int e = 0; e < 4; ++e) a[sb][e] *= near[e];
                    since[sb] = __builtin_amdgcn_exp2f((high - dec->high[16 * sb + 15]) + (low - dec->low[16 * sb + 15]));
                }
                largest = fmaxf(largest, fmaxf(fmaxf(fabsf(a[sb][0]), fabsf(a[sb][1])), fmaxf(fabsf(a[sb][2]), fabsf(a[sb][3]))) * since[sb]);
            }
            const Scale scale(MaxOver32(MaxOver16(largest)));
            attend4_t of_rows[DB]{};
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                if (2 * u > wave) continue;
                float weights[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) weights[e] = 2 * u + e / 4 <= wave ? a[2 * u + e / 4][e % 4] * (since[2 * u + e / 4] * scale.in) : 0.f;
                attend_half8_t p_hi, p_lo;
                Split<8>(weights, minus, &p_hi, &p_lo);
                const char* const at = vs + (32 * u + 4 * quarter + lane % 16 / 4) * Lds::kValuePitch + lane % 4 * 8;
                attend_half8_t v[DB];
#pragma unroll
                for (int d = 0; d < DB; ++d) v[d] = Join(ReadTurned(at + 32 * d), ReadTurned(at + 16 * Lds::kValuePitch + 32 * d));
#pragma unroll
                for (int d = 0; d < DB; ++d) of_rows[d] = Mfma(v[d], p_lo, of_rows[d]);
#pragma unroll
                for (int d = 0; d < DB; ++d) of_rows[d] = Mfma(v[d], p_hi, of_rows[d]);
            }
            const float from_rows = scale.out * kv_scale * run.out_scale;
            char* const to = yp + static_cast<int64_t>(own_row()) * y_row;
            const bool live = r0 + own_row() < rows;
            float dot = 0;
#pragma unroll
            for (int d = 0; d < DB; ++d) {
                const int j = 16 * d + 4 * quarter;
                AttendPiece<float, 4> out;
#pragma unroll
                for (int e = 0; e < 4; ++e) out.v[e] = __builtin_fmaf(of_rows[d][e], from_rows, y[d][e]);
                if (!live) continue;
                if (with_dots) {
                    const AttendPiece<T, 4> with = AttendPlace<WIDTHS>(AttendFetch<WIDTHS, 4>(dp + static_cast<int64_t>(own_row()) * d_row, j, cols), j, cols);
#pragma unroll
                    for (int e = 0; e < 4; ++e) dot += j + e < cols ? out.v[e] * static_cast<float>(with.v[e]) : 0.f;
                }
                if (EVEN ? j < cols : j + 4 <= cols) {
                    if (wide) {
                        *reinterpret_cast<AttendPiece<float, 4>*>(to + j * 4) = out;
                    } else {
                        AttendPiece<T, 4> o;
#pragma unroll
                        for (int e = 0; e < 4; ++e) o.v[e] = static_cast<T>(out.v[e]);
                        *reinterpret_cast<AttendPiece<T, 4>*>(to + j * 2) = o;
                    }
                } else if (!EVEN) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        if (j + e >= cols) continue;
                        if (wide) reinterpret_cast<float*>(to)[j + e] = out.v[e];
                        else reinterpret_cast<T*>(to)[j + e] = static_cast<T>(out.v[e]);
                    }
                }
            }
            if (with_dots) {
                dot += __shfl_xor(dot, 16);
                dot += __shfl_xor(dot, 32);
                if (quarter == 0 && live) dots()[row0 + way * (r0 + own_row())] = dot;
                dp += static_cast<int64_t>(d_row) * C;
            }
            yp += static_cast<int64_t>(y_row) * C;
        }
        if (!OUT && wave == 0 && more) sum_decays(r0 + C, decays + (turn ^ 1));
        __builtin_amdgcn_sched_barrier(0);
        load_q(r0 + C);
        {
            const char* const at = ks + block * Lds::kKeyPitch + piece;
            attend_half8_t k[2][NS / 2];
            const auto read = [&](int step, attend_half8_t (&to)[NS / 2]) {  // half of the keys of 32 rows
#pragma unroll
                for (int n = 0; n < NS / 2; ++n) {
                    const char* const row = at + 32 * (step / 2) * Lds::kKeyPitch + 32 * (step % 2 * (NS / 2) + n);
                    to[n] = Join(ReadTurned(row), ReadTurned(row + 16 * Lds::kKeyPitch));
                }
            };
            read(0, k[0]);
#pragma unroll
            for (int step = 0; step < 4; ++step) {
                if (step == 2 && here <= 32) break;
                if (step + 1 < 4) read(step + 1, k[step % 2 ^ 1]);
#pragma unroll
                for (int n = 0; n < NS / 2; ++n) s[step % 2 * (NS / 2) + n] = Mfma(k[step % 2][n], lo[step / 2], s[step % 2 * (NS / 2) + n]);
#pragma unroll
                for (int n = 0; n < NS / 2; ++n) s[step % 2 * (NS / 2) + n] = Mfma(k[step % 2][n], hi[step / 2], s[step % 2 * (NS / 2) + n]);
                __builtin_amdgcn_sched_barrier(0);
            }
        }
        find_most();
        __syncthreads();  // the copies of the state, and the rows of k and v, have been read
        if (OUT) keep_state();
    }

    if (OUT && r0 < rows) {
        // row by row, on a copy of the state in 32 bits in the place of the others
        float* const ss = reinterpret_cast<float*>(high_copy);  // [KD][VB]
#pragma unroll
        for (int n = 0; n < NS; ++n) {
#pragma unroll
            for (int r = 0; r < 4; ++r) ss[state_row(n, r) * VB + state_col()] = s[n][r] * Power(unit);
        }
        __syncthreads();
        const int j = lane;
        for (; r0 < rows; ++r0) {
            const int64_t row = row0 + way * r0;
            const T* const k = static_cast<const T*>(run.k.data) + b * run.k.batch + (h / run.k.share) * run.k.head + row * run.k.row;
            const T* const x = static_cast<const T*>(run.q.data) + b * run.q.batch + (h / run.q.share) * run.q.head + row * run.q.row;
            const T* const of_v = static_cast<const T*>(run.v.data) + b * run.v.batch + (h / run.v.share) * run.v.head + row * run.v.row + col0;
            const float step = gp != nullptr && r0 >= g_rows ? __builtin_amdgcn_exp2f(static_cast<float>(LogOfDecay(decay_at(r0)))) : 1.f, v = j < cols ? static_cast<float>(of_v[j]) * kv_scale : 0.f;
            float y = 0;
            for (int i = wave * (KD / 4); i < (wave + 1) * (KD / 4) && i < keys; ++i) {
                const float now = ss[i * VB + j] * step + static_cast<float>(k[i]) * v;
                ss[i * VB + j] = now;
                y += static_cast<float>(x[i]) * now;
            }
            sums[wave * VB + j] = y;
            __syncthreads();
            if (wave == 0) {
                y = (sums[j] + sums[VB + j] + sums[2 * VB + j] + sums[3 * VB + j]) * run.out_scale;
                const int64_t to = b * run.y.batch + h * run.y.head + row * run.y.row + col0 + j;
                if (j < cols) {
                    if (wide) static_cast<float*>(run.y.data)[to] = y;
                    else static_cast<T*>(run.y.data)[to] = static_cast<T>(y);
                }
                if (with_dots) {
                    float dot = 0;
                    if (j < cols) dot = y * static_cast<float>((static_cast<const T*>(run.dot.data) + b * run.dot.batch + (h / run.dot.share) * run.dot.head + row * run.dot.row + col0)[j]);
#pragma unroll
                    for (int o = 1; o < 64; o <<= 1) dot += __shfl_xor(dot, o);
                    if (lane == 0) dots()[row] = dot;
                }
            }
            __syncthreads();
        }
#pragma unroll
        for (int n = 0; n < NS; ++n) {
#pragma unroll
            for (int r = 0; r < 4; ++r) s[n][r] = ss[state_row(n, r) * VB + state_col()];
        }
        unit = 0;
    }
    if constexpr (!OUT) {
        float* const to = run.last.data + bh * run.last.head + segment * run.last.segment;
#pragma unroll
        for (int n = 0; n < NS; ++n) {
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int i = state_row(n, r);
                if (i < keys && state_col() < cols) to[i * run.last.i + (col0 + state_col()) * run.last.j] = s[n][r] * Power(unit);
            }
        }
        if (tid == 0 && block == run.first) run.decays[static_cast<int64_t>(bh) * p.segments + segment] = __builtin_amdgcn_exp2f(static_cast<float>(passed));
        return;
    }
    // rows behind the sequence's end
    for (int64_t row = (span.end > span.first ? span.end : span.first) + wave; row < span.whole; row += 4) {
        if (lane >= cols) continue;
        const int64_t to = b * run.y.batch + h * run.y.head + row * run.y.row + col0 + lane;
        if (wide) static_cast<float*>(run.y.data)[to] = 0.f;
        else static_cast<T*>(run.y.data)[to] = static_cast<T>(0);
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
                for (int r = 0; r < 4; ++r) dot += state_row(n, r) < keys && state_col() < cols ? s[n][r] * Power(unit) * other[n][r] : 0.f;
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
                if (i < keys && state_col() < cols) to[i * run.last.i + (col0 + state_col()) * run.last.j] = s[n][r] * Power(unit) * more;
            }
        }
    }
}

}  // namespace

void LaunchAttendHalf(const AttendArgs& p, int keys, int64_t blocks, bool states_alone, hipStream_t stream) {
    const AttendWidths widths = AttendWidthsOf(p, 8);
    const auto launch = [&](auto kd) {
        const auto kernel = [&](auto out, auto rows, auto grad) {
            constexpr int KD = decltype(kd)::value, kLds = AttendHalfLds<KD, decltype(out)::value>::kBytes;
            void (*const k)(AttendArgs) = AttendHalfKernel<KD, decltype(out)::value, decltype(rows)::value, decltype(grad)::value>;
            struct Tag {};  // a type of its own for every instantiation of this lambda
            EnsureDynamicLds<Tag>(reinterpret_cast<const void*>(k), kLds);
            hipLaunchKernelGGL(k, dim3(static_cast<unsigned>(blocks)), dim3(256), kLds, stream, p);
            CheckLaunch("linear_attention");
        };
        VisitWidths(widths, p.runs > 1, [&](auto rows, auto grad) { states_alone ? kernel(std::false_type{}, rows, grad) : kernel(std::true_type{}, rows, grad); });
    };
    if (keys <= 64) launch(std::integral_constant<int, 64>{});
    else if (keys <= 128) launch(std::integral_constant<int, 128>{});
    else launch(std::integral_constant<int, 256>{});
}

}  // namespace hipcx
