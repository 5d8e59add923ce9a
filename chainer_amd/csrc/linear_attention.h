// What linear attention and its gradients share.
//   S[t] = exp(g[t]) S[t-1] + k[t] v[t]^T,  y[t] = scale q[t] S[t]
// for every sequence and head, S being a matrix [keys, values] and g the logarithm of the decay.
//
// The gradients are passes of the same form with the arrays in other places, two of them from the last row to the first:
//   gq = scale S gy         is the pass of (gy, v, k) over the states' transposes,
//   R[t] = exp(g[t+1]) R[t+1] + scale q[t] gy[t]^T,  gk = R v, gv = R^T k  are passes backwards of (v, gy, q) and (k, q, gy),
//   gg[t] = <exp(g[t]) S[t-1], R[t]> = sum over u >= t of (q[u] gq[u] - k[u] gk[u]) and what the rows behind have of it.
// So one kernel does all of them (AttendRun).
#pragma once

#include "attend_decay_row.h"
#include "sequence.h"

namespace hipcx {

// Rows of [batch, time, head, element] whose last axis is dense; strides in elements.  `share` neighbouring heads read one.
struct AttendRows {
    void* data;
    int64_t batch, row, head;
    int share;
};

// Matrices [batch and head][segment][i][j]; strides in elements.
struct AttendStates {
    float* data;  // null: zeros, or not asked for
    int64_t head, segment, i, j;
};

// One pass: y[t] = out_scale sum over s of weight(t, s) kv_scale (q[t] k[s]) v[s] and the state that a segment begins with.
struct AttendRun {
    AttendRows q, k, v, y;
    AttendRows dot;        // rows like y's, whose products with y are wanted
    float* dots;           // [batch][head][blocks][length], or null
    AttendStates start, last;
    AttendStates other;    // the state's gradients behind each segment, whose products with the state there are wanted
    float* ends;           // [batch][head][segment][blocks], or null
    float* decays;         // [batch][head][segment]: a segment's own, of states alone
    float kv_scale, out_scale;
    int keys, values;      // extents of q and k, and of v and y
    int first, blocks;     // of kAttendColumns columns of v
    int back;              // from the last row to the first; the state decays by the row that follows
    int wide;              // y is float32
    int decay_last;        // `last` takes the first row's decay too
};

struct AttendArgs {
    AttendRun run[3];
    int runs, blocks;      // blocks of all runs
    const float* decay;    // null: none
    int64_t decay_batch, decay_row, decay_head;
    SequenceLengths lengths;
    int64_t batch, length, segment_rows;
    int heads, segments;
    int groups;            // of workgroups, all blocks of one head's segment, and the launch holds them eight times, rounded up
};

// The workgroup's number among those that have work, or -1: workgroups go to the eight chips in turn, and the blocks of a head's segment, which read the same rows, belong on one.
__device__ __forceinline__ int AttendNumber(const AttendArgs& p) {
    const int chip = static_cast<int>(blockIdx.x % 8), turn = static_cast<int>(blockIdx.x / 8), group = turn / p.blocks * 8 + chip;
    return group < p.groups ? group * p.blocks + turn % p.blocks : -1;
}

constexpr int kAttendTile = 64;      // rows that are taken at once
constexpr int kAttendColumns = 64;   // columns of v to a workgroup
constexpr int kMaxAttend = 256;      // keys, values

typedef float attend4_t __attribute__((ext_vector_type(4)));

template <typename T, int N>
struct __attribute__((packed, aligned(alignof(T)))) AttendPiece {
    T v[N];
};

// How the rows of a pass fall into pieces of 16 bytes: all whole; the last one not; rows of less than a piece.
enum AttendWidths { kAttendWhole, kAttendPart, kAttendNarrow };

// N elements of a row, a piece or less, without a branch, so that the loads of many are under way together: AttendFetch has them, from the row's end back where they reach over the end (a block of
// columns has at least one and may have others in front of it: where the row has a whole piece, so has what ends at its end), and AttendPlace brings them to their places when they are used.
template <int WIDTHS, int N, typename T>
__device__ __forceinline__ AttendPiece<T, N> AttendFetch(const T* row, int at, int end) {
    if constexpr (WIDTHS == kAttendNarrow) {
        AttendPiece<T, N> r;
#pragma unroll
        for (int e = 0; e < N; ++e) r.v[e] = row[min(at + e, end - 1)];
        return r;
    } else {
        return *reinterpret_cast<const AttendPiece<T, N>*>(row + (WIDTHS == kAttendWhole ? (at < end ? at : 0) : min(at, end - N)));
    }
}
template <int WIDTHS, typename T, int N>
__device__ __forceinline__ AttendPiece<T, N> AttendPlace(AttendPiece<T, N> r, int at, int end) {
    constexpr int one = 4 / sizeof(T), R = N / one;
    typedef uint32_t registers_t __attribute__((ext_vector_type(R)));
    registers_t d = __builtin_bit_cast(registers_t, r);
    if constexpr (WIDTHS == kAttendPart) {
        const int back = max(0, at + N - end);
        if constexpr (sizeof(T) == 2) {
#pragma unroll
            for (int i = 0; i < R; ++i) d[i] = back & 1 ? d[i] >> 16 | (i + 1 < R ? d[i + 1] << 16 : 0u) : d[i];
        }
#pragma unroll
        for (int step = 1; step < R; step *= 2) {
#pragma unroll
            for (int i = 0; i < R; ++i) d[i] = back & (step * one) ? (i + step < R ? d[i + step] : 0u) : d[i];
        }
    }
    if constexpr (WIDTHS == kAttendNarrow) {
        r = __builtin_bit_cast(AttendPiece<T, N>, d);
#pragma unroll
        for (int e = 0; e < N; ++e) r.v[e] = at + e < end ? r.v[e] : static_cast<T>(0);
        return r;
    }
#pragma unroll
    for (int i = 0; i < R; ++i) d[i] = at < end ? d[i] : 0u;
    return __builtin_bit_cast(AttendPiece<T, N>, d);
}

// A log decay in powers of two.  -infinity, a state that ends, is held at a number that no product of decays brings back.
__device__ __forceinline__ double LogOfDecay(float decay) {
    const double g = static_cast<double>(decay) * 1.4426950408889634;
    return g < -0x1p20 ? -0x1p20 : g;
}
// The one that takes the state to row t of a pass.
__device__ __forceinline__ double AttendDecay(const AttendArgs& p, int64_t b, int h, int64_t t) {
    return p.decay != nullptr ? LogOfDecay(p.decay[b * p.decay_batch + t * p.decay_row + h * p.decay_head]) : 0;
}

// The decays of a tile's rows, summed up from its first: as a float and what the float leaves out, so that differences are as good as a float's for any sum.
struct AttendDecays {
    alignas(16) float high[kAttendTile], low[kAttendTile];
    float end[kAttendTile];  // from a row to the tile's end, as a factor, times kv_scale
    float all;               // the tile's
    double sum;              // the tile's, in powers of two
};

__device__ __forceinline__ double ShflUpDouble(double v, int o) {
    const uint64_t b = __builtin_bit_cast(uint64_t, v);
    const uint32_t lo = __shfl_up(static_cast<uint32_t>(b), o), hi = __shfl_up(static_cast<uint32_t>(b >> 32), o);
    return __builtin_bit_cast(double, static_cast<uint64_t>(hi) << 32 | lo);
}
__device__ __forceinline__ double ShflDouble(double v, int lane) {
    const uint64_t b = __builtin_bit_cast(uint64_t, v);
    const uint32_t lo = __shfl(static_cast<uint32_t>(b), lane), hi = __shfl(static_cast<uint32_t>(b >> 32), lane);
    return __builtin_bit_cast(double, static_cast<uint64_t>(hi) << 32 | lo);
}

// Adds the value that a DPP move brings from another lane of the rows in ROWS, nothing elsewhere.
template <int MOVE, int ROWS>
__device__ __forceinline__ double AddMoved(double v) {
    const uint64_t b = __builtin_bit_cast(uint64_t, v);
    const uint32_t lo = __builtin_amdgcn_update_dpp(0, static_cast<int>(b), MOVE, ROWS, 0xf, false), hi = __builtin_amdgcn_update_dpp(0, static_cast<int>(b >> 32), MOVE, ROWS, 0xf, false);
    return v + __builtin_bit_cast(double, static_cast<uint64_t>(hi) << 32 | lo);
}

// By one wave, a lane to a row, of which `here` are there; g in powers of two, 0 for the others.  Returns the sum up to the lane's row.
__device__ __forceinline__ double SumDecays(AttendDecays* to, double g, int here, float kv_scale) {
    const int lane = threadIdx.x % 64;
    double sum = AddMoved<0x111, 0xf>(g);  // from 1, 2, 4 and 8 lanes before in the row of 16, then from the rows' last lanes
    sum = AddMoved<0x112, 0xf>(sum);
    sum = AddMoved<0x114, 0xf>(sum);
    sum = AddMoved<0x118, 0xf>(sum);
    sum = AddMoved<0x142, 0xa>(sum);
    sum = AddMoved<0x143, 0xc>(sum);
    const uint64_t b = __builtin_bit_cast(uint64_t, sum);
    const double all = __builtin_bit_cast(double, static_cast<uint64_t>(static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(b >> 32), 63))) << 32 |
                                                      static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(b), 63)));
    const float high = static_cast<float>(sum);
    to->high[lane] = high, to->low[lane] = static_cast<float>(sum - high);
    to->end[lane] = lane < here ? __builtin_amdgcn_exp2f(static_cast<float>(all - sum)) * kv_scale : 0.f;
    if (lane == 0) to->all = __builtin_amdgcn_exp2f(static_cast<float>(all)), to->sum = all;
    return sum;
}

// Rows of a segment: [first, end) of the sequence's.
struct AttendSpan {
    int64_t first, end, whole;  // whole: the end of the segment's rows in the padded batch
    __device__ __forceinline__ AttendSpan(const AttendArgs& p, int64_t length, int segment) {
        first = segment * p.segment_rows;
        whole = first + p.segment_rows < p.length ? first + p.segment_rows : p.length;
        end = whole < length ? whole : length;
        end = end < first ? first : end;
    }
};

// How the time axis is cut: into segments of whole tiles, two at least, of the number that costs least.  Costs are in a tile's time with the compute units full (`resident` workgroups to each):
// a round of workgroups takes a segment's tiles and three more for what comes before and behind them, 0.85 of that where there is a workgroup to a compute unit at most
// and between them in proportion; segments need the states that they start from first, which takes 0.4 of a tile each, and a pass over the states.  Of a padded batch half of the workgroups are taken to have work.
// `blocks`: workgroups to a head and segment; `states`: those of the states alone.
// One sequence of 16384 rows, 16 heads of 128 x 128 in float16, in 8, 16, 24 and 48 segments: 179, 141, 154 and 170 us, and 16 are taken; 20 padded ones of up to 777, 13 heads of 50 x 50 in
// float32, in 1, 2 and 3: 114, 110 and 95, and 3 are taken; 9 of 2533, 11 heads of 100 x 100 in float16, in 1, 2, 5 and 8: 186, 178, 161 and 179, and 5 are taken.
// float32 with up to 64 keys, cut for three workgroups to a compute unit where two fit, and for two: forward pass of 4 x 2048 rows of 8 heads 61 and 53 us, gradients of one sequence of 5000 rows of 10
// heads 127 and 115, of 2 x 3868 rows, 14 heads of 16 keys and 80 values, 331 and 298.
inline void CutAttend(AttendArgs* p, bool padded, int64_t blocks, int64_t states, int64_t resident, int64_t matrix) {
    const int64_t tiles = (p->length + kAttendTile - 1) / kAttendTile, heads = p->batch * p->heads, units = NumCUs();
    constexpr double alone = 0.85;
    const auto rounds = [&](int64_t workgroups, int64_t at_once) {
        if (padded) workgroups = (workgroups + 1) / 2;
        const int64_t rest = workgroups % at_once;
        const double part = at_once > units ? alone + (1 - alone) * static_cast<double>(std::max<int64_t>(0, rest - units)) / static_cast<double>(at_once - units) : 1;
        return static_cast<double>(workgroups / at_once) + (rest == 0 ? 0 : part);
    };
    int64_t best = 1;
    double least = 0;
    for (int64_t n = 1; n <= std::max<int64_t>(1, std::min<int64_t>(tiles / 2, 64)); ++n) {
        const int64_t each = (tiles + n - 1) / n;
        double cost = rounds(heads * blocks * n, units * resident) * static_cast<double>(each + 3);
        if (n > 1) cost += rounds(heads * states * (n - 1), units * 4) * (0.4 * static_cast<double>(each) + 2) + 0.6 + static_cast<double>(heads * n * matrix) * 3e-7;
        if (n == 1 || cost < least) best = n, least = cost;
    }
    p->segment_rows = std::max<int64_t>(1, (tiles + best - 1) / best) * kAttendTile;
    p->segments = static_cast<int>(std::max<int64_t>(1, (p->length + p->segment_rows - 1) / p->segment_rows));
}

// The sizes and arrays that the entries check alike.
struct AttendCall {
    AttendArgs p{};
    AttendRows q, k, v;
    int keys, values, key_heads, dtype;
    const float* state;
};
bool AttendSizesOf(const hipcx_array* q, const hipcx_array* v, AttendCall* c);
AttendCall DescribeAttend(const std::string& what, const hipcx_array* q, const hipcx_array* k, const hipcx_array* v, const hipcx_array* log_decay, double scale,
                          const hipcx_array* state, const hipcx_array* lengths);
// [batch, time, heads, width] with a dense last axis.
AttendRows DescribeAttendRows(const hipcx_array* a, const AttendCall& c, int64_t heads, int64_t width, int dtype, const std::string& what);
// [batch, heads, keys, values], or its transposes.
inline AttendStates AttendStatesOf(const float* data, int keys, int values, bool transposed) {
    const int64_t head = static_cast<int64_t>(keys) * values;
    return transposed ? AttendStates{const_cast<float*>(data), head, 0, 1, values} : AttendStates{const_cast<float*>(data), head, 0, values, 1};
}
// The segments' states of a pass in a workspace, [batch and head][segment][i][j].
inline AttendStates AttendSegments(float* data, const AttendArgs& p, int keys, int values) {
    const int64_t each = static_cast<int64_t>(keys) * values;
    return {data, each * p.segments, each, values, 1};
}
inline int AttendBlocks(int values) { return (values + kAttendColumns - 1) / kAttendColumns; }

inline AttendWidths AttendWidthsOf(const AttendArgs& p, int piece) {
    bool whole = true, narrow = false;
    for (int i = 0; i < p.runs; ++i) {
        for (const int width : {p.run[i].keys, p.run[i].values}) whole = whole && width % piece == 0, narrow = narrow || width < piece;
    }
    return whole ? kAttendWhole : narrow ? kAttendNarrow : kAttendPart;
}

// (narrow rows, which are few bytes, have no kernels without what the gradients need)
template <typename F>
void VisitWidths(AttendWidths widths, bool grad, F&& f) {
    if (widths == kAttendNarrow) f(std::integral_constant<int, kAttendNarrow>{}, std::true_type{});
    else if (widths == kAttendWhole) grad ? f(std::integral_constant<int, kAttendWhole>{}, std::true_type{}) : f(std::integral_constant<int, kAttendWhole>{}, std::false_type{});
    else grad ? f(std::integral_constant<int, kAttendPart>{}, std::true_type{}) : f(std::integral_constant<int, kAttendPart>{}, std::false_type{});
}

// Workgroups that a compute unit holds, as registers and LDS let them.
constexpr int kLdsOfUnit = 160 * 1024;
constexpr int AttendResident(bool half, int keys) { return keys <= 64 && half ? 3 : keys <= 128 ? 2 : 1; }

void LaunchAttend(const AttendArgs& p, int dtype, bool states_alone, hipStream_t stream);
void LaunchAttendHalf(const AttendArgs& p, int keys, int64_t blocks, bool states_alone, hipStream_t stream);  // float16
// What segments add to a state of zeros (`last` of a pass of states alone) becomes the state that they start from, in the order of the pass.
void LaunchAttendStarts(const AttendArgs& p, int run, const AttendStates& initial, hipStream_t stream);

}  // namespace hipcx
