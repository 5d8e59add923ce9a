// What the selective scan and its gradients share.
//   h[t][n] = exp(dt[t] a[n]) h[t-1][n] + dt[t] u[t] b[t][n],  y[t] = (sum over n of c[t][n] h[t][n] + d u[t]) silu(z[t])
// for every sequence and channel; dt = delta + bias, or softplus of it.  b and c belong to a group of channels.
#pragma once

#include <cfloat>

#include "sequence.h"

namespace hipcx {

// Rows of b or c, [batch, time, group, state]; strides in elements.
struct ScanShared {
    void* data;
    int64_t batch, row, group;
};

struct ScanArgs {
    SequenceRows u, delta, z, y;
    ScanShared b, c;
    const float *a, *d, *bias;  // [channels][states], [channels] or null
    const float* state;         // [batch][channels][states] or null
    float* new_state;
    SequenceLengths lengths;
    int64_t batch, length;
    int channels, states, group_channels;
    int group_blocks, blocks;   // workgroups along the channels of a group, of all groups
    int chunks, chunk_rows;     // of the time axis; whole tiles of rows
    float* ends;                // [batch][chunks][channels][states]: the state that the sequence starts from, then where each chunk but the last ends that starts from zeros
    float* steps;               // [batch][chunks - 1][channels]: dt summed over the chunk
    int softplus;
};

// Four lanes (a quad) belong to a channel: each keeps a quarter of its states, and they take the rows' other work in turns.  A wave has 16 channels.
constexpr int kScanChannels = 64;  // to a workgroup of four waves
constexpr int kScanTile = 16;      // rows whose b and c are in LDS

template <int S>
__device__ __forceinline__ float OfQuadLane(float v) {
    return __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, v), S * 0x55, 0xf, 0xf, true));
}
__device__ __forceinline__ float QuadSwap1(float v) { return __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, v), 0xB1, 0xf, 0xf, true)); }
__device__ __forceinline__ float QuadSwap2(float v) { return __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, v), 0x4E, 0xf, 0xf, true)); }

// Lane q of a quad gets the sum of v[q] over the quad.
__device__ __forceinline__ float QuadTransposedSum(const float (&v)[4], int q) {
    const bool odd = (q & 1) != 0, high = (q & 2) != 0;
    const float r0 = (odd ? v[1] : v[0]) + QuadSwap1(odd ? v[0] : v[1]);
    const float r1 = (odd ? v[3] : v[2]) + QuadSwap1(odd ? v[2] : v[3]);
    return (high ? r1 : r0) + QuadSwap2(high ? r0 : r1);
}

// log(1 + exp(x)) = max(x, 0) + log(1 + e), e = exp(-|x|); the logarithm as 2 artanh(s), s = e / (2 + e) <= 1/3, by seven terms of its series (the eighth is 1.4e-8 of
// the sum), so that a small e loses nothing in 1 + e.  Off by less than 10 + 4 |x| half steps, of which the roundings of x and of the exponential's argument are 3.3 |x|: at a step of 1e-3,
// x = -6.9, by some 30.
__device__ __forceinline__ float SoftplusOf(float x) {
    const float e = __builtin_amdgcn_exp2f(-kLog2E * __builtin_fabsf(x));
    const float s = e * __builtin_amdgcn_rcpf(2.f + e), q = s * s;
    float r = 1.f / 13;
    r = __builtin_fmaf(r, q, 1.f / 11);
    r = __builtin_fmaf(r, q, 1.f / 9);
    r = __builtin_fmaf(r, q, 1.f / 7);
    r = __builtin_fmaf(r, q, 1.f / 5);
    r = __builtin_fmaf(r, q, 1.f / 3);
    return __builtin_fmaxf(x, 0.f) + 2.f * __builtin_fmaf(s * q, r, s);
}

// States n0 .. n0 + NPL - 1 of `all`, which the padding follows; one access where they are all there.
template <int NPL>
struct __attribute__((packed, aligned(4))) LaneStates {
    float v[NPL];
};
template <int NPL>
__device__ __forceinline__ void LoadStates(const float* p, int n0, int all, float (&v)[NPL], float padding = 0.f) {
    if (n0 + NPL <= all) {
        const LaneStates<NPL> s = *reinterpret_cast<const LaneStates<NPL>*>(p + n0);
#pragma unroll
        for (int i = 0; i < NPL; ++i) v[i] = s.v[i];
    } else {
#pragma unroll
        for (int i = 0; i < NPL; ++i) v[i] = n0 + i < all ? p[n0 + i] : padding;
    }
}
// Exponents to base 2 of a step of 1.  -inf (a = -exp(a_log) overflows to it) as the lowest number: rows without a step, behind a sequence's last, multiply by exp(0) then, not by NaN.
// The padding's is next to 0 and below it: a finite step multiplies it by 2^-6 to 2^6, and an infinite one by 0, where exp(inf * 0) would make NaN of it and of the sums over states.
template <int NPL>
__device__ __forceinline__ void LoadExponents(const float* p, int n0, int all, float (&a)[NPL]) {
    LoadStates<NPL>(p, n0, all, a, -FLT_MIN);
#pragma unroll
    for (int i = 0; i < NPL; ++i) {
        a[i] *= kLog2E;
        a[i] = a[i] < -FLT_MAX ? -FLT_MAX : a[i];  // (NaN stays)
    }
}
template <int NPL>
__device__ __forceinline__ void StoreStates(float* p, int n0, int all, const float (&v)[NPL]) {
    if (n0 + NPL <= all) {
        LaneStates<NPL> s;
#pragma unroll
        for (int i = 0; i < NPL; ++i) s.v[i] = v[i];
        *reinterpret_cast<LaneStates<NPL>*>(p + n0) = s;
    } else {
#pragma unroll
        for (int i = 0; i < NPL; ++i) {
            if (n0 + i < all) p[n0 + i] = v[i];
        }
    }
}

// Fewer states than four lanes have room for, in a way that leaves no padding: a lane that has not enough of its own takes the last NPL states, one that has none takes the first ones, and a
// state that is there several times counts by a fraction.  (More than two lanes have states of their own unless NPL is 1.)
template <int NPL>
__device__ __forceinline__ int FirstOfLane(int lane, int all) {
    const int n0 = lane * NPL;
    if (n0 < all) return n0 + NPL <= all ? n0 : all - NPL;
    return NPL == 1 && all > 1 ? n0 - all : 0;
}
template <int NPL>
__device__ __forceinline__ float ShareOf(int n, int all) {
    if (NPL == 1) return all == 1 ? 0.25f : n < 4 - all ? 0.5f : 1.f;
    const bool of_first = all <= 3 * NPL && n < NPL, of_last = n >= all - NPL && n < all / NPL * NPL && all % NPL != 0;
    return of_first || of_last ? 0.5f : 1.f;
}

// s = exp(sum of dt) s + what the chunk adds, for `n` chunks one after another, `next` chunks apart (1 or -1): a state from the sequence's start to a chunk, or its gradient
// from the end back to one.  `adds` [chunk][per_chunk] and `steps` [chunk][channels] are read four chunks at a time.
template <int NPL>
__device__ __forceinline__ void ThroughChunks(float (&s)[NPL], const float (&a)[NPL], const float* adds, const float* steps, int n, int next, int64_t per_chunk, int64_t channels,
                                              int n0, int states) {
    for (int j = 0; j < n; j += 4) {
        float add[4][NPL], dt[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const int64_t at = static_cast<int64_t>(j + k < n ? j + k : n - 1) * next;
            LoadStates<NPL>(adds + at * per_chunk, n0, states, add[k]);
            dt[k] = steps[at * channels];
        }
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            if (j + k >= n) break;
#pragma unroll
            for (int i = 0; i < NPL; ++i) s[i] = __builtin_fmaf(__builtin_amdgcn_exp2f(dt[k] * a[i]), s[i], add[k][i]);
        }
    }
}

// Where a thread stands: its sequence, chunk, channel and lane of the quad.
struct ScanPlace {
    int64_t b;
    int chunk, group, channel, q;
    bool inside;  // else it repeats the group's last channel and stores nothing
    __device__ __forceinline__ ScanPlace(const ScanArgs& p, unsigned block, int chunks) {
        const unsigned line = block / static_cast<unsigned>(p.blocks), of_channels = block % static_cast<unsigned>(p.blocks);
        chunk = static_cast<int>(line % static_cast<unsigned>(chunks));
        b = line / static_cast<unsigned>(chunks);
        group = static_cast<int>(of_channels) / p.group_blocks;
        const int within = (static_cast<int>(of_channels) - group * p.group_blocks) * kScanChannels + (static_cast<int>(threadIdx.x) >> 2);
        inside = within < p.group_channels;
        channel = group * p.group_channels + (inside ? within : p.group_channels - 1);
        q = static_cast<int>(threadIdx.x) & 3;
    }
};

// A tile's rows of a channel, which a quad's lanes take in turns: the tile starts at an address that is the same for the whole workgroup, and a lane's place in it is a
// number of 32 bits, so that a load costs one more vector instruction at most.  `held`: what Fetch() has asked for.
template <typename T, int ROWS>
struct TileRows {
    static constexpr int kGroups = ROWS / 4;
    char* base;
    int group;  // bytes to the next four rows
    unsigned offset;
    T held[kGroups];
    __device__ __forceinline__ TileRows(const SequenceRows& r, const ScanPlace& at, int64_t t) {
        const int64_t row = r.row * static_cast<int64_t>(sizeof(T)), low = row < 0 ? (ROWS - 1) * row : 0;
        base = static_cast<char*>(r.data) + at.b * r.batch * static_cast<int64_t>(sizeof(T)) + t * row + low;
        group = static_cast<int>(4 * row);
        offset = static_cast<unsigned>(at.q * row - low + at.channel * static_cast<int64_t>(sizeof(T)));
        asm("" : "+v"(offset));  // (the compiler would put 64-bit addresses together)
#pragma unroll
        for (int g = 0; g < kGroups; ++g) held[g] = static_cast<T>(0);
    }
    __device__ __forceinline__ T& operator[](int g) const { return *reinterpret_cast<T*>(base + (offset + static_cast<unsigned>(g) * static_cast<unsigned>(group))); }
    // A lane's rows of the tile, all of them or those before `rows`.
    template <bool WHOLE>
    __device__ __forceinline__ void Fetch(int q, int rows) {
#pragma unroll
        for (int g = 0; g < kGroups; ++g) {
            T v = static_cast<T>(0);
            if (WHOLE || 4 * g + q < rows) v = (*this)[g];
            held[g] = v;
        }
    }
    __device__ __forceinline__ float Held(int g) const { return static_cast<float>(held[g]); }
    __device__ __forceinline__ void Move(int tiles) {
        base += static_cast<int64_t>(tiles) * kGroups * group;
        asm("" : "+v"(offset));  // else a register for each group's offset is kept from tile to tile
    }
};
constexpr int64_t kMaxScanLength = int64_t{1} << 30, kMaxScanChannels = int64_t{1} << 24, kMaxScanStates = 64;
constexpr int64_t kMaxScanRow = int64_t{1} << 26;  // elements from one row to the next: a tile and the channels fit those 32 bits

// A tile of b, or of b and c, on its way to LDS: workgroups of 256 threads take an element each, or a few.  REPEATS: states as FirstOfLane() deals them out, c times their share.
template <typename T, int NPL, int ROWS, int PARTS, bool REPEATS = false>
struct TileShared {
    static constexpr int kNP = 4 * NPL, kEach = (ROWS * kNP + 255) / 256;
    const T* from[PARTS][kEach];
    int64_t step[PARTS];
    bool is_state[kEach];
    float share[kEach];
    T held[PARTS][kEach];
    __device__ __forceinline__ TileShared(const ScanArgs& p, const ScanPlace& at, int64_t t) {
#pragma unroll
        for (int i = 0; i < kEach; ++i) {
            const int e = i * 256 + static_cast<int>(threadIdx.x), r = e / kNP, n = REPEATS ? FirstOfLane<NPL>(e % kNP / NPL, p.states) + e % NPL : e % kNP;
            is_state[i] = r < ROWS && n < p.states;
            if constexpr (REPEATS) share[i] = ShareOf<NPL>(n, p.states);
#pragma unroll
            for (int k = 0; k < PARTS; ++k) {
                const ScanShared& s = k == 0 ? p.b : p.c;
                from[k][i] = static_cast<const T*>(s.data) + at.b * s.batch + at.group * s.group + (t + r) * s.row + n;
                step[k] = ROWS * s.row;
                held[k][i] = static_cast<T>(0);
            }
        }
    }
    template <bool WHOLE>
    __device__ __forceinline__ void Fetch(int rows) {
#pragma unroll
        for (int i = 0; i < kEach; ++i) {
            const bool counts = is_state[i] && (WHOLE || (i * 256 + static_cast<int>(threadIdx.x)) / kNP < rows);
#pragma unroll
            for (int k = 0; k < PARTS; ++k) {
                T v = static_cast<T>(0);
                if (counts) v = *from[k][i];
                held[k][i] = v;
            }
        }
    }
    __device__ __forceinline__ void Move(int tiles) {
#pragma unroll
        for (int i = 0; i < kEach; ++i) {
#pragma unroll
            for (int k = 0; k < PARTS; ++k) from[k][i] += tiles * step[k];
        }
    }
    template <int K>
    __device__ __forceinline__ void Stage(float (&to)[ROWS][kNP]) const {
#pragma unroll
        for (int i = 0; i < kEach; ++i) {
            const int e = i * 256 + static_cast<int>(threadIdx.x);
            if (e < ROWS * kNP) to[e / kNP][e % kNP] = REPEATS && K == 1 ? static_cast<float>(held[K][i]) * share[i] : static_cast<float>(held[K][i]);
        }
    }
};

// The NPL of a call: a lane's share of the states, rounded up to a power of two.
template <typename F>
void VisitScan(int dtype, int states, F&& f) {
    const auto visit = [&](auto tag) {
        const int share = (states + 3) / 4;
        if (share <= 1) f(tag, std::integral_constant<int, 1>{});
        else if (share <= 2) f(tag, std::integral_constant<int, 2>{});
        else if (share <= 4) f(tag, std::integral_constant<int, 4>{});
        else if (share <= 8) f(tag, std::integral_constant<int, 8>{});
        else f(tag, std::integral_constant<int, 16>{});
    };
    if (dtype == HIPCX_FLOAT16) visit(Tag<half_t>{});
    else visit(Tag<float>{});
}

// [batch, time, ...] as TileRows reads it; of a single row, whatever its stride says of the next.
SequenceRows ScanRowsOf(const hipcx_array* a, const std::string& what);

// Cuts the time axis into chunks of `least` tiles or more, for `each` workgroups to a compute unit, where sequences and channels alone do not give it `enough`.
void CutScan(ScanArgs* p, int enough, int each, int least);

// The sizes that workspaces go by; false for what DescribeScan() refuses, which takes none.
bool ScanSizesOf(const hipcx_array* u, const hipcx_array* a, ScanArgs* p);

// Checks the inputs that the scan and its gradients share and describes them, except for the cut along time.
ScanArgs DescribeScan(const std::string& what, const hipcx_array* u, const hipcx_array* delta, const hipcx_array* a, const hipcx_array* b, const hipcx_array* c,
                      const hipcx_array* d, const hipcx_array* z, const hipcx_array* delta_bias, int delta_softplus, const hipcx_array* state,
                      const hipcx_array* lengths);

}  // namespace hipcx
