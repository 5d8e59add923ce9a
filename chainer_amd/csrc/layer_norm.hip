// Layer norm: rows normalised to mean 0 and variance 1, scaled and shifted by column, and its gradients.
//   m = sum x / n,  s = 1 / sqrt(sum (x - m)^2 / n + eps),  xh = (x - m) s,  y = xh gamma + beta
//   g = gy gamma,  gx = s (g - sum g / n - xh sum(g xh) / n),  ggamma = sum over rows of gy xh,  gbeta = sum over rows of gy
#include <algorithm>

#include "common.h"

namespace hipcx {
namespace {

struct NormArgs {
    const void* x;
    const void* gy;  // gradients alone
    const void* gamma;  // may be null: ones
    const void* beta;   // may be null: zeros
    void* out;          // y or gx, dense rows
    void* mean;
    void* inv_std;
    void* partial;  // [workgroups][2][cols]: sums of gy xh and of gy over a workgroup's rows
    int64_t rows, x_pitch, gy_pitch;  // pitches in elements
    int64_t cols;
    double eps;
    int weights;  // whether the weights' gradients are asked for
};

template <typename T>
constexpr int kPieceOf = 16 / sizeof(T);

template <typename T, int N>
struct __attribute__((packed, aligned(alignof(T)))) Elements {
    T v[N];
};

template <typename T>
using NormCompute = std::conditional_t<std::is_same<T, double>::value, double, float>;

// v and what a DPP move brings from another lane of the rows in ROWS, 0 elsewhere.
template <int MOVE, int ROWS>
__device__ __forceinline__ float AddMoved(float v) {
    return v + __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), MOVE, ROWS, 0xf, false));
}
template <int MOVE, int ROWS>
__device__ __forceinline__ double AddMoved(double v) {
    const uint64_t b = __builtin_bit_cast(uint64_t, v);
    const uint32_t lo = __builtin_amdgcn_update_dpp(0, static_cast<int>(b), MOVE, ROWS, 0xf, false), hi = __builtin_amdgcn_update_dpp(0, static_cast<int>(b >> 32), MOVE, ROWS, 0xf, false);
    return v + __builtin_bit_cast(double, static_cast<uint64_t>(hi) << 32 | lo);
}
__device__ __forceinline__ float OfLastLane(float v) { return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), 63)); }
__device__ __forceinline__ double OfLastLane(double v) {
    const uint64_t b = __builtin_bit_cast(uint64_t, v);
    return __builtin_bit_cast(double, static_cast<uint64_t>(static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(b >> 32), 63))) << 32 |
                                          static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(b), 63)));
}

// Sums over the G threads of a row, which all of them get, N at a time (of MOST): by moves inside the vector units, which are some ten times as quick as those through LDS.  Sixteen or 64 threads are
// neighbours in a wave; more are the whole workgroup, whose waves' sums meet in `meet` (two halves in turn: a wave that is still reading one half is waited for at the barrier of the other).
template <int G, int MOST, int N, typename C>
__device__ __forceinline__ void RowSum(C (&v)[N], C* meet, int& turn) {
    static_assert(G == 16 || G % 64 == 0, "rows of lanes, or waves");
    if constexpr (G == 16) {  // rotations by 8, 4, 2 and 1
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = AddMoved<0x128, 0xf>(v[i]);
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = AddMoved<0x124, 0xf>(v[i]);
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = AddMoved<0x122, 0xf>(v[i]);
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = AddMoved<0x121, 0xf>(v[i]);
        return;
    }
    // from 1, 2, 4 and 8 lanes before in the row of 16, then from the rows' last lanes
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = AddMoved<0x111, 0xf>(v[i]);
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = AddMoved<0x112, 0xf>(v[i]);
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = AddMoved<0x114, 0xf>(v[i]);
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = AddMoved<0x118, 0xf>(v[i]);
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = AddMoved<0x142, 0xa>(v[i]);
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = AddMoved<0x143, 0xc>(v[i]);
    if constexpr (G == 64) {
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = OfLastLane(v[i]);
    } else {
        constexpr int W = G / 64;
        C* const at = meet + turn * (W * MOST);
        turn ^= 1;
        if (threadIdx.x % 64 == 63) {
#pragma unroll
            for (int i = 0; i < N; ++i) at[threadIdx.x / 64 * N + i] = v[i];
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < N; ++i) {
            v[i] = 0;
#pragma unroll
            for (int w = 0; w < W; ++w) v[i] += at[w * N + i];
        }
    }
}

// A thread's pieces of a row: piece j of thread l covers columns (l + j G) E and on.  A piece that reaches over the row's end is moved back so that it is whole, and so are those behind it, so that no
// load waits for a branch; Counts tells which of a piece's elements are this thread's to count.  NARROW: rows of less than a piece, of which the first thread has all.
template <typename T, int G, bool NARROW>
struct RowPiece {
    static constexpr int E = kPieceOf<T>;
    int natural, at, cols;
    __device__ __forceinline__ RowPiece(int l, int j, int n) : natural((j * G + l) * E), at(NARROW ? 0 : min(natural, n - E)), cols(n) {}
    __device__ __forceinline__ bool Counts(int e) const { return NARROW ? natural == 0 && e < cols : e >= natural - at; }
    template <typename S>
    __device__ __forceinline__ Elements<S, E> Load(const S* row) const {
        if constexpr (!NARROW) return *reinterpret_cast<const Elements<S, E>*>(row + at);
        Elements<S, E> r;
#pragma unroll
        for (int e = 0; e < E; ++e) r.v[e] = row[min(e, cols - 1)];
        return r;
    }
    template <typename S, typename C>
    __device__ __forceinline__ void Store(S* row, const C (&v)[E]) const {
        if (natural >= cols) return;
        Elements<S, E> r;
#pragma unroll
        for (int e = 0; e < E; ++e) r.v[e] = static_cast<S>(v[e]);
        if constexpr (!NARROW) {
            *reinterpret_cast<Elements<S, E>*>(row + at) = r;
        } else {
#pragma unroll
            for (int e = 0; e < E; ++e) {
                if (e < cols) row[e] = r.v[e];
            }
        }
    }
};

// What a row's values are taken relative to: the mean, and 0 where that is less than half of the mean of their absolute values (`sum[1]`).  Values of one power of two have their last bit in one
// place, so that differences from a mean with bits beyond it are all rounded alike and shift the second sum by up to 2^-24 of the values, which is nothing next to a mean of their size, but more
// than the first sum's error next to a small one; and from a mean that small, cancellation takes less than half a bit of the variance.  float16's values, of eleven bits, are taken relative to
// the mean in twelve, from which their differences are exact.
template <typename C>
__device__ __forceinline__ void AddFirst(C* sum, C v) {
    sum[0] += v;
    sum[1] += __builtin_elementwise_abs(v);
}
template <typename T, typename C>
__device__ __forceinline__ C NearMean(const C* sum, C n) {
    if (__builtin_elementwise_abs(sum[0]) < static_cast<C>(0.5) * sum[1]) return static_cast<C>(0);
    const C mean = sum[0] / n;
    if constexpr (std::is_same<T, half_t>::value) return __builtin_bit_cast(float, __builtin_bit_cast(uint32_t, mean) & 0xfffff000u);
    else return mean;
}

// The first sum gives a number near the mean, and the sums of the differences from it and of their squares the mean and the variance: two passes over registers.  R rows at once: their loads
// are under way together, their sums meet together, and the parameters are read once for all of them.  Bound by memory: 16384 rows of 4096 in float16, parameters in float32, take 53 us
// (5.1 TB/s; one row at a time, 95 us: each row's parameters are four times its bytes from L2), 4480 rows of 650 in float32 7.0 us, of which some 3 are the launch.
template <typename T, typename P, int G, int V, int R, bool NARROW>
__global__ __launch_bounds__(G > 256 ? G : 256) void LayerNormKernel(NormArgs p) {
    using C = NormCompute<T>;
    using Piece = RowPiece<T, G, NARROW>;
    constexpr int E = kPieceOf<T>, THREADS = G > 256 ? G : 256, GROUPS = THREADS / G;
    __shared__ C meet[2 * 2 * R * (THREADS / 64)];
    const int l = threadIdx.x % G, cols = static_cast<int>(p.cols);
    const C n = static_cast<C>(cols);
    int turn = 0;
    const int64_t first = (static_cast<int64_t>(blockIdx.x) * GROUPS + threadIdx.x / G) * R;
    if (first >= p.rows) return;
    Elements<T, E> raw[R][V];
#pragma unroll
    for (int r = 0; r < R; ++r) {
        const T* const x = static_cast<const T*>(p.x) + (first + r < p.rows ? first + r : p.rows - 1) * p.x_pitch;
#pragma unroll
        for (int j = 0; j < V; ++j) raw[r][j] = Piece(l, j, cols).Load(x);
    }
    Elements<P, E> gamma[V], beta[V];
    const auto load = [&](int j) {
        if (p.gamma != nullptr) gamma[j] = Piece(l, j, cols).Load(static_cast<const P*>(p.gamma));
        if (p.beta != nullptr) beta[j] = Piece(l, j, cols).Load(static_cast<const P*>(p.beta));
    };
    constexpr bool kAhead = G < 1024;  // (sixteen waves have no registers for what is used later)
    if (kAhead) {
#pragma unroll
        for (int j = 0; j < V; ++j) load(j);
    }
    C v[R][V][E], sum[2 * R], more[2 * R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
        sum[2 * r] = sum[2 * r + 1] = 0;
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const Piece piece(l, j, cols);
            const bool all = !NARROW && (j + 1) * G * E <= cols;
#pragma unroll
            for (int e = 0; e < E; ++e) {
                v[r][j][e] = static_cast<C>(raw[r][j].v[e]);
                AddFirst(sum + 2 * r, all || piece.Counts(e) ? v[r][j][e] : static_cast<C>(0));
            }
        }
    }
    RowSum<G, 2 * R>(sum, meet, turn);
#pragma unroll
    for (int r = 0; r < R; ++r) {
        const C about = NearMean<T>(sum + 2 * r, n);
        sum[2 * r] = about;
        more[2 * r] = more[2 * r + 1] = 0;
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const Piece piece(l, j, cols);
            const bool all = !NARROW && (j + 1) * G * E <= cols;
#pragma unroll
            for (int e = 0; e < E; ++e) {
                v[r][j][e] -= about;
                const C d = all || piece.Counts(e) ? v[r][j][e] : static_cast<C>(0);
                more[2 * r] += d;
                more[2 * r + 1] = __builtin_elementwise_fma(d, d, more[2 * r + 1]);
            }
        }
    }
    RowSum<G, 2 * R>(more, meet, turn);
#pragma unroll
    for (int r = 0; r < R; ++r) {
        const int64_t row = first + r;
        if (row >= p.rows) continue;
        const C off = more[2 * r] / n;
        C var = more[2 * r + 1] / n - off * off;
        var = var < 0 ? static_cast<C>(0) : var;
        const C inv = static_cast<C>(1) / static_cast<C>(sqrt(var + static_cast<C>(p.eps)));
        if (l == 0) {
            static_cast<C*>(p.mean)[row] = sum[2 * r] + off;
            static_cast<C*>(p.inv_std)[row] = inv;
        }
#pragma unroll
        for (int j = 0; j < V; ++j) {
            if (!kAhead) load(j);
#pragma unroll
            for (int e = 0; e < E; ++e) {
                C y = (v[r][j][e] - off) * inv;
                if (p.gamma != nullptr) y *= static_cast<C>(gamma[j].v[e]);
                if (p.beta != nullptr) y += static_cast<C>(beta[j].v[e]);
                v[r][j][e] = y;
            }
            Piece(l, j, cols).Store(static_cast<T*>(p.out) + row * p.cols, v[r][j]);
        }
    }
}

// Rows that no workgroup holds in its registers, read three times.
template <typename T, typename P>
__global__ __launch_bounds__(1024) void LayerNormLongKernel(NormArgs p) {
    using C = NormCompute<T>;
    __shared__ C meet[2 * 2 * 16];
    const C n = static_cast<C>(p.cols);
    int turn = 0;
    for (int64_t row = blockIdx.x; row < p.rows; row += gridDim.x) {
        const T* const x = static_cast<const T*>(p.x) + row * p.x_pitch;
        T* const y = static_cast<T*>(p.out) + row * p.cols;
        C sum[2] = {0, 0}, more[2] = {0, 0};
        for (int64_t i = threadIdx.x; i < p.cols; i += 1024) AddFirst(sum, static_cast<C>(x[i]));
        RowSum<1024, 2>(sum, meet, turn);
        const C about = NearMean<T>(sum, n);
        for (int64_t i = threadIdx.x; i < p.cols; i += 1024) {
            const C d = static_cast<C>(x[i]) - about;
            more[0] += d;
            more[1] = __builtin_elementwise_fma(d, d, more[1]);
        }
        RowSum<1024, 2>(more, meet, turn);
        const C off = more[0] / n;
        C var = more[1] / n - off * off;
        var = var < 0 ? static_cast<C>(0) : var;
        const C inv = static_cast<C>(1) / static_cast<C>(sqrt(var + static_cast<C>(p.eps)));
        if (threadIdx.x == 0) {
            static_cast<C*>(p.mean)[row] = about + off;
            static_cast<C*>(p.inv_std)[row] = inv;
        }
        for (int64_t i = threadIdx.x; i < p.cols; i += 1024) {
            C v = (static_cast<C>(x[i]) - about - off) * inv;
            if (p.gamma != nullptr) v *= static_cast<C>(static_cast<const P*>(p.gamma)[i]);
            if (p.beta != nullptr) v += static_cast<C>(static_cast<const P*>(p.beta)[i]);
            y[i] = static_cast<T>(v);
        }
    }
}

// R rows' two sums, then their gradients, with the next rows on their way; a thread keeps its columns' sums over the rows that its workgroup walks through.  Bound by memory: 16384 rows of 4096 in
// float16 take 86 us (4.7 TB/s; without the next rows' loads ahead, one row at a time, 160), 4480 rows of 650 in float32 9.7 us.
template <typename T, typename P, int G, int V, int R, bool NARROW>
__global__ __launch_bounds__(G > 256 ? G : 256) void LayerNormGradKernel(NormArgs p) {
    using C = NormCompute<T>;
    using Piece = RowPiece<T, G, NARROW>;
    constexpr int E = kPieceOf<T>, THREADS = G > 256 ? G : 256, GROUPS = THREADS / G;
    __shared__ C meet[2 * 2 * R * (THREADS / 64)];
    __shared__ C shared_sums[GROUPS > 1 ? 2 * G * V * E : 1];
    const int l = threadIdx.x % G, cols = static_cast<int>(p.cols);
    const C n = static_cast<C>(cols);
    int turn = 0;
    C of_gamma[V][E], of_beta[V][E];
#pragma unroll
    for (int j = 0; j < V; ++j) {
#pragma unroll
        for (int e = 0; e < E; ++e) of_gamma[j][e] = of_beta[j][e] = 0;
    }
    Elements<T, E> x[R][V], gy[R][V];
    C mean[R], inv[R];
    const auto load = [&](int64_t first) {
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const int64_t row = first + r < p.rows ? first + r : p.rows - 1;
            mean[r] = static_cast<const C*>(p.mean)[row], inv[r] = static_cast<const C*>(p.inv_std)[row];
#pragma unroll
            for (int j = 0; j < V; ++j) {
                x[r][j] = Piece(l, j, cols).Load(static_cast<const T*>(p.x) + row * p.x_pitch);
                gy[r][j] = Piece(l, j, cols).Load(static_cast<const T*>(p.gy) + row * p.gy_pitch);
            }
        }
    };
    int64_t first = (static_cast<int64_t>(blockIdx.x) * GROUPS + threadIdx.x / G) * R;
    Elements<P, E> gamma[V];
    constexpr bool kAhead = G < 1024;  // (sixteen waves have no registers for what is used later)
    if (kAhead) {
        if (p.gamma != nullptr) {
#pragma unroll
            for (int j = 0; j < V; ++j) gamma[j] = Piece(l, j, cols).Load(static_cast<const P*>(p.gamma));
        }
        load(first);
    }
    for (; first < p.rows; first += static_cast<int64_t>(gridDim.x) * (GROUPS * R)) {
        if (!kAhead) load(first);
        C xh[kAhead ? R : 1][V][E], g[kAhead ? R : 1][V][E], sum[2 * R], scale[R];
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const bool live = first + r < p.rows;
            sum[2 * r] = sum[2 * r + 1] = 0;
            scale[r] = inv[r];
#pragma unroll
            for (int j = 0; j < V; ++j) {
                const Piece piece(l, j, cols);
                const bool all = !NARROW && (j + 1) * G * E <= cols;
                if (!kAhead && p.gamma != nullptr) gamma[j] = piece.Load(static_cast<const P*>(p.gamma));
#pragma unroll
                for (int e = 0; e < E; ++e) {
                    const C of_y = static_cast<C>(gy[r][j].v[e]), of_x = (static_cast<C>(x[r][j].v[e]) - mean[r]) * inv[r];
                    if (r == 0 || live) {  // (a group's first row is there)
                        of_gamma[j][e] = __builtin_elementwise_fma(of_y, of_x, of_gamma[j][e]);
                        of_beta[j][e] += of_y;
                    }
                    const C weighted = p.gamma != nullptr ? of_y * static_cast<C>(gamma[j].v[e]) : of_y;
                    if constexpr (kAhead) xh[r][j][e] = of_x, g[r][j][e] = weighted;
                    if (!all && !piece.Counts(e)) continue;
                    sum[2 * r] += weighted;
                    sum[2 * r + 1] = __builtin_elementwise_fma(weighted, of_x, sum[2 * r + 1]);
                }
            }
        }
        if (kAhead) load(first + static_cast<int64_t>(gridDim.x) * (GROUPS * R));
        RowSum<G, 2 * R>(sum, meet, turn);
#pragma unroll
        for (int r = 0; r < R; ++r) {
            if (first + r >= p.rows) continue;
            const C a = sum[2 * r] / n, b = sum[2 * r + 1] / n;
#pragma unroll
            for (int j = 0; j < V; ++j) {
                C out[E];
                if (!kAhead && p.gamma != nullptr) gamma[j] = Piece(l, j, cols).Load(static_cast<const P*>(p.gamma));
#pragma unroll
                for (int e = 0; e < E; ++e) {
                    if constexpr (kAhead) {
                        out[e] = scale[r] * (g[r][j][e] - a - xh[r][j][e] * b);
                    } else {
                        const C of_y = static_cast<C>(gy[r][j].v[e]), of_x = (static_cast<C>(x[r][j].v[e]) - mean[r]) * inv[r];
                        out[e] = scale[r] * ((p.gamma != nullptr ? of_y * static_cast<C>(gamma[j].v[e]) : of_y) - a - of_x * b);
                    }
                }
                Piece(l, j, cols).Store(static_cast<T*>(p.out) + (first + r) * p.cols, out);
            }
        }
    }
    if (!p.weights) return;
    C* const to = static_cast<C*>(p.partial) + static_cast<int64_t>(blockIdx.x) * 2 * p.cols;
    if constexpr (GROUPS == 1) {
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const Piece piece(l, j, cols);
#pragma unroll
            for (int e = 0; e < E; ++e) {
                if (piece.Counts(e)) to[piece.at + e] = of_gamma[j][e], to[p.cols + piece.at + e] = of_beta[j][e];
            }
        }
    } else {
        constexpr int WIDTH = G * V * E;
        for (int r = 0; r < GROUPS; ++r) {  // one of the groups after another: the order of the sums is always the same
            if (static_cast<int>(threadIdx.x / G) == r) {
#pragma unroll
                for (int j = 0; j < V; ++j) {
#pragma unroll
                    for (int e = 0; e < E; ++e) {
                        const int at = (j * G + l) * E + e;
                        shared_sums[at] = of_gamma[j][e] + (r > 0 ? shared_sums[at] : static_cast<C>(0));
                        shared_sums[WIDTH + at] = of_beta[j][e] + (r > 0 ? shared_sums[WIDTH + at] : static_cast<C>(0));
                    }
                }
            }
            __syncthreads();
        }
        if (static_cast<int>(threadIdx.x) < G) {
#pragma unroll
            for (int j = 0; j < V; ++j) {
                const Piece piece(l, j, cols);
#pragma unroll
                for (int e = 0; e < E; ++e) {
                    const int at = (j * G + l) * E + e;
                    if (piece.Counts(e)) to[piece.at + e] = shared_sums[at], to[p.cols + piece.at + e] = shared_sums[WIDTH + at];
                }
            }
        }
    }
}

template <typename T, typename P>
__global__ __launch_bounds__(1024) void LayerNormGradLongKernel(NormArgs p) {
    using C = NormCompute<T>;
    __shared__ C meet[2 * 2 * 16];
    const C n = static_cast<C>(p.cols);
    int turn = 0;
    for (int64_t row = blockIdx.x; row < p.rows; row += gridDim.x) {
        const T* const x = static_cast<const T*>(p.x) + row * p.x_pitch;
        const T* const gy = static_cast<const T*>(p.gy) + row * p.gy_pitch;
        const C mean = static_cast<const C*>(p.mean)[row], inv = static_cast<const C*>(p.inv_std)[row];
        const auto xh = [&](int64_t i) { return (static_cast<C>(x[i]) - mean) * inv; };
        const auto g = [&](int64_t i) { return static_cast<C>(gy[i]) * (p.gamma != nullptr ? static_cast<C>(static_cast<const P*>(p.gamma)[i]) : static_cast<C>(1)); };
        C sum[2] = {0, 0};
        for (int64_t i = threadIdx.x; i < p.cols; i += 1024) {
            sum[0] += g(i);
            sum[1] = __builtin_elementwise_fma(g(i), xh(i), sum[1]);
        }
        RowSum<1024, 2>(sum, meet, turn);
        const C a = sum[0] / n, b = sum[1] / n;
        for (int64_t i = threadIdx.x; i < p.cols; i += 1024) static_cast<T*>(p.out)[row * p.cols + i] = static_cast<T>(inv * (g(i) - a - xh(i) * b));
    }
}

// The weights' sums over the rows of a slice, of rows that LayerNormGradLongKernel walks through.
template <typename T>
__global__ __launch_bounds__(256) void LayerNormColumnsKernel(NormArgs p, int64_t slice_rows) {
    using C = NormCompute<T>;
    const int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
    if (i >= p.cols) return;
    const int64_t first = blockIdx.y * slice_rows, last = first + slice_rows < p.rows ? first + slice_rows : p.rows;
    C of_gamma = 0, of_beta = 0;
    for (int64_t row = first; row < last; ++row) {
        const C gy = static_cast<C>(static_cast<const T*>(p.gy)[row * p.gy_pitch + i]);
        const C xh = (static_cast<C>(static_cast<const T*>(p.x)[row * p.x_pitch + i]) - static_cast<const C*>(p.mean)[row]) * static_cast<const C*>(p.inv_std)[row];
        of_gamma = __builtin_elementwise_fma(gy, xh, of_gamma);
        of_beta += gy;
    }
    C* const to = static_cast<C*>(p.partial) + static_cast<int64_t>(blockIdx.y) * 2 * p.cols;
    to[i] = of_gamma, to[p.cols + i] = of_beta;
}

// Partial sums of workgroups -> gradients, added up in 64 bits: COLS columns to a workgroup, slices of the partial sums to its threads, which ask for sixteen at a time.
template <typename C, typename P, int COLS>
__global__ __launch_bounds__(256) void LayerNormSumKernel(const C* partial, int64_t parts, int64_t cols, P* ggamma, P* gbeta) {
    constexpr int S = 256 / COLS, N = 16;
    __shared__ double sums[S][2][COLS];
    const int c = threadIdx.x % COLS, s = threadIdx.x / COLS;
    const int64_t i = static_cast<int64_t>(blockIdx.x) * COLS + c, col = i < cols ? i : cols - 1;
    double of_gamma = 0, of_beta = 0;
    for (int64_t first = s; first < parts; first += S * N) {
        C a[N], b[N];
#pragma unroll
        for (int k = 0; k < N; ++k) {
            const int64_t part = first + k * S < parts ? first + k * S : parts - 1;
            a[k] = partial[part * 2 * cols + col], b[k] = partial[(part * 2 + 1) * cols + col];
        }
#pragma unroll
        for (int k = 0; k < N; ++k) {
            of_gamma += first + k * S < parts ? a[k] : static_cast<C>(0);
            of_beta += first + k * S < parts ? b[k] : static_cast<C>(0);
        }
    }
    sums[s][0][c] = of_gamma, sums[s][1][c] = of_beta;
    __syncthreads();
    if (s < 2 && i < cols) {
        double v = 0;
#pragma unroll
        for (int k = 0; k < S; ++k) v += sums[k][s][c];
        P* const to = s == 0 ? ggamma : gbeta;
        if (to != nullptr) to[i] = static_cast<P>(static_cast<C>(v));
    }
}

// ---------------------------------------------------------------------------------------------
// host
// ---------------------------------------------------------------------------------------------
// Threads of a row and pieces of each: the least that hold it; 0 pieces for rows of less than one, 0 threads for rows that nothing holds.
struct NormPlan {
    int threads, pieces;
};

NormPlan PlanNorm(int64_t cols, int64_t item) {
    if (cols * item < 16) return {16, 0};
    const int64_t pieces = (cols * item + 15) / 16;
    for (const NormPlan plan : {NormPlan{16, 1}, {16, 2}, {64, 1}, {64, 2}, {64, 3}, {64, 4}, {256, 2}, {256, 4}, {1024, 2}, {1024, 4}}) {
        if (pieces <= static_cast<int64_t>(plan.threads) * plan.pieces) return plan;
    }
    return {0, 0};
}

// f(threads, pieces, whether rows are narrow)
template <typename F>
void VisitNorm(NormPlan plan, F&& f) {
    const auto visit = [&](auto threads, auto pieces) { f(threads, pieces, std::false_type{}); };
    if (plan.pieces == 0) f(std::integral_constant<int, 16>{}, std::integral_constant<int, 1>{}, std::true_type{});
    else if (plan.threads == 16) plan.pieces == 1 ? visit(std::integral_constant<int, 16>{}, std::integral_constant<int, 1>{}) : visit(std::integral_constant<int, 16>{}, std::integral_constant<int, 2>{});
    else if (plan.threads == 1024) plan.pieces == 2 ? visit(std::integral_constant<int, 1024>{}, std::integral_constant<int, 2>{}) : visit(std::integral_constant<int, 1024>{}, std::integral_constant<int, 4>{});
    else if (plan.threads == 256) plan.pieces == 2 ? visit(std::integral_constant<int, 256>{}, std::integral_constant<int, 2>{}) : visit(std::integral_constant<int, 256>{}, std::integral_constant<int, 4>{});
    else if (plan.pieces == 1) visit(std::integral_constant<int, 64>{}, std::integral_constant<int, 1>{});
    else if (plan.pieces == 2) visit(std::integral_constant<int, 64>{}, std::integral_constant<int, 2>{});
    else if (plan.pieces == 3) visit(std::integral_constant<int, 64>{}, std::integral_constant<int, 3>{});
    else visit(std::integral_constant<int, 64>{}, std::integral_constant<int, 4>{});
}

// Rows at once, where there are enough that every compute unit still gets four workgroups' (or walks of a workgroup): as many as the registers hold, `elements` of a row to a thread.
constexpr int RowsAtOnce(int elements, int most) { return elements * 4 <= most ? 4 : elements * 2 <= most ? 2 : 1; }

int StatDtype(int dtype) { return dtype == HIPCX_FLOAT64 ? HIPCX_FLOAT64 : HIPCX_FLOAT32; }

// Workgroups that walk through all rows in the gradients, each with partial sums of its own.
int64_t GradWorkgroups(int64_t rows, int64_t cols, int64_t item) {
    const NormPlan plan = PlanNorm(cols, item);
    if (plan.threads == 0) return std::min<int64_t>(rows, 64);
    const int64_t each = plan.threads < 256 ? 256 / plan.threads : 1;
    return std::min<int64_t>((rows + each - 1) / each, (plan.threads > 256 ? 1 : 2) * static_cast<int64_t>(NumCUs()));
}

int64_t RowsOfAll(const hipcx_array* x) {
    int64_t n = 1;
    for (int i = 0; i + 1 < x->ndim; ++i) n *= x->shape[i];
    return n;
}

// Elements from one row to the next, of an array whose last axis is dense and whose other axes lie one behind the other.
int64_t PitchOf(const hipcx_array* x, const char* what) {
    const int64_t it = ItemSize(x->dtype);
    const int last = x->ndim - 1;
    if (TotalSize(x) == 0) return x->shape[last];
    HIPCX_REQUIRE(x->shape[last] == 1 || x->strides[last] == it, HIPCX_DIMENSION_ERROR, std::string("layer_norm: ") + what + " must have a dense last axis");
    int64_t pitch = 0, expect = 0;
    bool seen = false;  // an inner axis (of a stride of 0, perhaps)
    for (int i = last - 1; i >= 0; --i) {
        if (x->shape[i] == 1) continue;
        if (!seen) {
            HIPCX_REQUIRE(x->strides[i] % it == 0, HIPCX_DIMENSION_ERROR, std::string("layer_norm: strides of ") + what + " must be whole elements");
            pitch = x->strides[i] / it;
        } else {
            HIPCX_REQUIRE(x->strides[i] == expect, HIPCX_DIMENSION_ERROR, std::string("layer_norm: rows of ") + what + " must be equally far apart");
        }
        seen = true;
        expect = x->strides[i] * x->shape[i];
    }
    return pitch;
}

void RequireStats(const hipcx_array* a, const hipcx_array* x, const char* what) {
    ValidateArray(a, what);
    HIPCX_REQUIRE(a->dtype == StatDtype(x->dtype), HIPCX_DTYPE_ERROR, std::string("layer_norm: ") + what + " must be " + DtypeName(StatDtype(x->dtype)));
    bool same = a->ndim == x->ndim - 1;
    for (int i = 0; same && i < a->ndim; ++i) same = a->shape[i] == x->shape[i];
    HIPCX_REQUIRE(same, HIPCX_DIMENSION_ERROR, std::string("layer_norm: ") + what + " must have x's shape without its last axis, got " + ShapeStr(a));
    HIPCX_REQUIRE(IsContiguous(a), HIPCX_DIMENSION_ERROR, std::string("layer_norm: ") + what + " must be C-contiguous");
}

// Parameters are of x's dtype or, for float16, of float32; all of one.
void RequireWeights(const hipcx_array* a, const hipcx_array* x, int& dtype, const char* what) {
    if (a == nullptr) return;
    ValidateArray(a, what);
    HIPCX_REQUIRE(a->dtype == x->dtype || (x->dtype == HIPCX_FLOAT16 && a->dtype == HIPCX_FLOAT32), HIPCX_DTYPE_ERROR,
                  std::string("layer_norm: ") + what + " must have x's dtype, or float32 where x is float16");
    HIPCX_REQUIRE(dtype == 0 || a->dtype == dtype, HIPCX_DTYPE_ERROR, "layer_norm: parameters and their gradients must share a dtype");
    dtype = a->dtype;
    HIPCX_REQUIRE(a->ndim == 1 && a->shape[0] == x->shape[x->ndim - 1], HIPCX_DIMENSION_ERROR, std::string("layer_norm: ") + what + " must have one value per column, got " + ShapeStr(a));
    HIPCX_REQUIRE(IsContiguous(a), HIPCX_DIMENSION_ERROR, std::string("layer_norm: ") + what + " must be dense");
}

void RequireResult(const hipcx_array* a, const hipcx_array* x, const char* what) {
    ValidateArray(a, what);
    HIPCX_REQUIRE(a->dtype == x->dtype, HIPCX_DTYPE_ERROR, std::string("layer_norm: ") + what + " must have x's dtype");
    HIPCX_REQUIRE(SameShape(a, x), HIPCX_DIMENSION_ERROR, std::string("layer_norm: ") + what + " must have x's shape, got " + ShapeStr(a));
}

void RequireInput(const hipcx_array* x) {
    ValidateArray(x, "x");
    HIPCX_REQUIRE(IsFloatDtype(x->dtype), HIPCX_DTYPE_ERROR, std::string("layer_norm: floating point arrays only, got ") + DtypeName(x->dtype));
    HIPCX_REQUIRE(x->ndim >= 1, HIPCX_DIMENSION_ERROR, "layer_norm: x needs an axis");
}

// f(T, P) with the types of x and of its parameters.
template <typename F>
void VisitNormTypes(int x, int params, F&& f) {
    if (x == HIPCX_FLOAT64) f(Tag<double>{}, Tag<double>{});
    else if (x == HIPCX_FLOAT32) f(Tag<float>{}, Tag<float>{});
    else if (params == HIPCX_FLOAT32) f(Tag<half_t>{}, Tag<float>{});
    else f(Tag<half_t>{}, Tag<half_t>{});
}

}  // namespace
}  // namespace hipcx

using namespace hipcx;

extern "C" int hipcx_layer_norm(const hipcx_array* x, const hipcx_array* gamma, const hipcx_array* beta, double eps, const hipcx_array* y, const hipcx_array* mean,
                                const hipcx_array* inv_std, void* stream) {
    return Guard([&] {
        RequireInput(x);
        RequireResult(y, x, "y");
        HIPCX_REQUIRE(IsContiguous(y), HIPCX_DIMENSION_ERROR, "layer_norm: y must be C-contiguous");
        RequireStats(mean, x, "mean");
        RequireStats(inv_std, x, "inv_std");
        int params = 0;
        RequireWeights(gamma, x, params, "gamma");
        RequireWeights(beta, x, params, "beta");
        HIPCX_REQUIRE(eps >= 0 && eps < HUGE_VAL, HIPCX_CHAINERX_ERROR, "layer_norm: eps must be finite and not negative");
        NormArgs p{};
        p.x_pitch = PitchOf(x, "x");
        p.rows = RowsOfAll(x), p.cols = x->shape[x->ndim - 1], p.eps = eps;
        HIPCX_REQUIRE(p.cols > 0, HIPCX_DIMENSION_ERROR, "layer_norm: rows without elements have no mean");
        if (p.rows == 0) return;
        p.x = x->data, p.out = y->data, p.mean = mean->data, p.inv_std = inv_std->data;
        p.gamma = gamma != nullptr ? gamma->data : nullptr;
        p.beta = beta != nullptr ? beta->data : nullptr;
        const NormPlan plan = PlanNorm(p.cols, ItemSize(x->dtype));
        VisitNormTypes(x->dtype, params, [&](auto tx, auto tp) {
            using T = typename decltype(tx)::type;
            using P = typename decltype(tp)::type;
            if (plan.threads == 0) {
                hipLaunchKernelGGL((LayerNormLongKernel<T, P>), dim3(static_cast<unsigned>(std::min<int64_t>(p.rows, 1 << 20))), dim3(1024), 0, AsStream(stream), p);
            } else {
                VisitNorm(plan, [&](auto g, auto v, auto narrow) {
                    constexpr int G = decltype(g)::value, V = decltype(v)::value, threads = G > 256 ? G : 256, groups = threads / G;
                    const auto launch = [&](auto at_once) {
                        constexpr int R = decltype(at_once)::value;
                        const int64_t blocks = (p.rows + groups * R - 1) / (groups * R);
                        HIPCX_REQUIRE(blocks <= kBlocksPerLaunch, HIPCX_NOT_IMPLEMENTED_ERROR, "layer_norm: too many rows");
                        hipLaunchKernelGGL((LayerNormKernel<T, P, G, V, R, decltype(narrow)::value>), dim3(static_cast<unsigned>(blocks)), dim3(threads), 0, AsStream(stream), p);
                    };
                    constexpr int most = G == 1024 ? 1 : RowsAtOnce(V * kPieceOf<T> * static_cast<int>(sizeof(NormCompute<T>)) / 4, 64);
                    if (p.rows >= int64_t{4} * most * groups * NumCUs()) launch(std::integral_constant<int, most>{});
                    else launch(std::integral_constant<int, 1>{});
                });
            }
            CheckLaunch("layer_norm");
        });
    });
}

extern "C" size_t hipcx_layer_norm_grad_workspace_size(const hipcx_array* x) {
    size_t n = 0;
    Guard([&] {
        RequireInput(x);
        const int64_t rows = RowsOfAll(x), cols = x->shape[x->ndim - 1];
        if (rows <= 0 || cols <= 0 || cols >= (int64_t{1} << 40)) return;
        n = static_cast<size_t>(GradWorkgroups(rows, cols, ItemSize(x->dtype)) * 2 * cols * ItemSize(StatDtype(x->dtype)));
    });
    return n;
}

extern "C" int hipcx_layer_norm_grad(const hipcx_array* x, const hipcx_array* gamma, const hipcx_array* gy, const hipcx_array* mean, const hipcx_array* inv_std,
                                     const hipcx_array* gx, const hipcx_array* ggamma, const hipcx_array* gbeta, void* workspace, size_t workspace_bytes, void* stream) {
    return Guard([&] {
        RequireInput(x);
        RequireResult(gy, x, "gy");
        RequireResult(gx, x, "gx");
        HIPCX_REQUIRE(IsContiguous(gx), HIPCX_DIMENSION_ERROR, "layer_norm: gx must be C-contiguous");
        RequireStats(mean, x, "mean");
        RequireStats(inv_std, x, "inv_std");
        int params = 0;
        RequireWeights(gamma, x, params, "gamma");
        RequireWeights(ggamma, x, params, "ggamma");
        RequireWeights(gbeta, x, params, "gbeta");
        NormArgs p{};
        p.x_pitch = PitchOf(x, "x"), p.gy_pitch = PitchOf(gy, "gy");
        p.rows = RowsOfAll(x), p.cols = x->shape[x->ndim - 1];
        HIPCX_REQUIRE(p.cols > 0, HIPCX_DIMENSION_ERROR, "layer_norm: rows without elements have no mean");
        p.weights = ggamma != nullptr || gbeta != nullptr;
        const int64_t item = ItemSize(x->dtype), parts = p.rows == 0 ? 0 : GradWorkgroups(p.rows, p.cols, item);
        const size_t need = static_cast<size_t>(parts * 2 * p.cols * ItemSize(StatDtype(x->dtype)));
        if (p.weights && need > 0) {
            HIPCX_REQUIRE(workspace != nullptr && workspace_bytes >= need, HIPCX_CHAINERX_ERROR, "layer_norm_grad workspace too small: need " + std::to_string(need) + " bytes");
            HIPCX_REQUIRE(reinterpret_cast<uintptr_t>(workspace) % 16 == 0, HIPCX_CHAINERX_ERROR, "workspace must be 16-byte aligned");
        }
        p.x = x->data, p.gy = gy->data, p.out = gx->data, p.mean = mean->data, p.inv_std = inv_std->data, p.partial = workspace;
        p.gamma = gamma != nullptr ? gamma->data : nullptr;
        const NormPlan plan = PlanNorm(p.cols, item);
        VisitNormTypes(x->dtype, params, [&](auto tx, auto tp) {
            using T = typename decltype(tx)::type;
            using P = typename decltype(tp)::type;
            using C = NormCompute<T>;
            if (p.rows > 0 && plan.threads == 0) {
                hipLaunchKernelGGL((LayerNormGradLongKernel<T, P>), dim3(static_cast<unsigned>(std::min<int64_t>(p.rows, 1 << 20))), dim3(1024), 0, AsStream(stream), p);
                CheckLaunch("layer_norm_grad");
                if (p.weights) {
                    hipLaunchKernelGGL((LayerNormColumnsKernel<T>), dim3(static_cast<unsigned>((p.cols + 255) / 256), static_cast<unsigned>(parts)), dim3(256), 0, AsStream(stream), p,
                                       (p.rows + parts - 1) / parts);
                    CheckLaunch("layer_norm_grad");
                }
            } else if (p.rows > 0) {
                VisitNorm(plan, [&](auto g, auto v, auto narrow) {
                    constexpr int G = decltype(g)::value, V = decltype(v)::value, threads = G > 256 ? G : 256, groups = threads / G;
                    constexpr int most = G == 1024 ? 1 : RowsAtOnce(V * kPieceOf<T> * static_cast<int>(sizeof(NormCompute<T>)) / 4, 32);
                    if (p.rows >= int64_t{4} * most * groups * parts)
                        hipLaunchKernelGGL((LayerNormGradKernel<T, P, G, V, most, decltype(narrow)::value>), dim3(static_cast<unsigned>(parts)), dim3(threads), 0, AsStream(stream), p);
                    else
                        hipLaunchKernelGGL((LayerNormGradKernel<T, P, G, V, 1, decltype(narrow)::value>), dim3(static_cast<unsigned>(parts)), dim3(threads), 0, AsStream(stream), p);
                });
                CheckLaunch("layer_norm_grad");
            }
            if (p.weights) {
                const auto sum = [&](auto columns) {
                    constexpr int COLS = decltype(columns)::value;
                    hipLaunchKernelGGL((LayerNormSumKernel<C, P, COLS>), dim3(static_cast<unsigned>((p.cols + COLS - 1) / COLS)), dim3(256), 0, AsStream(stream), static_cast<const C*>(workspace), parts,
                                       p.cols, ggamma != nullptr ? static_cast<P*>(ggamma->data) : nullptr, gbeta != nullptr ? static_cast<P*>(gbeta->data) : nullptr);
                };
                // few columns are spread over more workgroups (650 columns: 7.6 -> 4.0 us), many are read in whole lines (4096 columns: 12.4 -> 7.6 us)
                if (p.cols < 2048) sum(std::integral_constant<int, 8>{});
                else sum(std::integral_constant<int, 32>{});
                CheckLaunch("layer_norm_grad");
            }
        });
    });
}
