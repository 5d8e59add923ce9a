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

// Sums over the G threads of a row, which all of them get.  Up to 64 are neighbours in a wave; more are the whole workgroup, whose waves' sums meet in `meet` (two halves in
// turn: a wave that is still reading one half is waited for at the barrier of the other).
template <int G, int N, typename C>
__device__ __forceinline__ void RowSum(C (&v)[N], C* meet, int& turn) {
#pragma unroll
    for (int o = 1; o < (G < 64 ? G : 64); o <<= 1) {
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] += __shfl_xor(v[i], o);
    }
    if constexpr (G > 64) {
        constexpr int W = G / 64;
        C* const at = meet + turn * (W * 2);
        turn ^= 1;
        if (threadIdx.x % 64 == 0) {
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

// A thread's pieces of a row: piece j of thread l covers columns (l + j G) E and on.  The row's last piece is moved back so that it is whole where the row has a whole piece at all;
// `lo` and `hi` tell which of its elements are this thread's to count.
template <typename T, int G>
struct RowPiece {
    static constexpr int E = kPieceOf<T>;
    int64_t at;
    int lo, hi;
    bool live, whole;
    __device__ __forceinline__ RowPiece(int l, int j, int64_t cols) {
        at = (static_cast<int64_t>(j) * G + l) * E;
        live = at < cols;
        lo = 0, hi = E;
        whole = cols >= E;
        if (live && at + E > cols) {
            if (whole) {
                lo = static_cast<int>(at + E - cols);
                at = cols - E;
            } else {
                hi = static_cast<int>(cols);
            }
        }
    }
    __device__ __forceinline__ bool Counts(int e) const { return live && e >= lo && e < hi; }
};

template <typename S, typename C, int E, typename Piece>
__device__ __forceinline__ void LoadPiece(const S* from, const Piece& p, C (&v)[E]) {
    if (!p.live) {
#pragma unroll
        for (int e = 0; e < E; ++e) v[e] = 0;
    } else if (p.whole) {
        const Elements<S, E> r = *reinterpret_cast<const Elements<S, E>*>(from + p.at);
#pragma unroll
        for (int e = 0; e < E; ++e) v[e] = static_cast<C>(r.v[e]);
    } else {
#pragma unroll
        for (int e = 0; e < E; ++e) v[e] = e < p.hi ? static_cast<C>(from[p.at + e]) : static_cast<C>(0);
    }
}

template <typename S, typename C, int E, typename Piece>
__device__ __forceinline__ void StorePiece(S* to, const Piece& p, const C (&v)[E]) {
    if (!p.live) return;
    if (p.whole) {
        Elements<S, E> r;
#pragma unroll
        for (int e = 0; e < E; ++e) r.v[e] = static_cast<S>(v[e]);
        *reinterpret_cast<Elements<S, E>*>(to + p.at) = r;
    } else {
#pragma unroll
        for (int e = 0; e < E; ++e) {
            if (e < p.hi) to[p.at + e] = static_cast<S>(v[e]);
        }
    }
}

// The first sum gives a mean that is off by its rounding, and the sum of the differences from it corrects both the mean and the variance: two passes over registers.
template <typename T, typename P, int G, int V>
__global__ __launch_bounds__(G > 256 ? G : 256) void LayerNormKernel(NormArgs p) {
    using C = NormCompute<T>;
    constexpr int E = kPieceOf<T>, THREADS = G > 256 ? G : 256, ROWS = THREADS / G;
    __shared__ C meet[2 * 2 * (THREADS / 64)];
    const int l = threadIdx.x % G;
    const C n = static_cast<C>(p.cols);
    int turn = 0;
    for (int64_t row = static_cast<int64_t>(blockIdx.x) * ROWS + threadIdx.x / G; row < p.rows; row += static_cast<int64_t>(gridDim.x) * ROWS) {
        const T* const x = static_cast<const T*>(p.x) + row * p.x_pitch;
        C v[V][E], sum[1] = {0};
#pragma unroll
        for (int j = 0; j < V; ++j) LoadPiece(x, RowPiece<T, G>(l, j, p.cols), v[j]);
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const RowPiece<T, G> piece(l, j, p.cols);
            if (static_cast<int64_t>(j + 1) * G * E <= p.cols) {
#pragma unroll
                for (int e = 0; e < E; ++e) sum[0] += v[j][e];
            } else {
#pragma unroll
                for (int e = 0; e < E; ++e) sum[0] += piece.Counts(e) ? v[j][e] : static_cast<C>(0);
            }
        }
        RowSum<G>(sum, meet, turn);
        const C about = sum[0] / n;
        C more[2] = {0, 0};
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const RowPiece<T, G> piece(l, j, p.cols);
            if (static_cast<int64_t>(j + 1) * G * E <= p.cols) {
#pragma unroll
                for (int e = 0; e < E; ++e) {
                    v[j][e] -= about;
                    more[0] += v[j][e];
                    more[1] = __builtin_elementwise_fma(v[j][e], v[j][e], more[1]);
                }
            } else {
#pragma unroll
                for (int e = 0; e < E; ++e) {
                    v[j][e] -= about;
                    const C d = piece.Counts(e) ? v[j][e] : static_cast<C>(0);
                    more[0] += d;
                    more[1] = __builtin_elementwise_fma(d, d, more[1]);
                }
            }
        }
        RowSum<G>(more, meet, turn);
        const C off = more[0] / n;
        C var = more[1] / n - off * off;
        var = var < 0 ? static_cast<C>(0) : var;
        const C inv = static_cast<C>(1) / static_cast<C>(sqrt(var + static_cast<C>(p.eps)));
        if (l == 0) {
            static_cast<C*>(p.mean)[row] = about + off;
            static_cast<C*>(p.inv_std)[row] = inv;
        }
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const RowPiece<T, G> piece(l, j, p.cols);
            C gamma[E], beta[E];
            if (p.gamma != nullptr) LoadPiece(static_cast<const P*>(p.gamma), piece, gamma);
            if (p.beta != nullptr) LoadPiece(static_cast<const P*>(p.beta), piece, beta);
#pragma unroll
            for (int e = 0; e < E; ++e) {
                C y = (v[j][e] - off) * inv;
                if (p.gamma != nullptr) y *= gamma[e];
                if (p.beta != nullptr) y += beta[e];
                v[j][e] = y;
            }
            StorePiece(static_cast<T*>(p.out) + row * p.cols, piece, v[j]);
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
        C sum[1] = {0}, more[2] = {0, 0};
        for (int64_t i = threadIdx.x; i < p.cols; i += 1024) sum[0] += static_cast<C>(x[i]);
        RowSum<1024>(sum, meet, turn);
        const C about = sum[0] / n;
        for (int64_t i = threadIdx.x; i < p.cols; i += 1024) {
            const C d = static_cast<C>(x[i]) - about;
            more[0] += d;
            more[1] = __builtin_elementwise_fma(d, d, more[1]);
        }
        RowSum<1024>(more, meet, turn);
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

// A row's two sums, then its gradients; a thread keeps its columns' sums over the rows that its workgroup walks through.
template <typename T, typename P, int G, int V>
__global__ __launch_bounds__(G > 256 ? G : 256) void LayerNormGradKernel(NormArgs p) {
    using C = NormCompute<T>;
    constexpr int E = kPieceOf<T>, THREADS = G > 256 ? G : 256, ROWS = THREADS / G;
    __shared__ C meet[2 * 2 * (THREADS / 64)];
    __shared__ C shared_sums[ROWS > 1 ? 2 * G * V * E : 1];
    const int l = threadIdx.x % G;
    const C n = static_cast<C>(p.cols);
    int turn = 0;
    C of_gamma[V][E], of_beta[V][E];
#pragma unroll
    for (int j = 0; j < V; ++j) {
#pragma unroll
        for (int e = 0; e < E; ++e) of_gamma[j][e] = of_beta[j][e] = 0;
    }
    for (int64_t row = static_cast<int64_t>(blockIdx.x) * ROWS + threadIdx.x / G; row < p.rows; row += static_cast<int64_t>(gridDim.x) * ROWS) {
        const T* const x = static_cast<const T*>(p.x) + row * p.x_pitch;
        const T* const gy = static_cast<const T*>(p.gy) + row * p.gy_pitch;
        const C mean = static_cast<const C*>(p.mean)[row], inv = static_cast<const C*>(p.inv_std)[row];
        C xh[V][E], g[V][E], sum[2] = {0, 0};
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const RowPiece<T, G> piece(l, j, p.cols);
            LoadPiece(x, piece, xh[j]);
            LoadPiece(gy, piece, g[j]);
        }
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const RowPiece<T, G> piece(l, j, p.cols);
            C gamma[E];
            if (p.gamma != nullptr) LoadPiece(static_cast<const P*>(p.gamma), piece, gamma);
            const bool all = static_cast<int64_t>(j + 1) * G * E <= p.cols;
#pragma unroll
            for (int e = 0; e < E; ++e) {
                xh[j][e] = (xh[j][e] - mean) * inv;
                of_gamma[j][e] = __builtin_elementwise_fma(g[j][e], xh[j][e], of_gamma[j][e]);
                of_beta[j][e] += g[j][e];
                if (p.gamma != nullptr) g[j][e] *= gamma[e];
            }
            if (all) {
#pragma unroll
                for (int e = 0; e < E; ++e) {
                    sum[0] += g[j][e];
                    sum[1] = __builtin_elementwise_fma(g[j][e], xh[j][e], sum[1]);
                }
            } else {
#pragma unroll
                for (int e = 0; e < E; ++e) {
                    if (!piece.Counts(e)) continue;
                    sum[0] += g[j][e];
                    sum[1] = __builtin_elementwise_fma(g[j][e], xh[j][e], sum[1]);
                }
            }
        }
        RowSum<G>(sum, meet, turn);
        const C a = sum[0] / n, b = sum[1] / n;
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const RowPiece<T, G> piece(l, j, p.cols);
#pragma unroll
            for (int e = 0; e < E; ++e) g[j][e] = inv * (g[j][e] - a - xh[j][e] * b);
            StorePiece(static_cast<T*>(p.out) + row * p.cols, piece, g[j]);
        }
    }
    if (!p.weights) return;
    C* const to = static_cast<C*>(p.partial) + static_cast<int64_t>(blockIdx.x) * 2 * p.cols;
    if constexpr (ROWS == 1) {
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const RowPiece<T, G> piece(l, j, p.cols);
#pragma unroll
            for (int e = 0; e < E; ++e) {
                if (piece.Counts(e)) to[piece.at + e] = of_gamma[j][e], to[p.cols + piece.at + e] = of_beta[j][e];
            }
        }
    } else {
        constexpr int WIDTH = G * V * E;
        for (int r = 0; r < ROWS; ++r) {  // one of the rows' threads after another: the order of the sums is always the same
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
                const RowPiece<T, G> piece(l, j, p.cols);
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
        RowSum<1024>(sum, meet, turn);
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

// Partial sums of workgroups -> gradients, added up in 64 bits: 32 columns to a workgroup, eight slices of the partial sums.
template <typename C, typename P>
__global__ __launch_bounds__(256) void LayerNormSumKernel(const C* partial, int64_t parts, int64_t cols, P* ggamma, P* gbeta) {
    __shared__ double sums[8][2][32];
    const int c = threadIdx.x % 32, s = threadIdx.x / 32;
    const int64_t i = static_cast<int64_t>(blockIdx.x) * 32 + c;
    double of_gamma = 0, of_beta = 0;
    if (i < cols) {
#pragma unroll 4
        for (int64_t k = s; k < parts; k += 8) {
            of_gamma += partial[k * 2 * cols + i];
            of_beta += partial[(k * 2 + 1) * cols + i];
        }
    }
    sums[s][0][c] = of_gamma, sums[s][1][c] = of_beta;
    __syncthreads();
    if (s < 2 && i < cols) {
        double v = 0;
#pragma unroll
        for (int k = 0; k < 8; ++k) v += sums[k][s][c];
        P* const to = s == 0 ? ggamma : gbeta;
        if (to != nullptr) to[i] = static_cast<P>(static_cast<C>(v));
    }
}

// ---------------------------------------------------------------------------------------------
// host
// ---------------------------------------------------------------------------------------------
// Threads of a row and pieces of each: the least that hold it, 0 threads for rows that nothing holds.
struct NormPlan {
    int threads, pieces;
};

NormPlan PlanNorm(int64_t cols, int64_t item) {
    const int64_t pieces = (cols * item + 15) / 16;
    for (const NormPlan plan : {NormPlan{16, 1}, {16, 2}, {64, 1}, {64, 2}, {64, 4}, {256, 2}, {256, 4}, {1024, 4}}) {
        if (pieces <= static_cast<int64_t>(plan.threads) * plan.pieces) return plan;
    }
    return {0, 0};
}

template <typename F>
void VisitNorm(NormPlan plan, F&& f) {
    const auto is = [&](int threads, int pieces) { return plan.threads == threads && plan.pieces == pieces; };
    if (is(16, 1)) f(std::integral_constant<int, 16>{}, std::integral_constant<int, 1>{});
    else if (is(16, 2)) f(std::integral_constant<int, 16>{}, std::integral_constant<int, 2>{});
    else if (is(64, 1)) f(std::integral_constant<int, 64>{}, std::integral_constant<int, 1>{});
    else if (is(64, 2)) f(std::integral_constant<int, 64>{}, std::integral_constant<int, 2>{});
    else if (is(64, 4)) f(std::integral_constant<int, 64>{}, std::integral_constant<int, 4>{});
    else if (is(256, 2)) f(std::integral_constant<int, 256>{}, std::integral_constant<int, 2>{});
    else if (is(256, 4)) f(std::integral_constant<int, 256>{}, std::integral_constant<int, 4>{});
    else f(std::integral_constant<int, 1024>{}, std::integral_constant<int, 4>{});
}

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
    for (int i = last - 1; i >= 0; --i) {
        if (x->shape[i] == 1) continue;
        if (expect == 0) {
            HIPCX_REQUIRE(x->strides[i] % it == 0, HIPCX_DIMENSION_ERROR, std::string("layer_norm: strides of ") + what + " must be whole elements");
            pitch = x->strides[i] / it;
        } else {
            HIPCX_REQUIRE(x->strides[i] == expect, HIPCX_DIMENSION_ERROR, std::string("layer_norm: rows of ") + what + " must be equally far apart");
        }
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
                VisitNorm(plan, [&](auto g, auto v) {
                    constexpr int G = decltype(g)::value, V = decltype(v)::value, threads = G > 256 ? G : 256;
                    const int64_t blocks = std::min<int64_t>((p.rows + threads / G - 1) / (threads / G), 1 << 20);
                    hipLaunchKernelGGL((LayerNormKernel<T, P, G, V>), dim3(static_cast<unsigned>(blocks)), dim3(threads), 0, AsStream(stream), p);
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
                VisitNorm(plan, [&](auto g, auto v) {
                    constexpr int G = decltype(g)::value, V = decltype(v)::value, threads = G > 256 ? G : 256;
                    hipLaunchKernelGGL((LayerNormGradKernel<T, P, G, V>), dim3(static_cast<unsigned>(parts)), dim3(threads), 0, AsStream(stream), p);
                });
                CheckLaunch("layer_norm_grad");
            }
            if (p.weights) {
                hipLaunchKernelGGL((LayerNormSumKernel<C, P>), dim3(static_cast<unsigned>((p.cols + 31) / 32)), dim3(256), 0, AsStream(stream), static_cast<const C*>(workspace), parts, p.cols,
                                   ggamma != nullptr ? static_cast<P*>(ggamma->data) : nullptr, gbeta != nullptr ? static_cast<P*>(gbeta->data) : nullptr);
                CheckLaunch("layer_norm_grad");
            }
        });
    });
}
