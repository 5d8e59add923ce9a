// A short convolution of every channel along time that sees the past alone, with the rows that a sequence's next piece needs, and its gradients.
#include "sequence.h"

namespace hipcx {
namespace {

constexpr int kMaxTaps = 8;

struct ConvArgs {
    SequenceRows x, y, state, new_state;  // state and new_state: taps - 1 rows, the oldest first
    SequenceRows gy, gnew, gx, gstate;
    const void *w, *b;  // [channels][taps], [channels] or null
    float* parts;       // gradients of w and b by parts, [part][taps + 1][channels]
    SequenceLengths lengths;
    int64_t batch, length, channels;
    int64_t first;        // the launch's first thread
    int pieces, chunks;   // of 16 bytes of a row, of rows
    int rows;             // to a chunk, taps - 1 at least where there is more than one
    int piece_bits;       // gradients: log2 of the pieces that a workgroup spans
    int silu;
};

template <typename T>
struct __attribute__((packed, aligned(alignof(T)))) Piece {
    static constexpr int kSize = 16 / sizeof(T);
    T v[kSize];
};

// `n` channels of a row, all of them in one access.
template <typename T>
__device__ __forceinline__ Piece<T> LoadPiece(const T* p, int n) {
    if (n >= Piece<T>::kSize) return *reinterpret_cast<const Piece<T>*>(p);
    Piece<T> v{};
#pragma unroll
    for (int e = 0; e < Piece<T>::kSize; ++e) {
        if (e < n) v.v[e] = p[e];
    }
    return v;
}
template <typename T>
__device__ __forceinline__ void StorePiece(T* p, const Piece<T>& v, int n) {
    if (n >= Piece<T>::kSize) {
        *reinterpret_cast<Piece<T>*>(p) = v;
        return;
    }
#pragma unroll
    for (int e = 0; e < Piece<T>::kSize; ++e) {
        if (e < n) p[e] = v.v[e];
    }
}

template <typename T>
__device__ __forceinline__ T* RowOf(const SequenceRows& r, int64_t b, int64_t row, int64_t channel) {
    return static_cast<T*>(r.data) + b * r.batch + row * r.row + channel;
}

// Row `i` of the state and x behind it.
template <typename T, int K>
__device__ __forceinline__ Piece<T> InputRow(const ConvArgs& p, int64_t b, int64_t i, int64_t channel, int n) {
    if (i >= K - 1) return LoadPiece(RowOf<T>(p.x, b, i - (K - 1), channel), n);
    if (p.state.data == nullptr) return Piece<T>{};
    return LoadPiece(RowOf<T>(p.state, b, i, channel), n);
}

template <typename T, int K>
struct Filter {
    T w[Piece<T>::kSize][K];
    T b[Piece<T>::kSize];
    __device__ __forceinline__ Filter(const ConvArgs& p, int64_t channel, int n) {
        const T* const from = static_cast<const T*>(p.w) + channel * K;
        const T* const bias = static_cast<const T*>(p.b);
#pragma unroll
        for (int e = 0; e < Piece<T>::kSize; ++e) {
#pragma unroll
            for (int k = 0; k < K; ++k) w[e][k] = e < n ? from[e * K + k] : static_cast<T>(0);
            b[e] = bias != nullptr && e < n ? bias[channel + e] : static_cast<T>(0);
        }
    }
    // The sum of `window`'s rows `at` to at + K - 1, in 32 bits.
    template <int N>
    __device__ __forceinline__ float Sum(const Piece<T> (&window)[N], int at, int e) const {
        float s = static_cast<float>(b[e]);
#pragma unroll
        for (int k = 0; k < K; ++k) s = __builtin_fmaf(static_cast<float>(w[e][k]), static_cast<float>(window[at + k].v[e]), s);
        return s;
    }
};

constexpr int kAhead = 8;  // rows whose loads are issued together

template <typename T, int K>
__global__ __launch_bounds__(256) void CausalConvKernel(ConvArgs p) {
    constexpr int E = Piece<T>::kSize;
    const int64_t index = p.first + static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
    if (index >= p.batch * p.chunks * p.pieces) return;
    const unsigned line = static_cast<unsigned>(index) / static_cast<unsigned>(p.pieces), piece = static_cast<unsigned>(index) % static_cast<unsigned>(p.pieces);
    const int64_t b = line / static_cast<unsigned>(p.chunks), t0 = static_cast<int64_t>(line % static_cast<unsigned>(p.chunks)) * p.rows, channel = static_cast<int64_t>(piece) * E;
    const int n = static_cast<int>(std::min<int64_t>(E, p.channels - channel));
    const int64_t len = LengthOf(p.lengths, b, p.length), end = std::min(t0 + p.rows, p.length);
    const Filter<T, K> f(p, channel, n);
    Piece<T> window[K - 1 + kAhead];
#pragma unroll
    for (int j = 0; j < K - 1; ++j) window[j] = t0 + j < len + K - 1 ? InputRow<T, K>(p, b, t0 + j, channel, n) : Piece<T>{};
    for (int64_t t = t0; t < end; t += kAhead) {
#pragma unroll
        for (int j = 0; j < kAhead; ++j) {
            window[K - 1 + j] = Piece<T>{};
            if (t + j < len && t + j < end) window[K - 1 + j] = LoadPiece(RowOf<T>(p.x, b, t + j, channel), n);
        }
#pragma unroll
        for (int j = 0; j < kAhead; ++j) {
            if (t + j >= end) break;
            Piece<T> y{};
            if (t + j < len) {
#pragma unroll
                for (int e = 0; e < E; ++e) {
                    const float s = f.Sum(window, j, e);
                    y.v[e] = static_cast<T>(p.silu != 0 ? s * LogisticOf(s) : s);
                }
            }
            StorePiece(RowOf<T>(p.y, b, t + j, channel), y, n);
        }
#pragma unroll
        for (int j = 0; j < K - 1; ++j) window[j] = window[kAhead + j];
    }
    // new_state may be state: the only thread that reads these channels of it moves its rows forward, the first one first
    if (t0 == 0) {
        for (int j = 0; j < K - 1; ++j) StorePiece(RowOf<T>(p.new_state, b, j, channel), InputRow<T, K>(p, b, len + j, channel, n), n);
    }
}

// gp = gy act'(sum) where a row counts, else 0.  The gradient of input row i (state and x behind it) is w[k] gp[i - k] summed over the taps: a thread
// goes through its rows and taps - 1 more, computes every sum again from x, and is done with input row i as soon as it has gp[i].
template <typename T, int K>
__global__ __launch_bounds__(256) void CausalConvGradKernel(ConvArgs p) {
    constexpr int E = Piece<T>::kSize, kRows = 4;
    __shared__ float sums[256 * E];
    const int span = 1 << p.piece_bits, lines = 256 >> p.piece_bits;
    const unsigned piece_blocks = (static_cast<unsigned>(p.pieces) + span - 1) >> p.piece_bits;
    const unsigned part = blockIdx.x / piece_blocks, piece_block = blockIdx.x % piece_blocks;
    const int64_t piece = static_cast<int64_t>(piece_block) * span + (threadIdx.x & (span - 1));
    const int64_t line = static_cast<int64_t>(part) * lines + (threadIdx.x >> p.piece_bits);
    const int64_t b = line / p.chunks, t0 = line % p.chunks * p.rows, channel = piece * E;
    float gw[E][K] = {}, gb[E] = {};
    if (piece < p.pieces && b < p.batch) {
        const int n = static_cast<int>(std::min<int64_t>(E, p.channels - channel));
        const int64_t len = LengthOf(p.lengths, b, p.length), end = std::min(t0 + p.rows, p.length);
        const Filter<T, K> f(p, channel, n);
        Piece<T> window[K - 1 + kRows];
        float gp[K - 1 + kRows][E] = {};
#pragma unroll
        for (int j = 0; j < K - 1; ++j) window[j] = t0 + j < len + K - 1 ? InputRow<T, K>(p, b, t0 + j, channel, n) : Piece<T>{};
        for (int64_t t = t0; t < end + K - 1; t += kRows) {
            Piece<T> gy[kRows];
#pragma unroll
            for (int j = 0; j < kRows; ++j) {
                window[K - 1 + j] = gy[j] = Piece<T>{};
                if (t + j < len && t + j < end + K - 1) {
                    window[K - 1 + j] = LoadPiece(RowOf<T>(p.x, b, t + j, channel), n);
                    gy[j] = LoadPiece(RowOf<T>(p.gy, b, t + j, channel), n);
                }
            }
#pragma unroll
            for (int j = 0; j < kRows; ++j) {
                const int64_t row = t + j;
#pragma unroll
                for (int e = 0; e < E; ++e) {
                    float g = 0.f;
                    if (row < len) {
                        g = static_cast<float>(gy[j].v[e]);
                        if (p.silu != 0) {
                            const float s = f.Sum(window, j, e), l = LogisticOf(s);
                            g *= l * __builtin_fmaf(s, 1.f - l, 1.f);
                        }
                    }
                    gp[K - 1 + j][e] = g;
                    if (row < end && row < len) {
                        gb[e] += g;
#pragma unroll
                        for (int k = 0; k < K; ++k) gw[e][k] = __builtin_fmaf(g, static_cast<float>(window[j + k].v[e]), gw[e][k]);
                    }
                }
                const bool of_state = row < K - 1;  // t0 is 0 there, or the row belongs to the chunk before
                if (row < end + K - 1 && row >= (t0 == 0 ? 0 : t0 + K - 1) && (!of_state || p.gstate.data != nullptr)) {
                    Piece<T> g{}, last{};
                    const bool ends = p.gnew.data != nullptr && row >= len && row < len + K - 1;
                    if (ends) last = LoadPiece(RowOf<T>(p.gnew, b, row - len, channel), n);
#pragma unroll
                    for (int e = 0; e < E; ++e) {
                        float s = static_cast<float>(last.v[e]);
#pragma unroll
                        for (int k = 0; k < K; ++k) s = __builtin_fmaf(static_cast<float>(f.w[e][k]), gp[K - 1 + j - k][e], s);
                        g.v[e] = static_cast<T>(s);
                    }
                    StorePiece(of_state ? RowOf<T>(p.gstate, b, row, channel) : RowOf<T>(p.gx, b, row - (K - 1), channel), g, n);
                }
            }
#pragma unroll
            for (int j = 0; j < K - 1; ++j) {
                window[j] = window[kRows + j];
#pragma unroll
                for (int e = 0; e < E; ++e) gp[j][e] = gp[kRows + j][e];
            }
        }
    }
    // the lines of a workgroup are added up one after another, the same way every time
#pragma unroll
    for (int k = 0; k <= K; ++k) {
        __syncthreads();
#pragma unroll
        for (int e = 0; e < E; ++e) sums[threadIdx.x * E + e] = k < K ? gw[e][k < K ? k : 0] : gb[e];
        __syncthreads();
        for (int c = threadIdx.x; c < span * E; c += 256) {
            const int64_t at = static_cast<int64_t>(piece_block) * span * E + c;
            if (at >= p.channels) continue;
            float s = 0.f;
            for (int i = 0; i < lines; ++i) s += sums[i * span * E + c];
            p.parts[(static_cast<int64_t>(part) * (K + 1) + k) * p.channels + at] = s;
        }
    }
}

// A column of partial sums to a thread, four threads to a column.
template <typename T>
__global__ __launch_bounds__(256) void CausalConvSumKernel(const float* parts, int64_t n_parts, int64_t channels, int taps, T* gw, T* gb) {
    __shared__ float sums[256];
    const int64_t width = (taps + 1) * channels, c = static_cast<int64_t>(blockIdx.x) * 64 + (threadIdx.x & 63);
    float s = 0.f;
    if (c < width) {
        for (int64_t i = threadIdx.x >> 6; i < n_parts; i += 4) s += parts[i * width + c];
    }
    sums[threadIdx.x] = s;
    __syncthreads();
    if (threadIdx.x >= 64 || c >= width) return;
    const float all = (sums[threadIdx.x] + sums[threadIdx.x + 64]) + (sums[threadIdx.x + 128] + sums[threadIdx.x + 192]);
    const int64_t k = c / channels, channel = c % channels;
    if (k < taps) gw[channel * taps + k] = static_cast<T>(all);
    else if (gb != nullptr) gb[channel] = static_cast<T>(all);
}

// Rows to a chunk: `most`, or the fewest powers of two of it that leave every compute unit four waves, down to the rows whose loads are issued together.
int ChunkRows(int64_t length, int64_t lines, int most) {
    int rows = most;
    while (rows > kAhead && lines * ((length + rows - 1) / rows) < int64_t{NumCUs()} * 1024) rows /= 2;
    return rows;
}

constexpr int kGradRows = 64;

int GradPieceBits(int64_t pieces) {
    int bits = 0;
    while (bits < 6 && (int64_t{1} << bits) < pieces) ++bits;
    return bits;
}

struct ConvSizes {
    int64_t batch, length, channels, taps, pieces;
    ConvSizes(const hipcx_array* x, const hipcx_array* w) : batch(x->shape[0]), length(x->shape[1]), channels(x->shape[2]), taps(w->shape[1]) {
        const int64_t each = 16 / ItemSize(x->dtype);
        pieces = (channels + each - 1) / each;
    }
    int64_t GradChunks() const {
        const int rows = ChunkRows(length, batch * pieces, kGradRows);
        return std::max<int64_t>(1, (length + rows - 1) / rows);
    }
    int64_t GradParts() const {
        const int lines = 256 >> GradPieceBits(pieces);
        return (batch * GradChunks() + lines - 1) / lines;
    }
};

void RequireConv(const hipcx_array* x, const hipcx_array* w, const char* name) {
    const std::string what = name;
    ValidateArray(x, "x");
    ValidateArray(w, "w");
    HIPCX_REQUIRE(x->dtype == HIPCX_FLOAT16 || x->dtype == HIPCX_FLOAT32, HIPCX_DTYPE_ERROR, what + ": float16 and float32 only, got " + DtypeName(x->dtype));
    HIPCX_REQUIRE(x->ndim == 3, HIPCX_DIMENSION_ERROR, what + ": x must be [batch, time, channels], got " + ShapeStr(x));
    HIPCX_REQUIRE(w->ndim == 2 && w->shape[0] == x->shape[2], HIPCX_DIMENSION_ERROR, what + ": w must be [channels, taps], got " + ShapeStr(w));
    HIPCX_REQUIRE(w->shape[1] >= 1 && w->shape[1] <= kMaxTaps, HIPCX_NOT_IMPLEMENTED_ERROR, what + ": 1 to 8 taps, got " + std::to_string(w->shape[1]));
    HIPCX_REQUIRE(w->dtype == x->dtype, HIPCX_DTYPE_ERROR, what + ": x and w must share a dtype");
    RequireDense(w, what + ": w");
}

template <typename F>
void VisitConv(int dtype, int64_t taps, F&& f) {
    const auto visit = [&](auto tag) {
        switch (taps) {
            case 1: f(tag, std::integral_constant<int, 1>{}); break;
            case 2: f(tag, std::integral_constant<int, 2>{}); break;
            case 3: f(tag, std::integral_constant<int, 3>{}); break;
            case 4: f(tag, std::integral_constant<int, 4>{}); break;
            case 5: f(tag, std::integral_constant<int, 5>{}); break;
            case 6: f(tag, std::integral_constant<int, 6>{}); break;
            case 7: f(tag, std::integral_constant<int, 7>{}); break;
            default: f(tag, std::integral_constant<int, 8>{}); break;
        }
    };
    if (dtype == HIPCX_FLOAT16) visit(Tag<half_t>{});
    else visit(Tag<float>{});
}

}  // namespace
}  // namespace hipcx

using namespace hipcx;

extern "C" {

int hipcx_causal_conv(const hipcx_array* x, const hipcx_array* w, const hipcx_array* b, const hipcx_array* state, const hipcx_array* lengths, int activation,
                      const hipcx_array* y, const hipcx_array* new_state, void* stream) {
    return Guard([&] {
        RequireConv(x, w, "causal_conv");
        const ConvSizes s(x, w);
        HIPCX_REQUIRE(y != nullptr && new_state != nullptr, HIPCX_CHAINERX_ERROR, "causal_conv: y and new_state are needed");
        HIPCX_REQUIRE(activation == HIPCX_ACTIVATION_NONE || activation == HIPCX_ACTIVATION_SILU, HIPCX_CHAINERX_ERROR, "causal_conv: unknown activation");
        RequireShape(b, {s.channels}, x->dtype, "causal_conv: b");
        RequireShape(state, {s.batch, s.taps - 1, s.channels}, x->dtype, "causal_conv: state");
        RequireShape(new_state, {s.batch, s.taps - 1, s.channels}, x->dtype, "causal_conv: new_state");
        RequireShape(y, {s.batch, s.length, s.channels}, x->dtype, "causal_conv: y");
        RequireDense(b, "causal_conv: b");
        ConvArgs p{};
        p.x = RowsOf(x, "causal_conv: x"), p.state = RowsOf(state, "causal_conv: state");
        p.y = RowsOf(y, "causal_conv: y"), p.new_state = RowsOf(new_state, "causal_conv: new_state");
        p.lengths = LengthsOf(lengths, s.batch, "causal_conv");
        p.w = w->data, p.b = b != nullptr ? b->data : nullptr;
        p.batch = s.batch, p.length = s.length, p.channels = s.channels, p.silu = activation;
        if (s.batch == 0 || s.channels == 0) return;
        p.rows = ChunkRows(s.length, s.batch * s.pieces, 32);
        const int64_t chunks = std::max<int64_t>(1, (s.length + p.rows - 1) / p.rows), threads = s.batch * chunks * s.pieces;
        HIPCX_REQUIRE(threads < (int64_t{1} << 31), HIPCX_NOT_IMPLEMENTED_ERROR, "causal_conv: too many elements");
        p.pieces = static_cast<int>(s.pieces), p.chunks = static_cast<int>(chunks);
        VisitConv(x->dtype, s.taps, [&](auto tag, auto taps) {
            using T = typename decltype(tag)::type;
            ForLaunches(threads, [&](dim3 grid, int64_t first) {
                p.first = first;
                hipLaunchKernelGGL((CausalConvKernel<T, decltype(taps)::value>), grid, dim3(256), 0, AsStream(stream), p);
                CheckLaunch("causal_conv");
            });
        });
    });
}

size_t hipcx_causal_conv_grad_workspace_size(const hipcx_array* x, const hipcx_array* w) {
    if (x == nullptr || w == nullptr || x->ndim != 3 || w->ndim != 2 || (x->dtype != HIPCX_FLOAT16 && x->dtype != HIPCX_FLOAT32)) return 0;
    const ConvSizes s(x, w);
    if (s.batch <= 0 || s.channels <= 0) return 0;
    return static_cast<size_t>(s.GradParts() * (s.taps + 1) * s.channels) * sizeof(float);
}

int hipcx_causal_conv_grad(const hipcx_array* x, const hipcx_array* w, const hipcx_array* b, const hipcx_array* state, const hipcx_array* lengths, int activation,
                           const hipcx_array* gy, const hipcx_array* gnew_state, const hipcx_array* gx, const hipcx_array* gw, const hipcx_array* gb,
                           const hipcx_array* gstate, void* workspace, size_t workspace_bytes, void* stream) {
    return Guard([&] {
        RequireConv(x, w, "causal_conv_grad");
        const ConvSizes s(x, w);
        HIPCX_REQUIRE(gy != nullptr && gx != nullptr && gw != nullptr, HIPCX_CHAINERX_ERROR, "causal_conv_grad: gy, gx and gw are needed");
        HIPCX_REQUIRE(activation == HIPCX_ACTIVATION_NONE || activation == HIPCX_ACTIVATION_SILU, HIPCX_CHAINERX_ERROR, "causal_conv_grad: unknown activation");
        RequireShape(b, {s.channels}, x->dtype, "causal_conv_grad: b");
        RequireShape(gb, {s.channels}, x->dtype, "causal_conv_grad: gb");
        RequireShape(gw, {s.channels, s.taps}, x->dtype, "causal_conv_grad: gw");
        RequireShape(gy, {s.batch, s.length, s.channels}, x->dtype, "causal_conv_grad: gy");
        RequireShape(gx, {s.batch, s.length, s.channels}, x->dtype, "causal_conv_grad: gx");
        for (const hipcx_array* a : {state, gnew_state, gstate}) RequireShape(a, {s.batch, s.taps - 1, s.channels}, x->dtype, "causal_conv_grad: state and its gradients");
        for (const hipcx_array* a : {b, gb, gw}) RequireDense(a, "causal_conv_grad: b, gb and gw");
        ConvArgs p{};
        p.x = RowsOf(x, "causal_conv_grad: x"), p.state = RowsOf(state, "causal_conv_grad: state"), p.gy = RowsOf(gy, "causal_conv_grad: gy");
        p.gnew = RowsOf(gnew_state, "causal_conv_grad: gnew_state"), p.gx = RowsOf(gx, "causal_conv_grad: gx"), p.gstate = RowsOf(gstate, "causal_conv_grad: gstate");
        p.lengths = LengthsOf(lengths, s.batch, "causal_conv_grad");
        p.w = w->data, p.b = b != nullptr ? b->data : nullptr;
        p.batch = s.batch, p.length = s.length, p.channels = s.channels, p.silu = activation;
        if (s.channels == 0) return;
        const size_t need = hipcx_causal_conv_grad_workspace_size(x, w);
        HIPCX_REQUIRE(workspace_bytes >= need && (need == 0 || workspace != nullptr), HIPCX_CHAINERX_ERROR, "causal_conv_grad: the workspace is too small");
        p.parts = static_cast<float*>(workspace);
        const int64_t parts = s.batch == 0 ? 0 : s.GradParts();
        p.piece_bits = GradPieceBits(s.pieces);
        p.pieces = static_cast<int>(s.pieces), p.chunks = static_cast<int>(s.GradChunks());
        p.rows = ChunkRows(s.length, s.batch * s.pieces, kGradRows);
        const int64_t blocks = parts * ((s.pieces + (1 << p.piece_bits) - 1) >> p.piece_bits);
        HIPCX_REQUIRE(blocks <= kBlocksPerLaunch, HIPCX_NOT_IMPLEMENTED_ERROR, "causal_conv_grad: too many elements");
        VisitConv(x->dtype, s.taps, [&](auto tag, auto taps) {
            using T = typename decltype(tag)::type;
            if (blocks != 0) {
                hipLaunchKernelGGL((CausalConvGradKernel<T, decltype(taps)::value>), dim3(static_cast<unsigned>(blocks)), dim3(256), 0, AsStream(stream), p);
                CheckLaunch("causal_conv_grad");
            }
            const int64_t columns = (s.taps + 1) * s.channels;
            hipLaunchKernelGGL(CausalConvSumKernel<T>, dim3(static_cast<unsigned>((columns + 63) / 64)), dim3(256), 0, AsStream(stream), p.parts, parts, s.channels,
                               static_cast<int>(s.taps), static_cast<T*>(gw->data), static_cast<T*>(gb != nullptr ? gb->data : nullptr));
            CheckLaunch("causal_conv_grad");
        });
    });
}

}  // extern "C"
