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
    int pieces, chunks;   // of a row's channels, of rows
    int rows;             // to a chunk, taps - 1 at least where there is more than one
    int piece_bits;       // gradients: log2 of the pieces that a workgroup spans
    int silu;
};

// E channels of a row, in one access at any address.
template <typename T, int E>
struct __attribute__((packed, aligned(alignof(T)))) Piece {
    T v[E];
};

template <typename T>
__device__ __forceinline__ T* RowOf(const SequenceRows& r, int64_t b, int64_t row, int64_t channel) {
    return static_cast<T*>(r.data) + b * r.batch + row * r.row + channel;
}

// A thread's part: E channels of a chunk of a sequence.  The last E channels of a row overlap those of the thread before where E does not divide the row, by `skip`:
// both compute these and store the same values, unless the state may have been moved forward under this one's reads, whose stores of them are left out then.
template <typename T, int K, int E>
struct ConvPart {
    using P = Piece<T, E>;
    const ConvArgs& p;
    int64_t b, t0, channel, len, end;
    int skip;
    float w[E][K], bias[E];

    __device__ __forceinline__ ConvPart(const ConvArgs& args, int64_t sequence, int64_t row, int64_t piece)
        : p(args), b(sequence), t0(row), channel(std::min(piece * E, args.channels - E)), len(LengthOf(args.lengths, sequence, args.length)),
          end(std::min(row + args.rows, args.length)), skip(static_cast<int>(piece * E - channel)) {
        const Piece<T, E * K> all = *reinterpret_cast<const Piece<T, E * K>*>(static_cast<const T*>(p.w) + channel * K);
        P of_bias{};
        if (p.b != nullptr) of_bias = *reinterpret_cast<const P*>(static_cast<const T*>(p.b) + channel);
#pragma unroll
        for (int i = 0; i < E * K; ++i) w[i / K][i % K] = static_cast<float>(all.v[i]);
#pragma unroll
        for (int e = 0; e < E; ++e) bias[e] = static_cast<float>(of_bias.v[e]);
    }
    __device__ __forceinline__ P Load(const SequenceRows& r, int64_t row) const { return *reinterpret_cast<const P*>(RowOf<T>(r, b, row, channel)); }
    __device__ __forceinline__ void Store(const SequenceRows& r, int64_t row, const P& v) const { *reinterpret_cast<P*>(RowOf<T>(r, b, row, channel)) = v; }
    __device__ __forceinline__ void StoreOwn(const SequenceRows& r, int64_t row, const P& v) const {
        T* const to = RowOf<T>(r, b, row, channel);
        if (skip == 0) {
            *reinterpret_cast<P*>(to) = v;
        } else {
#pragma unroll
            for (int e = 1; e < E; ++e) {
                if (e >= skip) to[e] = v.v[e];
            }
        }
    }
    // Row `i` of the state and x behind it.
    __device__ __forceinline__ P Input(int64_t i) const {
        P v{};
        if (i >= K - 1) v = Load(p.x, i - (K - 1));
        else if (p.state.data != nullptr) v = Load(p.state, i);
        return v;
    }
    // The taps - 1 rows before the chunk's first.
    template <int N>
    __device__ __forceinline__ void Before(P (&window)[N]) const {
#pragma unroll
        for (int j = 0; j < K - 1; ++j) {
            window[j] = P{};
            if (t0 + j < len + K - 1) window[j] = Input(t0 + j);
        }
    }
    // The sum of `window`'s rows `at` to at + K - 1, in 32 bits.
    template <int N>
    __device__ __forceinline__ float Sum(const P (&window)[N], int at, int e) const {
        float s = bias[e];
#pragma unroll
        for (int k = 0; k < K; ++k) s = __builtin_fmaf(static_cast<float>(window[at + k].v[e]), w[e][k], s);
        return s;
    }
};

// Bound by memory: x read once and y written once, beside taps - 1 rows of the chunk before.  A thread keeps its window in registers and walks down the rows of 16 bytes of
// channels, kAhead of whose loads are in flight.  A batch of 16 x 2048 x 4096 float16, four taps, SiLU: 107 us, 5.0 TB/s; with sequences half as long on average 89.  kAhead of 8:
// 110 and 94.  One token of 1300 channels 4.8 us, a launch and two trips to memory.  float16 windows of five taps take 146 registers (three waves), of six to eight 176 to 235 (two), and
// bound those by latency: 8 x 2048 x 2048 31 us with four taps, 35, 39, 43 and 46 with five to eight; float32 46 to 50.
constexpr int kAhead = 4;      // rows whose loads are issued together
constexpr int kFewestRows = 8; // to a chunk, taps - 1 at least

template <typename T, int K, int E>
__global__ __launch_bounds__(256, K <= 4 ? 4 : 2) void CausalConvKernel(ConvArgs p) {
    using P = Piece<T, E>;
    const int64_t index = p.first + static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
    if (index >= p.batch * p.chunks * p.pieces) return;
    const unsigned line = static_cast<unsigned>(index) / static_cast<unsigned>(p.pieces), piece = static_cast<unsigned>(index) % static_cast<unsigned>(p.pieces);
    const ConvPart<T, K, E> c(p, line / static_cast<unsigned>(p.chunks), static_cast<int64_t>(line % static_cast<unsigned>(p.chunks)) * p.rows, piece);
    const int64_t stop = std::min(c.end, c.len);
    P window[K - 1 + kAhead];
    c.Before(window);
    const auto row = [&](int64_t t, int j, auto own) __attribute__((always_inline)) {
        P y;
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const float s = c.Sum(window, j, e);
            y.v[e] = static_cast<T>(p.silu != 0 ? s * LogisticOf(s) : s);
        }
        if constexpr (decltype(own)::value) c.StoreOwn(p.y, t, y);
        else c.Store(p.y, t, y);
    };
    int64_t t = c.t0;
    // up to kAhead rows: a chunk's first ones and its last ones
    const auto edge = [&]() __attribute__((always_inline)) {
#pragma unroll
        for (int j = 0; j < kAhead; ++j) {
            P v{};
            if (t + j < stop) v = c.Load(p.x, t + j);
            window[K - 1 + j] = v;
        }
#pragma unroll
        for (int j = 0; j < kAhead; ++j) {
            if (t + j >= stop) break;
            row(t + j, j, std::true_type{});
        }
#pragma unroll
        for (int j = 0; j < K - 1; ++j) window[j] = window[kAhead + j];
        t += kAhead;
    };
    edge();
    if (K - 1 > kAhead && t < stop) edge();  // all rows whose sums take the state's in
    for (; t + kAhead <= stop; t += kAhead) {
#pragma unroll
        for (int j = 0; j < kAhead; ++j) window[K - 1 + j] = c.Load(p.x, t + j);
#pragma unroll
        for (int j = 0; j < kAhead; ++j) row(t + j, j, std::false_type{});
#pragma unroll
        for (int j = 0; j < K - 1; ++j) window[j] = window[kAhead + j];
    }
    if (t < stop) edge();
    for (t = std::max(c.t0, c.len); t < c.end; ++t) c.Store(p.y, t, P{});
    if (c.t0 == 0) {  // new_state may be state: this thread alone reads and writes these channels of it, all of them before it writes any
        P last[K];
#pragma unroll
        for (int j = 0; j < K - 1; ++j) last[j] = c.Input(c.len + j);
#pragma unroll
        for (int j = 0; j < K - 1; ++j) c.StoreOwn(p.new_state, j, last[j]);
    }
}

// gp = gy act'(sum) where a row counts, else 0.  The gradient of input row i (state and x behind it) is w[k] gp[i - k] summed over the taps: a thread
// goes through its rows and taps - 1 more, computes every sum again from x, and is done with input row i as soon as it has gp[i].  Bound by memory, x and gy in and gx out:
// 8 x 2048 x 2048 float16 50 to 55 us, 3.7 to 4.0 TB/s, of float32 87 us, 4.6.  Registers decide: 124 to 128 of them with four taps, four waves (4 spilled outside the rows in
// float16), where the compiler has no reason to hold more (blocks of rows with masks instead of single ones at the ends: 150 to 180, 62 to 69 us; held to 128 it spills in the rows, 300 to
// 490).  Five and six taps take 142 to 166, three waves, seven and eight 180 to 210, two: 64, 73, 88 and 97 us in float16, 100, 112, 110 and 117 in float32.
template <typename T, int K, int E>
__global__ __launch_bounds__(256, K <= 4 ? 4 : 2) void CausalConvGradKernel(ConvArgs p) {
    using P = Piece<T, E>;
    constexpr int kRows = 4;
    __shared__ float sums[256 * E];
    const int span = 1 << p.piece_bits, lines = 256 >> p.piece_bits;
    const unsigned piece_blocks = (static_cast<unsigned>(p.pieces) + span - 1) >> p.piece_bits;
    const unsigned part = blockIdx.x / piece_blocks, piece_block = blockIdx.x % piece_blocks;
    const int64_t piece = static_cast<int64_t>(piece_block) * span + (threadIdx.x & (span - 1));
    const int64_t line = static_cast<int64_t>(part) * lines + (threadIdx.x >> p.piece_bits);
    float gw[E][K] = {}, gb[E] = {};
    int skip = 0;
    if (piece < p.pieces && line < p.batch * p.chunks) {
        const ConvPart<T, K, E> c(p, line / p.chunks, line % p.chunks * p.rows, piece);
        skip = c.skip;
        P window[K - 1 + kRows], gy[kRows];
        float gp[K - 1 + kRows][E] = {};
        c.Before(window);
        // row j of the window: gp, and the row's share of the sums over rows
        const auto slope = [&](int j, bool own) __attribute__((always_inline)) {
#pragma unroll
            for (int e = 0; e < E; ++e) {
                float g = static_cast<float>(gy[j].v[e]);
                if (p.silu != 0) {
                    const float s = c.Sum(window, j, e), l = LogisticOf(s);
                    g *= l * __builtin_fmaf(s, 1.f - l, 1.f);
                }
                gp[K - 1 + j][e] = g;
                if (own) {
                    gb[e] += g;
#pragma unroll
                    for (int k = 0; k < K; ++k) gw[e][k] = __builtin_fmaf(static_cast<float>(window[j + k].v[e]), g, gw[e][k]);
                }
            }
        };
        const auto of_input = [&](int j, const P& last) __attribute__((always_inline)) {
            P g;
#pragma unroll
            for (int e = 0; e < E; ++e) {
                float s = static_cast<float>(last.v[e]);
#pragma unroll
                for (int k = 0; k < K; ++k) s = __builtin_fmaf(c.w[e][k], gp[K - 1 + j - k][e], s);
                g.v[e] = static_cast<T>(s);
            }
            return g;
        };
        const auto shift = [&](auto by) __attribute__((always_inline)) {
            constexpr int kBy = decltype(by)::value;
#pragma unroll
            for (int j = 0; j < K - 1; ++j) {
                window[j] = window[kBy + j];
#pragma unroll
                for (int e = 0; e < E; ++e) gp[j][e] = gp[kBy + j][e];
            }
        };
        // row by row where a sequence or a chunk begins or ends
        const auto single = [&](int64_t t) __attribute__((always_inline)) {
            const bool counts = t < c.len;
            P x{}, g{};
            if (counts) x = c.Load(p.x, t), g = c.Load(p.gy, t);
            window[K - 1] = x, gy[0] = g;
            slope(0, counts && t < c.end);
#pragma unroll
            for (int e = 0; e < E; ++e) gp[K - 1][e] = counts ? gp[K - 1][e] : 0.f;  // (whatever the rows before have made of the sum)
            const bool of_state = t < K - 1;  // of the first chunk: what comes before a later one's rows belongs to the chunk before
            if ((c.t0 == 0 || t >= c.t0 + K - 1) && (!of_state || p.gstate.data != nullptr)) {
                P last{};
                if (p.gnew.data != nullptr && t >= c.len && t < c.len + K - 1) last = c.Load(p.gnew, t - c.len);
                if (of_state) c.Store(p.gstate, t, of_input(0, last));
                else c.Store(p.gx, t - (K - 1), of_input(0, last));
            }
            shift(std::integral_constant<int, 1>{});
        };
        int64_t t = c.t0;
        for (const int64_t stop = std::min(c.t0, c.end) + K - 1; t < stop; ++t) single(t);
        for (const int64_t stop = std::min(c.end, c.len); t + kRows <= stop; t += kRows) {
#pragma unroll
            for (int j = 0; j < kRows; ++j) window[K - 1 + j] = c.Load(p.x, t + j), gy[j] = c.Load(p.gy, t + j);
#pragma unroll
            for (int j = 0; j < kRows; ++j) {
                slope(j, true);
                c.Store(p.gx, t + j - (K - 1), of_input(j, P{}));
            }
            shift(std::integral_constant<int, kRows>{});
        }
        for (; t < c.end + K - 1; ++t) single(t);
    }
    // the lines of a workgroup are added up one after another, the same way every time
#pragma unroll
    for (int k = 0; k <= K; ++k) {
        __syncthreads();
#pragma unroll
        for (int e = 0; e < E; ++e) {
            if (e >= skip) sums[threadIdx.x * E + e - skip] = k < K ? gw[e][k < K ? k : 0] : gb[e];
        }
        __syncthreads();
        for (int i = threadIdx.x; i < span * E; i += 256) {
            const int64_t at = static_cast<int64_t>(piece_block) * span * E + i;
            if (at >= p.channels) continue;
            float s = 0.f;
            for (int j = 0; j < lines; ++j) s += sums[j * span * E + i];
            p.parts[(static_cast<int64_t>(part) * (K + 1) + k) * p.channels + at] = s;
        }
    }
}

// Columns of partial sums, eight threads to a column.
template <typename T>
__global__ __launch_bounds__(256) void CausalConvSumKernel(const float* parts, int64_t n_parts, int64_t channels, int taps, T* gw, T* gb) {
    __shared__ float sums[8][32];
    const int64_t width = (taps + 1) * channels, c = static_cast<int64_t>(blockIdx.x) * 32 + (threadIdx.x & 31);
    const int slice = static_cast<int>(threadIdx.x) >> 5;
    float s = 0.f;
    if (c < width) {
#pragma unroll 8
        for (int64_t i = slice; i < n_parts; i += 8) s += parts[i * width + c];
    }
    sums[slice][threadIdx.x & 31] = s;
    __syncthreads();
    if (slice != 0 || c >= width) return;
    float all = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) all += sums[i][threadIdx.x];
    const int64_t k = c / channels, channel = c % channels;
    if (k < taps) gw[channel * taps + k] = static_cast<T>(all);
    else if (gb != nullptr) gb[channel] = static_cast<T>(all);
}

// Rows to a chunk: 32, or 16 or 8 where that leaves a compute unit fewer than 16 waves.  A chunk reads taps - 1 rows of the one before again, mostly from the caches.
// us, 32 and 64 rows: 16 x 2048 x 4096 float16 109, 114; gradients at 8 x 2048 x 2048, with the forward call, 84, 87.
int ChunkRows(int64_t length, int64_t lines) {
    int rows = 32;
    while (rows > kFewestRows && lines * ((length + rows - 1) / rows) < int64_t{NumCUs()} * 1024) rows /= 2;
    return rows;
}

// Channels to a thread: 16 bytes, and four of either type for the gradients, whose sums over rows and windows fill the registers; one where a row has fewer.
int ConvChannels(const hipcx_array* x) {
    const int64_t each = 16 / ItemSize(x->dtype);
    return x->shape[2] >= each ? static_cast<int>(each) : 1;
}
int GradChannels(int64_t channels) { return channels >= 4 ? 4 : 1; }

int GradPieceBits(int64_t pieces) {
    int bits = 0;
    while (bits < 6 && (int64_t{1} << bits) < pieces) ++bits;
    return bits;
}

struct ConvSizes {
    int64_t batch, length, channels, taps;
    ConvSizes(const hipcx_array* x, const hipcx_array* w) : batch(x->shape[0]), length(x->shape[1]), channels(x->shape[2]), taps(w->shape[1]) {}
    int64_t GradPieces() const { return (channels + GradChannels(channels) - 1) / GradChannels(channels); }
    int GradRows() const { return ChunkRows(length, batch * GradPieces()); }
    int64_t GradChunks() const { return std::max<int64_t>(1, (length + GradRows() - 1) / GradRows()); }
    int64_t GradParts() const {
        const int lines = 256 >> GradPieceBits(GradPieces());
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
        const int64_t each = ConvChannels(x), pieces = (s.channels + each - 1) / each;
        p.rows = ChunkRows(s.length, s.batch * pieces);
        const int64_t chunks = std::max<int64_t>(1, (s.length + p.rows - 1) / p.rows), threads = s.batch * chunks * pieces;
        HIPCX_REQUIRE(threads < (int64_t{1} << 31), HIPCX_NOT_IMPLEMENTED_ERROR, "causal_conv: too many elements");
        p.pieces = static_cast<int>(pieces), p.chunks = static_cast<int>(chunks);
        VisitConv(x->dtype, s.taps, [&](auto tag, auto taps) {
            using T = typename decltype(tag)::type;
            ForLaunches(threads, [&](dim3 grid, int64_t first) {
                p.first = first;
                if (each == 1) hipLaunchKernelGGL((CausalConvKernel<T, decltype(taps)::value, 1>), grid, dim3(256), 0, AsStream(stream), p);
                else hipLaunchKernelGGL((CausalConvKernel<T, decltype(taps)::value, 16 / static_cast<int>(sizeof(T))>), grid, dim3(256), 0, AsStream(stream), p);
                CheckLaunch("causal_conv");
            });
        });
    });
}

size_t hipcx_causal_conv_grad_workspace_size(const hipcx_array* x, const hipcx_array* w) {
    if (x == nullptr || w == nullptr || x->ndim != 3 || w->ndim != 2 || (x->dtype != HIPCX_FLOAT16 && x->dtype != HIPCX_FLOAT32)) return 0;
    const ConvSizes s(x, w);
    if (s.batch <= 0 || s.channels <= 0 || w->shape[0] != s.channels || s.taps < 1 || s.taps > kMaxTaps) return 0;  // (none for what the call refuses)
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
        const int64_t pieces = s.GradPieces();
        p.piece_bits = GradPieceBits(pieces);
        p.pieces = static_cast<int>(pieces), p.chunks = static_cast<int>(s.GradChunks());
        p.rows = s.GradRows();
        const int64_t blocks = parts * ((pieces + (1 << p.piece_bits) - 1) >> p.piece_bits);
        HIPCX_REQUIRE(blocks <= kBlocksPerLaunch, HIPCX_NOT_IMPLEMENTED_ERROR, "causal_conv_grad: too many elements");
        VisitConv(x->dtype, s.taps, [&](auto tag, auto taps) {
            using T = typename decltype(tag)::type;
            if (blocks != 0) {
                const dim3 grid(static_cast<unsigned>(blocks));
                if (GradChannels(s.channels) == 1) hipLaunchKernelGGL((CausalConvGradKernel<T, decltype(taps)::value, 1>), grid, dim3(256), 0, AsStream(stream), p);
                else hipLaunchKernelGGL((CausalConvGradKernel<T, decltype(taps)::value, 4>), grid, dim3(256), 0, AsStream(stream), p);
                CheckLaunch("causal_conv_grad");
            }
            const int64_t columns = (s.taps + 1) * s.channels;
            hipLaunchKernelGGL(CausalConvSumKernel<T>, dim3(static_cast<unsigned>((columns + 31) / 32)), dim3(256), 0, AsStream(stream), p.parts, parts, s.channels,
                               static_cast<int>(s.taps), static_cast<T*>(gw->data), static_cast<T*>(gb != nullptr ? gb->data : nullptr));
            CheckLaunch("causal_conv_grad");
        });
    });
}

}  // extern "C"
