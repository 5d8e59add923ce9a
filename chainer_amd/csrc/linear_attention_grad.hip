// The gradients of linear attention: its three passes (linear_attention.h), and what they have of the log decays.
#include <utility>

#include "linear_attention.h"

namespace hipcx {
namespace {

struct AttendDecayArgs {
    const float *of_q, *of_k;  // [batch][head][blocks][length]: parts of q gq and k gk
    const float* ends;         // [batch][head][segment][blocks]: what the rows behind a segment have of the decays in it
    float* out;                // [batch][length][head], or null
    double* totals;            // [batch][head][segment], or null
    SequenceLengths lengths;
    int64_t length, segment_rows;
    int blocks, heads, segments;
};

// gg[t] = sum over u >= t of (q[u] gq[u] - k[u] gk[u]): sums from a segment's last row to its first, in 64 bits, on top of what lies behind the segment.
template <int THREADS>
__global__ __launch_bounds__(THREADS) void AttendDecayKernel(AttendDecayArgs p) {
    __shared__ double waves[THREADS / 64];
    const int segment = static_cast<int>(blockIdx.x % p.segments);
    const int64_t bh = blockIdx.x / p.segments, b = bh / p.heads;
    const int h = static_cast<int>(bh % p.heads), tid = threadIdx.x, lane = tid % 64;
    const int64_t length = LengthOf(p.lengths, b, p.length), first = segment * p.segment_rows;
    const int64_t whole = first + p.segment_rows < p.length ? first + p.segment_rows : p.length, end = whole < length ? whole : length;
    double behind = 0, total = 0;
    for (int i = 0; i < p.blocks; ++i) behind += p.ends[(bh * p.segments + segment) * p.blocks + i];
    for (int64_t last = end; last > first; last -= THREADS) {
        const int64_t t = last - 1 - tid;
        double sum = 0;
        if (t >= first) {
            for (int i = 0; i < p.blocks; ++i) sum += static_cast<double>(p.of_q[(bh * p.blocks + i) * p.length + t]) - p.of_k[(bh * p.blocks + i) * p.length + t];
        }
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const double before = ShflUpDouble(sum, o);
            if (lane >= o) sum += before;
        }
        __syncthreads();
        if (lane == 63) waves[tid / 64] = sum;
        __syncthreads();
        for (int w = 0; w < tid / 64; ++w) sum += waves[w];
        sum += behind;
        if (t >= first) {
            if (p.out != nullptr) p.out[(b * p.length + t) * p.heads + h] = static_cast<float>(sum);
            total += sum;
        }
#pragma unroll
        for (int w = 0; w < THREADS / 64; ++w) behind += waves[w];
    }
    if (p.out != nullptr) {
        for (int64_t t = (end > first ? end : first) + tid; t < whole; t += THREADS) p.out[(b * p.length + t) * p.heads + h] = 0.f;
    }
    if (p.totals == nullptr) return;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const double other = ShflDouble(total, lane ^ o);
        total += other;
    }
    __syncthreads();
    if (lane == 0) waves[tid / 64] = total;
    __syncthreads();
    if (tid == 0) {
        total = 0;
#pragma unroll
        for (int w = 0; w < THREADS / 64; ++w) total += waves[w];
        p.totals[bh * p.segments + segment] = total;
    }
}

// One decay for all rows of a head: the sum over sequences and segments, a wave to a head.
__global__ __launch_bounds__(64) void AttendHeadDecayKernel(const double* totals, float* out, int64_t batch, int heads, int segments) {
    const int h = blockIdx.x, lane = threadIdx.x;
    double sum = 0;
    for (int64_t i = lane; i < batch * segments; i += 64) sum += totals[(i / segments * heads + h) * segments + i % segments];
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const double other = ShflDouble(sum, lane ^ o);
        sum += other;
    }
    if (lane == 0) out[h] = static_cast<float>(sum);
}

// The heads' gradients of what they share, [row][head][element] in 32 bits, added up in the order of the heads and rounded once.
template <typename T>
__global__ __launch_bounds__(256) void AttendShareKernel(const float* parts, AttendRows out, int64_t rows, int64_t length, int key_heads, int share, int width) {
    const int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
    if (i >= rows * key_heads * width) return;
    const int e = static_cast<int>(i % width);
    const int64_t head = i / width, row = head / key_heads;
    const int h = static_cast<int>(head % key_heads);
    const float* const from = parts + (row * key_heads + h) * share * width + e;
    float sum = 0;
    for (int s = 0; s < share; ++s) sum += from[static_cast<int64_t>(s) * width];
    static_cast<T*>(out.data)[row / length * out.batch + row % length * out.row + h * out.head + e] = static_cast<T>(sum);
}

// Offsets of the workspace's parts, in bytes.
struct GradWorkspace {
    size_t states, gradients, decays, of_q, of_k, ends, totals, gq, gk, bytes = 0;
    size_t Take(int64_t floats) {
        const size_t at = bytes;
        bytes += (static_cast<size_t>(floats) * 4 + 255) / 256 * 256;
        return at;
    }
    GradWorkspace(const AttendCall& c, bool of_decays, bool of_heads) {
        const AttendArgs& p = c.p;
        const int64_t bh = p.batch * p.heads, each = static_cast<int64_t>(c.keys) * c.values, blocks = AttendBlocks(c.keys);
        states = Take(p.segments > 1 ? bh * p.segments * each : 0), gradients = Take(p.segments > 1 ? bh * p.segments * each : 0);
        decays = Take(p.segments > 1 ? 2 * bh * p.segments : 0);
        of_q = Take(of_decays ? bh * p.length * blocks : 0), of_k = Take(of_decays ? bh * p.length * blocks : 0);
        ends = Take(of_decays ? bh * p.segments * blocks : 0), totals = Take(of_heads ? bh * p.segments * 2 : 0);
        const int64_t shared = c.key_heads < p.heads ? bh * p.length * c.keys : 0;
        gq = Take(shared), gk = Take(shared);
    }
};

void CutGrad(AttendCall* c, bool padded) {
    const int64_t keys = AttendBlocks(c->keys), values = AttendBlocks(c->values);
    CutAttend(&c->p, padded, 2 * keys + values, keys + values, AttendResident(c->dtype == HIPCX_FLOAT16, std::max(c->keys, c->values)), 2 * static_cast<int64_t>(c->keys) * c->values);
}

}  // namespace
}  // namespace hipcx

using namespace hipcx;

extern "C" {

size_t hipcx_linear_attention_grad_workspace_size(const hipcx_array* q, const hipcx_array* v, const hipcx_array* log_decay, const hipcx_array* lengths) {
    AttendCall c;
    if (!AttendSizesOf(q, v, &c)) return 0;
    CutGrad(&c, lengths != nullptr);
    return GradWorkspace(c, log_decay != nullptr, log_decay != nullptr && log_decay->ndim == 1).bytes;
}

int hipcx_linear_attention_grad(const hipcx_array* q, const hipcx_array* k, const hipcx_array* v, const hipcx_array* log_decay, double scale, const hipcx_array* state,
                                const hipcx_array* lengths, const hipcx_array* gy, const hipcx_array* gnew_state, const hipcx_array* gq, const hipcx_array* gk,
                                const hipcx_array* gv, const hipcx_array* glog_decay, const hipcx_array* gstate, void* workspace, size_t workspace_bytes, void* stream) {
    return Guard([&] {
        const std::string what = "linear_attention_grad";
        AttendCall c = DescribeAttend(what, q, k, v, log_decay, scale, state, lengths);
        HIPCX_REQUIRE(gy != nullptr && gq != nullptr && gk != nullptr && gv != nullptr, HIPCX_CHAINERX_ERROR, what + ": gy, gq, gk and gv are needed");
        HIPCX_REQUIRE(glog_decay == nullptr || log_decay != nullptr, HIPCX_CHAINERX_ERROR, what + ": glog_decay goes with log_decay");
        AttendArgs& p = c.p;
        const int dtype = q->dtype;
        const AttendRows from = DescribeAttendRows(gy, c, p.heads, c.values, dtype, what + ": gy");
        const AttendRows to_q = DescribeAttendRows(gq, c, c.key_heads, c.keys, dtype, what + ": gq"), to_k = DescribeAttendRows(gk, c, c.key_heads, c.keys, dtype, what + ": gk");
        const AttendRows to_v = DescribeAttendRows(gv, c, p.heads, c.values, dtype, what + ": gv");
        for (const hipcx_array* a : {gnew_state, gstate}) {
            RequireShape(a, {p.batch, p.heads, c.keys, c.values}, HIPCX_FLOAT32, what + ": gnew_state and gstate");
            RequireDense(a, what + ": gnew_state and gstate");
        }
        if (glog_decay != nullptr) {
            if (log_decay->ndim == 1) RequireShape(glog_decay, {p.heads}, HIPCX_FLOAT32, what + ": glog_decay");
            else RequireShape(glog_decay, {p.batch, p.length, p.heads}, HIPCX_FLOAT32, what + ": glog_decay");
            RequireDense(glog_decay, what + ": glog_decay");
        }
        CutGrad(&c, lengths != nullptr);
        const bool of_heads = glog_decay != nullptr && glog_decay->ndim == 1;
        const GradWorkspace w(c, log_decay != nullptr, log_decay != nullptr && log_decay->ndim == 1);
        HIPCX_REQUIRE(workspace_bytes >= w.bytes && (w.bytes == 0 || workspace != nullptr), HIPCX_CHAINERX_ERROR, what + ": the workspace is too small");
        HIPCX_REQUIRE(reinterpret_cast<uintptr_t>(workspace) % 16 == 0, HIPCX_CHAINERX_ERROR, "workspace must be 16-byte aligned");
        const bool shared = c.key_heads < p.heads;
        HIPCX_REQUIRE(!shared || p.batch * p.length * c.key_heads * c.keys < (int64_t{1} << 31), HIPCX_NOT_IMPLEMENTED_ERROR, what + ": too many elements");
        HIPCX_REQUIRE(p.batch * p.heads * p.segments <= kBlocksPerLaunch, HIPCX_NOT_IMPLEMENTED_ERROR, what + ": too many elements");
        char* const ws = static_cast<char*>(workspace);
        const auto floats = [&](size_t at) { return reinterpret_cast<float*>(ws + at); };
        const hipStream_t s = AsStream(stream);
        const float* const gnew = gnew_state != nullptr ? static_cast<const float*>(gnew_state->data) : nullptr;
        const int64_t bh = p.batch * p.heads;
        if (bh > 0) {
            const AttendRows wide{nullptr, p.length * p.heads * c.keys, static_cast<int64_t>(p.heads) * c.keys, c.keys, 1};
            const float f_scale = static_cast<float>(scale);
            AttendRun &of_q = p.run[0], &of_k = p.run[1], &of_v = p.run[2];
            of_q.q = from, of_q.k = c.v, of_q.v = c.k, of_q.y = to_q, of_q.kv_scale = 1, of_q.out_scale = f_scale;
            of_k.q = c.v, of_k.k = from, of_k.v = c.q, of_k.y = to_k, of_k.kv_scale = f_scale, of_k.out_scale = 1, of_k.back = 1;
            of_v.q = c.k, of_v.k = c.q, of_v.v = from, of_v.y = to_v, of_v.kv_scale = f_scale, of_v.out_scale = 1, of_v.back = 1;
            for (AttendRun* run : {&of_q, &of_k}) run->keys = c.values, run->values = c.keys;
            of_v.keys = c.keys, of_v.values = c.values;
            if (shared) {
                of_q.y = of_k.y = wide;
                of_q.y.data = ws + w.gq, of_k.y.data = ws + w.gk;
                of_q.wide = of_k.wide = 1;
            }
            if (glog_decay != nullptr) {
                of_q.dot = c.q, of_q.dots = floats(w.of_q), of_q.ends = floats(w.ends);
                of_k.dot = c.k, of_k.dots = floats(w.of_k);
            }
            const AttendStates state_t = AttendStatesOf(c.state, c.keys, c.values, true), gnew_plain = AttendStatesOf(gnew, c.keys, c.values, false),
                               gnew_t = AttendStatesOf(gnew, c.keys, c.values, true);
            of_q.start = state_t, of_q.other = gnew_t, of_k.start = gnew_t, of_v.start = gnew_plain;
            if (p.segments > 1) {
                // the states and their gradients that the segments start from; those of v's pass serve k's too, as transposes
                AttendArgs states = p;
                states.run[0] = of_q, states.run[1] = of_v;
                states.runs = 2;
                states.run[0].last = AttendSegments(floats(w.states), p, c.values, c.keys), states.run[1].last = AttendSegments(floats(w.gradients), p, c.keys, c.values);
                states.run[0].decays = floats(w.decays), states.run[1].decays = floats(w.decays) + bh * p.segments;
                states.run[0].first = 0, states.run[0].blocks = AttendBlocks(c.keys), states.run[1].first = states.run[0].blocks, states.run[1].blocks = AttendBlocks(c.values);
                states.blocks = states.run[0].blocks + states.run[1].blocks;
                LaunchAttend(states, dtype, true, s);
                LaunchAttendStarts(states, 0, state_t, s);
                LaunchAttendStarts(states, 1, gnew_plain, s);
                of_q.start = states.run[0].last, of_v.start = of_k.start = of_q.other = states.run[1].last;
                std::swap(of_k.start.i, of_k.start.j), std::swap(of_q.other.i, of_q.other.j);
            }
            if (gstate != nullptr) of_v.last = AttendStatesOf(static_cast<const float*>(gstate->data), c.keys, c.values, false), of_v.decay_last = 1;
            p.runs = 3, p.blocks = 0;
            for (int i = 0; i < 3; ++i) {
                p.run[i].first = p.blocks, p.run[i].blocks = AttendBlocks(p.run[i].values);
                p.blocks += p.run[i].blocks;
            }
            LaunchAttend(p, dtype, false, s);
            if (shared && p.length > 0) {
                const int64_t rows = p.batch * p.length, n = rows * c.key_heads * c.keys;
                for (const auto& [at, to] : {std::pair<size_t, const AttendRows*>{w.gq, &to_q}, {w.gk, &to_k}}) {
                    const dim3 grid(static_cast<unsigned>((n + 255) / 256));
                    if (dtype == HIPCX_FLOAT16) hipLaunchKernelGGL((AttendShareKernel<half_t>), grid, dim3(256), 0, s, floats(at), *to, rows, p.length, c.key_heads, p.heads / c.key_heads, c.keys);
                    else hipLaunchKernelGGL((AttendShareKernel<float>), grid, dim3(256), 0, s, floats(at), *to, rows, p.length, c.key_heads, p.heads / c.key_heads, c.keys);
                    CheckLaunch("linear_attention_grad");
                }
            }
            if (glog_decay != nullptr) {
                AttendDecayArgs d{};
                d.of_q = floats(w.of_q), d.of_k = floats(w.of_k), d.ends = floats(w.ends);
                d.lengths = p.lengths, d.length = p.length, d.segment_rows = p.segment_rows, d.heads = p.heads, d.segments = p.segments;
                d.blocks = AttendBlocks(c.keys);
                if (of_heads) d.totals = reinterpret_cast<double*>(ws + w.totals);
                else d.out = static_cast<float*>(glog_decay->data);
                // (segments of 2048 rows: 12 us with 256 threads)
                if (p.segment_rows > 256) hipLaunchKernelGGL(AttendDecayKernel<1024>, dim3(static_cast<unsigned>(bh * p.segments)), dim3(1024), 0, s, d);
                else hipLaunchKernelGGL(AttendDecayKernel<256>, dim3(static_cast<unsigned>(bh * p.segments)), dim3(256), 0, s, d);
                CheckLaunch("linear_attention_grad");
            }
        }
        if (of_heads) {
            hipLaunchKernelGGL(AttendHeadDecayKernel, dim3(static_cast<unsigned>(p.heads)), dim3(64), 0, s, reinterpret_cast<const double*>(ws + w.totals),
                               static_cast<float*>(glog_decay->data), p.batch, p.heads, p.segments);
            CheckLaunch("linear_attention_grad");
        }
    });
}

}  // extern "C"
