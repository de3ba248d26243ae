// The gradients of linear attention over many steps (linear_attention.h).
#include "linear_attention.h"

namespace layers {
namespace {

// One wavefront takes a span of a head: two steps a lane. Backwards from the product of the memory at the span's end
// and its gradient, each step adds q.dq - k.dk without its own product to the gradient of the step after it,
// unless an episode starts there. It reads two dots a slice, head and step, and no more: 20 us for 16,384 heads of 64 steps.
struct DecayArgs {
    const float *queryDots, *keyDots, *crossings;  // [slices][head][time], and [slices][head][span]
    int querySlices, keySlices, time, heads, spans;
    unsigned allHeads;
    const float *decay;
    const unsigned char *resets;
    long long decayStrides[3], resetStrides[2];
    float *out;      // [batch][time][head], or null
    double *totals;  // [head][span]
};
__global__ __launch_bounds__(256) void DecayKernel(DecayArgs a) {
    static_assert(kSpan == 128, "two steps a lane");
    const int lane = threadIdx.x & 63;
    const long long items = (long long)a.allHeads * a.spans;
    for (long long item = blockIdx.x * 4ll + (threadIdx.x >> 6); item < items; item += gridDim.x * 4ll) {
        const int span = item % a.spans;
        const unsigned head = item / a.spans;
        const int h = head % a.heads, b = head / a.heads, begin = span * kSpan, end = min(begin + kSpan, a.time);
        double step[2];
        bool starts[3];
#pragma unroll
        for (int i = 0; i < 3; i++) {
            const int t = begin + 2 * lane + i;
            starts[i] = false;
            // What the first step of the next span starts with is in that span's memory already.
            if (t < end) {
                starts[i] = a.decay[b * a.decayStrides[0] + t * a.decayStrides[1] + h * a.decayStrides[2]] < kNothingKept;
                if (a.resets) starts[i] |= a.resets[b * a.resetStrides[0] + t * a.resetStrides[1]] != 0;
            }
            if (i == 2) break;
            step[i] = 0;
            if (t >= end) continue;
            for (int n = 0; n < a.querySlices; n++) step[i] += a.queryDots[((long long)n * a.allHeads + head) * a.time + t];
            for (int n = 0; n < a.keySlices; n++) step[i] -= a.keyDots[((long long)n * a.allHeads + head) * a.time + t];
        }
        double crossing = 0;
        for (int n = 0; n < a.querySlices; n++) crossing += a.crossings[((long long)n * a.allHeads + head) * a.spans + span];
        if (lane == 63) step[1] += crossing;
        // The gradients of a lane's first step, and whether they take what comes after the lane.
        double sum = starts[1] ? step[0] : step[0] + step[1];
        int open = !starts[1] && !starts[2];
        for (int d = 1; d < 64; d *= 2) {
            const double later = __shfl_down(sum, d);
            const int more = __shfl_down(open, d);
            if (lane + d < 64 && open) sum += later, open = more;
        }
        const double after = __shfl_down(sum, 1);
        const double second = lane < 63 && !starts[2] ? step[1] + after : step[1];
        const double found[2] = {starts[0] ? 0.0 : starts[1] ? step[0] : step[0] + second, starts[1] ? 0.0 : second};
        double total = 0;
#pragma unroll
        for (int i = 0; i < 2; i++) {
            const int t = begin + 2 * lane + i;
            if (t >= end) continue;
            if (a.out) a.out[((long long)b * a.time + t) * a.heads + h] = (float)found[i];
            total += found[i];
        }
        if (a.totals) {
            for (int d = 32; d; d /= 2) total += __shfl_xor(total, d);
            if (lane == 0) a.totals[item] = total;
        }
    }
}

// The totals of one head over the batch and its spans, always in the same order.
__global__ __launch_bounds__(256) void TotalKernel(const double *totals, float *out, int batch, int heads, int spans) {
    __shared__ double sums[256];
    double sum = 0;
    const long long count = (long long)batch * spans;
    for (long long i = threadIdx.x; i < count; i += 256) sum += totals[(i / spans * heads + blockIdx.x) * spans + i % spans];
    sums[threadIdx.x] = sum;
    __syncthreads();
    for (unsigned d = 128; d; d /= 2) {
        if (threadIdx.x < d) sums[threadIdx.x] += sums[threadIdx.x + d];
        __syncthreads();
    }
    if (threadIdx.x == 0) out[blockIdx.x] = (float)sums[0];
}

// Gradients of keys and queries that `share` heads share, from a part of each of them.
template <class T>
__global__ __launch_bounds__(256) void SharedKernel(const float *parts, T *out, long long count, int size, int share) {
    const long long step = (long long)gridDim.x * 256;
    for (long long i = blockIdx.x * 256ll + threadIdx.x; i < count; i += step) {
        const float *from = parts + i / size * share * size + i % size;
        float sum = 0;
        for (int n = 0; n < share; n++) sum += from[(long long)n * size];
        out[i] = As<T>(sum);
    }
}

// What lies where in the workspace, in floats.
struct Layout {
    long long memories, factors, dots, crossings, totals, parts, end;
};
Layout LayoutOf(const Attention &a) {
    const Runs runs = RunsOf(a);
    const long long heads = runs.allHeads, kept = heads * (runs.spans - 1), size = (long long)a.key_size * a.value_size;
    const long long slices = (a.key_size + 15) / 16;
    const auto four = [](long long x) { return (x + 3) / 4 * 4; };
    Layout at{};
    at.factors = four(kept * size);
    at.dots = at.factors + four(2 * kept);
    at.crossings = at.dots + (a.d_decay ? four(2 * slices * heads * a.time) : 0);
    at.totals = at.crossings + (a.d_decay ? four(slices * heads * runs.spans) : 0);
    at.parts = at.totals + (a.d_decay && a.decay_of_head ? four(2 * heads * runs.spans) : 0);
    at.end = at.parts + (a.heads != a.key_heads ? 2 * heads * a.time * a.key_size : 0);
    return at;
}

template <class T>
void Backward(const Attention &a, hipStream_t stream) {
    Runs runs = RunsOf(a);
    const Layout at = LayoutOf(a);
    float *work = static_cast<float *>(a.workspace);
    const int share = a.heads / a.key_heads;
    const long long size = (long long)a.key_size * a.value_size, heads = runs.allHeads, tokens = heads * a.time;
    const bool whole = IsWhole(a);
    const Tensor query = TensorOf(a.query, a.query_strides, share), key = TensorOf(a.key, a.key_strides, share);
    const Tensor value = TensorOf(a.value, a.value_strides, 1), output = TensorOf(a.d_output, a.d_output_strides, 1);
    const auto put = [&](Run &r, void *to, bool floats) {
        r.output = to, r.floats = floats;
        r.outputStrides[0] = (long long)a.time * a.heads * r.columns, r.outputStrides[1] = (long long)a.heads * r.columns;
        r.outputStrides[2] = r.columns;
    };

    if (runs.spans > 1) {
        Runs memories = runs;
        Run &r = memories.run[0];
        r.key = query, r.value = output;
        r.rows = a.key_size, r.columns = a.value_size, r.reverse = true, r.in = a.scale;
        r.last = work + at.memories;
        memories.firstSpan = 1, memories.spanCount = runs.spans - 1;
        memories.factors = runs.factors = reinterpret_cast<double *>(work + at.factors);
        RunMemories(memories, a.type, whole, stream);
        JoinMemories(runs, static_cast<const float *>(a.d_last), work + at.memories, size, true, stream);
    }

    Run &dq = runs.run[0], &dk = runs.run[1], &dv = runs.run[2];
    dq.query = output, dq.key = value, dq.value = key, dq.weight = query;
    dq.rows = a.value_size, dq.columns = a.key_size, dq.transposed = true, dq.in = 1, dq.out = a.scale;
    dq.first = static_cast<const float *>(a.state), dq.starts = static_cast<const float *>(a.checkpoints);
    put(dq, share > 1 ? work + at.parts : a.d_query, share > 1);

    dk.query = value, dk.key = output, dk.value = query, dk.weight = key;
    dk.rows = a.value_size, dk.columns = a.key_size, dk.reverse = dk.transposed = true, dk.in = a.scale, dk.out = 1;
    dk.first = static_cast<const float *>(a.d_last), dk.starts = work + at.memories;
    put(dk, share > 1 ? work + at.parts + tokens * a.key_size : a.d_key, share > 1);

    dv.query = key, dv.key = query, dv.value = output;
    dv.rows = a.key_size, dv.columns = a.value_size, dv.reverse = true, dv.in = a.scale, dv.out = 1;
    dv.first = static_cast<const float *>(a.d_last), dv.starts = work + at.memories, dv.last = static_cast<float *>(a.d_state);
    put(dv, a.d_value, false);

    // A launch has one number of rows, in tiles of 32, and kernels of full tiles take no other. Where keys and values differ in
    // it, or one of them fills its tiles alone, and with enough wavefronts, the values' run has a launch of its own. (bfloat16, 64
    // steps: 4,096 heads of 128 x 64 take 274 against 755 us, 512 of 32 x 64 28 against 37; 256 of 48 x 64 33 against 29.)
    const bool full = a.key_size % 16 == 0 && a.value_size % 16 == 0 && (a.key_size % 32 == 0 || a.value_size % 32 == 0);
    const bool apart = a.key_size != a.value_size && ((whole && full) || (a.key_size + 31) / 32 != (a.value_size + 31) / 32) &&
                       heads * runs.spans * ((2 * a.key_size + a.value_size) / 16) >= 11 * 256;
    if (a.d_decay) {
        const long long slices = (a.key_size + 15) / 16;
        dq.dots = work + at.dots, dk.dots = work + at.dots + slices * tokens;
        dq.crossings = work + at.crossings, dq.against = work + at.memories, dq.againstLast = static_cast<const float *>(a.d_last);
        LaunchRuns<T, kGradient>(runs, apart ? 2 : 3, whole, stream);
        DecayArgs d{dq.dots, dk.dots, dq.crossings, runs.slices[0], runs.slices[1], a.time, a.heads, runs.spans, runs.allHeads, runs.decay,
                    runs.resets, {}, {}, a.decay_of_head ? nullptr : static_cast<float *>(a.d_decay),
                    a.decay_of_head ? reinterpret_cast<double *>(work + at.totals) : nullptr};
        for (int i = 0; i < 3; i++) d.decayStrides[i] = runs.decayStrides[i];
        for (int i = 0; i < 2; i++) d.resetStrides[i] = runs.resetStrides[i];
        const long long items = heads * runs.spans;
        hipLaunchKernelGGL(DecayKernel, dim3((unsigned)(items < (1 << 22) ? (items + 3) / 4 : 1 << 20)), dim3(256), 0, stream, d);
        if (a.decay_of_head)
            hipLaunchKernelGGL(TotalKernel, dim3(a.heads), dim3(256), 0, stream, d.totals, static_cast<float *>(a.d_decay), a.batch,
                               a.heads, runs.spans);
    } else {
        RunOutputs(runs, apart ? 2 : 3, a.type, whole, stream);
    }
    if (apart) {
        runs.run[0] = dv;
        RunOutputs(runs, 1, a.type, whole, stream);
    }
    if (share > 1) {
        const long long count = tokens / share * a.key_size;
        const unsigned blocks = (unsigned)(count > (1ll << 24) ? 1 << 16 : (count + 255) / 256);
        for (const bool keys : {false, true})
            if (count)
                hipLaunchKernelGGL((SharedKernel<T>), dim3(blocks), dim3(256), 0, stream,
                                   work + at.parts + (keys ? tokens * a.key_size : 0),
                                   static_cast<T *>(keys ? a.d_key : a.d_query), count, a.key_size, share);
    }
}

}  // namespace
}  // namespace layers

using namespace layers;

extern "C" __attribute__((visibility("default"))) unsigned long long cuju_linear_attention_backward_workspace(
    const struct cuju_linear_attention *attention) {
    if (!Fits(attention)) return 0;
    return LayoutOf(*attention).end * sizeof(float);
}

extern "C" __attribute__((visibility("default"))) int cuju_linear_attention_backward(const struct cuju_linear_attention *attention, void *stream) {
    if (!Fits(attention)) return -1;
    const Attention &a = *attention;
    if (a.batch == 0) return 0;
    if (a.time > 0 && (!a.query || !a.key || !a.value || !a.decay || !a.d_output || !a.d_query || !a.d_key || !a.d_value))
        return Failed("expected inputs and their gradients");
    if (a.time > kSpan && !a.checkpoints) return Failed("expected the checkpoints of the forward pass");
    if (LayoutOf(a).end && !a.workspace) return Failed("expected a workspace");
    ForType(a.type, [&](auto x) { Backward<decltype(x)>(a, static_cast<hipStream_t>(stream)); });
    return Launched("the gradients of linear attention");
}
