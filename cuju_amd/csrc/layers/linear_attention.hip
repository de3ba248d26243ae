// Linear attention with decays: one step of it for acting, and its forward pass over many steps (linear_attention.h).
#include "linear_attention.h"

namespace layers {
namespace {

// ---------------------------------------------------------------------------------------- one step

// One wavefront takes a head's memory, or a part of its columns: `Lanes` lanes of four columns each side by side,
// 64 / Lanes groups of rows. The memory is read once and written once, which bounds it: 360,448 heads of 64 x 64 take 2,290 us,
// 12.0 GB, 5.2 TB/s (an update in place of 4 GiB reaches 5.9).
template <class T, int Keys, int Lanes, bool Whole>
__global__ __launch_bounds__(256) void StepKernel(Attention a, View<const T> query, View<const T> key, View<const T> value,
                                                  int slices, int columns, unsigned waves) {
    constexpr int kGroups = 64 / Lanes, kRows = Keys / kGroups;
    __shared__ float sharedKeys[4][2][Keys];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const unsigned id = blockIdx.x * 4 + wave;
    float *keys = sharedKeys[wave][0], *queries = sharedKeys[wave][1];
    if (id >= waves) return;
    const unsigned slice = id % slices, head = id / slices;
    const int h = head % a.heads, b = head / a.heads, kh = h / (a.heads / a.key_heads);
    const int dk = a.key_size, dv = a.value_size;
    // All loads start before the first is waited for. A memory that is cleared is loaded too, and dropped: what it
    // held, infinities among it, is gone.
    const float decay = Global(static_cast<const float *>(a.decay))[b * a.decay_strides[0] + h * a.decay_strides[2]];
    const bool reset = a.resets && Global(a.resets)[b * a.reset_strides[0]];
    const int first = slice * columns + (lane % Lanes) * 4, row0 = (lane / Lanes) * kRows;
    const int valid = min(columns - (lane % Lanes) * 4, dv - first);
    float *at = static_cast<float *>(a.state) + ((long long)head * dk + row0) * dv + first;
    Pack<float, 4> s[kRows];
#pragma unroll
    for (int i = 0; i < kRows; i++) s[i] = Load<4, Whole>(at + i * dv, row0 + i < dk ? valid : 0);
    const auto v = Load<4, Whole>(value.At(b, 0, h) + first, valid);
    const T *key0 = key.At(b, 0, kh), *query0 = query.At(b, 0, kh);
#pragma unroll
    for (int i = lane; i < Keys; i += 64) {
        keys[i] = i < dk ? Float(key0[i]) : 0.f;
        queries[i] = i < dk ? Float(query0[i]) : 0.f;
    }
    // Only this wavefront reads them, and its LDS accesses keep their order.
    Forget();
    const bool cleared = reset || decay < kNothingKept;
    const float kept = cleared ? 0.f : expf(decay);
    float out[4] = {0, 0, 0, 0};
#pragma unroll
    for (int i = 0; i < kRows; i++) {
        const float k = keys[row0 + i], q = queries[row0 + i];
#pragma unroll
        for (int c = 0; c < 4; c++) {
            s[i].x[c] = fmaf(k, Float(v.x[c]), cleared ? 0.f : s[i].x[c] * kept);
            out[c] = fmaf(q, s[i].x[c], out[c]);
        }
        Store<4, Whole>(at + i * dv, s[i], row0 + i < dk ? valid : 0);
    }
#pragma unroll
    for (int d = Lanes; d < 64; d *= 2)
#pragma unroll
        for (int c = 0; c < 4; c++) out[c] += __shfl_xor(out[c], d);
    Pack<T, 4> o;
#pragma unroll
    for (int c = 0; c < 4; c++) o.x[c] = As<T>(a.scale * out[c]);
    if (row0 == 0) Store<4, Whole>(static_cast<T *>(a.output) + (long long)head * dv + first, o, valid);
}

template <class T, int Keys>
void LaunchStep(const Attention &a, hipStream_t stream) {
    const int slices = (a.value_size + 63) / 64, columns = min(a.value_size, 64);
    const unsigned waves = (unsigned)(a.batch * (long long)a.heads * slices);
    const auto query = ViewOf<const T>(a.query, a.query_strides, a.key_size);
    const auto key = ViewOf<const T>(a.key, a.key_strides, a.key_size);
    const auto value = ViewOf<const T>(a.value, a.value_strides, a.value_size);
    const bool whole = value.whole && Aligned(16, a.state) && Aligned(4 * sizeof(T), a.output);
    const auto launch = [&](auto kernel) {
        hipLaunchKernelGGL(kernel, dim3((waves + 3) / 4), dim3(256), 0, stream, a, query, key, value, slices, columns, waves);
    };
    if (!whole) launch(StepKernel<T, Keys, 16, false>);
    else if (columns <= 16) launch(StepKernel<T, Keys, 4, true>);
    else if (columns <= 32) launch(StepKernel<T, Keys, 8, true>);
    else launch(StepKernel<T, Keys, 16, true>);
}

// ------------------------------------------------------------------------------------- many steps

constexpr int kJoined = 8;
// A thread takes an element of a head's memory through the spans. It waits for memory: eight spans' loads are on their way
// together (44 heads of 128 x 128 through 24 spans 21 us, 66 MB each way).
__global__ __launch_bounds__(256) void JoinKernel(const float *first, float *memories, const double *factors, long long size,
                                                  long long elements, int spans, bool reverse) {
    const long long step = (long long)gridDim.x * blockDim.x;
    for (long long i = (long long)blockIdx.x * blockDim.x + threadIdx.x; i < elements; i += step) {
        const long long head = i / size, element = i % size;
        float memory = first ? first[i] : 0.f;
        float *at = memories + head * (spans - 1) * size + element;
        const double *factor = factors + head * (spans - 1);
        // Some spans' loads at a time, so that each is not waited for by itself.
        for (int n = 0; n + 1 < spans; n += kJoined) {
            float own[kJoined];
            double kept[kJoined];
#pragma unroll
            for (int x = 0; x < kJoined; x++)
                if (n + x + 1 < spans) {
                    const int place = reverse ? spans - 2 - n - x : n + x;
                    own[x] = at[place * size], kept[x] = factor[place];
                }
#pragma unroll
            for (int x = 0; x < kJoined; x++)
                if (n + x + 1 < spans) {
                    memory = kept[x] < 0. ? own[x] : (float)fma(kept[x], (double)memory, (double)own[x]);
                    at[(reverse ? spans - 2 - n - x : n + x) * size] = memory;
                }
        }
    }
}

// Few heads are cut into spans, so that more wavefronts run: the memories at the spans' ends cost more than half of the
// outputs. Cut and whole, with square memories of 16, 32, 64 and 128 and 1,024 steps, in us: bfloat16 of 1,024 tiles 85 and 102, 64
// and 93, 71 and 108, 126 and 148, of 2,048 159 and 126, 115 and 106, 134 and 130, 248 and 164; float32 of 512 tiles 72 and 119,
// 52 and 105, 95 and 128, 210 and 213, of 1,024 132 and 127, 94 and 128, 169 and 161, 390 and 275. 384 steps gain less: 43
// and 45 in bfloat16 of 1,024 tiles of 64. The largest memories would take half the limit: 384 steps of 128 in float16 of
// 1,024 tiles 106 and 90, in float32 of 512 97 and 86.
bool Splits(const Attention &a) {
    const long long heads = (long long)a.batch * a.heads;
    return a.time >= 3 * kSpan && heads * ((a.value_size + 15) / 16) < (a.type == 0 ? 1024 : 2048);
}

template <class T>
void Forward(const Attention &a, hipStream_t stream) {
    Runs runs = RunsOf(a);
    Run &run = runs.run[0];
    const int share = a.heads / a.key_heads;
    run.query = TensorOf(a.query, a.query_strides, share), run.key = TensorOf(a.key, a.key_strides, share);
    run.value = TensorOf(a.value, a.value_strides, 1);
    run.rows = a.key_size, run.columns = a.value_size, run.in = 1, run.out = a.scale;
    run.output = a.output;
    run.outputStrides[0] = (long long)a.time * a.heads * a.value_size, run.outputStrides[1] = (long long)a.heads * a.value_size;
    run.outputStrides[2] = a.value_size;
    run.first = static_cast<const float *>(a.state);
    const bool whole = IsWhole(a);
    if (Splits(a)) {
        const long long size = (long long)a.key_size * a.value_size, kept = (long long)runs.allHeads * (runs.spans - 1);
        float *memories = static_cast<float *>(a.checkpoints ? a.checkpoints : a.workspace);
        runs.factors = static_cast<double *>(a.workspace) + (a.checkpoints ? 0 : (kept * size + 1) / 2);
        run.last = memories, runs.spanCount = runs.spans - 1;
        LaunchRuns<T, kMemory>(runs, 1, whole, stream);
        JoinMemories(runs, run.first, memories, size, false, stream);
        run.starts = memories, runs.spanCount = runs.spans;
    } else {
        run.kept = static_cast<float *>(a.checkpoints);
        runs.length = a.time > 0 ? a.time : 1, runs.spans = runs.spanCount = 1;
    }
    run.last = static_cast<float *>(a.last);
    LaunchRuns<T, kOutputs>(runs, 1, whole, stream);
}

}  // namespace

void RunMemories(Runs &runs, int type, bool whole, hipStream_t stream) {
    ForType(type, [&](auto x) { LaunchRuns<decltype(x), kMemory>(runs, 1, whole, stream); });
}
void RunOutputs(Runs &runs, int count, int type, bool whole, hipStream_t stream) {
    ForType(type, [&](auto x) { LaunchRuns<decltype(x), kOutputs>(runs, count, whole, stream); });
}
void JoinMemories(const Runs &runs, const float *first, float *memories, long long size, bool reverse, hipStream_t stream) {
    const long long elements = runs.allHeads * size;
    const unsigned blocks = (unsigned)(elements > (1ll << 24) ? 1 << 16 : (elements + 255) / 256);
    hipLaunchKernelGGL(JoinKernel, dim3(blocks), dim3(256), 0, stream, first, memories, runs.factors, size, elements, runs.spans, reverse);
}

}  // namespace layers

using namespace layers;

extern "C" __attribute__((visibility("default"))) int cuju_linear_attention_step(const struct cuju_linear_attention *attention, void *stream) {
    if (!Fits(attention)) return -1;
    const Attention &a = *attention;
    if (a.time != 1) return Failed("expected one step");
    if (a.batch == 0) return 0;
    if (!a.query || !a.key || !a.value || !a.decay || !a.state || !a.output) return Failed("expected a memory and an output");
    ForType(a.type, [&](auto x) {
        using T = decltype(x);
        const auto s = static_cast<hipStream_t>(stream);
        if (a.key_size <= 32) LaunchStep<T, 32>(a, s);
        else if (a.key_size <= 64) LaunchStep<T, 64>(a, s);
        else LaunchStep<T, 128>(a, s);
    });
    return Launched("the step of linear attention");
}

extern "C" __attribute__((visibility("default"))) unsigned long long cuju_linear_attention_forward_workspace(
    const struct cuju_linear_attention *attention) {
    if (!Fits(attention) || !Splits(*attention)) return 0;
    const Attention &a = *attention;
    const unsigned long long kept = (unsigned long long)a.batch * a.heads * ((a.time - 1) / kSpan);
    const unsigned long long memories = a.checkpoints ? 0 : (kept * a.key_size * a.value_size + 1) / 2;
    return (memories + kept) * sizeof(double);
}

extern "C" __attribute__((visibility("default"))) int cuju_linear_attention_forward(const struct cuju_linear_attention *attention, void *stream) {
    if (!Fits(attention)) return -1;
    const Attention &a = *attention;
    if (a.batch == 0) return 0;
    if (a.time > 0 && (!a.query || !a.key || !a.value || !a.decay || !a.output)) return Failed("expected inputs and an output");
    if (cuju_linear_attention_forward_workspace(attention) && !a.workspace) return Failed("expected a workspace");
    ForType(a.type, [&](auto x) { Forward<decltype(x)>(a, static_cast<hipStream_t>(stream)); });
    return Launched("linear attention over many steps");
}
