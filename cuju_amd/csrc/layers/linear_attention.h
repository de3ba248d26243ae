// Linear attention with decays, as runs of one recurrence: its forward pass, and its gradients, which are the same
// recurrence with the tensors in other roles.
//
//   S_t = a_t S_{t-1} + k_t v_t^T,  o_t = scale S_t^T q_t,  a_t = exp(decay_t), 0 where an episode starts.
//
// With dS_t the gradient of S_t, dS_t = scale q_t do_t^T + a_{t+1} dS_{t+1}:
//   dq_t = scale S_t do_t:  query do, key v, value k, memory S^T;
//   dv_t = dS_t^T k_t:      backwards in time, query k, key q, value do, memory dS;
//   dk_t = dS_t v_t:        backwards in time, query v, key do, value q, memory dS^T.
// A run's own columns (of the memory and of the outputs) are its value's, its rows its key's. The log decay of step t
// gets <dS_t, a_t S_{t-1}>, which is that of step t + 1 and q_t.dq_t - k_t.dk_t without the step's own product; so the
// runs for dq and dk leave those dots, and a sum backwards over time, begun anew at the end of every span and episode,
// finds the decays' gradients.
//
// Steps are cut into spans of 128 (kSpan). With the memories at the ends of spans known, the spans are played side by
// side: that is how gradients are found, and how few long sequences fill the chip.
#pragma once
#include "../../../include/cuju_amd.h"
#include "steps.h"

namespace layers {

using Attention = cuju_linear_attention;
constexpr int kSpan = 128;

// One run of the recurrence over all heads.
struct Run {
    const void *query, *key, *value, *weight;  // weight: what the outputs' dots are taken with, or null
    long long queryStrides[3], keyStrides[3], valueStrides[3], weightStrides[3];
    int queryHeads, keyHeads, valueHeads, weightHeads;  // heads that share one of the tensor's
    int rows, columns, slices;
    bool reverse, transposed;  // whether steps go backwards, and memories lie [column][row]
    float in, out;             // factors of what is written and of what is read
    void *output;
    long long outputStrides[3];
    bool floats;          // whether the output is float, whatever the type
    const float *first;   // the memory at the run's start, or null for zeros
    const float *starts;  // at the start of its other spans, [head][spans - 1], in the order of time
    float *last;          // the memory at the end of the run, or null (backwards: before the first step)
    float *kept;          // the memory before every span but the first, in a run of one piece; or null
    float *dots;          // [slice][head][time]
    const float *against, *againstLast;  // memories at the ends of spans, and the last one's: their products with the run's
    float *crossings;                    // [slice][head][span]
};
struct Runs {
    int time, heads, length, spans, firstSpan, spanCount, units;  // length: steps of a span; units: slices of all runs
    unsigned firstHead, allHeads;
    const float *decay;
    const unsigned char *resets;
    long long decayStrides[3], resetStrides[2];
    float *factors;  // [head][spans - 1]: the product of a span's factors, or -1 where an episode starts in it
    Run run[3];
};

enum Mode {
    kMemory,   // the memory alone, from zeros, at the end of every span that has another behind it
    kOutputs,  // outputs
    kGradient  // outputs, and their dots with the weights
};

struct Step {
    float decay;
    bool cleared;
};

template <class T, int KeyTiles, int Tiles, bool Whole, Mode mode>
__global__ __launch_bounds__(64) void RunKernel(Runs a) {
    const int lane = threadIdx.x, m = lane & 15, g = lane >> 4;
    unsigned id = Place(blockIdx.x, gridDim.x);
    int slice = id % a.units, which = 0;
    id /= a.units;
    const int span = a.firstSpan + id % a.spanCount;
    const unsigned head = a.firstHead + id / a.spanCount;
    while (slice >= a.run[which].slices) slice -= a.run[which++].slices;
    const Run &run = a.run[which];
    const int h = head % a.heads, b = head / a.heads;
    const int rows = run.rows, columns = run.columns;
    const int column = slice * 16 * Tiles + m * Tiles, mine = max(0, min(Tiles, columns - column));
    const int begin = span * a.length, count = min(a.length, a.time - begin);
    const long long size = (long long)rows * columns, before = (long long)head * (a.spans - 1);

    F4 s[KeyTiles][Tiles];
#pragma unroll
    for (int t = 0; t < KeyTiles; t++)
#pragma unroll
        for (int c = 0; c < Tiles; c++) s[t][c] = F4{0, 0, 0, 0};
    // take(element of the run's memory, element of another) in its place.
    const auto read = [&](const float *memory, auto take) {
#pragma unroll
        for (int t = 0; t < KeyTiles; t++) {
            const int row = 16 * t + 4 * g;
            if (run.transposed) {
#pragma unroll
                for (int c = 0; c < Tiles; c++) {
                    const auto x = Load<4, Whole>(memory + (long long)(column + c) * rows + row, c < mine ? rows - row : 0);
#pragma unroll
                    for (int r = 0; r < 4; r++) s[t][c][r] = take(s[t][c][r], x.x[r]);
                }
            } else {
#pragma unroll
                for (int r = 0; r < 4; r++) {
                    const auto x = Load<Tiles, Whole>(memory + (long long)(row + r) * columns + column, row + r < rows ? mine : 0);
#pragma unroll
                    for (int c = 0; c < Tiles; c++) s[t][c][r] = take(s[t][c][r], x.x[c]);
                }
            }
        }
    };
    const auto write = [&](float *memory) {
#pragma unroll
        for (int t = 0; t < KeyTiles; t++)
#pragma unroll
            for (int r = 0; r < 4; r++) {
                const int row = 16 * t + 4 * g + r;
                Pack<float, Tiles> x;
#pragma unroll
                for (int c = 0; c < Tiles; c++) x.x[c] = s[t][c][r];
                Store<Tiles, Whole>(memory + (long long)row * columns + column, x, row < rows ? mine : 0);
            }
    };
    if constexpr (mode != kMemory) {
        const bool starts = run.reverse ? span == a.spans - 1 : span == 0;
        const float *memory = starts ? run.first : run.starts;
        if (memory)
            read(memory + (starts ? (long long)head : before + (run.reverse ? span : span - 1)) * size, [](float, float y) { return y; });
    }

    // The time of the span's step i, and what the memory is scaled by on the way to it: backwards in time that is the
    // factor of the step that comes after it in time.
    const auto timeOf = [&](int i) { return run.reverse ? begin + count - 1 - i : begin + i; };
    const auto gateAt = [&](int t) {
        Step step{Global(a.decay)[b * a.decayStrides[0] + t * a.decayStrides[1] + h * a.decayStrides[2]], false};
        if (a.resets) step.cleared = Global(a.resets)[b * a.resetStrides[0] + t * a.resetStrides[1]];
        step.cleared |= step.decay < kNothingKept;
        return step;
    };
    const auto scale = [&](Step gate) {
        const float kept = gate.cleared ? 0.f : expf(gate.decay);
#pragma unroll
        for (int t = 0; t < KeyTiles; t++)
#pragma unroll
            for (int c = 0; c < Tiles; c++)
#pragma unroll
                for (int r = 0; r < 4; r++) s[t][c][r] = gate.cleared ? 0.f : kept * s[t][c][r];
    };
    const auto at = [&](const void *p, const long long *strides, int heads, int t) {
        return Global(static_cast<const T *>(p)) + b * strides[0] + t * strides[1] + h / heads * strides[2];
    };

#pragma unroll 1
    for (int i = 0; i < count; i++) {
        const int t = timeOf(i);
        if constexpr (mode == kOutputs)
            if (run.kept && i > 0 && i % kSpan == 0)
                write(run.kept + ((long long)head * ((a.time - 1) / kSpan) + i / kSpan - 1) * size);
        const auto v = Load<Tiles, Whole>(at(run.value, run.valueStrides, run.valueHeads, t) + column, mine);
        if (!run.reverse) scale(gateAt(t));
        else if (i > 0) scale(gateAt(t + 1));
        const T *key = at(run.key, run.keyStrides, run.keyHeads, t), *query = at(run.query, run.queryStrides, run.queryHeads, t);
        float strict[Tiles] = {}, own = 0;
#pragma unroll
        for (int x = 0; x < KeyTiles; x++) {
            const int row = 16 * x + 4 * g;
            const auto k = Load<4, Whole>(key + row, rows - row);
            Pack<T, 4> q{};
            if constexpr (mode != kMemory) q = Load<4, Whole>(query + row, rows - row);
#pragma unroll
            for (int r = 0; r < 4; r++) {
                if constexpr (mode == kGradient) {
                    own = fmaf(Float(q.x[r]), Float(k.x[r]), own);
#pragma unroll
                    for (int c = 0; c < Tiles; c++) strict[c] = fmaf(Float(q.x[r]), s[x][c][r], strict[c]);
                }
#pragma unroll
                for (int c = 0; c < Tiles; c++) {
                    s[x][c][r] = fmaf(Float(k.x[r]) * run.in, Float(v.x[c]), s[x][c][r]);
                    if constexpr (mode == kOutputs) strict[c] = fmaf(Float(q.x[r]), s[x][c][r], strict[c]);
                }
            }
        }
        if constexpr (mode != kMemory) {
            own += __shfl_xor(own, 16);
            own += __shfl_xor(own, 32);
            Pack<T, Tiles> w{}, o;
            Pack<float, Tiles> wide;
            if constexpr (mode == kGradient)
                if (run.weight) w = Load<Tiles, Whole>(at(run.weight, run.weightStrides, run.weightHeads, t) + column, mine);
            float dot = 0;
#pragma unroll
            for (int c = 0; c < Tiles; c++) {
                strict[c] += __shfl_xor(strict[c], 16);
                strict[c] += __shfl_xor(strict[c], 32);
                strict[c] *= run.out;
                if constexpr (mode == kGradient) {
                    if (c < mine) dot = fmaf(strict[c], Float(w.x[c]), dot);
                    strict[c] = fmaf(run.out * run.in * own, Float(v.x[c]), strict[c]);
                }
                o.x[c] = As<T>(strict[c]);
                wide.x[c] = strict[c];
            }
            const long long to = b * run.outputStrides[0] + t * run.outputStrides[1] + h * run.outputStrides[2] + column;
            if (run.floats) Store<Tiles, Whole>(static_cast<float *>(run.output) + to, wide, g == 0 ? mine : 0);
            else Store<Tiles, Whole>(static_cast<T *>(run.output) + to, o, g == 0 ? mine : 0);
            if constexpr (mode == kGradient) {
                dot = RowSum(dot);
                if (run.weight && lane == 0) run.dots[((long long)slice * a.allHeads + head) * a.time + t] = dot;
            }
        }
    }

    if constexpr (mode == kMemory) {
        if (run.reverse && count > 0) scale(gateAt(begin));
        write(run.last + (before + (run.reverse ? span - 1 : span)) * size);
        if (slice == 0) {
            // The span's factors.
            double sum = 0;
            bool cleared = false;
            for (int t = begin + lane; t < begin + count; t += 64) {
                const Step gate = gateAt(t);
                cleared |= gate.cleared;
                sum += gate.decay;
            }
            for (int d = 32; d; d /= 2) sum += __shfl_xor(sum, d);
            const float factor = __ballot(cleared) ? -1.f : (float)exp(sum);
            if (lane == 0) a.factors[before + (run.reverse ? span - 1 : span)] = factor;
        }
    } else {
        if constexpr (mode == kGradient)
            if (run.crossings) {
                const bool ends = span == a.spans - 1;
                const float *memory = ends ? run.againstLast : run.against;
                float sum = 0;
                if (memory) read(memory + (ends ? (long long)head : before + span) * size, [&](float x, float y) { return sum = fmaf(x, y, sum), x; });
                sum = WaveSum(sum);
                if (lane == 0) run.crossings[((long long)slice * a.allHeads + head) * a.spans + span] = sum;
            }
        if (run.last && span == (run.reverse ? 0 : a.spans - 1)) {
            if (run.reverse && count > 0) scale(gateAt(0));
            write(run.last + (long long)head * size);
        }
    }
}

// A tensor's place in a run; `heads` share one of its heads.
inline bool IsWhole(const void *p, const long long *strides, int size, size_t bytes) {
    return strides[0] % 4 == 0 && strides[1] % 4 == 0 && strides[2] % 4 == 0 && size % 4 == 0 && Aligned(4 * bytes, p);
}
inline void Take(const void *&p, long long (&strides)[3], int &heads, const void *from, const long long *fromStrides, int share) {
    p = from, heads = share;
    for (int i = 0; i < 3; i++) strides[i] = fromStrides[i];
}
inline Runs RunsOf(const Attention &a) {
    Runs r{};
    r.time = a.time, r.heads = a.heads, r.length = kSpan, r.spans = a.time > kSpan ? (a.time + kSpan - 1) / kSpan : 1;
    r.spanCount = r.spans, r.allHeads = (unsigned)(a.batch * (long long)a.heads);
    r.decay = static_cast<const float *>(a.decay), r.resets = a.resets;
    for (int i = 0; i < 3; i++) r.decayStrides[i] = a.decay_strides[i];
    for (int i = 0; i < 2; i++) r.resetStrides[i] = a.reset_strides[i];
    return r;
}
// Whether every pack of four of the call's tensors is aligned and none is cut.
inline bool IsWhole(const Attention &a) {
    const size_t bytes = a.type == 0 ? 4 : 2;
    for (const void *p : {a.output, static_cast<void *>(a.d_query), static_cast<void *>(a.d_key), static_cast<void *>(a.d_value)})
        if (!Aligned(4 * bytes, p)) return false;
    for (const void *p : {static_cast<const void *>(a.state), static_cast<const void *>(a.last), static_cast<const void *>(a.checkpoints),
                          a.d_last, static_cast<const void *>(a.d_state), static_cast<const void *>(a.workspace)})
        if (!Aligned(16, p)) return false;
    return IsWhole(a.query, a.query_strides, a.key_size, bytes) && IsWhole(a.key, a.key_strides, a.key_size, bytes) &&
           IsWhole(a.value, a.value_strides, a.value_size, bytes) &&
           (!a.d_output || IsWhole(a.d_output, a.d_output_strides, a.value_size, bytes));
}

// The tiles of 16 columns that a wavefront of a launch takes, 0 to 2 as powers of two.
template <class T>
int TilesOf(const Runs &runs, int count, int keyTiles, bool whole) {
    if (!whole) return 1;
    const int most = kPieces<T> * keyTiles > 12 ? 1 : kPieces<T> * keyTiles > 4 ? 2 : 4;
    for (int tiles = most; tiles > 1; tiles /= 2) {
        long long slices = 0;
        bool wide = false;
        for (int i = 0; i < count; i++) {
            slices += (runs.run[i].columns + 16 * tiles - 1) / (16 * tiles);
            wide |= runs.run[i].columns > 8 * tiles;
        }
        if (wide && runs.allHeads * slices * runs.spanCount >= 1024) return tiles;
    }
    return 1;
}
inline int KeyTilesOf(const Runs &runs, int count) {
    int rows = 0;
    for (int i = 0; i < count; i++) rows = rows > runs.run[i].rows ? rows : runs.run[i].rows;
    return rows <= 32 ? 2 : rows <= 64 ? 4 : rows <= 96 ? 6 : 8;
}
// Cuts the columns of the runs for wavefronts of `tiles` tiles.
inline void Cut(Runs &runs, int count, int tiles) {
    runs.units = 0;
    for (int i = 0; i < count; i++) {
        runs.run[i].slices = (runs.run[i].columns + 16 * tiles - 1) / (16 * tiles);
        runs.units += runs.run[i].slices;
    }
}

template <class T, Mode mode, int KeyTiles>
void LaunchTiles(Runs &runs, int count, bool whole, hipStream_t stream) {
    constexpr int most = kPieces<T> * KeyTiles > 12 ? 1 : kPieces<T> * KeyTiles > 4 ? 2 : 4;
    const int tiles = TilesOf<T>(runs, count, KeyTiles, whole);
    Cut(runs, count, tiles);
    const auto launch = [&](auto kernel) {
        // A grid has fewer than 2^32 threads.
        const unsigned blocks = runs.units * runs.spanCount, most = (1u << 25) / blocks < 1 ? 1 : (1u << 25) / blocks;
        for (unsigned first = 0; first < runs.allHeads; first += most) {
            runs.firstHead = first;
            const unsigned heads = runs.allHeads - first < most ? runs.allHeads - first : most;
            hipLaunchKernelGGL(kernel, dim3(heads * blocks), dim3(64), 0, stream, runs);
        }
    };
    if (!whole) launch(RunKernel<T, KeyTiles, 1, false, mode>);
    else if (tiles == 4) launch(RunKernel<T, KeyTiles, most >= 4 ? 4 : 1, true, mode>);
    else if (tiles == 2) launch(RunKernel<T, KeyTiles, most >= 2 ? 2 : 1, true, mode>);
    else launch(RunKernel<T, KeyTiles, 1, true, mode>);
}
template <class T, Mode mode>
void LaunchRuns(Runs &runs, int count, bool whole, hipStream_t stream) {
    switch (KeyTilesOf(runs, count)) {
    case 2: LaunchTiles<T, mode, 2>(runs, count, whole, stream); break;
    case 4: LaunchTiles<T, mode, 4>(runs, count, whole, stream); break;
    case 6: LaunchTiles<T, mode, 6>(runs, count, whole, stream); break;
    default: LaunchTiles<T, mode, 8>(runs, count, whole, stream); break;
    }
}
// Of the element type `type`; defined in linear_attention.hip and, for gradients, in linear_attention_backward.hip.
void RunMemories(Runs &runs, int type, bool whole, hipStream_t stream);
void RunOutputs(Runs &runs, int count, int type, bool whole, hipStream_t stream);
// The memories at the ends of spans, from those that each span leaves by itself: [head][spans - 1].
void JoinMemories(const Runs &runs, const float *first, float *memories, long long size, bool reverse, hipStream_t stream);

// Whether a call's arguments fit the kernels; the failure is kept otherwise.
inline bool Fits(const Attention *a) {
    if (!a || a->type < 0 || a->type > 2) return Failed("expected linear attention of the type 0, 1 or 2"), false;
    if (a->batch < 0 || a->time < 0 || a->heads < 1 || a->key_heads < 1 || a->heads % a->key_heads)
        return Failed("expected heads that are a multiple of the key heads"), false;
    // A grid has room for all spans of a head.
    if (a->time >= (1 << 24) || a->heads >= (1 << 16)) return Failed("expected fewer than 2^24 steps and 2^16 heads"), false;
    if (a->batch * (long long)a->heads >= (1ll << 23)) return Failed("expected fewer than 2^23 heads in the batch"), false;
    if (a->key_size < 1 || a->key_size > kMaxKey || a->value_size < 1 || a->value_size > kMaxValue)
        return Failed("expected key and value sizes from 1 to 128"), false;
    return true;
}

}  // namespace layers
