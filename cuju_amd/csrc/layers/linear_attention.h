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

#include <array>

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

// A step's gate; what is loaded is looked at only when it is used.
struct Step {
    float decay;
    unsigned char reset;
    __device__ __forceinline__ bool Cleared() const { return reset | (decay < kNothingKept); }
    // Whether 32 steps of such factors could leave the range of 32 bits on the way to a product that does not.
    __device__ __forceinline__ bool Steep() const { return !(decay <= 2.f); }
};

// Wavefronts that a SIMD has to hold.
template <class T, int KeyTiles, int Tiles, Mode mode>
constexpr int kRunWaves = 2;

constexpr int kSteps = 2 * kChunk;  // steps that are played together: two tiles of the matrix instruction

// Sums over the products of pieces whose places add up to less than `Most`.
template <int Most, int A, int B>
__device__ __forceinline__ F4 MfmaMost(const B8 (&a)[A], const B8 (&b)[B], F4 c) {
#pragma unroll
    for (int i = A - 1; i >= 0; i--)
#pragma unroll
        for (int j = B - 1; j >= 0; j--)
            if (i + j < Most) c = Mfma32(a[i], b[j], c);
    return c;
}
// The same of 16 contracted indices, two products to an instruction.
template <int Most, int A, int B>
__device__ __forceinline__ F4 MfmaHalves(const Four (&a)[A], const Four (&b)[B], F4 c) {
    Four left{}, right{};
    bool half = false;
#pragma unroll
    for (int i = A - 1; i >= 0; i--)
#pragma unroll
        for (int j = B - 1; j >= 0; j--) {
            if (i + j >= Most) continue;
            if (half) c = Mfma32(Eight(left, a[i]), Eight(right, b[j]), c);
            left = a[i], right = b[j], half = !half;
        }
    return half ? Mfma32(Eight(left, left), Eight(right, Four{}), c) : c;
}
template <int Pieces>
__device__ __forceinline__ void SplitPair(F4 lo, F4 hi, B8 (&x)[Pieces]) {
    const float first[4] = {lo[0], lo[1], lo[2], lo[3]}, second[4] = {hi[0], hi[1], hi[2], hi[3]};
    Four a[Pieces], b[Pieces];
    Split<Pieces>(first, a), Split<Pieces>(second, b);
    Eights(a, b, x);
}
// Eight elements in memory.
template <class T>
__device__ __forceinline__ void PiecesOf(const Pack<T, 8> &x, B8 (&piece)[kPieces<T>]) {
    struct Halves {
        Pack<T, 4> x[2];
    };
    const Halves h = __builtin_bit_cast(Halves, x);
    Pair<T>(h.x[0], h.x[1], piece);
}

// One wavefront takes 16 * Tiles columns of a head's memory through a span, 32 steps at a time, with the memory in
// registers. The columns never mix, so the wavefronts of a head share nothing.
//
// With the steps i, j of a chunk, G_i the product of the factors up to i and D_ij of those from j + 1 to i (0 across an
// episode's start), O = out (G Q S + in (D o Q K^T) V), and the memory becomes G_C S + K^T (in D_C V). The products
// are sums of products of bfloat16 pieces (common.h), 32 indices an instruction. A 16-bit output takes the memory and the
// scores in two pieces, 16 bits: the 2^-16 that is lost of a term is less than the output's rounding by 2^-9 or
// 2^-12. The memory itself, and outputs whose dots are taken for the decays, keep all three.
//
// A lane holds eight neighbouring rows of a pair of tiles: rows 32 p + 8 g + 4 x + r of the tiles 2 p + x, so that its
// keys are 16 bytes of memory. Which rows a tile has is free as long as queries, keys and memory agree.
//
// The products over a chunk's steps take a NaN or an infinity of a key or value, times a zero, to all of them. A chunk
// that has one, or factors past e^2, is played step by step.
template <class T, int KeyTiles, int Tiles, bool Whole, Mode mode>
__global__ __launch_bounds__(64) __attribute__((amdgpu_waves_per_eu(kRunWaves<T, KeyTiles, Tiles, mode>))) void RunKernel(Runs a) {
    constexpr int P = kPieces<T>, kPairs = KeyTiles / 2;
    constexpr int kHeld = mode == kGradient || P == kFloatPieces ? kFloatPieces : 2;
    __shared__ double reach[kSteps];
    __shared__ __align__(16) float wholes[kSteps], afters[kSteps], diagonal[kSteps];
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
    const bool reverse = run.reverse;
    const int column = slice * 16 * Tiles + m * Tiles, mine = max(0, min(Tiles, columns - column));
    const int begin = span * a.length, count = min(a.length, a.time - begin);
    const long long size = (long long)rows * columns, before = (long long)head * (a.spans - 1);
    const auto rowOf = [&](int t) { return 32 * (t >> 1) + 8 * g + 4 * (t & 1); };

    F4 s[KeyTiles][Tiles];
#pragma unroll
    for (int t = 0; t < KeyTiles; t++)
#pragma unroll
        for (int c = 0; c < Tiles; c++) s[t][c] = F4{0, 0, 0, 0};
    // take(element of the run's memory, element of another) in its place.
    const auto read = [&](const float *memory, auto take) {
#pragma unroll
        for (int t = 0; t < KeyTiles; t++) {
            const int row = rowOf(t);
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
                const int row = rowOf(t) + r;
                Pack<float, Tiles> x;
#pragma unroll
                for (int c = 0; c < Tiles; c++) x.x[c] = s[t][c][r];
                Store<Tiles, Whole>(memory + (long long)row * columns + column, x, row < rows ? mine : 0);
            }
    };
    if constexpr (mode != kMemory) {
        const bool starts = reverse ? span == a.spans - 1 : span == 0;
        const float *memory = starts ? run.first : run.starts;
        if (memory)
            read(memory + (starts ? (long long)head : before + (reverse ? span : span - 1)) * size, [](float, float y) { return y; });
    }

    // The time of the span's step i, and what the memory is scaled by on the way to it: backwards in time that is the
    // factor of the step that comes after it in time, and none for the first.
    const auto timeOf = [&](int i) { return reverse ? begin + count - 1 - i : begin + i; };
    const auto gateAt = [&](int t) {
        Step step{Global(a.decay)[b * a.decayStrides[0] + t * a.decayStrides[1] + h * a.decayStrides[2]], 0};
        if (a.resets) step.reset = Global(a.resets)[b * a.resetStrides[0] + t * a.resetStrides[1]];
        return step;
    };
    const auto gateOf = [&](int i) {
        return i < count && (i > 0 || !reverse) ? gateAt(reverse ? timeOf(i) + 1 : timeOf(i)) : Step{0.f, 0};
    };
    const auto scale = [&](Step gate) {
        const bool cleared = gate.Cleared();
        const float kept = cleared ? 0.f : expf(gate.decay);
#pragma unroll
        for (int t = 0; t < KeyTiles; t++)
#pragma unroll
            for (int c = 0; c < Tiles; c++)
#pragma unroll
                for (int r = 0; r < 4; r++) s[t][c][r] = cleared ? 0.f : kept * s[t][c][r];
    };
    const auto at = [&](const void *p, const long long *strides, int heads, int t) {
        return Global(static_cast<const T *>(p)) + b * strides[0] + t * strides[1] + h / heads * strides[2];
    };
    const auto put = [&](int t, const float (&x)[Tiles], int valid) {
        const long long to = b * run.outputStrides[0] + t * run.outputStrides[1] + h * run.outputStrides[2] + column;
        if (run.floats) {
            Pack<float, Tiles> o;
#pragma unroll
            for (int c = 0; c < Tiles; c++) o.x[c] = x[c];
            Store<Tiles, Whole>(Global(static_cast<float *>(run.output)) + to, o, valid);
        } else {
            Pack<T, Tiles> o;
#pragma unroll
            for (int c = 0; c < Tiles; c++) o.x[c] = As<T>(x[c]);
            Store<Tiles, Whole>(Global(static_cast<T *>(run.output)) + to, o, valid);
        }
    };

    // Steps one after the other.
    const auto playSteps = [&](int first, int past) {
#pragma unroll 1
        for (int i = first; i < past; i++) {
            const int t = timeOf(i);
            const auto v = Load<Tiles, Whole>(at(run.value, run.valueStrides, run.valueHeads, t) + column, mine);
            if (i > 0 || !reverse) scale(gateOf(i));
            const T *key = at(run.key, run.keyStrides, run.keyHeads, t);
            const T *query = mode == kMemory ? nullptr : at(run.query, run.queryStrides, run.queryHeads, t);
            float strict[Tiles] = {}, own = 0;
#pragma unroll
            for (int x = 0; x < KeyTiles; x++) {
                const int row = rowOf(x);
                const auto k = Load<4, Whole>(key + row, rows - row);
                Pack<T, 4> q{};
                if constexpr (mode != kMemory) q = Load<4, Whole>(query + row, rows - row);
#pragma unroll
                for (int r = 0; r < 4; r++) {
                    if constexpr (mode != kMemory) own = fmaf(Float(q.x[r]), Float(k.x[r]), own);
#pragma unroll
                    for (int c = 0; c < Tiles; c++) {
                        if constexpr (mode != kMemory) strict[c] = fmaf(Float(q.x[r]), s[x][c][r], strict[c]);
                        s[x][c][r] = fmaf(Float(k.x[r]) * run.in, Float(v.x[c]), s[x][c][r]);
                    }
                }
            }
            if constexpr (mode != kMemory) {
                own += __shfl_xor(own, 16);
                own += __shfl_xor(own, 32);
                Pack<T, Tiles> w{};
                if constexpr (mode == kGradient)
                    if (run.weight) w = Load<Tiles, Whole>(at(run.weight, run.weightStrides, run.weightHeads, t) + column, mine);
                float dot = 0;
#pragma unroll
                for (int c = 0; c < Tiles; c++) {
                    strict[c] += __shfl_xor(strict[c], 16);
                    strict[c] += __shfl_xor(strict[c], 32);
                    strict[c] *= run.out;
                    if (c < mine) dot = fmaf(strict[c], Float(w.x[c]), dot);
                    strict[c] = fmaf(run.out * run.in * own, Float(v.x[c]), strict[c]);
                }
                put(t, strict, g == 0 ? mine : 0);
                if constexpr (mode == kGradient) {
                    dot = RowSum(dot);
                    if (run.weight && lane == 0) run.dots[((long long)slice * a.allHeads + head) * a.time + t] = dot;
                }
            }
        }
    };

    // The inputs of the steps from `first`: of a lane's steps m and 16 + m the keys and queries, of its steps 4 g + r and
    // 16 + 4 g + r the values. Past the end the last step is read again.
    Pack<T, 8> nextK[2][kPairs], nextQ[2][kPairs];
    Pack<T, Tiles> nextV[2][4];
    Step nextGate[2];
    const auto eight = [&](const T *p, int row) {
        struct Halves {
            Pack<T, 4> x[2];
        } h{Load<4, Whole>(p + row, rows - row), Load<4, Whole>(p + row + 4, rows - row - 4)};
        return __builtin_bit_cast(Pack<T, 8>, h);
    };
    const auto fetchKeys = [&](int first) {
#pragma unroll
        for (int n = 0; n < 2; n++) {
            const int t = timeOf(min(first + 16 * n + m, count - 1));
            const T *key = at(run.key, run.keyStrides, run.keyHeads, t);
#pragma unroll
            for (int p = 0; p < kPairs; p++) nextK[n][p] = eight(key, rowOf(2 * p));
            if constexpr (mode != kMemory) {
                const T *query = at(run.query, run.queryStrides, run.queryHeads, t);
#pragma unroll
                for (int p = 0; p < kPairs; p++) nextQ[n][p] = eight(query, rowOf(2 * p));
            }
        }
    };
    const auto fetchValues = [&](int first) {
#pragma unroll
        for (int n = 0; n < 2; n++) {
            nextGate[n] = gateOf(first + 16 * n + m);
#pragma unroll
            for (int r = 0; r < 4; r++) {
                const int t = timeOf(min(first + 16 * n + 4 * g + r, count - 1));
                nextV[n][r] = Load<Tiles, Whole>(at(run.value, run.valueStrides, run.valueHeads, t) + column, mine);
            }
        }
    };

    const Eyes eyes = EyesOf(m, g);
    const auto ones = __builtin_bit_cast(B8, std::array<uint32_t, 4>{0x3f803f80u, 0x3f803f80u, 0x3f803f80u, 0x3f803f80u});
    if (count > 0) fetchKeys(0), fetchValues(0);
#pragma unroll 1
    for (int first = 0; first < count; first += kSteps) {
        const int valid = min(kSteps, count - first);
        if constexpr (mode == kOutputs)
            if (run.kept && first > 0 && first % kSpan == 0)
                write(run.kept + ((long long)head * ((a.time - 1) / kSpan) + first / kSpan - 1) * size);

        // Pieces of the keys and queries; products with the memory, the scores, and the keys' transpose.
        F4 mark = {0, 0, 0, 0}, scores[3], o[2][Tiles];  // scores: of the tiles 00, 10 and 11, in row order
        Four turned[2][KeyTiles][P];
#pragma unroll
        for (int x = 0; x < 3; x++) scores[x] = F4{0, 0, 0, 0};
#pragma unroll
        for (int n = 0; n < 2; n++)
#pragma unroll
            for (int c = 0; c < Tiles; c++) o[n][c] = F4{0, 0, 0, 0};
#pragma unroll
        for (int p = 0; p < kPairs; p++) {
            B8 kp[2][P], qp[2][P];
#pragma unroll
            for (int n = 0; n < 2; n++) {
                PiecesOf<T>(nextK[n][p], kp[n]);
                mark = Mfma32(ones, kp[n][0], mark);
                Turn<P>(kp[n], eyes.half[0], turned[n][2 * p]);
                Turn<P>(kp[n], eyes.half[1], turned[n][2 * p + 1]);
            }
            if constexpr (mode != kMemory) {
#pragma unroll
                for (int n = 0; n < 2; n++) PiecesOf<T>(nextQ[n][p], qp[n]);
                scores[0] = MfmaMost<3>(kp[0], qp[0], scores[0]);
                scores[1] = MfmaMost<3>(kp[0], qp[1], scores[1]);
                scores[2] = MfmaMost<3>(kp[1], qp[1], scores[2]);
#pragma unroll
                for (int c = 0; c < Tiles; c++) {
                    B8 sp[kHeld];
                    SplitPair<kHeld>(s[2 * p][c], s[2 * p + 1][c], sp);
#pragma unroll
                    for (int n = 0; n < 2; n++) o[n][c] = MfmaMost<kHeld>(qp[n], sp, o[n][c]);
                }
            }
        }
        Pack<T, Tiles> v[2][4];
#pragma unroll
        for (int n = 0; n < 2; n++)
#pragma unroll
            for (int r = 0; r < 4; r++) v[n][r] = 16 * n + 4 * g + r < valid ? nextV[n][r] : Pack<T, Tiles>{};
        const Step gate[2] = {nextGate[0], nextGate[1]};
        Pack<T, Tiles> w[2][4];
        if constexpr (mode == kGradient)
            if (run.weight)
#pragma unroll
                for (int n = 0; n < 2; n++)
#pragma unroll
                    for (int r = 0; r < 4; r++)
                        w[n][r] = Load<Tiles, Whole>(at(run.weight, run.weightStrides, run.weightHeads,
                                                        timeOf(min(first + 16 * n + 4 * g + r, count - 1))) + column, mine);
        if (first + kSteps < count) fetchKeys(first + kSteps), fetchValues(first + kSteps);

        // The values as right operands, [piece].
        B8 vp[Tiles][P];
#pragma unroll
        for (int c = 0; c < Tiles; c++) {
            Four half[2][P];
#pragma unroll
            for (int n = 0; n < 2; n++) {
                const Pack<T, 4> x{{v[n][0].x[c], v[n][1].x[c], v[n][2].x[c], v[n][3].x[c]}};
                Split<T>(x, half[n]);
            }
            Eights(half[0], half[1], vp[c]);
            mark = Mfma32(ones, vp[c][0], mark);
        }
        if (__ballot(mark[0] * 0.f != 0.f || gate[0].Steep() || gate[1].Steep())) {
            playSteps(first, first + valid);
            continue;
        }

        // How the chunk is cut, and the products of its factors.
        const bool cleared[2] = {gate[0].Cleared(), gate[1].Cleared()};
        const unsigned cuts = (unsigned)(__ballot(cleared[0]) & 0xffff) | (unsigned)(__ballot(cleared[1]) & 0xffff) << 16;
        double G[2];
        G[0] = RowUpTo(cleared[0] ? 0.0 : gate[0].decay * kLog2E);
        G[1] = RowUpTo(cleared[1] ? 0.0 : gate[1].decay * kLog2E) + __shfl(G[0], 15);
        const double last = __shfl(G[1], 15);
        int start[2];  // where the episode of a lane's steps starts, or -1 before the chunk
#pragma unroll
        for (int n = 0; n < 2; n++) {
            const unsigned upTo = cuts & ((2u << (16 * n + m)) - 1);
            start[n] = upTo ? 31 - __builtin_clz(upTo) : -1;
        }
        const int latest = cuts ? 31 - __builtin_clz(cuts) : -1;
        __syncthreads();
        if (g == 0) {
#pragma unroll
            for (int n = 0; n < 2; n++) {
                const int i = 16 * n + m;
                reach[i] = G[n];
                wholes[i] = start[n] < 0 ? run.out * Exp2(G[n]) : -1.f;
                afters[i] = i >= latest ? run.in * Exp2(last - G[n]) : 0.f;
            }
        }
        __syncthreads();

        if constexpr (mode != kMemory) {
            const float both = run.in * run.out;
            const bool strict = mode == kGradient;
            F4 mixed[3];
#pragma unroll
            for (int x = 0; x < 3; x++) {
                const int n = x > 0, j0 = x == 2 ? 16 : 0;
#pragma unroll
                for (int r = 0; r < 4; r++) {
                    const int i = 16 * n + m, j = j0 + 4 * g + r;
                    const float d = both * Exp2(G[n] - reach[j]);
                    if (mode == kGradient && x != 1 && i == j) diagonal[i] = both * scores[x][r];
                    mixed[x][r] = j >= start[n] && (strict ? j < i : j <= i) ? d * scores[x][r] : 0.f;
                }
            }
            Four lower[3][kHeld];
#pragma unroll
            for (int x = 0; x < 3; x++) {
                const float f[4] = {mixed[x][0], mixed[x][1], mixed[x][2], mixed[x][3]};
                Split<kHeld>(f, lower[x]);
            }
            B8 second[kHeld];
            Eights(lower[1], lower[2], second);
            __syncthreads();
#pragma unroll
            for (int n = 0; n < 2; n++) {
                const F4 whole = *reinterpret_cast<const F4 *>(wholes + 16 * n + 4 * g);
#pragma unroll
                for (int c = 0; c < Tiles; c++) {
#pragma unroll
                    for (int r = 0; r < 4; r++) o[n][c][r] = whole[r] < 0.f ? 0.f : whole[r] * o[n][c][r];
                    if (n == 1) {
                        o[n][c] = MfmaMost<kHeld>(second, vp[c], o[n][c]);
                    } else {
                        Four half[P];
#pragma unroll
                        for (int i = 0; i < P; i++) {
                            struct Both {
                                Four lo, hi;
                            };
                            half[i] = __builtin_bit_cast(Both, vp[c][i]).lo;
                        }
                        o[n][c] = MfmaHalves<kHeld>(lower[0], half, o[n][c]);
                    }
                }
            }
#pragma unroll
            for (int n = 0; n < 2; n++) {
                F4 own = {0, 0, 0, 0};
                if constexpr (mode == kGradient) own = *reinterpret_cast<const F4 *>(diagonal + 16 * n + 4 * g);
#pragma unroll
                for (int r = 0; r < 4; r++) {
                    const int i = 16 * n + 4 * g + r, t = timeOf(first + i);
                    float x[Tiles], dot = 0;
#pragma unroll
                    for (int c = 0; c < Tiles; c++) {
                        x[c] = o[n][c][r];
                        if constexpr (mode == kGradient) {
                            if (c < mine) dot = fmaf(x[c], Float(w[n][r].x[c]), dot);
                            x[c] = fmaf(own[r], Float(v[n][r].x[c]), x[c]);
                        }
                    }
                    put(t, x, i < valid ? mine : 0);
                    if constexpr (mode == kGradient)
                        if (run.weight) {
                            dot = RowSum(dot);
                            if (m == 0 && i < valid) run.dots[((long long)slice * a.allHeads + head) * a.time + t] = dot;
                        }
                }
            }
        }

        const float kept = Exp2(last);
        B8 kt[KeyTiles][P];
#pragma unroll
        for (int t = 0; t < KeyTiles; t++) Eights(turned[0][t], turned[1][t], kt[t]);
#pragma unroll
        for (int c = 0; c < Tiles; c++) {
            F4 x[2];
#pragma unroll
            for (int n = 0; n < 2; n++) {
                const F4 after = *reinterpret_cast<const F4 *>(afters + 16 * n + 4 * g);
#pragma unroll
                for (int r = 0; r < 4; r++) x[n][r] = after[r] * Float(v[n][r].x[c]);
            }
            B8 written[kFloatPieces];
            SplitPair<kFloatPieces>(x[0], x[1], written);
#pragma unroll
            for (int t = 0; t < KeyTiles; t++) {
                F4 held;
#pragma unroll
                for (int r = 0; r < 4; r++) held[r] = cuts ? 0.f : kept * s[t][c][r];
                s[t][c] = MfmaMost<3>(kt[t], written, held);
            }
        }
    }

    if constexpr (mode == kMemory) {
        if (reverse && count > 0) scale(gateAt(begin));
        write(run.last + (before + (reverse ? span - 1 : span)) * size);
        if (slice == 0) {
            // The span's factors.
            double sum = 0;
            bool cleared = false;
            for (int t = begin + lane; t < begin + count; t += 64) {
                const Step gate = gateAt(t);
                cleared |= gate.Cleared();
                sum += gate.decay;
            }
            for (int d = 32; d; d /= 2) sum += __shfl_xor(sum, d);
            const float factor = __ballot(cleared) ? -1.f : (float)exp(sum);
            if (lane == 0) a.factors[before + (reverse ? span - 1 : span)] = factor;
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
        if (run.last && span == (reverse ? 0 : a.spans - 1)) {
            if (reverse && count > 0) scale(gateAt(0));
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
