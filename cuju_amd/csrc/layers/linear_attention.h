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

struct Tensor {
    const void *p;
    long long strides[3];  // [batch][time][head]
    int share;             // heads that share one of its heads
};
// One run of the recurrence over all heads.
struct Run {
    Tensor query, key, value, weight;  // weight: what the outputs' dots are taken with, or null
    int rows, columns;
    bool reverse, transposed;  // whether steps go backwards, and memories lie [column][row]
    bool floats;               // whether the output is float, whatever the type
    float in, out;             // factors of what is written and of what is read
    void *output;
    long long outputStrides[3];
    const float *first;   // the memory at the run's start, or null for zeros
    const float *starts;  // at the start of its other spans, [head][spans - 1], in the order of time
    float *last;          // the memory at the end of the run, or null (backwards: before the first step)
    float *kept;          // the memory before every span but the first, in a run of one piece; or null
    float *dots;          // [slice][head][time]
    const float *against, *againstLast;  // memories at the ends of spans, and the last one's: their products with the run's
    float *crossings;                    // [slice][head][span]
};
struct Runs {
    int time, heads, length, spans, firstSpan, spanCount;  // length: steps of a span
    int units, slices[3];                                  // slices of all runs and of each
    unsigned firstHead, allHeads;
    const float *decay;
    const unsigned char *resets;
    long long decayStrides[3], resetStrides[2];
    bool near;       // whether 32 steps of every tensor are within 2^31 bytes
    double *factors;  // [head][spans - 1]: the product of a span's factors, or -1 where an episode starts in it
    Run run[3];
};
// A run out of the kernel's arguments, where an index that the compiler does not know would copy them all, read anew
// at every call: few of its words are needed over the long loop, and all would not fit the scalar registers.
__device__ __forceinline__ Run RunAt(int which) {
    using Word = const __attribute__((address_space(4))) uint32_t;
    Word *p = (Word *)((const __attribute__((address_space(4))) char *)__builtin_amdgcn_kernarg_segment_ptr() + offsetof(Runs, run)) +
              which * (sizeof(Run) / 4);
    asm volatile("" : "+s"(p));
    struct Words {
        uint32_t x[sizeof(Run) / 4];
    } words;
#pragma unroll
    for (int i = 0; i < (int)(sizeof(Run) / 4); i++) words.x[i] = p[i];
    return __builtin_bit_cast(Run, words);
}
// A tensor's steps of one head, in the order in which a run plays them.
template <class T>
struct Line {
    const T *p;
    long long step;
    __device__ __forceinline__ const T *At(int i) const { return p + i * step; }
};
// The same within 32 steps, counted in the order of time from the first of them.
template <class T>
struct Near {
    const T *p;
    int step;
    __device__ __forceinline__ const T *At(int i) const { return p + i * step; }
};

enum Shape {
    kLoose,  // sizes and strides that packs of four elements do not fit
    kWhole,  // that they fit
    kFull    // and sizes that the tiles fit
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

// Wavefronts that a SIMD has to hold: two hide each other's waits, and the largest memories of floats leave registers for
// one. With one and two, 4,096 heads and 64 steps: float32 64 x 64 forward 227 and 141 us, gradients 657 and 385; float16
// 128 x 128 603 and 440, 1,486 and 1,114; float32 96 x 96 425 and 574, 1,160 and 1,533.
template <class T, int KeyTiles, Mode mode>
constexpr int kRunWaves = mode != kMemory && KeyTiles * kPieces<T> >= 18 ? 1 : 2;
constexpr int kSteps = 2 * kChunk;  // steps that are played together: two tiles of the matrix instruction

// The transpose of a lane's first or second four of eight values, piece by piece, by a product with the identity: the
// instruction of 16 contracted indices, half the time of the one of 32.
template <int P>
__device__ __forceinline__ void TurnHalf(const B8 (&x)[P], int which, Four eye, Four (&turned)[P]) {
    using S4 = __attribute__((ext_vector_type(4))) short;
    struct Halves {
        S4 x[2];
    };
#pragma unroll
    for (int i = 0; i < P; i++) {
        const F4 t = __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(__builtin_bit_cast(Halves, x[i]).x[which], __builtin_bit_cast(S4, eye),
                                                               F4{0, 0, 0, 0}, 0, 0, 0);
        const float f[4] = {t[0], t[1], t[2], t[3]};
        Four whole[1];
        Split<1>(f, whole);
        turned[i] = whole[0];
    }
}
template <int Pieces>
__device__ __forceinline__ void SplitPair(F4 lo, F4 hi, B8 (&x)[Pieces]) {
    const float first[4] = {lo[0], lo[1], lo[2], lo[3]}, second[4] = {hi[0], hi[1], hi[2], hi[3]};
    Four a[Pieces], b[Pieces];
    Split<Pieces>(first, a), Split<Pieces>(second, b);
    Eights(a, b, x);
}
// Elements as the 32-bit words of memory: an array of 16-bit elements would take a register for each of them.
template <int N>
struct Words {
    uint32_t x[N];
};
template <class T, int N>
constexpr int kWords = N * (int)sizeof(T) < 4 ? 1 : N * (int)sizeof(T) / 4;
// N elements from a place aligned to `Aligned` of them, the first `valid` real and the others zero. `Whole`: either all or none.
template <class T, int N, bool Whole, int Aligned = N>
__device__ __forceinline__ Words<kWords<T, N>> LoadWords(const T *p, int valid = N) {
    constexpr int kElements = 4 / sizeof(T);
    Words<kWords<T, N>> w{};
    if constexpr (!Whole) {
#pragma unroll
        for (int i = 0; i < N; i++)
            if (i < valid) w.x[i / kElements] |= Bits(p[i]) << (16 * (i % kElements));
    } else if constexpr (N * sizeof(T) < 4) {
        if (valid > 0) w.x[0] = Bits(*p);
    } else {
        struct __attribute__((packed, aligned(Aligned * sizeof(T)))) InMemory {
            Words<kWords<T, N>> w;
        };
        if (valid > 0) w = reinterpret_cast<const InMemory *>(p)->w;
    }
    return w;
}
template <class T, int N>
__device__ __forceinline__ Words<kWords<T, N>> WordsOf(const float (&x)[N]) {
    Pack<T, N> p;
#pragma unroll
    for (int i = 0; i < N; i++) p.x[i] = As<T>(x[i]);
    if constexpr (N * sizeof(T) < 4) return {{Bits(p.x[0])}};
    else return __builtin_bit_cast(Words<kWords<T, N>>, p);
}
template <class T, int N>
__device__ __forceinline__ Pack<T, N> PackOf(const Words<kWords<T, N>> &w) {
    if constexpr (N * sizeof(T) < 4) return __builtin_bit_cast(Pack<T, N>, (uint16_t)w.x[0]);
    else return __builtin_bit_cast(Pack<T, N>, w);
}
// The same at `base`, which all lanes share, and a lane's `place` in bytes. The place is made anew where it is used: an
// address of a scalar and one register is only found within a block of the program.
template <class T, int N, bool Whole>
__device__ __forceinline__ Words<kWords<T, N>> WordsAt(const T *base, int place, int valid) {
    if constexpr (!Whole) {
        return LoadWords<T, N, false>(Lane(base, place), valid);
    } else {
        Words<kWords<T, N>> w{};
        if (valid > 0) w = LoadWords<T, N, true>(Lane(base, Renewed(place)));
        return w;
    }
}
template <int N, bool Whole, class T>
__device__ __forceinline__ Pack<T, N> LoadAt(const T *base, int place, int valid) {
    if constexpr (!Whole) {
        return Load<N, false>(Lane(base, place), valid);
    } else {
        Pack<T, N> x{};
        if (valid > 0) x = Load<N, true>(Lane(base, Renewed(place)), N);
        return x;
    }
}
template <int N, bool Whole, class T>
__device__ __forceinline__ void StoreAt(T *base, int place, const Pack<T, N> &x, int valid) {
    if constexpr (!Whole) Store<N, false>(Lane(base, place), x, valid);
    else if (valid > 0) Store<N, true>(Lane(base, Renewed(place)), x, N);
}
// The words are made here, and not where they are used first, from values that take more registers.
template <class X>
__device__ __forceinline__ void Made(X &x) {
    Words<sizeof(X) / 4> w = __builtin_bit_cast(Words<sizeof(X) / 4>, x);
#pragma unroll
    for (int i = 0; i < (int)(sizeof(X) / 4); i++) asm volatile("" : "+v"(w.x[i]));
    x = __builtin_bit_cast(X, w);
}
// Element i of such words.
template <class T, int N>
__device__ __forceinline__ float ElementOf(const Words<N> &w, int i) {
    return OfWord<T>(w.x[i * (int)sizeof(T) / 4], i);
}
// The pieces of a lane's eight neighbouring elements, and of the elements i of four places.
template <class T, int N>
__device__ __forceinline__ void PiecesOf(const Words<N> &w, B8 (&piece)[kPieces<T>]) {
    if constexpr (kPieces<T> == 1) {
        piece[0] = __builtin_bit_cast(B8, w);
    } else {
        F4 half[2];
#pragma unroll
        for (int i = 0; i < 8; i++) half[i / 4][i % 4] = ElementOf<T>(w, i);
        SplitPair<kPieces<T>>(half[0], half[1], piece);
    }
}
template <class T, int N>
__device__ __forceinline__ void PiecesOf(const Words<N> (&w)[4], int i, Four (&piece)[kPieces<T>]) {
    if constexpr (kPieces<T> == 1) {
#pragma unroll
        for (int j = 0; j < 2; j++)
            piece[0].x[j] = __builtin_amdgcn_perm(w[2 * j + 1].x[i / 2], w[2 * j].x[i / 2], i % 2 ? 0x07060302 : 0x05040100);
    } else {
        const float f[4] = {ElementOf<T>(w[0], i), ElementOf<T>(w[1], i), ElementOf<T>(w[2], i), ElementOf<T>(w[3], i)};
        Split<kPieces<T>>(f, piece);
    }
}

// One wavefront takes 16 * Tiles columns of a head's memory through a span, 32 steps at a time, with the memory in
// registers. The columns never mix, so the wavefronts of a head share nothing.
//
// What bounds it: memory where heads are many and products few: 16,384 heads of 64 x 64 and 64 steps in bfloat16, forward,
// move 1.07 GB in 256 us, 4.2 TB/s (a copy reaches 4.8), and the three runs of their gradients 1.75 GB in 590, 3.0 TB/s.
// There the vector instructions between the products show: two wavefronts a SIMD are all that the registers hold. Few long
// sequences wait for the chain of chunks: 3,000 steps of 44 heads of 128 x 128 take 38 us for the spans' own memories, 21 to
// join them and 86 for the outputs.
//
// With the steps i, j of a chunk, G_i the product of the factors up to i and D_ij of those from j + 1 to i (0 across an
// episode's start), O = out (G Q S + in (D o Q K^T) V), and the memory becomes G_C S + K^T (in D_C V). The products
// are sums of products of bfloat16 pieces (common.h), 32 indices an instruction. Memories and scores have all three pieces
// whatever the type: with two of them, cut off, a term would lose up to 2^-15 of itself, always towards zero, and terms that cancel
// would leave that of themselves.
//
// A lane holds eight neighbouring rows of a pair of tiles: rows 32 p + 8 g + 4 x + r of the tiles 2 p + x, so that its
// keys are 16 bytes of memory. Which rows a tile has is free as long as queries, keys and memory agree.
//
// The products over a chunk's steps take a NaN or an infinity of a key or value, times a zero, to all of them. A wavefront
// that meets one, or a factor past e^2, begins its span again and plays it step by step.
template <class T, int KeyTiles, int Tiles, Shape shape, Mode mode>
__global__ __launch_bounds__(64) __attribute__((amdgpu_waves_per_eu(kRunWaves<T, KeyTiles, mode>))) void RunKernel(Runs a) {
    constexpr int P = kPieces<T>, kPairs = KeyTiles / 2;
    constexpr bool Whole = shape != kLoose, full = shape == kFull;
    // By step: the factors' sum up to it in two floats, and the factors of what it reads (NaN behind a reset) and writes.
    __shared__ __align__(16) float reach[2][kSteps], wholes[kSteps], afters[kSteps], diagonal[kSteps];
    const int lane = threadIdx.x, m = lane & 15, g = lane >> 4;
    unsigned head = Place(blockIdx.x, gridDim.x);
    int slice = head % a.units, which = 0;
    head /= a.units;
    const int span = a.firstSpan + head % a.spanCount;
    head = a.firstHead + head / a.spanCount;
    while (slice >= a.slices[which]) slice -= a.slices[which++];
    const int h = head % a.heads, b = head / a.heads;
    const int begin = span * a.length, count = min(a.length, a.time - begin);
    const bool reverse = RunAt(which).reverse;
    const int sign = reverse ? -1 : 1, late = reverse ? 1 : 0, opens = reverse ? begin + count - 1 : begin;
    const int column = slice * 16 * Tiles + m * Tiles;
    const int ownColumns = full ? Tiles : max(0, min(Tiles, RunAt(which).columns - column));
    const auto ownRows = [&] { return full ? 16 * KeyTiles : RunAt(which).rows; };

    F4 s[KeyTiles][Tiles];
    // take(element of the run's memory, element of another) in its place.
    const auto read = [&](const float *memory, auto take) {
        const int rows = ownRows(), columns = RunAt(which).columns;
        const bool transposed = RunAt(which).transposed;
        const int lanes = (transposed ? column * rows + 8 * g : 8 * g * columns + column) * 4;
#pragma unroll
        for (int t = 0; t < KeyTiles; t++) {
            const int row = 32 * (t >> 1) + 4 * (t & 1);
            if (transposed) {
#pragma unroll
                for (int c = 0; c < Tiles; c++) {
                    const auto x = LoadAt<4, Whole>(memory + c * rows + row, lanes, c < ownColumns ? rows - row - 8 * g : 0);
#pragma unroll
                    for (int r = 0; r < 4; r++) s[t][c][r] = take(s[t][c][r], x.x[r]);
                }
            } else {
#pragma unroll
                for (int r = 0; r < 4; r++) {
                    const auto x = LoadAt<Tiles, Whole>(memory + (row + r) * columns, lanes, row + r + 8 * g < rows ? ownColumns : 0);
#pragma unroll
                    for (int c = 0; c < Tiles; c++) s[t][c][r] = take(s[t][c][r], x.x[c]);
                }
            }
        }
    };
    const auto write = [&](float *memory) {
        const int rows = ownRows(), columns = RunAt(which).columns, mine = full ? Tiles : Renewed(ownColumns);
        const int lanes = (8 * g * columns + Renewed(column)) * 4;
#pragma unroll
        for (int t = 0; t < KeyTiles; t++)
#pragma unroll
            for (int r = 0; r < 4; r++) {
                const int row = 32 * (t >> 1) + 4 * (t & 1) + r;
                Pack<float, Tiles> x;
#pragma unroll
                for (int c = 0; c < Tiles; c++) x.x[c] = s[t][c][r];
                StoreAt<Tiles, Whole>(memory + row * columns, lanes, x, row + 8 * g < rows ? mine : 0);
            }
    };
    // Places of memories of a head, and of spans, in floats.
    const auto memoryAt = [&](long long index) {
        const Run run = RunAt(which);
        return index * run.rows * run.columns;
    };
    const auto between = [&](int index) { return memoryAt((long long)head * (Argument<Runs>().spans - 1) + index); };
    const auto begins = [&] {
#pragma unroll
        for (int t = 0; t < KeyTiles; t++)
#pragma unroll
            for (int c = 0; c < Tiles; c++) s[t][c] = F4{0, 0, 0, 0};
        if constexpr (mode != kMemory) {
            const Run run = RunAt(which);
            const bool starts = reverse ? span == Argument<Runs>().spans - 1 : span == 0;
            if (const float *memory = starts ? run.first : run.starts)
                read(memory + (starts ? memoryAt(head) : between(reverse ? span : span - 1)), [](float, float y) { return y; });
        }
    };
    const bool keeps = mode == kOutputs && RunAt(which).kept;
    const auto keep = [&](int i) {
        if (keeps && i > 0 && i % kSpan == 0)
            write(RunAt(which).kept + memoryAt((long long)head * ((Argument<Runs>().time - 1) / kSpan) + i / kSpan - 1));
    };

    // A tensor's line of this head, from the span's first step on. What the memory is scaled by on the way to a step is,
    // backwards in time, the factor of the step that comes after it in time, and nothing for the first.
    const auto lineOf = [&](const Tensor &x, auto type) {
        using Element = decltype(type);
        return Line<Element>{Global(static_cast<const Element *>(x.p)) + b * x.strides[0] + opens * x.strides[1] + h / x.share * x.strides[2],
                             sign * x.strides[1]};
    };
    const auto decayLine = [&] {
        const Runs a = Argument<Runs>();
        return Line<float>{Global(a.decay) + b * a.decayStrides[0] + (opens + late) * a.decayStrides[1] + h * a.decayStrides[2],
                           sign * a.decayStrides[1]};
    };
    const auto resetLine = [&] {
        const Runs a = Argument<Runs>();
        return Line<unsigned char>{a.resets ? Global(a.resets) + b * a.resetStrides[0] + (opens + late) * a.resetStrides[1] : nullptr,
                                   sign * a.resetStrides[1]};
    };
    const auto outputLine = [&] {
        const Run run = RunAt(which);
        const int bytes = run.floats ? 4 : (int)sizeof(T);
        const long long first = b * run.outputStrides[0] + opens * run.outputStrides[1] + h * run.outputStrides[2];
        return Line<char>{static_cast<const char *>(run.output) + first * bytes, sign * run.outputStrides[1] * bytes};
    };
    const auto dotsAt = [&] {
        const Runs a = Argument<Runs>();
        return RunAt(which).dots + ((long long)slice * a.allHeads + head) * a.time + opens;
    };
    const auto gateAt = [&](int i) {
        Step step{*decayLine().At(i), 0};
        const auto resets = resetLine();
        if (resets.p) step.reset = *resets.At(i);
        return step;
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
    const bool floats = mode != kMemory && RunAt(which).floats, weighs = mode == kGradient && RunAt(which).weight.p;
    // Stores the outputs of a step at a lane's `place` in bytes, as floats or as elements.
    const auto putFloats = [&](const char *base, int place, const float (&x)[Tiles], int valid) {
        Pack<float, Tiles> o;
#pragma unroll
        for (int c = 0; c < Tiles; c++) o.x[c] = x[c];
        StoreAt<Tiles, Whole>(reinterpret_cast<float *>(const_cast<char *>(base)), place + 4 * column, o, valid);
    };
    const auto put = [&](const char *base, int place, const Words<kWords<T, Tiles>> &x, int valid) {
        StoreAt<Tiles, Whole>(reinterpret_cast<T *>(const_cast<char *>(base)), place + (int)sizeof(T) * column, PackOf<T, Tiles>(x), valid);
    };

    // All steps, one after the other.
    const auto playSteps = [&] {
        const Run run = RunAt(which);
        const int rows = ownRows(), mine = ownColumns;
        const Line<T> keys = lineOf(run.key, T()), values = lineOf(run.value, T());
        const Line<T> queries = mode != kMemory ? lineOf(run.query, T()) : Line<T>{}, weights = weighs ? lineOf(run.weight, T()) : Line<T>{};
        const Line<char> outputs = outputLine();
        float *dots = dotsAt();
#pragma unroll 1
        for (int i = 0; i < count; i++) {
            keep(i);
            const auto v = Load<Tiles, Whole>(values.At(i) + column, mine);
            if (i >= late) scale(gateAt(i));
            const T *key = keys.At(i), *query = mode == kMemory ? nullptr : queries.At(i);
            float strict[Tiles] = {}, own = 0;
#pragma unroll
            for (int x = 0; x < KeyTiles; x++) {
                const int row = 32 * (x >> 1) + 8 * g + 4 * (x & 1);
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
                if (weighs) w = Load<Tiles, Whole>(weights.At(i) + column, mine);
                float dot = 0;
#pragma unroll
                for (int c = 0; c < Tiles; c++) {
                    strict[c] += __shfl_xor(strict[c], 16);
                    strict[c] += __shfl_xor(strict[c], 32);
                    strict[c] *= run.out;
                    if (c < mine) dot = fmaf(strict[c], Float(w.x[c]), dot);
                    strict[c] = fmaf(run.out * run.in * own, Float(v.x[c]), strict[c]);
                }
                if (floats) putFloats(outputs.At(i), 0, strict, g == 0 ? mine : 0);
                else put(outputs.At(i), 0, WordsOf<T>(strict), g == 0 ? mine : 0);
                dot = RowSum(dot);
                if (weighs && lane == 0) dots[sign * i] = dot;
            }
        }
    };

    // The inputs of the next 32 steps: of a lane's steps m and 16 + m the keys and queries, of its steps 4 g + r and
    // 16 + 4 g + r the values and weights. Past the end the last step is read again. An address is one that all lanes
    // share, that of the chunk's first step in time, and a lane's offset of 32 bits.
    using RowWords = Words<kWords<T, 8>>;
    using ColumnWords = Words<kWords<T, Tiles>>;
    RowWords nextK[2][kPairs], nextQ[2][kPairs];
    ColumnWords nextV[2][4];
    Step nextGate[2];
    const auto nearOf = [&](const auto &line) {
        Near<std::remove_const_t<std::remove_pointer_t<decltype(line.p)>>> near{line.p, sign * (int)line.step};
        if (reverse && near.p) near.p -= (kSteps - 1) * near.step;
        return near;
    };
    const auto advance = [&](auto &near) { near.p += sign * kSteps * near.step; };
    Near<T> keys{}, queries{}, values{}, weights{};
    Near<float> decays{};
    Near<unsigned char> resets{};
    Near<char> outputs{};
    const float *dots = nullptr;
    const auto placeOf = [&](int i) { return reverse ? kSteps - 1 - i : i; };
    const auto rowsAt = [&](const Near<T> &line, int left, RowWords(&x)[2][kPairs]) {
#pragma unroll
        for (int n = 0; n < 2; n++) {
            const int place = (placeOf(min(16 * n + Renewed(m), left - 1)) * line.step + 8 * g) * (int)sizeof(T);
            if constexpr (full) {
                const uint32_t lanes = Renewed(place);
#pragma unroll
                for (int q = 0; q < kPairs; q++) x[n][q] = LoadWords<T, 8, true, 4>(Lane(line.p + 32 * q, lanes));
            } else {
                const int rest = ownRows() - 8 * g;
#pragma unroll
                for (int q = 0; q < kPairs; q++) {
                    struct Halves {
                        Words<kWords<T, 4>> x[2];
                    } half;
#pragma unroll
                    for (int i = 0; i < 2; i++) half.x[i] = WordsAt<T, 4, Whole>(line.p + 32 * q + 4 * i, place, rest - 32 * q - 4 * i);
                    x[n][q] = __builtin_bit_cast(RowWords, half);
                }
            }
        }
    };
    const auto columnsAt = [&](const Near<T> &line, int left, ColumnWords(&x)[2][4]) {
        if (full && left >= kSteps) {
            const uint32_t lanes = Renewed(((reverse ? 12 - 4 * g : 4 * g) * line.step + Renewed(column)) * (int)sizeof(T));
#pragma unroll
            for (int n = 0; n < 2; n++)
#pragma unroll
                for (int r = 0; r < 4; r++) x[n][r] = LoadWords<T, Tiles, true>(Lane(line.At(reverse ? 19 - 16 * n - r : 16 * n + r), lanes));
        } else {
            const int mine = full ? Tiles : Renewed(ownColumns);
#pragma unroll
            for (int n = 0; n < 2; n++)
#pragma unroll
                for (int r = 0; r < 4; r++)
                    x[n][r] = WordsAt<T, Tiles, Whole>(line.p, (placeOf(min(16 * n + 4 * g + r, left - 1)) * line.step + Renewed(column)) * (int)sizeof(T), mine);
        }
    };
    // Where nothing is left nothing is fetched, and what was fetched before is given up: its registers are free until then.
    const auto fetchRows = [&](int left) {
        if (left <= 0) {
#pragma unroll
            for (int n = 0; n < 2; n++)
#pragma unroll
                for (int q = 0; q < kPairs; q++) nextK[n][q] = nextQ[n][q] = RowWords{};
            return;
        }
        rowsAt(keys, left, nextK), advance(keys);
        if constexpr (mode != kMemory) rowsAt(queries, left, nextQ), advance(queries);
    };
    const auto fetchColumns = [&](int first) {
        if (first >= count) {
#pragma unroll
            for (int n = 0; n < 2; n++) {
                nextGate[n] = Step{};
#pragma unroll
                for (int r = 0; r < 4; r++) nextV[n][r] = ColumnWords{};
            }
            return;
        }
        columnsAt(values, count - first, nextV), advance(values);
#pragma unroll
        for (int n = 0; n < 2; n++) {
            const int i = 16 * n + Renewed(m);
            nextGate[n] = Step{0.f, 0};
            if (first + i < count && first + i >= late) {
                nextGate[n].decay = *Lane(decays.p, Renewed(placeOf(i) * decays.step * 4));
                if (resets.p) nextGate[n].reset = *Lane(resets.p, Renewed(placeOf(i) * resets.step));
            }
        }
        advance(decays);
        if (resets.p) advance(resets);
    };

    // The identity as a right operand of four values a lane.
    Four eye;
#pragma unroll
    for (int j = 0; j < 2; j++) eye.x[j] = (4 * g + 2 * j == m ? 0x3f80u : 0u) | (4 * g + 2 * j + 1 == m ? 0x3f800000u : 0u);
    // Steps that are too far apart for 32 bits are played one by one.
    bool finite = Argument<Runs>().near;
    begins();
    if (finite) {
        const Run run = RunAt(which);
        keys = nearOf(lineOf(run.key, T())), values = nearOf(lineOf(run.value, T()));
        decays = nearOf(decayLine()), resets = nearOf(resetLine());
        if constexpr (mode != kMemory) queries = nearOf(lineOf(run.query, T())), outputs = nearOf(outputLine());
        if (weighs) weights = nearOf(lineOf(run.weight, T())), dots = dotsAt() - (reverse ? kSteps - 1 : 0);
        fetchRows(count), fetchColumns(0);
    }
    const float in = RunAt(which).in, out = RunAt(which).out;
#pragma unroll 1
    for (int first = 0; first < count && finite; first += kSteps) {
        const int valid = min(kSteps, count - first);
        keep(first);

        // Pieces of the keys and queries; products with the memory, the scores, and the keys' transpose.
        F4 mark = {0, 0, 0, 0}, scores[3], o[2][Tiles];  // scores: of the tiles 00, 10 and 11, in row order
        B8 turned[KeyTiles][P];
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
            for (int n = 0; n < 2; n++) PiecesOf<T>(nextK[n][p], kp[n]);
            mark = Mfma32(kp[0][0], kp[1][0], mark);
#pragma unroll
            for (int x = 0; x < 2; x++) {
                Four half[2][P];
#pragma unroll
                for (int n = 0; n < 2; n++) TurnHalf<P>(kp[n], x, eye, half[n]);
                Eights(half[0], half[1], turned[2 * p + x]);
#pragma unroll
                for (int i = 0; i < P; i++) Made(turned[2 * p + x][i]);
            }
            if constexpr (mode != kMemory) {
#pragma unroll
                for (int n = 0; n < 2; n++) PiecesOf<T>(nextQ[n][p], qp[n]);
                scores[0] = Mfma32(kp[0], qp[0], scores[0]);
                scores[1] = Mfma32(kp[0], qp[1], scores[1]);
                scores[2] = Mfma32(kp[1], qp[1], scores[2]);
#pragma unroll
                for (int c = 0; c < Tiles; c++) {
                    B8 sp[kFloatPieces];
                    SplitPair<kFloatPieces>(s[2 * p][c], s[2 * p + 1][c], sp);
#pragma unroll
                    for (int n = 0; n < 2; n++) o[n][c] = Mfma32(qp[n], sp, o[n][c]);
                }
            }
            __builtin_amdgcn_sched_barrier(0);
        }
        ColumnWords v[2][4], w[2][4];
#pragma unroll
        for (int n = 0; n < 2; n++)
#pragma unroll
            for (int r = 0; r < 4; r++) v[n][r] = nextV[n][r], w[n][r] = ColumnWords{};
        if (valid < kSteps)
#pragma unroll
            for (int n = 0; n < 2; n++)
#pragma unroll
                for (int r = 0; r < 4; r++) v[n][r] = 16 * n + 4 * g + r < valid ? v[n][r] : ColumnWords{};
        const Step gate[2] = {nextGate[0], nextGate[1]};
        if (weighs) columnsAt(weights, valid, w), advance(weights);
        // Products of keys, and of values, tell whether one is not finite.
#pragma unroll
        for (int c = 0; c < Tiles; c++) {
            Four half[2][P];
#pragma unroll
            for (int n = 0; n < 2; n++) PiecesOf<T>(v[n], c, half[n]);
            const B8 both = Eight(half[0][0], half[1][0]);
            mark = Mfma32(both, both, mark);
        }
        if (__ballot(((mark[0] + mark[1]) + (mark[2] + mark[3])) * 0.f != 0.f || gate[0].Steep() || gate[1].Steep())) {
            finite = false;
            break;
        }

        __builtin_amdgcn_sched_barrier(0);
        // How the chunk is cut, and the products of its factors.
        const bool cleared[2] = {gate[0].Cleared(), gate[1].Cleared()};
        const unsigned cuts = (unsigned)(__ballot(cleared[0]) & 0xffff) | (unsigned)(__ballot(cleared[1]) & 0xffff) << 16;
        float high[2], low[2], kept;
        int start[2];  // where the episode of a lane's steps starts, or -1 before the chunk
        {
            double G[2];
            G[0] = RowUpTo(cleared[0] ? 0.0 : gate[0].decay * kLog2E);
            G[1] = RowUpTo(cleared[1] ? 0.0 : gate[1].decay * kLog2E) + __shfl(G[0], 15);
            const double last = __shfl(G[1], 15);
            const int latest = cuts ? 31 - __builtin_clz(cuts) : -1;
            kept = Exp2(last);
            __syncthreads();
#pragma unroll
            for (int n = 0; n < 2; n++) {
                const int i = 16 * n + m;
                const unsigned upTo = cuts & ((2u << i) - 1);
                start[n] = upTo ? 31 - __builtin_clz(upTo) : -1;
                high[n] = (float)G[n], low[n] = (float)(G[n] - high[n]);
                if (g == 0) {
                    reach[0][i] = high[n], reach[1][i] = low[n];
                    wholes[i] = start[n] < 0 ? out * Exp2(G[n]) : __builtin_nanf("");
                    afters[i] = i >= latest ? in * Exp2(last - G[n]) : 0.f;
                }
            }
            __syncthreads();
        }

        ColumnWords done[2][4];
        if constexpr (mode != kMemory) {
            const float factor = in * out;
#pragma unroll
            for (int n = 0; n < 2; n++) {
                // The scores of the tile's steps with those of each tile up to it; for dots without a step's own.
                Four lower[2][kFloatPieces];
#pragma unroll
                for (int x = 0; x <= n; x++) {
                    const F4 high4 = *reinterpret_cast<const F4 *>(reach[0] + 16 * x + 4 * g);
                    const F4 low4 = *reinterpret_cast<const F4 *>(reach[1] + 16 * x + 4 * g);
                    float mixed[4];
#pragma unroll
                    for (int r = 0; r < 4; r++) {
                        const int i = 16 * n + m, j = 16 * x + 4 * g + r;
                        const float score = factor * scores[n + x][r];
                        if (mode == kGradient && x == n && i == j) diagonal[i] = score;
                        const float d = __builtin_amdgcn_exp2f((high[n] - high4[r]) + (low[n] - low4[r])) * score;
                        mixed[r] = x < n || (mode == kGradient ? j < i : j <= i) ? d : 0.f;
                    }
                    if (cuts)
#pragma unroll
                        for (int r = 0; r < 4; r++) mixed[r] = 16 * x + 4 * g + r >= start[n] ? mixed[r] : 0.f;
                    Split<kFloatPieces>(mixed, lower[x]);
                }
                B8 both[kFloatPieces];
                if (n == 1) Eights(lower[0], lower[1], both);
                __builtin_amdgcn_sched_barrier(0);
                const F4 whole = *reinterpret_cast<const F4 *>(wholes + 16 * n + 4 * g);
#pragma unroll
                for (int c = 0; c < Tiles; c++)
#pragma unroll
                    for (int r = 0; r < 4; r++) o[n][c][r] *= whole[r];
                if (cuts)
#pragma unroll
                    for (int c = 0; c < Tiles; c++)
#pragma unroll
                        for (int r = 0; r < 4; r++) o[n][c][r] = whole[r] != whole[r] ? 0.f : o[n][c][r];
#pragma unroll
                for (int c = 0; c < Tiles; c++) {
                    Four half[2][P];
                    PiecesOf<T>(v[0], c, half[0]);
                    if (n == 0) {
                        o[n][c] = Mfma16(lower[0], half[0], o[n][c]);
                    } else {
                        B8 both2[P];
                        PiecesOf<T>(v[1], c, half[1]);
                        Eights(half[0], half[1], both2);
                        o[n][c] = Mfma32(both, both2, o[n][c]);
                    }
                }
                F4 own = {0, 0, 0, 0};
                if constexpr (mode == kGradient) {
                    __syncthreads();
                    own = *reinterpret_cast<const F4 *>(diagonal + 16 * n + 4 * g);
                }
                const int mine = full ? Tiles : Renewed(ownColumns), place = (reverse ? 12 - 4 * g : 4 * g);
#pragma unroll
                for (int r = 0; r < 4; r++) {
                    const bool real = valid == kSteps || 16 * n + 4 * g + r < valid;
                    const int later = reverse ? 19 - 16 * n - r : 16 * n + r;
                    float x[Tiles], dot = 0;
#pragma unroll
                    for (int c = 0; c < Tiles; c++) {
                        x[c] = o[n][c][r];
                        if constexpr (mode == kGradient) {
                            if (full || c < mine) dot = fmaf(x[c], ElementOf<T>(w[n][r], c), dot);
                            x[c] = fmaf(own[r], ElementOf<T>(v[n][r], c), x[c]);
                        }
                    }
                    done[n][r] = WordsOf<T>(x);
                    Made(done[n][r]);
                    if (floats) putFloats(outputs.At(later), place * outputs.step, x, real ? mine : 0);
                    if (weighs) {
                        dot = RowSum(dot);
                        if (m == 0 && real) *Lane(const_cast<float *>(dots) + later, Renewed(place * 4)) = dot;
                    }
                }
                __builtin_amdgcn_sched_barrier(0);
            }
            if (weighs) dots += sign * kSteps;
        }

        fetchRows(count - first - kSteps);
        if (cuts)
#pragma unroll
            for (int t = 0; t < KeyTiles; t++)
#pragma unroll
                for (int c = 0; c < Tiles; c++) s[t][c] = F4{0, 0, 0, 0};
        F4 after[2];
#pragma unroll
        for (int n = 0; n < 2; n++) after[n] = *reinterpret_cast<const F4 *>(afters + 16 * n + 4 * g);
#pragma unroll
        for (int c = 0; c < Tiles; c++) {
            F4 x[2];
#pragma unroll
            for (int n = 0; n < 2; n++)
#pragma unroll
                for (int r = 0; r < 4; r++) x[n][r] = after[n][r] * ElementOf<T>(v[n][r], c);
            B8 written[kFloatPieces];
            SplitPair<kFloatPieces>(x[0], x[1], written);
#pragma unroll
            for (int t = 0; t < KeyTiles; t++) s[t][c] = Mfma32(turned[t], written, s[t][c] * kept);
        }
        fetchColumns(first + kSteps);
        // Outputs leave behind the next steps' loads: the wait for loads, which are answered in the order in which loads and
        // stores were sent, does not wait for them.
        if constexpr (mode != kMemory) {
            __builtin_amdgcn_sched_barrier(0);
            if (!floats) {
                const int mine = full ? Tiles : Renewed(ownColumns), place = (reverse ? 12 - 4 * g : 4 * g) * outputs.step;
#pragma unroll
                for (int n = 0; n < 2; n++)
#pragma unroll
                    for (int r = 0; r < 4; r++)
                        put(outputs.At(reverse ? 19 - 16 * n - r : 16 * n + r), place, done[n][r],
                            valid == kSteps || 16 * n + 4 * g + r < valid ? mine : 0);
            }
            advance(outputs);
            __builtin_amdgcn_sched_barrier(0);
        }
    }
    if (!finite) {
        begins();
        playSteps();
    }

    const Runs all = Argument<Runs>();
    const Run run = RunAt(which);
    if constexpr (mode == kMemory) {
        if (reverse && count > 0) scale(gateAt(count));
        const int place = reverse ? span - 1 : span;
        write(run.last + between(place));
        if (slice == 0) {
            // The span's factors.
            double sum = 0;
            bool cleared = false;
            for (int i = lane; i < count; i += 64) {
                const Step gate = gateAt(i + late);
                cleared |= gate.Cleared();
                sum += gate.decay;
            }
            for (int d = 32; d; d /= 2) sum += __shfl_xor(sum, d);
            // In 64 bits: 128 factors may leave the range of 32 where a memory times them does not. Those that leave 64 leave 32
            // with the least memory, but not with one of zero.
            const double factor = __ballot(cleared) ? -1. : exp(sum > 700. && sum < __builtin_inf() ? 700. : sum);
            if (lane == 0) all.factors[(long long)head * (all.spans - 1) + place] = factor;
        }
    } else {
        if constexpr (mode == kGradient)
            if (run.crossings) {
                const bool ends = span == all.spans - 1;
                float sum = 0;
                if (const float *memory = ends ? run.againstLast : run.against)
                    read(memory + (ends ? memoryAt(head) : between(span)), [&](float x, float y) { return sum = fmaf(x, y, sum), x; });
                sum = WaveSum(sum);
                if (lane == 0) run.crossings[((long long)slice * all.allHeads + head) * all.spans + span] = sum;
            }
        if (run.last && span == (reverse ? 0 : all.spans - 1)) {
            if (reverse && count > 0) scale(gateAt(count));
            write(run.last + memoryAt(head));
        }
    }
}

// Whether a tensor's packs of four are aligned and none is cut.
inline bool IsWhole(const void *p, const long long *strides, int size, size_t bytes) {
    return strides[0] % 4 == 0 && strides[1] % 4 == 0 && strides[2] % 4 == 0 && size % 4 == 0 && Aligned(4 * bytes, p);
}
inline Tensor TensorOf(const void *p, const long long *strides, int share) { return {p, {strides[0], strides[1], strides[2]}, share}; }
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

// The most tiles of 16 columns whose memory fits a wavefront's registers beside the rest: the keys of a chunk are turned once
// for all of them. With half of them 4,096 heads and 64 steps of bfloat16 64 x 64 take 68 us for 56, gradients 186 for 137;
// 128 x 128 310 for 232, 719 for 543; float16 96 x 96 223 for 165, 590 for 429. Float32 64 x 64 with two 169 for 141.
template <class T, int KeyTiles>
constexpr int kMostTiles = KeyTiles * kPieces<T> <= 4 ? 4 : KeyTiles * kPieces<T> <= (kPieces<T> == kFloatPieces ? 8 : 12) ? 2 : 1;
// The tiles that a wavefront of a launch takes: as many as leave a wavefront for each of the chip's 1,024 SIMDs. (bfloat16
// 64 x 64, 64 steps, forward, with one tile and with four: 256 heads 11.1 and 12.6 us, 2,048 heads 38 and 24.)
template <class T>
int TilesOf(const Runs &runs, int count, int keyTiles) {
    const int most = keyTiles == 2 ? kMostTiles<T, 2> : keyTiles == 4 ? kMostTiles<T, 4> : keyTiles == 6 ? kMostTiles<T, 6> : kMostTiles<T, 8>;
    for (int tiles = most; tiles > 1; tiles /= 2) {
        long long slices = 0;
        bool full = true;
        for (int i = 0; i < count; i++) {
            slices += runs.run[i].columns / (16 * tiles);
            full &= runs.run[i].rows == 16 * keyTiles && runs.run[i].columns % (16 * tiles) == 0;
        }
        if (full && runs.allHeads * slices * runs.spanCount >= 1024) return tiles;
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
        runs.slices[i] = (runs.run[i].columns + 16 * tiles - 1) / (16 * tiles);
        runs.units += runs.slices[i];
    }
}

inline bool IsNear(const Runs &runs, int count, size_t bytes) {
    const auto near = [](long long stride, size_t bytes) { return stride >= 0 && stride < (1 << 26) / (long long)bytes; };
    if (!near(runs.decayStrides[1], sizeof(float)) || !near(runs.resetStrides[1], 1)) return false;
    for (int i = 0; i < count; i++) {
        const Run &r = runs.run[i];
        if (!near(r.query.strides[1], bytes) || !near(r.key.strides[1], bytes) || !near(r.value.strides[1], bytes) ||
            !near(r.weight.strides[1], bytes) || !near(r.outputStrides[1], r.floats ? sizeof(float) : bytes))
            return false;
    }
    return true;
}

template <class T, Mode mode, int KeyTiles>
void LaunchTiles(Runs &runs, int count, bool whole, hipStream_t stream) {
    runs.near = IsNear(runs, count, sizeof(T));
    constexpr int most = kMostTiles<T, KeyTiles>;
    const int tiles = whole ? TilesOf<T>(runs, count, KeyTiles) : 1;
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
    bool full = whole;
    for (int i = 0; i < count; i++) full &= runs.run[i].rows == 16 * KeyTiles && runs.run[i].columns % (16 * tiles) == 0;
    if (!whole) launch(RunKernel<T, KeyTiles, 1, kLoose, mode>);
    else if (!full) launch(RunKernel<T, KeyTiles, 1, kWhole, mode>);
    else if (tiles == 4) launch(RunKernel<T, KeyTiles, most >= 4 ? 4 : 1, kFull, mode>);
    else if (tiles == 2) launch(RunKernel<T, KeyTiles, most >= 2 ? 2 : 1, kFull, mode>);
    else launch(RunKernel<T, KeyTiles, 1, kFull, mode>);
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
