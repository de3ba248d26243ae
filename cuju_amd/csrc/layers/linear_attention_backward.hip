// The gradients of linear attention over many steps (linear_attention.h).
#include "linear_attention.h"

namespace layers {
namespace {

// A step whose log decay is below this passes on so little that differences of the dots around it would not hold its gradient.
// Beside steps that forget nothing, in 64 x 64, the gradient at a decay of -0.5 is 3e-6 of its terms' 2-norm off, of -2 9e-6, of
// -3.99 5e-5; what SharpKernel finds is 7e-7 off at any.
constexpr float kSharp = -4.f;
// One wavefront takes a span of a head: two steps a lane. Backwards from the product of the memory at the span's end
// and its gradient, each step adds q.dq - k.dk without its own product to the gradient of the step after it,
// unless an episode starts there. It reads two dots a slice, head and step, and no more: 20 us for 16,384 heads of 64 steps.
// Spans with sharp steps are left to the next kernel.
struct DecayArgs {
    const float *queryDots, *keyDots, *crossings;  // [slices][head][time], and [slices][head][span]
    int querySlices, keySlices, time, heads, spans;
    unsigned allHeads;
    const float *decay;
    const unsigned char *resets;
    long long decayStrides[3], resetStrides[2];
    float *out;            // [batch][time][head], or null
    double *totals;        // [head][span]
    unsigned char *sharp;  // [head][span]: whether a span has a sharp step
    bool empty;            // whether the first step starts with nothing
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
        bool starts[3], steep = false;
#pragma unroll
        for (int i = 0; i < 3; i++) {
            const int t = begin + 2 * lane + i;
            starts[i] = false;
            // What the first step of the next span starts with is in that span's memory already.
            if (t < end) {
                const float decay = a.decay[b * a.decayStrides[0] + t * a.decayStrides[1] + h * a.decayStrides[2]];
                starts[i] = decay < kNothingKept || (a.empty && t == 0);
                if (a.resets) starts[i] |= a.resets[b * a.resetStrides[0] + t * a.resetStrides[1]] != 0;
                steep |= !starts[i] && decay < kSharp;
            }
            if (i == 2) break;
            step[i] = 0;
            if (t >= end) continue;
            for (int n = 0; n < a.querySlices; n++) step[i] += a.queryDots[((long long)n * a.allHeads + head) * a.time + t];
            for (int n = 0; n < a.keySlices; n++) step[i] -= a.keyDots[((long long)n * a.allHeads + head) * a.time + t];
        }
        const bool sharp = __ballot(steep);
        if (lane == 0) a.sharp[item] = sharp;
        if (sharp) continue;
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

// x 2^power, and zero where x is, whatever the power.
__device__ __forceinline__ float Scaled(float x, double power) {
    const float whole = rintf((float)power);
    return ldexpf(x * __builtin_amdgcn_exp2f((float)(power - whole)), (int)fminf(fmaxf(whole, -4096.f), 4096.f));
}
__device__ __forceinline__ double BlockSum(double x, double (&sums)[4]) {
    for (int d = 32; d; d /= 2) x += __shfl_xor(x, d);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) sums[threadIdx.x >> 6] = x;
    __syncthreads();
    return (sums[0] + sums[1]) + (sums[2] + sums[3]);
}
// A lane's eight elements of each pair of tiles of a step's row, zeros past its end; 16 bytes at once, for the lines of the cache
// that a load touches (by eight bytes the kernel below takes 675 us for 518).
template <class T, int kPairs, bool Whole>
struct Row {
    Words<kWords<T, 8>> pair[kPairs];
    __device__ __forceinline__ void Load(const T *row, int g, int size) {
#pragma unroll
        for (int p = 0; p < kPairs; p++) {
            const int at = 32 * p + 8 * g;
            if (Whole && sizeof(T) == 2 && at + 8 <= size) {
                pair[p] = LoadWords<T, 8, true, 4>(row + at);
            } else {
                struct Halves {
                    Words<kWords<T, 4>> x[2];
                } half;
#pragma unroll
                for (int i = 0; i < 2; i++) half.x[i] = LoadWords<T, 4, Whole>(row + at + 4 * i, size - at - 4 * i);
                pair[p] = __builtin_bit_cast(Words<kWords<T, 8>>, half);
            }
        }
    }
    __device__ __forceinline__ void Pieces(int p, B8 (&piece)[kPieces<T>]) const { PiecesOf<T>(pair[p], piece); }
};

// The gradients of the decays of spans with sharp steps, as sums of what passes each step: no difference of large sums. Of an
// earlier and a later step j < t <= i of the span (i) scale (q_i.k_j) (do_i.v_j) F_ij passes step t, of the memory S before the
// span (ii) scale q_i S do_i F_i, of the gradient D of the memory behind it (iii) k_j D v_j F_j, and of both (iv) <S, D> F, where F
// are the products of the factors in between. A step that is cleared ends all of them. The products are of pieces (common.h). A tile
// of 16 x 16 pairs is summed by row and by column, for the steps within its later and its earlier steps, and whole, for
// those between. 16,384 heads of 64 x 64 and 64 steps in bfloat16, each with a sharp step, take 500 to 520 us, and 5 where none has
// one. Wavefronts wait for loads for 72 % of their cycles: a load of steps' rows touches 16 lines of the cache, one after the other.
struct SharpArgs {
    DecayArgs decays;
    Tensor query, key, value, output;  // output: its gradient
    int rows, columns;                 // of a memory
    float scale;
    const float *first, *starts, *ends, *last;  // memories before spans, and their gradients behind them; first and last or null
};
constexpr long long kSharpBlocks = 1024;  // as many as the chip holds: each takes every 1,024th span
template <class T, int kPairs>
constexpr int kSharpWaves = kPairs * kPieces<T> <= 2 ? 4 : kPairs * kPieces<T> <= 6 ? 3 : 2;
template <class T, int kPairs, bool Whole>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(kSharpWaves<T, kPairs>))) void SharpKernel(SharpArgs s) {
    constexpr int kTiles = kSpan / kChunk, P = kPieces<T>;
    __shared__ double level[kSpan];  // the sum of log decays, in base 2, but those of steps that are cleared or past any range
    __shared__ int episode[kSpan];   // how many steps were cleared up to this, and how many were past any range in the upper half
    __shared__ float rows[kTiles][kTiles][kChunk], columns[kTiles][kTiles][kChunk], diagonal[kTiles][kChunk][kChunk + 1];
    __shared__ float parts[2][kTiles][kSpan];  // (ii) and (iii), by 16 columns of the memory
    __shared__ double sums[4], tiled[2][kTiles], between[kTiles][kTiles];
    const DecayArgs &a = s.decays;
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6, m = lane & 15, g = lane >> 4, own = t / kChunk, step = t % kChunk;
    const long long items = (long long)a.allHeads * a.spans, size = (long long)s.rows * s.columns;

    const auto find = [&](long long item) {
        const int span = item % a.spans;
        const unsigned head = item / a.spans;
        const int h = head % a.heads, b = head / a.heads, begin = span * kSpan, count = min(kSpan, a.time - begin);
        const int tiles = (count + kChunk - 1) / kChunk;
        const auto lineOf = [&](const Tensor &x) {
            return Line<T>{Global(static_cast<const T *>(x.p)) + b * x.strides[0] + begin * x.strides[1] + h / x.share * x.strides[2],
                           x.strides[1]};
        };
        const long long place = (long long)head * (a.spans - 1) + span;
        const float *start = span ? s.starts + (place - 1) * size : s.first ? s.first + head * size : nullptr;
        const float *end = span < a.spans - 1 ? s.ends + place * size : s.last ? s.last + head * size : nullptr;

        // The two wavefronts of the span's steps; what the first one has seen is added to the second's.
        __syncthreads();
        double sum = 0;
        int seen = 0;
        if (wave < 2) {
            float decay = 0;
            bool cleared = false;
            if (t < count) {
                decay = a.decay[b * a.decayStrides[0] + (begin + t) * a.decayStrides[1] + h * a.decayStrides[2]];
                cleared = decay < kNothingKept || (a.resets && a.resets[b * a.resetStrides[0] + (begin + t) * a.resetStrides[1]]);
            }
            const bool far = !cleared && !(decay <= 1024.f);
            sum = RowUpTo(cleared || far ? 0. : decay * kLog2E);
            const double row = __shfl(sum, 15), second = __shfl(sum, 31), third = __shfl(sum, 47);
            sum += (g > 0 ? row : 0.) + (g > 1 ? second : 0.) + (g > 2 ? third : 0.);
            const unsigned long long upTo = ~0ull >> (63 - lane);
            seen = __popcll(__ballot(cleared) & upTo) | __popcll(__ballot(far) & upTo) << 16;
            if (t == 63) sums[0] = sum, episode[63] = seen;
        }
        __syncthreads();
        const double firstSum = sums[0];
        const int firstSeen = episode[63];
        __syncthreads();
        if (wave < 2) level[t] = sum + (wave ? firstSum : 0.), episode[t] = seen + (wave ? firstSeen : 0);
        __syncthreads();
        const int episodes = episode[count - 1] & 0xffff;
        // x times the factors behind step j, or the span's start, up to step i.
        const auto passed = [&](float x, int i, int j) {
            const bool far = (episode[i] ^ (j < 0 ? 0 : episode[j])) >> 16;
            return far ? __builtin_nanf("") : Scaled(x, level[i] - (j < 0 ? 0. : level[j]));
        };

        // (i) Pairs of steps: a wavefront takes two tiles of later steps with all earlier ones; a lane has the later steps 4 g + r
        // and the earlier step m.
        const Line<T> queries = lineOf(s.query), keys = lineOf(s.key), values = lineOf(s.value), outputs = lineOf(s.output);
        for (int late = wave; late < tiles; late = late < 4 ? 7 - late : kTiles) {
            const int i0 = min(kChunk * late + m, count - 1);
            Row<T, kPairs, Whole> query, output;
            query.Load(queries.At(i0), g, s.rows), output.Load(outputs.At(i0), g, s.columns);
            for (int early = 0; early <= late; early++) {
                const int j0 = min(kChunk * early + m, count - 1);
                // Products of a lane's later and earlier step.
                const auto product = [&](const Row<T, kPairs, Whole> &left, const Line<T> &right, int size) {
                    Row<T, kPairs, Whole> row;
                    row.Load(right.At(j0), g, size);
                    F4 found = {0, 0, 0, 0};
#pragma unroll
                    for (int p = 0; p < kPairs; p++) {
                        B8 x[P], y[P];
                        left.Pieces(p, x), row.Pieces(p, y), found = Mfma32(x, y, found);
                    }
                    __builtin_amdgcn_sched_barrier(0);
                    return found;
                };
                const F4 scores = product(query, keys, s.rows), answers = product(output, values, s.columns);
                float column = 0;
#pragma unroll
                for (int r = 0; r < 4; r++) {
                    const int i = kChunk * late + 4 * g + r, j = kChunk * early + m;
                    float pair = 0;
                    if (i < count && j < i && !((episode[i] ^ episode[j]) & 0xffff)) pair = passed(scores[r], i, j) * (answers[r] * s.scale);
                    column += pair;
                    if (late == early) diagonal[late][4 * g + r][m] = pair;
                    const float row = RowSum(pair);
                    if (m == 0) rows[late][early][4 * g + r] = row;
                }
                column += __shfl_xor(column, 16);
                column += __shfl_xor(column, 32);
                if (g == 0) columns[late][early][m] = column;
            }
        }
        // (ii) and (iii): a step's row times a memory, times its answer. A wavefront takes 16 columns of the memory. (iv): their
        // products with those of another.
        double both = 0;
        const auto pass = [&](const Line<T> &left, const float *memory, const Line<T> &right, const float *other, float (&out)[kTiles][kSpan]) {
            for (int first = wave * kChunk; first < s.columns; first += 4 * kChunk) {
                const int column = min(first + m, s.columns - 1);
                B8 held[kPairs][kFloatPieces];
#pragma unroll
                for (int p = 0; p < kPairs; p++) {
                    F4 x[2], y[2] = {{0, 0, 0, 0}, {0, 0, 0, 0}};
#pragma unroll
                    for (int r = 0; r < 8; r++) {
                        const int row = 32 * p + 8 * g + r;
                        x[r / 4][r % 4] = row < s.rows ? memory[row * s.columns + column] : 0.f;
                        if (other) y[r / 4][r % 4] = row < s.rows && first + m < s.columns ? other[row * s.columns + column] : 0.f;
                    }
                    if (other)
#pragma unroll
                        for (int r = 0; r < 8; r++)
                            if (first + m < s.columns) both += (double)x[r / 4][r % 4] * y[r / 4][r % 4];
                    SplitPair<kFloatPieces>(x[0], x[1], held[p]);
                }
                for (int tile = 0; tile < tiles; tile++) {
                    Row<T, kPairs, Whole> row;
                    row.Load(left.At(min(kChunk * tile + m, count - 1)), g, s.rows);
                    float answer[4];
#pragma unroll
                    for (int r = 0; r < 4; r++) answer[r] = Float(right.At(min(kChunk * tile + 4 * g + r, count - 1))[column]);
                    F4 products = {0, 0, 0, 0};
#pragma unroll
                    for (int p = 0; p < kPairs; p++) {
                        B8 x[P];
                        row.Pieces(p, x), products = Mfma32(x, held[p], products);
                    }
#pragma unroll
                    for (int r = 0; r < 4; r++) {
                        const float sum = RowSum(first + m < s.columns ? products[r] * answer[r] : 0.f);
                        if (m == 0) out[first / kChunk][kChunk * tile + 4 * g + r] = sum;
                    }
                }
            }
        };
        if (start) pass(queries, start, outputs, nullptr, parts[0]);
        if (end) pass(keys, end, values, episodes == 0 ? start : nullptr, parts[1]);
        both = BlockSum(both, sums);

        // Everything within the steps' own tiles, 16 threads each: what later steps read, and what earlier steps wrote.
        float later = 0, earlier = 0;
        if (t < count) {
            float found[2] = {};
            for (int x = 0; x * kChunk < s.columns; x++) found[0] += start ? parts[0][x][t] : 0.f, found[1] += end ? parts[1][x][t] : 0.f;
            if (!(episode[t] & 0xffff)) later = passed(s.scale * found[0], t, -1);
            if ((episode[t] & 0xffff) == episodes) earlier = passed(found[1], count - 1, t);
        }
        if (wave < 2) {
            const double allLater = RowSum(later), allEarlier = RowSum(earlier);
            if (step == 0) tiled[0][own] = allLater, tiled[1][own] = allEarlier;
            // The diagonal tiles' sums from each later step on, by earlier step.
            float down = 0;
            if (own < tiles)
#pragma unroll
                for (int i = kChunk - 1; i >= 0; i--) down += diagonal[own][i][step], diagonal[own][i][step] = down;
        } else if (t - 128 < kTiles * kTiles) {
            const int late = (t - 128) / kTiles, early = (t - 128) % kTiles;
            double all = 0;
            if (late < tiles && early < late)
#pragma unroll
                for (int j = 0; j < kChunk; j++) all += columns[late][early][j];
            between[late][early] = all;
        }
        __syncthreads();
        double found = 0;
        if (wave < 2) {
            for (int n = 0; n < own && own < tiles; n++) later += rows[own][n][step];
            for (int n = own + 1; n < tiles; n++) earlier += columns[n][own][step];
            found = (double)RowFrom(later) + Dpp<kRowShiftRight + 1>(RowUpTo(earlier));
            if (t < count) {
                float near = 0;
#pragma unroll
                for (int j = 0; j < kChunk; j++) near += j < step ? diagonal[own][step][j] : 0.f;
                found += near;
                for (int n = own + 1; n < tiles; n++) found += tiled[0][n];
                for (int n = 0; n < own; n++) found += tiled[1][n];
                for (int late = own + 1; late < tiles; late++)
                    for (int early = 0; early < own; early++) found += between[late][early];
                if (episodes == 0) found += passed((float)both, count - 1, -1);
                if (a.out) a.out[((long long)b * a.time + begin + t) * a.heads + h] = (float)found;
            } else {
                found = 0;
            }
        }
        if (a.totals) {
            found = BlockSum(found, sums);
            if (t == 0) a.totals[item] = found;
        }
    };

    // Every workgroup looks for its spans 64 at a time.
    for (long long first = blockIdx.x; first < items; first += 64ll * gridDim.x) {
        const long long mine = first + (long long)lane * gridDim.x;
        unsigned long long sharp = __ballot(mine < items && a.sharp[mine < items ? mine : first]);
        for (; sharp; sharp &= sharp - 1) find(first + (long long)__builtin_ctzll(sharp) * gridDim.x);
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
    long long memories, factors, dots, crossings, totals, sharp, parts, end;
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
    at.sharp = at.totals + (a.d_decay && a.decay_of_head ? four(2 * heads * runs.spans) : 0);
    at.parts = at.sharp + (a.d_decay ? four((heads * runs.spans + 3) / 4) : 0);
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
    // it, or one of them fills its tiles alone, and with enough wavefronts, the values' run has a launch of its own. Enough
    // are 11 of 16 columns for each of the 256 compute units, where the two cross: apart and together, 64 steps, of 1,408, 2,816 and
    // 8,192 wavefronts in all, in us: bfloat16 128 x 64 39 and 34, 40 and 50, 54 and 96; 32 x 64 28 and 26, 34 and 33, 53 and 65;
    // float16 64 x 128 41 and 41, 52 and 63, 103 and 121; float32 32 x 128 39 and 48, 49 and 70, 106 and 176. Sizes like 48 x 80 in
    // 16 bits (95 and 83 of 8,192) and 48 x 64 in 32 (96 and 84) would be better off together.
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
                    a.decay_of_head ? reinterpret_cast<double *>(work + at.totals) : nullptr, reinterpret_cast<unsigned char *>(work + at.sharp),
                    !a.state};
        for (int i = 0; i < 3; i++) d.decayStrides[i] = runs.decayStrides[i];
        for (int i = 0; i < 2; i++) d.resetStrides[i] = runs.resetStrides[i];
        const long long items = heads * runs.spans;
        hipLaunchKernelGGL(DecayKernel, dim3((unsigned)(items < (1 << 22) ? (items + 3) / 4 : 1 << 20)), dim3(256), 0, stream, d);
        const SharpArgs sharp{d, query, key, value, output, a.key_size, a.value_size, a.scale, dq.first, dq.starts, dq.against, dq.againstLast};
        const dim3 grid((unsigned)(items < kSharpBlocks ? items : kSharpBlocks));
        const auto launch = [&](auto kernel) { hipLaunchKernelGGL(kernel, grid, dim3(256), 0, stream, sharp); };
        const bool small = a.key_size <= 64 && a.value_size <= 64;
        if (whole) launch(small ? SharpKernel<T, 2, true> : SharpKernel<T, 4, true>);
        else launch(small ? SharpKernel<T, 2, false> : SharpKernel<T, 4, false>);
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
