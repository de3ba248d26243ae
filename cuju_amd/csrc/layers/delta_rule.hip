// The gated delta rule: one step of it for acting, and its forward pass over many steps.
//
// A head's memory is a matrix S [key][value]. A step scales it by exp(decay) (or clears it, where an
// episode starts), reads what it holds under the key, and writes the part of the value that is
// missing: u = beta (v - S^T k), S += k u^T; the output is scale * S^T q.
#include "delta_rule.h"

namespace layers {
namespace {

// ---------------------------------------------------------------------------------------- one step

// One wavefront takes a head's memory, or a part of its columns: `Lanes` lanes of four columns each
// side by side, 64 / Lanes groups of rows. The memory is read once and written once, which bounds it;
// both products with it come from one pass over the registers, since S_new^T q = (a S)^T q + (q.k) u.
// 360,448 heads of 64 x 64 in bfloat16, 12.0 GB, take 2,275 us: 5.3 TB/s, where an update in place of one
// large tensor reaches 5.9. 44 heads take 6 us.
template <class T, int Keys, int Lanes, bool Whole>
__global__ __launch_bounds__(256) void StepKernel(Rule rule, View<const T> query, View<const T> key, View<const T> value,
                                                  Gates gates, float *memory, T *output, int slices, int columns,
                                                  unsigned waves) {
    constexpr int kGroups = 64 / Lanes, kRows = Keys / kGroups;
    __shared__ float sharedKeys[4][2][Keys];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const unsigned id = blockIdx.x * 4 + wave;
    float *keys = sharedKeys[wave][0], *queries = sharedKeys[wave][1];
    if (id >= waves) return;
    const unsigned slice = id % slices, head = id / slices;
    const int h = head % rule.heads, b = head / rule.heads, kh = h / (rule.heads / rule.key_heads);
    const int dk = rule.key_size, dv = rule.value_size;
    // All loads start before the first is waited for. A memory that is cleared is loaded too, and
    // dropped: what it held, infinities among it, is gone.
    const StepGates gate = LoadGates(gates, b, 0, 1, h);
    const int first = slice * columns + (lane % Lanes) * 4, row0 = (lane / Lanes) * kRows;
    const int valid = min(columns - (lane % Lanes) * 4, dv - first);
    float *at = memory + ((long long)head * dk + row0) * dv + first;
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
    const bool cleared = gate.Reset();
    const float kept = cleared ? 0.f : expf(gate.decay);
    float seen[4] = {0, 0, 0, 0}, out[4] = {0, 0, 0, 0}, both = 0;
#pragma unroll
    for (int i = 0; i < kRows; i++) {
        const float k = keys[row0 + i], q = queries[row0 + i];
        both = fmaf(k, q, both);
#pragma unroll
        for (int c = 0; c < 4; c++) {
            s[i].x[c] = cleared ? 0.f : s[i].x[c] * kept;
            seen[c] = fmaf(k, s[i].x[c], seen[c]);
            out[c] = fmaf(q, s[i].x[c], out[c]);
        }
    }
#pragma unroll
    for (int d = Lanes; d < 64; d *= 2) {
        both += __shfl_xor(both, d);
#pragma unroll
        for (int c = 0; c < 4; c++) {
            seen[c] += __shfl_xor(seen[c], d);
            out[c] += __shfl_xor(out[c], d);
        }
    }
    Pack<T, 4> o;
#pragma unroll
    for (int c = 0; c < 4; c++) {
        const float u = gate.beta * (Float(v.x[c]) - seen[c]);
        o.x[c] = As<T>(rule.scale * fmaf(both, u, out[c]));
        seen[c] = u;
    }
#pragma unroll
    for (int i = 0; i < kRows; i++) {
        const float k = keys[row0 + i];
#pragma unroll
        for (int c = 0; c < 4; c++) s[i].x[c] = fmaf(k, seen[c], s[i].x[c]);
        Store<4, Whole>(at + i * dv, s[i], row0 + i < dk ? valid : 0);
    }
    if (row0 == 0) Store<4, Whole>(output + (long long)head * dv + first, o, valid);
}

template <class T, int Keys>
void LaunchStep(const Rule &r, hipStream_t stream) {
    // At most 64 columns a wavefront, so that keys of 128 fit its registers. 16,384 heads with 64 against 32
    // columns a wavefront: 89 against 88 us (64 x 64), 114 against 136 (64 x 72), 383 against 415 (128 x 128).
    const int slices = (r.value_size + 63) / 64, columns = min(r.value_size, 64);
    const unsigned waves = (unsigned)(r.batch * (long long)r.heads * slices);
    const auto query = ViewOf<const T>(r.query, r.query_strides, r.key_size);
    const auto key = ViewOf<const T>(r.key, r.key_strides, r.key_size);
    const auto value = ViewOf<const T>(r.value, r.value_strides, r.value_size);
    const bool whole = value.whole && Aligned(16, r.state) && Aligned(4 * sizeof(T), r.output);
    const auto launch = [&](auto kernel) {
        hipLaunchKernelGGL(kernel, dim3((waves + 3) / 4), dim3(256), 0, stream, r, query, key, value, GatesOf(r),
                           static_cast<float *>(r.state), static_cast<T *>(r.output), slices, columns, waves);
    };
    if (!whole) launch(StepKernel<T, Keys, 16, false>);
    else if (columns <= 16) launch(StepKernel<T, Keys, 4, true>);
    else if (columns <= 32) launch(StepKernel<T, Keys, 8, true>);
    else launch(StepKernel<T, Keys, 16, true>);
}

// ------------------------------------------------------------------------------------- many steps

// One wavefront takes a head, or 16 * Tiles columns of its memory, through all its steps, 16 at a
// time, with the memory in registers. The columns of the memory never mix, so the wavefronts of a
// head share nothing; what depends on the keys alone each computes for itself.
//
// With the steps of a chunk i, j, G_i the product of the decays up to i and D_ij of those from j + 1
// to i, the values written solve (I + A) U = B with A_ij = beta_i D_ij k_i.k_j (j < i) and
// B_i = beta_i (v_i - G_i S^T k_i); then O = scale (G Q S + (D o Q K^T) U), and the memory becomes
// G_C S + K^T (D_C U). The memory and U are results of the matrix instruction and its right operands
// next, in the same registers; the keys are turned by a product with the identity.
//
// A reset within the chunk cuts it: the parts are played one after the other with the other steps'
// keys, values and gates zero, so nothing of one episode, not even a NaN, meets the next. Each part costs
// what a chunk does.
//
// The products over a chunk's steps take a later step's NaN or infinity, times a zero, into the outputs before
// it. A wavefront that has written values to its memory that are not finite finds the outputs that are not again when
// it is through, step by step from the definition.
//
// Many short sequences are bound by memory: 16,384 heads of 64 steps, 64 x 64 in bfloat16, with the
// memories kept for the gradients, 1.35 GB, take 310 us, 4.4 TB/s. A wavefront on a SIMD by itself is
// bound by its own instructions, some 750 a chunk of keys of 128: 44 heads of 3,000 steps, 128 x 128,
// take 410 us, 2.2 us a chunk.
template <class T>
struct ForwardArgs {
    Rule rule;
    View<const T> query, key, value;
    Gates gates;
    int slices;
    bool inPlace;  // whether the last memory goes where the first one is
};

// Those outputs of a wavefront's columns that are not finite, one step after the other: the chunk at `chunk` is the
// first that has some for a value written that is not, and where memories are kept the last one before it is
// the start. From where the columns hold nothing finite to the end of the episode no output is, and steps are passed
// over. 44 heads of 128 x 128 take 2.3 us a step.
template <class T, int KeyTiles, int Tiles, bool Whole>
__device__ __forceinline__ void OutputsByStep(int chunk) {
    const ForwardArgs<T> a = Argument<ForwardArgs<T>>();
    const Rule &rule = a.rule;
    // The lane, found anew: the thread's number would take a register all the way here.
    const int lane = __builtin_amdgcn_mbcnt_hi(~0u, __builtin_amdgcn_mbcnt_lo(~0u, 0)), m = lane & 15, g = lane >> 4;
    const unsigned id = Place(blockIdx.x, gridDim.x), head = id / a.slices;
    const int h = head % rule.heads, b = head / rule.heads, kh = h / (rule.heads / rule.key_heads);
    const int dk = rule.key_size, dv = rule.value_size, time = rule.time;
    const int column = id % a.slices * 16 * Tiles + m * Tiles, columns = max(0, min(Tiles, dv - column));
    // What other lanes of the wavefront have put down is read.
    __threadfence_block();
    const int segment = rule.checkpoints ? chunk / kSegment : 0;
    const float *memory = static_cast<const float *>(segment ? rule.checkpoints : rule.state);
    const long long index = segment ? (long long)head * ((time - 1) / kSegment) + segment - 1 : head;
    float s[KeyTiles][4][Tiles] = {};
    if (memory)
#pragma unroll
        for (int t = 0; t < KeyTiles; t++)
#pragma unroll
            for (int r = 0; r < 4; r++) {
                const int row = 16 * t + 4 * g + r;
                const auto x = Load<Tiles, Whole>(memory + (index * dk + row) * dv + column, row < dk ? columns : 0);
#pragma unroll
                for (int c = 0; c < Tiles; c++) s[t][r][c] = x.x[c];
            }
    bool lost = false;
#pragma unroll 1
    for (int step = segment * kSegment; step < time; step++) {
        if (lost) {
            // To the next start of an episode, 64 steps at a time.
            const unsigned long long starts = __ballot(LoadGates(a.gates, b, step + lane, time, h).Reset());
            if (!starts) {
                step += 63;
                continue;
            }
            step += __builtin_ctzll(starts);
        }
        // All loads start before the first is waited for.
        const StepGates gate = LoadGates(a.gates, b, step, time, h);
        T *at = static_cast<T *>(rule.output) + (((long long)b * time + step) * rule.heads + h) * dv + column;
        Pack<T, Tiles> o = Load<Tiles, Whole>(at, columns);
        const auto v = Load<Tiles, Whole>(a.value.At(b, step, h) + column, columns);
        Pack<T, 4> k[KeyTiles], q[KeyTiles];
#pragma unroll
        for (int t = 0; t < KeyTiles; t++) {
            k[t] = Load<4, Whole>(a.key.At(b, step, kh) + 16 * t + 4 * g, dk - 16 * t - 4 * g);
            q[t] = Load<4, Whole>(a.query.At(b, step, kh) + 16 * t + 4 * g, dk - 16 * t - 4 * g);
        }
        const bool starts = gate.Reset();
        const float kept = starts ? 0.f : expf(gate.decay);
        float written[Tiles] = {}, out[Tiles] = {};
#pragma unroll
        for (int t = 0; t < KeyTiles; t++)
#pragma unroll
            for (int r = 0; r < 4; r++)
#pragma unroll
                for (int c = 0; c < Tiles; c++) {
                    s[t][r][c] = starts ? 0.f : kept * s[t][r][c];
                    written[c] = fmaf(Float(k[t].x[r]), s[t][r][c], written[c]);
                }
#pragma unroll
        for (int c = 0; c < Tiles; c++) {
            written[c] += __shfl_xor(written[c], 16);
            written[c] += __shfl_xor(written[c], 32);
            written[c] = gate.beta * (Float(v.x[c]) - written[c]);
        }
#pragma unroll
        for (int t = 0; t < KeyTiles; t++)
#pragma unroll
            for (int r = 0; r < 4; r++)
#pragma unroll
                for (int c = 0; c < Tiles; c++) {
                    s[t][r][c] = fmaf(Float(k[t].x[r]), written[c], s[t][r][c]);
                    out[c] = fmaf(Float(q[t].x[r]), s[t][r][c], out[c]);
                }
        bool holds = false, found = false;
#pragma unroll
        for (int c = 0; c < Tiles; c++) {
            out[c] += __shfl_xor(out[c], 16);
            out[c] += __shfl_xor(out[c], 32);
            if (Float(o.x[c]) * 0.f != 0.f) o.x[c] = As<T>(rule.scale * out[c]), found = true;
            holds |= c < columns && written[c] * 0.f == 0.f;
        }
        // A store where there is nothing to change would hold up the next step's loads.
        if (found && g == 0) Store<Tiles, Whole>(at, o, columns);
        lost = __ballot(holds) == 0;
    }
    if (a.inPlace)
#pragma unroll
        for (int t = 0; t < KeyTiles; t++)
#pragma unroll
            for (int r = 0; r < 4; r++) {
                const int row = 16 * t + 4 * g + r;
                Pack<float, Tiles> x;
#pragma unroll
                for (int c = 0; c < Tiles; c++) x.x[c] = s[t][r][c];
                Store<Tiles, Whole>(static_cast<float *>(rule.last) + ((long long)head * dk + row) * dv + column, x, row < dk ? columns : 0);
            }
}

// Wavefronts that a SIMD has to hold: of short keys and narrow pieces more, which they come to with a few registers
// less (16,000 heads of 32 x 32 in half, 20 steps: 79 us with three, 89 with two).
template <class T, int KeyTiles, int Tiles>
constexpr int kForwardWaves = KeyTiles == 2 && Tiles == 1 && kPieces<T> == 1                                ? 4
                              : KeyTiles == 2 && (Tiles == 1 || (Tiles == 2 && kPieces<T> < kFloatPieces)) ? 3
                                                                                                            : 2;

template <class T, int KeyTiles, int Tiles, bool Whole>
__global__ __launch_bounds__(64) __attribute__((amdgpu_waves_per_eu(kForwardWaves<T, KeyTiles, Tiles>))) void ForwardKernel(ForwardArgs<T> a) {
    const Rule &rule = a.rule;
    const View<const T> &query = a.query, &key = a.key, &value = a.value;
    const Gates &gates = a.gates;
    const int slices = a.slices;
    __shared__ double reach[kChunk];
    __shared__ float betas[kChunk];
    const int lane = threadIdx.x, m = lane & 15, g = lane >> 4;
    const unsigned id = Place(blockIdx.x, gridDim.x);
    const int slice = id % slices;
    const unsigned head = id / slices;
    const int h = head % rule.heads, b = head / rule.heads, kh = h / (rule.heads / rule.key_heads);
    const int dk = rule.key_size, dv = rule.value_size, time = rule.time;
    // Lane m's columns lie side by side, one in each tile.
    const int column = slice * 16 * Tiles + m * Tiles, columns = max(0, min(Tiles, dv - column));

    F4 s[KeyTiles][Tiles];
    if (rule.state) {
        const float *first = static_cast<const float *>(rule.state) + ((long long)head * dk + 4 * g) * dv + column;
#pragma unroll
        for (int t = 0; t < KeyTiles; t++)
#pragma unroll
            for (int r = 0; r < 4; r++) {
                const bool real = 16 * t + 4 * g + r < dk;
                const auto x = Load<Tiles, Whole>(first + (16 * t + r) * dv, real ? columns : 0);
#pragma unroll
                for (int c = 0; c < Tiles; c++) s[t][c][r] = x.x[c];
            }
    } else {
#pragma unroll
        for (int t = 0; t < KeyTiles; t++)
#pragma unroll
            for (int c = 0; c < Tiles; c++) s[t][c] = F4{0, 0, 0, 0};
    }
    const auto keep = [&](void *memories, long long index) {
        const int rows = Opaque(dk) - 4 * g, stride = Opaque(dv);
        float *to = static_cast<float *>(memories) + (index * dk + 4 * g) * stride + column;
#pragma unroll
        for (int t = 0; t < KeyTiles; t++)
#pragma unroll
            for (int r = 0; r < 4; r++) {
                Pack<float, Tiles> x;
#pragma unroll
                for (int c = 0; c < Tiles; c++) x.x[c] = s[t][c][r];
                Store<Tiles, Whole>(to + (16 * t + r) * stride, x, 16 * t + r < rows ? columns : 0);
            }
    };

    // The next part's inputs are on their way while one is computed. Past the end of time the last
    // step is read again, and masked.
    Pack<T, 4> nextK[KeyTiles], nextQ[KeyTiles];
    Pack<T, Tiles> nextV[4];
    StepGates next;
    const bool full = Whole && dk == 16 * KeyTiles && dv % (16 * Tiles) == 0;
    // Where the lane reads and writes next: pointers that move on by a chunk, since a lone wavefront's
    // time is its number of instructions.
    const long long ahead = kChunk;
    const T *atK = key.At(b, m, kh) + 4 * g, *atQ = query.At(b, m, kh) + 4 * g, *atV = value.At(b, 4 * g, h) + column;
    const float *atDecay = gates.decay + b * gates.decayStrides[0] + m * gates.decayStrides[1] + h * gates.decayStrides[2];
    const float *atBeta = gates.beta + b * gates.betaStrides[0] + m * gates.betaStrides[1] + h * gates.betaStrides[2];
    T *atOut = static_cast<T *>(rule.output) + (((long long)b * time + 4 * g) * rule.heads + h) * dv + column;
    const unsigned char *atReset = gates.resets ? gates.resets + b * gates.resetStrides[0] + m * gates.resetStrides[1] : nullptr;
    const auto fetch = [&](int t0) {
        const int left = time - t0;  // steps that are left
        if (full && left >= kChunk) {
#pragma unroll
            for (int i = 0; i < KeyTiles; i++) {
                nextK[i] = *reinterpret_cast<const Pack<T, 4> *>(Global(atK) + 16 * i);
                nextQ[i] = *reinterpret_cast<const Pack<T, 4> *>(Global(atQ) + 16 * i);
            }
            const T *v = atV;
#pragma unroll
            for (int r = 0; r < 4; r++, v += value.time) nextV[r] = *reinterpret_cast<const Pack<T, Tiles> *>(Global(v));
            next.decay = *Global(atDecay), next.beta = *Global(atBeta);
            next.cleared = gates.resets ? *Global(atReset) : 0;
        } else {
            const int sizes = Opaque(dk) - 4 * g, back = min(0, left - 1 - m);
            const T *k = Global(atK) + back * key.time, *q = Global(atQ) + back * query.time;
#pragma unroll
            for (int i = 0; i < KeyTiles; i++) {
                nextK[i] = Load<4, Whole>(k + 16 * i, sizes - 16 * i);
                nextQ[i] = Load<4, Whole>(q + 16 * i, sizes - 16 * i);
            }
#pragma unroll
            for (int r = 0; r < 4; r++)
                nextV[r] = Load<Tiles, Whole>(Global(atV) + min(r, left - 1 - 4 * g) * value.time, columns);
            next = LoadGates(gates, b, t0 + m, time, h);
        }
    };
    const auto advance = [&] {
        atK += ahead * key.time, atQ += ahead * query.time, atV += ahead * value.time;
        atDecay += ahead * gates.decayStrides[1], atBeta += ahead * gates.betaStrides[1];
        if (gates.resets) atReset += ahead * gates.resetStrides[1];
    };

    constexpr int P = kPieces<T>;
    const Eyes eyes = EyesOf(m, g);

    // A part's outputs leave with the next part's loads: the wait for loads, which are answered in the order in
    // which loads and stores were sent, then finds them gone.
    Pack<T, Tiles> done[4];
    int doneLow = 0, doneHigh = 0;
    // Values written: a sum that is not finite where one is not, lanes that had such a one, and the chunk up to which
    // none had. Looked at a part later, the sum waits for no product.
    float mark = 0;
    unsigned long long odd = 0;
    int clean = 0;
    const auto put = [&] {
        T *out = Global(atOut);
        const int stride = rule.heads * dv;
        if (full && doneHigh - doneLow == kChunk) {
#pragma unroll
            for (int r = 0; r < 4; r++, out += stride) *reinterpret_cast<Pack<T, Tiles> *>(out) = done[r];
        } else {
#pragma unroll
            for (int r = 0; r < 4; r++, out += stride)
                Store<Tiles, Whole>(out, done[r], 4 * g + r >= doneLow && 4 * g + r < doneHigh ? columns : 0);
        }
        if (doneHigh == kChunk) atOut += ahead * stride;
    };

    if (time > 0) fetch(0);
    for (int t0 = 0, low = 0, high; t0 < time; low = high) {
        // The part: steps [low, high) of the chunk at t0. The others are masked.
        const unsigned cuts = (unsigned)(__ballot(next.Reset()) & 0xffff);
        const int count = min(kChunk, time - t0);
        const unsigned later = cuts >> (low + 1);
        high = later ? min(count, low + 1 + __builtin_ctz(later)) : count;
        const bool starts = (cuts >> low) & 1, mine = m >= low && m < high;
        if (rule.checkpoints && low == 0 && t0 > 0 && t0 % kSegment == 0)
            keep(rule.checkpoints, (long long)head * ((time - 1) / kSegment) + t0 / kSegment - 1);
        if (starts) {
#pragma unroll
            for (int t = 0; t < KeyTiles; t++)
#pragma unroll
                for (int c = 0; c < Tiles; c++) s[t][c] = F4{0, 0, 0, 0};
        }
        const double G = RowUpTo(mine && !(starts && m == low) ? next.decay * kLog2E : 0.0);
        const float beta = mine ? next.beta : 0.f;
        Pack<T, 4> k[KeyTiles], q[KeyTiles];
        Pack<T, Tiles> v[4];
#pragma unroll
        for (int i = 0; i < KeyTiles; i++) k[i] = nextK[i], q[i] = nextQ[i];
#pragma unroll
        for (int r = 0; r < 4; r++) v[r] = nextV[r];
        if (high - low < kChunk) {
#pragma unroll
            for (int i = 0; i < KeyTiles; i++) k[i] = Masked(k[i], mine), q[i] = Masked(q[i], mine);
#pragma unroll
            for (int r = 0; r < 4; r++)
                if (4 * g + r < low || 4 * g + r >= high) v[r] = Pack<T, Tiles>{};
        }
        put();
        odd |= __ballot(mark * 0.f != 0.f);
        if (!odd) clean = t0;
        const int end = high;
        if (high == count) t0 += kChunk, high = 0, advance();
        if (t0 < time) fetch(t0);

        __syncthreads();
        if (g == 0) reach[m] = G, betas[m] = beta;
        __syncthreads();

        // Products with the memory, of k_i.k_j, and of q_i.k_j in row order; the keys' transpose.
        F4 kk = {0, 0, 0, 0}, qk = {0, 0, 0, 0}, u[Tiles], o[Tiles];
        Four turned[KeyTiles][P];
#pragma unroll
        for (int c = 0; c < Tiles; c++) u[c] = o[c] = F4{0, 0, 0, 0};
#pragma unroll
        for (int p = 0; p < KeyTiles / 2; p++) {
            B8 kp[P], qp[P];
            Pair<T>(k[2 * p], k[2 * p + 1], kp), Pair<T>(q[2 * p], q[2 * p + 1], qp);
            kk = Mfma32<P, P>(kp, kp, kk);
            qk = Mfma32<P, P>(kp, qp, qk);
            Turn<P>(kp, eyes.half[0], turned[2 * p]);
            Turn<P>(kp, eyes.half[1], turned[2 * p + 1]);
#pragma unroll
            for (int c = 0; c < Tiles; c++) {
                B8 sp[kFloatPieces];
                Pair(s[2 * p][c], s[2 * p + 1][c], sp);
                u[c] = Mfma32<P, kFloatPieces>(kp, sp, u[c]);
                o[c] = Mfma32<P, kFloatPieces>(qp, sp, o[c]);
            }
        }

        const double last = reach[kChunk - 1];
        double Gj[4];
        float betaj[4];
#pragma unroll
        for (int r = 0; r < 4; r++) Gj[r] = reach[4 * g + r], betaj[r] = betas[4 * g + r];
        F4 aA, dA, aP;
#pragma unroll
        for (int r = 0; r < 4; r++) {
            const int j = 4 * g + r;
            // Either way round, the later step minus the earlier one.
            const float d = Exp2(j <= m ? G - Gj[r] : Gj[r] - G);
            aP[r] = j <= m ? rule.scale * d * qk[r] : 0.f;
            aA[r] = j < m ? beta * d * kk[r] : 0.f;
            dA[r] = m < j ? betaj[r] * d * kk[r] : 0.f;
        }
        const F4 aT = UnitLowerInverse(aA, dA, m, g);
#pragma unroll
        for (int r = 0; r < 4; r++) {
            const float whole = Exp2(Gj[r]), asked = -whole * betaj[r], out = rule.scale * whole;
#pragma unroll
            for (int c = 0; c < Tiles; c++) {
                u[c][r] = fmaf(asked, u[c][r], betaj[r] * Float(v[r].x[c]));
                o[c][r] *= out;
            }
        }
#pragma unroll
        for (int c = 0; c < Tiles; c++) {
            u[c] = Product(aT, u[c]);
            o[c] = Product(aP, u[c], o[c]);
        }
#pragma unroll
        for (int r = 0; r < 4; r++) {
#pragma unroll
            for (int c = 0; c < Tiles; c++) done[r].x[c] = As<T>(o[c][r]);
            const float after = Exp2(last - Gj[r]);
#pragma unroll
            for (int c = 0; c < Tiles; c++) u[c][r] *= after;
        }
        mark = 0;
#pragma unroll
        for (int c = 0; c < Tiles; c++) mark += (u[c][0] + u[c][1]) + (u[c][2] + u[c][3]);
        doneLow = low, doneHigh = end;
        const float kept = Exp2(last);
        Four up[Tiles][kFloatPieces];
#pragma unroll
        for (int c = 0; c < Tiles; c++) Split(u[c], up[c]);
#pragma unroll
        for (int t = 0; t < KeyTiles; t++)
#pragma unroll
            for (int c = 0; c < Tiles; c++) s[t][c] = Mfma16(turned[t], up[c], s[t][c] * kept);
    }
    put();
    odd |= __ballot(mark * 0.f != 0.f);
    // A last memory in the first one's place leaves that for the steps to be found again from, which end in it too.
    if (rule.last && !(odd && a.inPlace)) keep(rule.last, head);
    if (odd) OutputsByStep<T, KeyTiles, Tiles, Whole>(clean);
}

template <class T, int KeyTiles>
void LaunchForward(const Rule &r, hipStream_t stream) {
    const auto query = ViewOf<const T>(r.query, r.query_strides, r.key_size);
    const auto key = ViewOf<const T>(r.key, r.key_strides, r.key_size);
    const auto value = ViewOf<const T>(r.value, r.value_strides, r.value_size);
    const bool whole = query.whole && key.whole && value.whole && Aligned(4 * sizeof(T), r.output) &&
                       Aligned(16, r.state) && Aligned(16, r.last) && Aligned(16, r.checkpoints);
    const auto launch = [&](auto kernel, int tiles) {
        const int slices = (r.value_size + 16 * tiles - 1) / (16 * tiles);
        hipLaunchKernelGGL(kernel, dim3((unsigned)(r.batch * (long long)r.heads * slices)), dim3(64), 0, stream,
                           ForwardArgs<T>{r, query, key, value, GatesOf(r), slices, r.last && r.last == r.state});
    };
    // Wide pieces repeat less of the keys' work; narrow ones give few heads more wavefronts. The chip
    // has 1,024 SIMDs, and the widest pieces that fill them are the fastest: 64 x 64 in bfloat16, 128 steps,
    // pieces of 64, 32 and 16 columns, 1,024 heads 40, 41 and 62 us; 256 heads 33, 33 and 25. Four tiles of
    // a float's or a long key's pieces are more than the registers hold.
    constexpr int most = kPieces<T> * KeyTiles > 12 ? 1 : kPieces<T> * KeyTiles > 4 ? 2 : 4;
    const long long heads = (long long)r.batch * r.heads;
    const auto fills = [&](int tiles) {
        return tiles <= most && r.value_size > 8 * tiles && heads * ((r.value_size + 16 * tiles - 1) / (16 * tiles)) >= 1024;
    };
    if (!whole) launch(ForwardKernel<T, KeyTiles, 1, false>, 1);
    else if (fills(4)) launch(ForwardKernel<T, KeyTiles, most >= 4 ? 4 : 1, true>, 4);
    else if (fills(2)) launch(ForwardKernel<T, KeyTiles, most >= 2 ? 2 : 1, true>, 2);
    else launch(ForwardKernel<T, KeyTiles, 1, true>, 1);
}

}  // namespace
}  // namespace layers

using namespace layers;

extern "C" __attribute__((visibility("default"))) int cuju_delta_rule_step(const struct cuju_delta_rule *rule, void *stream) {
    if (!Fits(rule)) return -1;
    const Rule &r = *rule;
    if (r.time != 1) return Failed("expected one step");
    if (r.batch == 0) return 0;
    if (!r.query || !r.key || !r.value || !r.decay || !r.beta || !r.state || !r.output) return Failed("expected a memory and an output");
    ForType(r.type, [&](auto x) {
        using T = decltype(x);
        const auto s = static_cast<hipStream_t>(stream);
        if (r.key_size <= 32) LaunchStep<T, 32>(r, s);
        else if (r.key_size <= 64) LaunchStep<T, 64>(r, s);
        else LaunchStep<T, 128>(r, s);
    });
    return Launched("the delta rule's step");
}

extern "C" __attribute__((visibility("default"))) int cuju_delta_rule_forward(const struct cuju_delta_rule *rule, void *stream) {
    if (!Fits(rule)) return -1;
    const Rule &r = *rule;
    if (r.batch == 0) return 0;
    if (r.time > 0 && (!r.query || !r.key || !r.value || !r.decay || !r.beta || !r.output))
        return Failed("expected inputs and an output");
    ForType(r.type, [&](auto x) {
        using T = decltype(x);
        const auto s = static_cast<hipStream_t>(stream);
        if (r.key_size <= 32) LaunchForward<T, 2>(r, s);
        else if (r.key_size <= 64) LaunchForward<T, 4>(r, s);
        else if (r.key_size <= 96) LaunchForward<T, 6>(r, s);
        else LaunchForward<T, 8>(r, s);
    });
    return Launched("the delta rule over many steps");
}
