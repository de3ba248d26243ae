// The gradients of the gated delta rule over many steps.
//
// With the forward pass's chunk (delta_rule.hip), R = (I + A)^-1, P = scale D o Q K^T, the chunk's
// outputs' gradient dO and the gradient dS of the memory after it:
//   dU = P^T dO + D_C K dS          dB = R^T dU           dv = beta dB
//   dP = dO U^T                     dA = -dB U^T
//   dq = scale G S0 dO + (scale D o dP) K
//   dk = D_C dS U - beta G S0 dB + (scale D o dP)^T Q + (N + N^T) K,   N = beta D o dA
//   dbeta_i = dB_i.(v_i - G_i S0^T k_i) + sum_j dA_ij D_ij k_i.k_j
//   dS0 = G_C dS + scale Q^T (G dO) - K^T (beta G dB)
// and the log decay of step l, which every product from before l to after it carries, gets
//   sum_{i>=l} e_i + sum_{j<l<=i} E_ij + sum_{j<l} f_j + G_C <dS, S0>,
// e_i = q_i.(scale G S0 dO)_i - k_i.(beta G S0 dB)_i, E = dP o P + dA o A, f_j = k_j.(D_C dS U)_j:
// sums of like terms, with no difference of totals that would cost a strong decay its precision.
#include "delta_rule.h"

namespace layers {
namespace {

// One workgroup takes a head backwards through its steps, a segment of two chunks at a time. A
// wavefront holds 16 columns of the memory. The segment's inputs lie in LDS while the next segment's
// are on their way to registers. Two wavefronts first build a chunk's triangular matrices each; then
// the first chunk is played forward from the segment's checkpoint, and the chunks are taken in
// reverse. The products that contract the columns (S0 dO, S0 dB, dS U) go through LDS, each wavefront
// taking whole tiles of keys.
template <class T>
struct BackwardArgs {
    Rule rule;
    View<const T> query, key, value, dOutput;
    Gates gates;
    void *dQuery, *dKey;  // of T with the key heads, or of float with the heads where `shared`
    bool shared;
};

constexpr int kMatrixRow = 16, kMatrix = kChunk * kMatrixRow;  // a 16x16 matrix in LDS
constexpr int kMostShared = 160 * 1024;

// LDS for keys of up to `KeyTiles` tiles and values of up to `Pairs` pairs of them, in floats.
template <int KeyTiles, int Pairs, int ElementSize>
struct BackwardShared {
    static constexpr int kWaves = 2 * Pairs;
    static constexpr int kMemoryRow = Pairs * 32 + 4;     // floats of a row of the memory
    static constexpr int kRow = Pairs * 32 + 8;           // 16-bit elements of a step's row of pieces
    static constexpr int kKeyRow = KeyTiles * 16 + 4, kValueRow = Pairs * 32 + 4;  // elements of a step's inputs
    static constexpr int kMatrices = kSegment / kChunk * kMatrix, kPieceRows = kFloatPieces * kChunk * kRow / 2;
    static constexpr int kMemory1 = KeyTiles * 16 * kMemoryRow;
    static constexpr int kKeyRows = kSegment * kKeyRow * ElementSize / 4, kValueRows = kSegment * kValueRow * ElementSize / 4;
    static constexpr int kReach = 0, kBetas = kReach + 2 * kSegment, kCuts = kBetas + kSegment, kInverse = kCuts + 4,
                         kMixed = kInverse + kMatrices, kProducts = kMixed + kMatrices, kU = kProducts + kMatrices,
                         kB = kU + kPieceRows, kDots = kB + kPieceRows, kK = kDots + 2 * kWaves * 4 * kChunk, kQ = kK + kKeyRows,
                         kO = kQ + kKeyRows, kMemory = kO + kValueRows,
                         // The values are read before any memory is put down.
                         kV = kMemory;
    // Both the memory and its gradient where they fit, else one after the other, with the tiles' sums
    // kept between.
    static constexpr bool kBoth = (kMemory + 2 * kMemory1) * 4 <= kMostShared;
    static constexpr int kSecond = kBoth ? kMemory + kMemory1 : kMemory, kTiles = kMemory + kMemory1;
    static constexpr int kFloats = kMemory + (kBoth ? 2 * kMemory1 : kMemory1 + KeyTiles * 256);
    static_assert(kValueRows <= kMemory1 + (kBoth ? kMemory1 : 0), "room for the values");
};

__device__ __forceinline__ F4 RowOrder(const float *matrix, int m, int g) {
    return *reinterpret_cast<const F4 *>(matrix + m * kMatrixRow + 4 * g);
}
__device__ __forceinline__ F4 ColumnOrder(const float *matrix, int m, int g) {
    F4 x;
#pragma unroll
    for (int r = 0; r < 4; r++) x[r] = matrix[(4 * g + r) * kMatrixRow + m];
    return x;
}

template <class T, int KeyTiles, int Pairs, bool Whole>
__global__ __launch_bounds__(128 * Pairs) __attribute__((amdgpu_waves_per_eu(2))) void BackwardKernel(BackwardArgs<T> a) {
    using At = BackwardShared<KeyTiles, Pairs, sizeof(T)>;
    using Args = BackwardArgs<T>;
    extern __shared__ __align__(16) float shared[];
    constexpr int P = kPieces<T>, kThreads = 128 * Pairs, kWaves = 2 * Pairs;
    const Rule &rule = a.rule;
    const int lane = threadIdx.x & 63, m = lane & 15, g = lane >> 4, wave = threadIdx.x >> 6;
    constexpr int ms = At::kMemoryRow, rs = At::kRow, ks = At::kKeyRow, vs = At::kValueRow;
    double *reach = reinterpret_cast<double *>(shared + At::kReach);
    float *betas = shared + At::kBetas, *memory = shared + At::kMemory, *second = shared + At::kSecond;
    unsigned *cutsOf = reinterpret_cast<unsigned *>(shared + At::kCuts);
    // Rows of values by step, [piece][step][column].
    uint16_t *sharedU = reinterpret_cast<uint16_t *>(shared + At::kU), *sharedB = reinterpret_cast<uint16_t *>(shared + At::kB);
    T *keys = reinterpret_cast<T *>(shared + At::kK), *queries = reinterpret_cast<T *>(shared + At::kQ);
    T *values = reinterpret_cast<T *>(shared + At::kV), *outputs = reinterpret_cast<T *>(shared + At::kO);

    const unsigned head = Place(blockIdx.x, gridDim.x);
    const int h = head % rule.heads, b = head / rule.heads, kh = h / (rule.heads / rule.key_heads);
    const int dk = rule.key_size, dv = rule.value_size, time = rule.time;
    const int column = 16 * wave + m;       // the column of a lane in column order
    const int column4 = 16 * wave + 4 * g;  // its first of four in row order
    const int segments = (time + kSegment - 1) / kSegment;
    const Four eye = Eye(m, g);
    F4 one;
#pragma unroll
    for (int r = 0; r < 4; r++) one[r] = m == 4 * g + r ? 1.f : 0.f;

    const auto loadMemory = [&](const void *memories, long long index, F4(&s)[KeyTiles]) {
        const int rows = Opaque(dk) - 4 * g, stride = Opaque(dv);
        const float *from = static_cast<const float *>(memories) + (index * dk + 4 * g) * stride + column;
#pragma unroll
        for (int t = 0; t < KeyTiles; t++)
#pragma unroll
            for (int r = 0; r < 4; r++) {
                s[t][r] = 0.f;
                if (memories && 16 * t + r < rows && column < dv) s[t][r] = from[(16 * t + r) * stride];
            }
    };

    // A segment's inputs: packs of four elements, thread by thread, on the way from memory to LDS. Past
    // the end of time the last step is read again, and masked.
    constexpr int kKeyPacks = (kSegment * KeyTiles * 4 + kThreads - 1) / kThreads, kValuePacks = kSegment * Pairs * 8 / kThreads;
    Pack<T, 4> nextK[kKeyPacks], nextQ[kKeyPacks], nextV[kValuePacks], nextO[kValuePacks];
    StepGates nextGate;
    const auto fetch = [&](int s0) {
        const Args now = Argument<Args>();
        int i = threadIdx.x;
#pragma unroll
        for (int j = 0; j < kKeyPacks; j++, i += kThreads) {
            const int t = min(s0 + i / (KeyTiles * 4), time - 1), d = i % (KeyTiles * 4) * 4;
            const int valid = i < kSegment * KeyTiles * 4 ? dk - d : 0;
            nextK[j] = Load<4, Whole>(now.key.At(b, t, kh) + d, valid);
            nextQ[j] = Load<4, Whole>(now.query.At(b, t, kh) + d, valid);
        }
        i = threadIdx.x;
#pragma unroll
        for (int j = 0; j < kValuePacks; j++, i += kThreads) {
            const int t = min(s0 + i / (Pairs * 8), time - 1), d = i % (Pairs * 8) * 4;
            nextV[j] = Load<4, Whole>(now.value.At(b, t, h) + d, dv - d);
            nextO[j] = Load<4, Whole>(now.dOutput.At(b, t, h) + d, dv - d);
        }
        if (wave < kSegment / kChunk) nextGate = LoadGates(now.gates, b, s0 + wave * kChunk + m, time, h);
    };
    const auto stage = [&] {
        int i = threadIdx.x;
#pragma unroll
        for (int j = 0; j < kKeyPacks; j++, i += kThreads) {
            const int to = i / (KeyTiles * 4) * ks + i % (KeyTiles * 4) * 4;
            if (i < kSegment * KeyTiles * 4) {
                *reinterpret_cast<Pack<T, 4> *>(keys + to) = nextK[j];
                *reinterpret_cast<Pack<T, 4> *>(queries + to) = nextQ[j];
            }
        }
        i = threadIdx.x;
#pragma unroll
        for (int j = 0; j < kValuePacks; j++, i += kThreads) {
            const int to = i / (Pairs * 8) * vs + i % (Pairs * 8) * 4;
            *reinterpret_cast<Pack<T, 4> *>(values + to) = nextV[j];
            *reinterpret_cast<Pack<T, 4> *>(outputs + to) = nextO[j];
        }
    };
    // Step m of chunk c, where it is of this part.
    const auto keyTile = [&](const T *rows, int c, int t, bool mine) {
        return Masked(*reinterpret_cast<const Pack<T, 4> *>(rows + (c * kChunk + m) * ks + 16 * t + 4 * g), mine);
    };
    const auto valueTile = [&](const T *rows, int c, int x, bool mine) {
        return Masked(*reinterpret_cast<const Pack<T, 4> *>(rows + (c * kChunk + m) * vs + 16 * x + 4 * g), mine);
    };

    F4 dS[KeyTiles];
    loadMemory(rule.d_last, head, dS);
    if (segments > 0) fetch((segments - 1) * kSegment);
    int turn = 0;  // which half of `dots`

    for (int segment = segments - 1; segment >= 0; segment--) {
        const int s0 = segment * kSegment;
        const int chunks = min(kSegment / kChunk, (time - s0 + kChunk - 1) / kChunk);
        const auto checkpoint = [&](F4(&s)[KeyTiles]) {
            const Args now = Argument<Args>();
            if (segment > 0) loadMemory(now.rule.checkpoints, (long long)head * (segments - 1) + segment - 1, s);
            else loadMemory(now.rule.state, head, s);
        };
        __syncthreads();
        stage();
        const StepGates gate = nextGate;
        F4 start[KeyTiles];
        checkpoint(start);
        if (segment > 0) fetch(s0 - kSegment);
        __syncthreads();
        // ---- The chunks' matrices, one wavefront a chunk.
        if (wave < chunks) {
            const int c = wave, count = min(kChunk, time - s0 - c * kChunk);
            const unsigned cuts = (unsigned)(__ballot(gate.Reset()) & 0xffff);
            if (g == 0) betas[c * kChunk + m] = gate.beta;
            if (lane == 0) cutsOf[c] = cuts;
            for (int low = 0, high; low < count; low = high) {
                const unsigned later = cuts >> (low + 1);
                high = later ? min(count, low + 1 + __builtin_ctz(later)) : count;
                const bool starts = (cuts >> low) & 1, mine = m >= low && m < high;
                const double G = RowUpTo(mine && !(starts && m == low) ? gate.decay * kLog2E : 0.0);
                const float beta = mine ? gate.beta : 0.f;
                if (mine && g == 0) reach[c * kChunk + m] = G;
                F4 kk = {0, 0, 0, 0}, qk = {0, 0, 0, 0};
#pragma unroll
                for (int p = 0; p < KeyTiles / 2; p++) {
                    B8 kp[P], qp[P];
                    Pair<T>(keyTile(keys, c, 2 * p, mine), keyTile(keys, c, 2 * p + 1, mine), kp);
                    Pair<T>(keyTile(queries, c, 2 * p, mine), keyTile(queries, c, 2 * p + 1, mine), qp);
                    kk = Mfma32<P, P>(kp, kp, kk);
                    qk = Mfma32<P, P>(kp, qp, qk);
                }
                F4 aA, dA, aP, aKK;
#pragma unroll
                for (int r = 0; r < 4; r++) {
                    const int j = 4 * g + r;
                    const double Gj = __shfl(G, j);
                    const float betaj = __shfl(beta, j);
                    const float d = Exp2(j <= m ? G - Gj : Gj - G);
                    aP[r] = j <= m ? rule.scale * d * qk[r] : 0.f;
                    aKK[r] = j < m ? d * kk[r] : 0.f;
                    aA[r] = beta * aKK[r];
                    dA[r] = m < j ? betaj * d * kk[r] : 0.f;
                }
                const F4 aT = UnitLowerInverse<false>(aA, dA, m, g).rows;
                if (mine) {
                    const int to = c * kMatrix + m * kMatrixRow + 4 * g;
                    *reinterpret_cast<F4 *>(shared + At::kInverse + to) = aT;
                    *reinterpret_cast<F4 *>(shared + At::kMixed + to) = aP;
                    *reinterpret_cast<F4 *>(shared + At::kProducts + to) = aKK;
                }
            }
        }
        __syncthreads();

        // The values that chunk c writes and their errors, from the memory `s` before it; with `advance`
        // the memory goes on to the next chunk.
        const auto play = [&](int c, bool advance, F4(&s)[KeyTiles], F4 &wrote, F4 &errors) {
            const int count = min(kChunk, time - s0 - c * kChunk);
            const unsigned cuts = cutsOf[c];
            wrote = errors = F4{0, 0, 0, 0};
            for (int low = 0, high; low < count; low = high) {
                const unsigned later = cuts >> (low + 1);
                high = later ? min(count, low + 1 + __builtin_ctz(later)) : count;
                const bool starts = (cuts >> low) & 1, mine = m >= low && m < high;
                Four v[P];
                Split<T>(valueTile(values, c, wave, mine), v);
                F4 seen = {0, 0, 0, 0}, error = Turn<P>(v, eye), written;
                if (!starts) {
#pragma unroll
                    for (int p = 0; p < KeyTiles / 2; p++) {
                        B8 kp[P], sp[kFloatPieces];
                        Pair<T>(keyTile(keys, c, 2 * p, mine), keyTile(keys, c, 2 * p + 1, mine), kp);
                        Pair(s[2 * p], s[2 * p + 1], sp);
                        seen = Mfma32<P, kFloatPieces>(kp, sp, seen);
                    }
                }
                F4 aT = RowOrder(shared + At::kInverse + c * kMatrix, m, g);
                bool in[4];
                double Gj[4];
#pragma unroll
                for (int r = 0; r < 4; r++) {
                    in[r] = 4 * g + r >= low && 4 * g + r < high;
                    Gj[r] = in[r] ? reach[c * kChunk + 4 * g + r] : 0.0;
                    error[r] = fmaf(-Exp2(Gj[r]), seen[r], error[r]);
                    written[r] = in[r] ? betas[c * kChunk + 4 * g + r] * error[r] : 0.f;
                    aT[r] = mine && in[r] ? aT[r] : 0.f;
                }
                written = Product(aT, written);
                const double last = reach[c * kChunk + high - 1];
#pragma unroll
                for (int r = 0; r < 4; r++) {
                    wrote[r] = in[r] ? written[r] : wrote[r];
                    errors[r] = in[r] ? error[r] : errors[r];
                    written[r] *= in[r] ? Exp2(last - Gj[r]) : 0.f;
                }
                if (!advance) continue;
                Four wp[kFloatPieces];
                Split(written, wp);
                const float kept = Exp2(last);
#pragma unroll
                for (int t = 0; t < KeyTiles; t++) {
                    Forget();
                    Four x[P], turned[P];
                    Split<T>(keyTile(keys, c, t, mine), x);
                    Turn<P>(x, eye, turned);
                    F4 held = s[t] * kept;
                    if (starts) held = F4{0, 0, 0, 0};
                    s[t] = Mfma16(turned, wp, held);
                }
            }
        };
        F4 wroteFirst, errorsFirst;
        F4 wroteC, errorC;
#pragma unroll 1
        for (int c = 0; c < chunks; c++) {
            if (c) wroteFirst = wroteC, errorsFirst = errorC;
            play(c, c + 1 < chunks, start, wroteC, errorC);
        }
        __syncthreads();

        for (int c = chunks - 1; c >= 0; c--) {
            const int t0 = s0 + c * kChunk;
            const unsigned cuts = cutsOf[c];
            if (c + 1 < chunks) checkpoint(start), wroteC = wroteFirst, errorC = errorsFirst;
            for (int high = min(kChunk, time - t0), low; high > 0; high = low) {
                const unsigned below = cuts & ((1u << high) - 1);
                low = below ? 31 - __builtin_clz(below) : 0;
                const bool starts = (cuts >> low) & 1, mine = m >= low && m < high;
                float *dots = shared + At::kDots + turn * kWaves * 4 * kChunk;
                turn ^= 1;
                const double G = mine ? reach[c * kChunk + m] : 0.0, last = reach[c * kChunk + high - 1];
                const float beta = mine ? betas[c * kChunk + m] : 0.f;
                bool in[4];
                double Gj[4];
                float betaj[4], afterJ[4], wholeJ[4];
#pragma unroll
                for (int r = 0; r < 4; r++) {
                    in[r] = 4 * g + r >= low && 4 * g + r < high;
                    Gj[r] = in[r] ? reach[c * kChunk + 4 * g + r] : 0.0;
                    betaj[r] = in[r] ? betas[c * kChunk + 4 * g + r] : 0.f;
                    afterJ[r] = in[r] ? Exp2(last - Gj[r]) : 0.f;
                    wholeJ[r] = in[r] ? Exp2(Gj[r]) : 0.f;
                }

                // The gradients of the values written, and of the right side they solve.
                Four op[P];
                Split<T>(valueTile(outputs, c, wave, mine), op);
                const F4 dO = Turn<P>(op, eye);
                F4 dU = {0, 0, 0, 0};
#pragma unroll
                for (int p = 0; p < KeyTiles / 2; p++) {
                    B8 kp[P], sp[kFloatPieces];
                    Pair<T>(keyTile(keys, c, 2 * p, mine), keyTile(keys, c, 2 * p + 1, mine), kp);
                    Pair(dS[2 * p], dS[2 * p + 1], sp);
                    dU = Mfma32<P, kFloatPieces>(kp, sp, dU);
                }
                Forget();
                F4 dT = ColumnOrder(shared + At::kInverse + c * kMatrix, m, g);
                F4 dP = ColumnOrder(shared + At::kMixed + c * kMatrix, m, g), written;
#pragma unroll
                for (int r = 0; r < 4; r++) {
                    dU[r] *= afterJ[r];
                    dT[r] = in[r] && mine ? dT[r] : 0.f;
                    dP[r] = in[r] && mine ? dP[r] : 0.f;
                    written[r] = in[r] ? wroteC[r] : 0.f;
                }
                dU = Product(dP, dO, dU);
                const F4 dB = Product(dT, dU), aB = Product(dU, dT), aU = Product(written, one);
                Forget();
                {
                    Four up[kFloatPieces], bp[kFloatPieces];
                    Split(aU, up), Split(aB, bp);
#pragma unroll
                    for (int p = 0; p < kFloatPieces; p++) {
                        *reinterpret_cast<Four *>(sharedU + (p * kChunk + m) * rs + column4) = up[p];
                        *reinterpret_cast<Four *>(sharedB + (p * kChunk + m) * rs + column4) = bp[p];
                    }
                }
                F4 wrong;
#pragma unroll
                for (int r = 0; r < 4; r++) wrong[r] = RowSum(in[r] ? dB[r] * errorC[r] : 0.f);
                if (m == 0) *reinterpret_cast<F4 *>(dots + (wave * 4 + 0) * kChunk + 4 * g) = wrong;
                float held = 0;
#pragma unroll
                for (int t = 0; t < KeyTiles; t++)
#pragma unroll
                    for (int r = 0; r < 4; r++) {
                        memory[(16 * t + 4 * g + r) * ms + column] = dS[t][r];
                        if (starts) continue;
                        if (At::kBoth) second[(16 * t + 4 * g + r) * ms + column] = start[t][r];
                        held = fmaf(dS[t][r], start[t][r], held);
                    }
                held = WaveSum(held);
                if (lane == 0) dots[(wave * 4 + 3) * kChunk] = held;
                if (mine) {
                    Pack<T, 4> x;
#pragma unroll
                    for (int r = 0; r < 4; r++) x.x[r] = As<T>(beta * aB[r]);
                    Store<4, Whole>(static_cast<T *>(Argument<Args>().rule.d_value) +
                                        (((long long)b * time + t0 + m) * rule.heads + h) * dv + column4,
                                    x, dv - column4);
                }
                __syncthreads();

                // The matrices' gradients.
                const auto rowPieces = [&](const uint16_t *rows, int x, B8(&to)[kFloatPieces]) {
#pragma unroll
                    for (int p = 0; p < kFloatPieces; p++) {
                        const uint16_t *from = rows + (p * kChunk + m) * rs + 32 * x + 4 * g;
                        to[p] = Eight(*reinterpret_cast<const Four *>(from), *reinterpret_cast<const Four *>(from + 16));
                    }
                };
                const auto memoryPieces = [&](const float *from, int t, int x, B8(&to)[kFloatPieces]) {
                    from += (16 * t + m) * ms + 32 * x + 4 * g;
                    Pair(*reinterpret_cast<const F4 *>(from), *reinterpret_cast<const F4 *>(from + 16), to);
                };
                const auto outputPieces = [&](int x, B8(&to)[P]) {
                    Pair<T>(valueTile(outputs, c, 2 * x, mine), valueTile(outputs, c, 2 * x + 1, mine), to);
                };
                F4 gP = {0, 0, 0, 0}, gA = {0, 0, 0, 0};
#pragma unroll
                for (int x = 0; x < Pairs; x++) {
                    B8 uw[kFloatPieces], other[kFloatPieces], out[P];
                    rowPieces(sharedU, x, uw);
                    outputPieces(x, out);
                    gP = Mfma32<kFloatPieces, P>(uw, out, gP);
                    rowPieces(sharedB, x, other);
                    gA = Mfma32<kFloatPieces, kFloatPieces>(uw, other, gA);
                }
                Forget();
                const F4 aP = RowOrder(shared + At::kMixed + c * kMatrix, m, g);
                const F4 aKK = RowOrder(shared + At::kProducts + c * kMatrix, m, g);
                F4 aM, aN, E;
                float betaSum = 0;
#pragma unroll
                for (int r = 0; r < 4; r++) {
                    const int j = 4 * g + r;
                    const bool both = mine && in[r];
                    const float d = both && j <= m ? Exp2(G - Gj[r]) : 0.f;
                    aM[r] = rule.scale * d * gP[r];
                    aN[r] = j < m ? -beta * d * gA[r] : 0.f;
                    const float part = both && j < m ? -gA[r] * aKK[r] : 0.f;
                    betaSum += part;
                    E[r] = (both && j <= m ? gP[r] * aP[r] : 0.f) + beta * part;
                }
                Four mp[kFloatPieces], mt[kFloatPieces], np[kFloatPieces];
                Split(aM, mp), Split(Product(aM, one), mt), Split(aN + Product(aN, one), np);

                Forget();
                // This wavefront's tiles of keys: dS U, S0 dO and S0 dB.
                const auto written1 = [&](int t) {
                    F4 sum = {0, 0, 0, 0};
#pragma unroll
                    for (int x = 0; x < Pairs; x++) {
                        B8 uw[kFloatPieces], sp[kFloatPieces];
                        rowPieces(sharedU, x, uw);
                        memoryPieces(memory, t, x, sp);
                        sum = Mfma32<kFloatPieces, kFloatPieces>(uw, sp, sum);
                    }
                    return sum;
                };
                if (!At::kBoth) {
                    for (int t = wave; t < KeyTiles; t += kWaves)
                        *reinterpret_cast<F4 *>(shared + At::kTiles + (t * 64 + lane) * 4) = written1(t);
                    __syncthreads();
                    if (!starts) {
#pragma unroll
                        for (int t = 0; t < KeyTiles; t++)
#pragma unroll
                            for (int r = 0; r < 4; r++) second[(16 * t + 4 * g + r) * ms + column] = start[t][r];
                    }
                    __syncthreads();
                }
                F4 f = {0, 0, 0, 0}, e = {0, 0, 0, 0};
#pragma unroll 1
                for (int t = wave; t < KeyTiles; t += kWaves) {
                    F4 dQ = {0, 0, 0, 0}, y = {0, 0, 0, 0};
                    const F4 dKeys = At::kBoth ? written1(t) : *reinterpret_cast<const F4 *>(shared + At::kTiles + (t * 64 + lane) * 4);
                    Forget();
                    if (!starts)
#pragma unroll
                        for (int x = 0; x < Pairs; x++) {
                            B8 sp[kFloatPieces], other[kFloatPieces], out[P];
                            memoryPieces(second, t, x, sp);
                            outputPieces(x, out);
                            dQ = Mfma32<P, kFloatPieces>(out, sp, dQ);
                            rowPieces(sharedB, x, other);
                            y = Mfma32<kFloatPieces, kFloatPieces>(other, sp, y);
                        }
                    Forget();
                    Four kx[P], qx[P], kTurned[P], qTurned[P];
                    Split<T>(keyTile(keys, c, t, mine), kx), Split<T>(keyTile(queries, c, t, mine), qx);
                    Turn<P>(kx, eye, kTurned), Turn<P>(qx, eye, qTurned);
                    const F4 kf = Turn<P>(kx, eye), qf = Turn<P>(qx, eye);
                    F4 dK;
#pragma unroll
                    for (int r = 0; r < 4; r++) {
                        dK[r] = afterJ[r] * dKeys[r];
                        f[r] = fmaf(dK[r], kf[r], f[r]);
                        const float fromKey = -betaj[r] * wholeJ[r] * y[r];
                        dQ[r] *= rule.scale * wholeJ[r];
                        e[r] = fmaf(qf[r], dQ[r], fmaf(kf[r], fromKey, e[r]));
                        dK[r] += fromKey;
                    }
                    dQ = Mfma16(mp, kTurned, dQ);
                    dK = Mfma16(mt, qTurned, dK);
                    dK = Mfma16(np, kTurned, dK);
                    const Args now = Argument<Args>();
#pragma unroll
                    for (int r = 0; r < 4; r++) {
                        if (!in[r] || 16 * t + m >= dk) continue;
                        const long long row = (long long)b * time + t0 + 4 * g + r;
                        if (now.shared) {
                            const long long to = (row * rule.heads + h) * dk + 16 * t + m;
                            static_cast<float *>(now.dQuery)[to] = dQ[r];
                            static_cast<float *>(now.dKey)[to] = dK[r];
                        } else {
                            const long long to = (row * rule.key_heads + kh) * dk + 16 * t + m;
                            static_cast<T *>(now.dQuery)[to] = As<T>(dQ[r]);
                            static_cast<T *>(now.dKey)[to] = As<T>(dK[r]);
                        }
                    }
                }
                Forget();
                F4 eSum, fSum;
#pragma unroll
                for (int r = 0; r < 4; r++) eSum[r] = RowSum(e[r]), fSum[r] = RowSum(f[r]);
                if (m == 0) {
                    *reinterpret_cast<F4 *>(dots + (wave * 4 + 1) * kChunk + 4 * g) = eSum;
                    *reinterpret_cast<F4 *>(dots + (wave * 4 + 2) * kChunk + 4 * g) = fSum;
                }

                // The gradient of the memory before this part.
                const float kept = Exp2(last);
                if (starts) {
#pragma unroll
                    for (int t = 0; t < KeyTiles; t++) dS[t] = F4{0, 0, 0, 0};
                } else {
                    Four dOp[kFloatPieces], dBp[kFloatPieces];
                    F4 x, y;
#pragma unroll
                    for (int r = 0; r < 4; r++) x[r] = rule.scale * wholeJ[r] * dO[r], y[r] = -betaj[r] * wholeJ[r] * dB[r];
                    Split(x, dOp), Split(y, dBp);
#pragma unroll
                    for (int t = 0; t < KeyTiles; t++) {
                        Forget();
                        Four x[P], turned[P];
                        Split<T>(keyTile(queries, c, t, mine), x);
                        Turn<P>(x, eye, turned);
                        dS[t] = Mfma16(turned, dOp, dS[t] * kept);
                        Split<T>(keyTile(keys, c, t, mine), x);
                        Turn<P>(x, eye, turned);
                        dS[t] = Mfma16(turned, dBp, dS[t]);
                    }
                }
                __syncthreads();

                // The gates' gradients, a lane for each step.
                if (wave == 0) {
                    float eAll = 0, fAll = 0, bAll = 0, heldAll = 0;
#pragma unroll
                    for (int w = 0; w < kWaves; w++) {
                        bAll += dots[(w * 4 + 0) * kChunk + m];
                        eAll += dots[(w * 4 + 1) * kChunk + m];
                        fAll += dots[(w * 4 + 2) * kChunk + m];
                        heldAll += dots[(w * 4 + 3) * kChunk];
                    }
                    float across = 0;
#pragma unroll
                    for (int r = 0; r < 4; r++) {
                        const float x = RowFrom(E[r]);
                        across += 4 * g + r < m ? x : 0.f;
                    }
                    across += __shfl_xor(across, 16);
                    across += __shfl_xor(across, 32);
                    betaSum += __shfl_xor(betaSum, 16);
                    betaSum += __shfl_xor(betaSum, 32);
                    const float through = starts ? 0.f : kept * heldAll;
                    const float decay = RowFrom(eAll) + across + Dpp<kRowShiftRight + 1>(RowUpTo(fAll)) + through;
                    if (mine && g == 0) {
                        const long long to = ((long long)b * time + t0 + m) * rule.heads + h;
                        const Args now = Argument<Args>();
                        static_cast<float *>(now.rule.d_decay)[to] = starts && m == low ? 0.f : decay;
                        static_cast<float *>(now.rule.d_beta)[to] = bAll + betaSum;
                    }
                }
            }
        }
    }
    if (rule.d_state) {
        const int rows = dk - 4 * g;
        float *to = static_cast<float *>(rule.d_state) + ((long long)head * dk + 4 * g) * dv + column;
#pragma unroll
        for (int t = 0; t < KeyTiles; t++)
#pragma unroll
            for (int r = 0; r < 4; r++)
                if (16 * t + r < rows && column < dv) to[(16 * t + r) * dv] = dS[t][r];
    }
}

// The gradients of keys that several heads share: their sum, in the heads' order.
template <class T>
__global__ __launch_bounds__(256) void SharedKeysKernel(const float *parts, T *out, int group, int size, long long count) {
    for (long long i = blockIdx.x * 256ll + threadIdx.x; i < count; i += gridDim.x * 256ll) {
        const long long row = i / size;
        const float *p = parts + row * group * size + (i - row * size);
        float sum = 0;
        for (int n = 0; n < group; n++) sum += p[n * size];
        out[i] = As<T>(sum);
    }
}

template <class T, int KeyTiles>
bool LaunchBackward(const Rule &r, hipStream_t stream) {
    const bool shared = r.heads != r.key_heads;
    const long long steps = (long long)r.batch * r.time, each = steps * r.heads * r.key_size;
    float *parts = static_cast<float *>(r.workspace);
    BackwardArgs<T> a{r,
                      ViewOf<const T>(r.query, r.query_strides, r.key_size),
                      ViewOf<const T>(r.key, r.key_strides, r.key_size),
                      ViewOf<const T>(r.value, r.value_strides, r.value_size),
                      ViewOf<const T>(r.d_output, r.d_output_strides, r.value_size),
                      GatesOf(r),
                      shared ? parts : r.d_query,
                      shared ? parts + each : r.d_key,
                      shared};
    const bool whole = a.query.whole && a.key.whole && a.value.whole && a.dOutput.whole && Aligned(4 * sizeof(T), r.d_value);
    const auto launch = [&](auto wide, auto packed) {
        constexpr int Pairs = decltype(wide)::value;
        const auto kernel = BackwardKernel<T, KeyTiles, Pairs, decltype(packed)::value>;
        constexpr int bytes = BackwardShared<KeyTiles, Pairs, sizeof(T)>::kFloats * sizeof(float);
        static_assert(bytes <= kMostShared, "the memory of a head fits a compute unit's LDS");
        if (hipFuncSetAttribute(reinterpret_cast<const void *>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, bytes) !=
            hipSuccess)
            return false;
        hipLaunchKernelGGL(kernel, dim3((unsigned)(r.batch * (long long)r.heads)), dim3(128 * Pairs), bytes, stream, a);
        return true;
    };
    const int pairs = (r.value_size + 31) / 32;
    bool set;
    if (!whole) set = launch(std::integral_constant<int, 4>(), std::false_type());
    else if (pairs == 1) set = launch(std::integral_constant<int, 1>(), std::true_type());
    else if (pairs == 2) set = launch(std::integral_constant<int, 2>(), std::true_type());
    else if (pairs == 3) set = launch(std::integral_constant<int, 3>(), std::true_type());
    else set = launch(std::integral_constant<int, 4>(), std::true_type());
    if (!set) return false;
    if (shared && steps > 0) {
        const long long count = steps * r.key_heads * r.key_size;
        const unsigned blocks = (unsigned)(count < 256ll * 8192 ? (count + 255) / 256 : 8192);
        const int group = r.heads / r.key_heads;
        hipLaunchKernelGGL(SharedKeysKernel<T>, dim3(blocks), dim3(256), 0, stream, parts, static_cast<T *>(r.d_query), group,
                           r.key_size, count);
        hipLaunchKernelGGL(SharedKeysKernel<T>, dim3(blocks), dim3(256), 0, stream, parts + each,
                           static_cast<T *>(r.d_key), group, r.key_size, count);
    }
    return true;
}

}  // namespace
}  // namespace layers

using namespace layers;

extern "C" __attribute__((visibility("default"))) int cuju_delta_rule_backward(const struct cuju_delta_rule *rule, void *stream) {
    if (!Fits(rule)) return -1;
    const Rule &r = *rule;
    if (r.batch == 0) return 0;
    if (r.time > 0 && (!r.query || !r.key || !r.value || !r.decay || !r.beta || !r.d_output || !r.d_query || !r.d_key ||
                       !r.d_value || !r.d_decay || !r.d_beta))
        return Failed("expected inputs and their gradients");
    if (r.time > 0 && r.heads != r.key_heads && !r.workspace) return Failed("expected a workspace for shared keys");
    if (r.time > kSegment && !r.checkpoints) return Failed("expected the forward pass's checkpoints");
    bool set = true;
    ForType(r.type, [&](auto x) {
        using T = decltype(x);
        const auto s = static_cast<hipStream_t>(stream);
        if (r.key_size <= 32) set = LaunchBackward<T, 2>(r, s);
        else if (r.key_size <= 64) set = LaunchBackward<T, 4>(r, s);
        else if (r.key_size <= 96) set = LaunchBackward<T, 6>(r, s);
        else set = LaunchBackward<T, 8>(r, s);
    });
    if (!set) {
        (void)hipGetLastError();
        return Failed("hipFuncSetAttribute: the delta rule's gradients do not fit the shared memory");
    }
    return Launched("the delta rule's gradients");
}
