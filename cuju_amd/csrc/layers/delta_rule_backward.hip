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

// One workgroup takes a head, or a part of its columns, backwards through its steps, 32 at a time: two
// tiles of steps, from the memory that the forward pass kept before them. A wavefront holds 16 columns of the
// memory and of its gradient. The steps' inputs lie in LDS while the next ones are on their way to
// registers. Between barriers,
//  - the triangular matrices of the tiles (11, 22) and between them (21), a block to a wavefront;
//  - U, dU and dB by columns, put down in row order in pieces, with the memory's gradient;
//  - dP and dA, and from them the matrices the keys' and queries' gradients take, a block to a
//    wavefront; dS U by tiles of keys, whole tiles to a wavefront;
//  - with the memory in its gradient's place: S0 dO, S0 dB, and the keys' and queries' gradients.
// Heads that share keys, or whose columns take several workgroups, leave parts of the gradients of the keys,
// queries and gates that a second kernel adds up, in their order.
//
// 16,384 heads of 64 steps, 64 x 64 in bfloat16, 2.0 GB, take 1,076 us. Registers (215 of 256) and LDS hold
// it at two wavefronts on a SIMD, vector instructions take 46 % of the cycles, a third of them splits into
// pieces, and the wavefronts wait 42 % of theirs, for LDS between products that need one another and at the
// barriers.
template <class T>
struct BackwardArgs {
    Rule rule;
    View<const T> query, key, value, dOutput;
    Gates gates;
    void *dQuery, *dKey;    // of T, or parts of float by head and slice
    float *dDecay, *dBeta;  // or parts by slice
    int slices;
    bool parted;  // whether dQuery and dKey are parts
};

constexpr int kMatrix = kChunk * kChunk;                  // a 16x16 matrix in LDS
constexpr int kPieceMatrix = kFloatPieces * kMatrix / 2;  // its pieces
constexpr int kBlock = 2 * kMatrix;                       // a block's P and K K^T, and then the pieces of its N
enum Block { kFirst, kSecond, kAcross };                  // of two tiles of steps: 11, 22 and 21

// LDS for keys of up to `KeyTiles` tiles and `Waves` wavefronts of 16 columns, in floats.
template <int KeyTiles, int Waves, int ElementSize>
struct BackwardShared {
    static constexpr int kMemoryRow = Waves * 16 + 4;  // floats of a row of the memory
    static constexpr int kRow = Waves * 16 + 8;        // 16-bit elements of a step's row of pieces
    static constexpr int kKeyRow = KeyTiles * 16 + 4, kValueRow = Waves * 16 + 4;  // elements of a step's inputs
    static constexpr int kPieceRows = kFloatPieces * kSegment * kRow / 2;
    static constexpr int kKeyRows = kSegment * kKeyRow * ElementSize / 4, kValueRows = kSegment * kValueRow * ElementSize / 4;
    static constexpr int kReach = 0, kBetas = kReach + 2 * kSegment, kWhole = kBetas + kSegment, kAfter = kWhole + kSegment,
                         kInverse = kAfter + kSegment, kMixed = kInverse + 2 * kMatrix,
                         kProducts = kMixed + kMatrix, kM = kMixed + 3 * kBlock, kSums = kM + 3 * kPieceMatrix,
                         kDots = kSums + 8 * kChunk, kU = kDots + Waves * 4 * kSegment,
                         kB = kU + kPieceRows, kK = kB + kPieceRows, kQ = kK + kKeyRows, kO = kQ + kKeyRows,
                         kMemory = kO + kValueRows, kFloats = kMemory + KeyTiles * 16 * kMemoryRow;
};

__device__ __forceinline__ F4 RowOrder(const float *matrix, int m, int g) {
    return *reinterpret_cast<const F4 *>(matrix + m * kChunk + 4 * g);
}
__device__ __forceinline__ F4 ColumnOrder(const float *matrix, int m, int g) {
    F4 x;
#pragma unroll
    for (int r = 0; r < 4; r++) x[r] = matrix[(4 * g + r) * kChunk + m];
    return x;
}

// Wavefronts that a SIMD has to hold: two, but one where the registers of two would spill (keys over 64, and
// floats with more tiles of keys than wavefronts) and the workgroup has no more than a wavefront a SIMD.
template <class T, int KeyTiles, int Waves>
constexpr int kWavesPerSimd = KeyTiles > 4 || (sizeof(T) == 4 && Waves < KeyTiles) ? 1 : 2;

template <class T, int KeyTiles, int Waves, bool Whole>
__global__ __launch_bounds__(64 * Waves) __attribute__((amdgpu_waves_per_eu(kWavesPerSimd<T, KeyTiles, Waves>))) void BackwardKernel(
    BackwardArgs<T> a) {
    using At = BackwardShared<KeyTiles, Waves, sizeof(T)>;
    using Args = BackwardArgs<T>;
    extern __shared__ __align__(16) float shared[];
    constexpr int P = kPieces<T>, kThreads = 64 * Waves, kPairs = Waves / 2;
    const Rule &rule = a.rule;
    // The lane is read anew in every part: the addresses that follow from it would fill the registers.
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    int lane = threadIdx.x & 63, m = lane & 15, g = lane >> 4;
    constexpr int ms = At::kMemoryRow, rs = At::kRow, ks = At::kKeyRow, vs = At::kValueRow;
    double *reach = reinterpret_cast<double *>(shared + At::kReach);
    float *betas = shared + At::kBetas, *wholes = shared + At::kWhole, *afters = shared + At::kAfter;
    float *memory = shared + At::kMemory, *dots = shared + At::kDots, *sums = shared + At::kSums;
    // Rows of values by step, [piece][step][column].
    uint16_t *sharedU = reinterpret_cast<uint16_t *>(shared + At::kU), *sharedB = reinterpret_cast<uint16_t *>(shared + At::kB);
    uint16_t *sharedM = reinterpret_cast<uint16_t *>(shared + At::kM), *sharedN = reinterpret_cast<uint16_t *>(shared + At::kMixed);
    T *keys = reinterpret_cast<T *>(shared + At::kK), *queries = reinterpret_cast<T *>(shared + At::kQ);
    T *outputs = reinterpret_cast<T *>(shared + At::kO);

    const unsigned id = Place(blockIdx.x, gridDim.x);
    const unsigned slice = id % a.slices, head = id / a.slices;
    const int h = head % rule.heads, b = head / rule.heads, kh = h / (rule.heads / rule.key_heads);
    const int dk = rule.key_size, dv = rule.value_size, time = rule.time;
    const int base = slice * 16 * Waves;
    int column = base + 16 * wave + m;  // a lane's column in column order
    int column4 = 16 * wave + 4 * g;    // its first of four in row order, within the slice
    const int segments = (time + kSegment - 1) / kSegment;
    const Eyes eyes = EyesOf(m, g);

    const auto loadMemory = [&](const void *memories, long long index, F4(&s)[KeyTiles]) {
        const int rows = Opaque(dk) - 4 * g, stride = Opaque(dv);
        const float *from = static_cast<const float *>(memories) + index * dk * dv;
        const uint32_t at = (4 * g * stride + column) * sizeof(float);
#pragma unroll
        for (int t = 0; t < KeyTiles; t++)
#pragma unroll
            for (int r = 0; r < 4; r++) {
                s[t][r] = 0.f;
                if (memories && 16 * t + r < rows && column < dv) s[t][r] = *Lane(from + (16 * t + r) * stride, at);
            }
    };

    // The steps' inputs: packs of four elements, thread by thread, on the way from memory to LDS; the
    // values of a wavefront's own columns in row order. Past the end of time the last step is read again,
    // and masked.
    constexpr int kKeyPacks = (kSegment * KeyTiles * 4 + kThreads - 1) / kThreads, kValuePacks = kSegment * Waves * 4 / kThreads;
    Pack<T, 4> nextK[kKeyPacks], nextQ[kKeyPacks], nextV[2], nextO[kValuePacks];
    StepGates nextGates[2];
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
            const int t = min(s0 + i / (Waves * 4), time - 1), d = base + i % (Waves * 4) * 4;
            nextO[j] = Load<4, Whole>(now.dOutput.At(b, t, h) + d, dv - d);
        }
#pragma unroll
        for (int j = 0; j < 2; j++) {
            const int t = min(s0 + kChunk * j + m, time - 1), d = base + column4;
            nextV[j] = Load<4, Whole>(now.value.At(b, t, h) + d, dv - d);
            nextGates[j] = LoadGates(now.gates, b, s0 + kChunk * j + m, time, h);
        }
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
            const int to = i / (Waves * 4) * vs + i % (Waves * 4) * 4;
            *reinterpret_cast<Pack<T, 4> *>(outputs + to) = nextO[j];
        }
    };

    F4 dS[KeyTiles];
    loadMemory(rule.d_last, head, dS);
    if (segments > 0) fetch((segments - 1) * kSegment);

    for (int segment = segments - 1; segment >= 0; segment--) {
        const int s0 = segment * kSegment, count = min(kSegment, time - s0);
        __syncthreads();
        stage();
        const StepGates gates[2] = {nextGates[0], nextGates[1]};
        const Pack<T, 4> values[2] = {nextV[0], nextV[1]};
        F4 start[KeyTiles];
        {
            const Args now = Argument<Args>();
            if (segment > 0) loadMemory(now.rule.checkpoints, (long long)head * (segments - 1) + segment - 1, start);
            else loadMemory(now.rule.state, head, start);
        }
        if (segment > 0) fetch(s0 - kSegment);
        const unsigned cuts = (unsigned)(__ballot(gates[0].Reset()) & 0xffff) | (unsigned)(__ballot(gates[1].Reset()) & 0xffff) << 16;
        __syncthreads();

        // Parts between resets, last first; the steps of other parts are masked.
        for (int high = count, low; high > 0; high = low) {
            const unsigned below = cuts & (high < 32 ? (1u << high) - 1 : ~0u);
            low = below ? 31 - __builtin_clz(below) : 0;
            const bool starts = (cuts >> low) & 1;
#pragma unroll
            for (int t = 0; t < KeyTiles; t++) Renew(start[t]);
            lane = Renewed(lane), m = lane & 15, g = lane >> 4, column4 = 16 * wave + 4 * g;
            const auto mine = [&](int tile) { return kChunk * tile + m >= low && kChunk * tile + m < high; };
            const auto in = [&](int tile, int r) { return kChunk * tile + 4 * g + r >= low && kChunk * tile + 4 * g + r < high; };
            const auto keyPair = [&](const T *rows, int tile, int p, B8(&x)[P]) {
                const T *from = rows + (kChunk * tile + m) * ks + 32 * p + 4 * g;
                Pair<T>(Masked(*reinterpret_cast<const Pack<T, 4> *>(from), mine(tile)),
                        Masked(*reinterpret_cast<const Pack<T, 4> *>(from + 16), mine(tile)), x);
            };
            const auto valueTile = [&](const T *rows, int tile, int x) {
                return Masked(*reinterpret_cast<const Pack<T, 4> *>(rows + (kChunk * tile + m) * vs + 16 * x + 4 * g), mine(tile));
            };

            // ---- The triangular matrices.
            double G[2];
            {
                const auto kept = [&](int tile) {
                    return mine(tile) && !(starts && kChunk * tile + m == low) ? gates[tile].decay * kLog2E : 0.0;
                };
                G[0] = RowUpTo(kept(0));
                G[1] = RowUpTo(kept(1)) + __shfl(G[0], 15);
            }
            const double last = __shfl(high > kChunk ? G[1] : G[0], (high - 1) & 15);
            if (wave == 0 && g == 0)
#pragma unroll
                for (int tile = 0; tile < 2; tile++) {
                    const int at = kChunk * tile + m;
                    reach[at] = mine(tile) ? G[tile] : 0.0;
                    betas[at] = mine(tile) ? gates[tile].beta : 0.f;
                    wholes[at] = mine(tile) ? Exp2(G[tile]) : 0.f;
                    afters[at] = mine(tile) ? Exp2(last - G[tile]) : 0.f;
                }
#pragma unroll 1
            for (int block = wave; block < 3; block += Waves) {
                const int row = block == kFirst ? 0 : 1, col = block == kSecond ? 1 : 0;
                F4 kk = {0, 0, 0, 0}, qk = {0, 0, 0, 0};
#pragma unroll
                for (int p = 0; p < KeyTiles / 2; p++) {
                    B8 kj[P], ki[P], qi[P];
                    keyPair(keys, col, p, kj), keyPair(keys, row, p, ki), keyPair(queries, row, p, qi);
                    kk = Mfma32<P, P>(kj, ki, kk);
                    qk = Mfma32<P, P>(kj, qi, qk);
                }
                const double Gi = row ? G[1] : G[0], Gc = col ? G[1] : G[0];
                const float beta = mine(row) ? (row ? gates[1].beta : gates[0].beta) : 0.f;
                F4 aA, dA, aP, aKK;
#pragma unroll
                for (int r = 0; r < 4; r++) {
                    const int j = 4 * g + r;
                    const double Gj = __shfl(Gc, j);
                    const float betaj = __shfl(beta, j);
                    const bool later = block == kAcross || j <= m, before = block == kAcross || j < m;
                    // Either way round, the later step minus the earlier one.
                    const float d = mine(row) && in(col, r) ? Exp2(later ? Gi - Gj : Gj - Gi) : 0.f;
                    aP[r] = later ? rule.scale * d * qk[r] : 0.f;
                    aKK[r] = before ? d * kk[r] : 0.f;
                    aA[r] = beta * aKK[r];
                    dA[r] = m < j ? betaj * d * kk[r] : 0.f;
                }
                const int to = m * kChunk + 4 * g;
                *reinterpret_cast<F4 *>(shared + At::kMixed + block * kBlock + to) = aP;
                *reinterpret_cast<F4 *>(shared + At::kProducts + block * kBlock + to) = aKK;
                if (block != kAcross)
                    *reinterpret_cast<F4 *>(shared + At::kInverse + block * kMatrix + to) = UnitLowerInverse(aA, dA, m, g);
            }
            __syncthreads();

            // ---- By columns: U, what the steps wrote, with its errors, from the memory before, and dU and dB from
            // the gradient of the memory after. The two chains of products go side by side.
            F4 U[2], error[2], dO[2], dB[2], wrong[2];
            {
                F4 seen[2], dU[2];
                seen[0] = seen[1] = dU[0] = dU[1] = F4{0, 0, 0, 0};
#pragma unroll
                for (int p = 0; p < KeyTiles / 2; p++) {
                    B8 kp[2][P], sp[kFloatPieces];
                    keyPair(keys, 0, p, kp[0]), keyPair(keys, 1, p, kp[1]);
                    if (!starts) {
                        Pair(start[2 * p], start[2 * p + 1], sp);
                        seen[0] = Mfma32<P, kFloatPieces>(kp[0], sp, seen[0]);
                        seen[1] = Mfma32<P, kFloatPieces>(kp[1], sp, seen[1]);
                    }
                    Pair(dS[2 * p], dS[2 * p + 1], sp);
                    dU[0] = Mfma32<P, kFloatPieces>(kp[0], sp, dU[0]);
                    dU[1] = Mfma32<P, kFloatPieces>(kp[1], sp, dU[1]);
                }
                B8 v[P], o[P];
                Pair<T>(Masked(values[0], mine(0)), Masked(values[1], mine(1)), v);
                Pair<T>(valueTile(outputs, 0, wave), valueTile(outputs, 1, wave), o);
                F4 beta[2];
#pragma unroll
                for (int tile = 0; tile < 2; tile++) {
                    const F4 value = Turn<P>(v, eyes.half[tile]);
                    dO[tile] = Turn<P>(o, eyes.half[tile]);
                    const F4 whole = *reinterpret_cast<const F4 *>(wholes + kChunk * tile + 4 * g);
                    beta[tile] = *reinterpret_cast<const F4 *>(betas + kChunk * tile + 4 * g);
#pragma unroll
                    for (int r = 0; r < 4; r++) error[tile][r] = fmaf(-whole[r], seen[tile][r], value[r]);
                    U[tile] = beta[tile] * error[tile];
                    dU[tile] *= *reinterpret_cast<const F4 *>(afters + kChunk * tile + 4 * g);
                }
                const auto mixed = [&](int block) { return ColumnOrder(shared + At::kMixed + block * kBlock, m, g); };
                const auto inverse = [&](int block) { return shared + At::kInverse + block * kMatrix; };
                const float *across = shared + At::kProducts + kAcross * kBlock;
                dU[1] = Product(mixed(kSecond), dO[1], dU[1]);
                U[0] = Product(RowOrder(inverse(kFirst), m, g), U[0]);
                dU[0] = Product(mixed(kFirst), dO[0], dU[0]);
                dB[1] = Product(ColumnOrder(inverse(kSecond), m, g), dU[1]);
                U[1] = Product(RowOrder(across, m, g) * -betas[kChunk + m], U[0], U[1]);
                dU[0] = Product(mixed(kAcross), dO[1], dU[0]);
                U[1] = Product(RowOrder(inverse(kSecond), m, g), U[1]);
                dU[0] = Product(ColumnOrder(across, m, g) * -beta[1], dB[1], dU[0]);
                dB[0] = Product(ColumnOrder(inverse(kFirst), m, g), dU[0]);
            }
            float held = 0;
            if (!starts) {
#pragma unroll
                for (int t = 0; t < KeyTiles; t++)
#pragma unroll
                    for (int r = 0; r < 4; r++) held = fmaf(dS[t][r], start[t][r], held);
            }
            held = WaveSum(held);
#pragma unroll
            for (int tile = 0; tile < 2; tile++)
#pragma unroll
                for (int r = 0; r < 4; r++) wrong[tile][r] = RowSum(dB[tile][r] * error[tile][r]);
            if (m == 0) {
                *reinterpret_cast<F4 *>(dots + (wave * 4 + 0) * kSegment + 4 * g) = wrong[0];
                *reinterpret_cast<F4 *>(dots + (wave * 4 + 0) * kSegment + kChunk + 4 * g) = wrong[1];
            }
            if (lane == 0) dots[(wave * 4 + 3) * kSegment] = held;
            // In row order for the products over columns.
            {
                Four lo[kFloatPieces], hi[kFloatPieces];
                B8 x[kFloatPieces];
                const auto put = [&](uint16_t *rows) {
                    Eights<kFloatPieces>(lo, hi, x);
#pragma unroll
                    for (int tile = 0; tile < 2; tile++) {
                        Four turned[kFloatPieces];
                        Turn<kFloatPieces>(x, eyes.half[tile], turned);
#pragma unroll
                        for (int i = 0; i < kFloatPieces; i++)
                            *reinterpret_cast<Four *>(rows + (i * kSegment + kChunk * tile + m) * rs + column4) = turned[i];
                    }
                };
                Split(U[0], lo), Split(U[1], hi);
                put(sharedU);
                Split(dB[0], lo), Split(dB[1], hi);
                put(sharedB);
                T *to = static_cast<T *>(Argument<Args>().rule.d_value) + (((long long)b * time + s0) * rule.heads + h) * dv + base;
#pragma unroll
                for (int tile = 0; tile < 2; tile++) {
                    const F4 rows = Turn<kFloatPieces>(x, eyes.half[tile]);
                    Pack<T, 4> v;
#pragma unroll
                    for (int r = 0; r < 4; r++) v.x[r] = As<T>(betas[kChunk * tile + m] * rows[r]);
                    const uint32_t at = ((kChunk * tile + m) * rule.heads * dv + column4) * sizeof(T);
                    Store<4, Whole>(Lane(to, at), v, mine(tile) ? dv - base - column4 : 0);
                }
            }
#pragma unroll
            for (int t = 0; t < KeyTiles; t++)
#pragma unroll
                for (int r = 0; r < 4; r++) memory[(16 * t + 4 * g + r) * ms + 16 * wave + m] = dS[t][r];
            __syncthreads();

            const auto rowPieces = [&](const uint16_t *rows, int tile, int x, B8(&to)[kFloatPieces]) {
#pragma unroll
                for (int i = 0; i < kFloatPieces; i++) {
                    const uint16_t *from = rows + (i * kSegment + kChunk * tile + m) * rs + 32 * x + 4 * g;
                    to[i] = Eight(*reinterpret_cast<const Four *>(from), *reinterpret_cast<const Four *>(from + 16));
                }
            };
            const auto outputPieces = [&](int tile, int x, B8(&to)[P]) {
                Pair<T>(valueTile(outputs, tile, 2 * x), valueTile(outputs, tile, 2 * x + 1), to);
            };
            const auto memoryPieces = [&](int t, int x, B8(&to)[kFloatPieces]) {
                const float *from = memory + (16 * t + m) * ms + 32 * x + 4 * g;
                Pair(*reinterpret_cast<const F4 *>(from), *reinterpret_cast<const F4 *>(from + 16), to);
            };
            const auto putPieces = [&](uint16_t *pieces, F4 x) {
                Four p[kFloatPieces];
                Split(x, p);
#pragma unroll
                for (int i = 0; i < kFloatPieces; i++)
                    *reinterpret_cast<Four *>(pieces + i * kMatrix + m * kChunk + 4 * g) = p[i];
            };
            const auto getPieces = [&](const uint16_t *pieces, Four(&p)[kFloatPieces]) {
#pragma unroll
                for (int i = 0; i < kFloatPieces; i++)
                    p[i] = *reinterpret_cast<const Four *>(pieces + i * kMatrix + m * kChunk + 4 * g);
            };
            const auto getM = [&](int block, Four(&p)[kFloatPieces]) { getPieces(sharedM + block * 2 * kPieceMatrix, p); };
            const auto getN = [&](int block, Four(&p)[kFloatPieces]) { getPieces(sharedN + block * 2 * kBlock, p); };
            // ---- The matrices' gradients.
#pragma unroll 1
            for (int block = wave; block < 3; block += Waves) {
                const int row = block == kFirst ? 0 : 1, col = block == kSecond ? 1 : 0;
                F4 gP = {0, 0, 0, 0}, gA = {0, 0, 0, 0};
#pragma unroll
                for (int x = 0; x < kPairs; x++) {
                    B8 uw[kFloatPieces], bw[kFloatPieces], out[P];
                    rowPieces(sharedU, col, x, uw), rowPieces(sharedB, row, x, bw), outputPieces(row, x, out);
                    gP = Mfma32<kFloatPieces, P>(uw, out, gP);
                    gA = Mfma32<kFloatPieces, kFloatPieces>(uw, bw, gA);
                }
                const F4 aP = RowOrder(shared + At::kMixed + block * kBlock, m, g);
                const F4 aKK = RowOrder(shared + At::kProducts + block * kBlock, m, g);
                const float beta = betas[kChunk * row + m];
                const double Gi = row ? G[1] : G[0];
                F4 M, N, E;
                float betaSum = 0;
#pragma unroll
                for (int r = 0; r < 4; r++) {
                    const int j = 4 * g + r;
                    const bool both = mine(row) && in(col, r), later = block == kAcross || j <= m;
                    const float d = both && later ? Exp2(Gi - reach[kChunk * col + j]) : 0.f;
                    M[r] = rule.scale * d * gP[r];
                    N[r] = block == kAcross || j < m ? -beta * d * gA[r] : 0.f;
                    const float part = both ? -gA[r] * aKK[r] : 0.f;
                    betaSum += part;
                    E[r] = (both ? gP[r] * aP[r] : 0.f) + beta * part;
                }
                putPieces(sharedM + block * 2 * kPieceMatrix, M);
                if (block != kAcross) {
                    Four lo[kFloatPieces];
                    B8 x[kFloatPieces];
                    Split(N, lo);
                    Eights<kFloatPieces>(lo, lo, x);
                    N += Turn<kFloatPieces>(x, eyes.half[0]);
                }
                Forget();
                putPieces(sharedN + block * 2 * kBlock, N);
                betaSum += __shfl_xor(betaSum, 16);
                betaSum += __shfl_xor(betaSum, 32);
                if (g == 0) sums[block * kChunk + m] = betaSum;
                // What of E crosses each step: from before it to it or after, within the block; and the block
                // across by rows and by columns.
                float across = 0;
#pragma unroll
                for (int r = 0; r < 4; r++) {
                    const float from = block == kAcross ? E[r] : RowFrom(E[r]);
                    across += block == kAcross || 4 * g + r < m ? from : 0.f;
                }
                across += __shfl_xor(across, 16);
                across += __shfl_xor(across, 32);
                if (g == 0) sums[(3 + block) * kChunk + m] = across;
                if (block == kAcross) {
                    F4 columns;
#pragma unroll
                    for (int r = 0; r < 4; r++) columns[r] = RowSum(E[r]);
                    if (m == 0) *reinterpret_cast<F4 *>(sums + 6 * kChunk + 4 * g) = columns;
                }
            }
            // ---- dS U by tiles of keys, kept in registers until the memory is in dS's place.
            constexpr int kMine = (KeyTiles + Waves - 1) / Waves;
            F4 fromLater[kMine][2];
#pragma unroll
            for (int i = 0; i < kMine; i++) {
                const int t = wave + i * Waves;
                fromLater[i][0] = fromLater[i][1] = F4{0, 0, 0, 0};
                if (t < KeyTiles) {
#pragma unroll
                    for (int x = 0; x < kPairs; x++) {
                        B8 sp[kFloatPieces];
                        memoryPieces(t, x, sp);
#pragma unroll
                        for (int tile = 0; tile < 2; tile++) {
                            B8 uw[kFloatPieces];
                            rowPieces(sharedU, tile, x, uw);
                            fromLater[i][tile] = Mfma32<kFloatPieces, kFloatPieces>(uw, sp, fromLater[i][tile]);
                        }
                    }
                }
            }
            __syncthreads();
            if (!starts) {
#pragma unroll
                for (int t = 0; t < KeyTiles; t++)
#pragma unroll
                    for (int r = 0; r < 4; r++) memory[(16 * t + 4 * g + r) * ms + 16 * wave + m] = start[t][r];
            }

            // ---- The gradient of the memory before this part, by columns.
            const float kept = wholes[high - 1];
            if (starts) {
#pragma unroll
                for (int t = 0; t < KeyTiles; t++) dS[t] = F4{0, 0, 0, 0};
            } else {
                B8 op[kFloatPieces], bp[kFloatPieces];
                {
                    F4 x[2], y[2];
#pragma unroll
                    for (int tile = 0; tile < 2; tile++) {
                        const F4 whole = *reinterpret_cast<const F4 *>(wholes + kChunk * tile + 4 * g);
                        const F4 beta = *reinterpret_cast<const F4 *>(betas + kChunk * tile + 4 * g);
                        x[tile] = rule.scale * whole * dO[tile];
                        y[tile] = -beta * whole * dB[tile];
                    }
                    Pair(x[0], x[1], op), Pair(y[0], y[1], bp);
                }
#pragma unroll
                for (int p = 0; p < KeyTiles / 2; p++) {
                    B8 x0[P], x1[P], y0[P], y1[P];
                    keyPair(queries, 0, p, x0), keyPair(queries, 1, p, x1);
                    keyPair(keys, 0, p, y0), keyPair(keys, 1, p, y1);
#pragma unroll
                    for (int half = 0; half < 2; half++) {
                        Four lo[P], hi[P];
                        B8 turned[P];
                        F4 s = dS[2 * p + half] * kept;
                        Turn<P>(x0, eyes.half[half], lo), Turn<P>(x1, eyes.half[half], hi);
                        Eights<P>(lo, hi, turned);
                        s = Mfma32<P, kFloatPieces>(turned, op, s);
                        Turn<P>(y0, eyes.half[half], lo), Turn<P>(y1, eyes.half[half], hi);
                        Eights<P>(lo, hi, turned);
                        dS[2 * p + half] = Mfma32<P, kFloatPieces>(turned, bp, s);
                    }
                }
            }
            __syncthreads();

            // ---- The keys' and queries' gradients.
            F4 e[2], f[2];
            e[0] = e[1] = f[0] = f[1] = F4{0, 0, 0, 0};
#pragma unroll
            for (int i = 0; i < kMine; i++) {
                const int t = wave + i * Waves;
                if (t >= KeyTiles) continue;
                F4 dQ[2], dK[2], y[2];
                dQ[0] = dQ[1] = y[0] = y[1] = F4{0, 0, 0, 0};
                if (!starts) {
#pragma unroll
                    for (int x = 0; x < kPairs; x++) {
                        B8 sp[kFloatPieces];
                        memoryPieces(t, x, sp);
#pragma unroll
                        for (int tile = 0; tile < 2; tile++) {
                            B8 bw[kFloatPieces], out[P];
                            outputPieces(tile, x, out);
                            dQ[tile] = Mfma32<P, kFloatPieces>(out, sp, dQ[tile]);
                            rowPieces(sharedB, tile, x, bw);
                            y[tile] = Mfma32<kFloatPieces, kFloatPieces>(bw, sp, y[tile]);
                        }
                    }
                }
                // This tile's keys and queries, both tiles of steps side by side, and in column order.
                const auto tilePair = [&](const T *rows, B8(&x)[P]) {
                    const T *from = rows + m * ks + 16 * t + 4 * g;
                    Pair<T>(Masked(*reinterpret_cast<const Pack<T, 4> *>(from), mine(0)),
                            Masked(*reinterpret_cast<const Pack<T, 4> *>(from + kChunk * ks), mine(1)), x);
                };
                B8 kx[P], qx[P], kAll[P], qAll[P];
                Four k[2][P], q[2][P];
                tilePair(keys, kx), tilePair(queries, qx);
#pragma unroll
                for (int tile = 0; tile < 2; tile++) {
                    const F4 whole = *reinterpret_cast<const F4 *>(wholes + kChunk * tile + 4 * g);
                    const F4 beta = *reinterpret_cast<const F4 *>(betas + kChunk * tile + 4 * g);
                    const F4 kf = Turn<P>(kx, eyes.half[tile]), qf = Turn<P>(qx, eyes.half[tile]);
                    Turn<P>(kx, eyes.half[tile], k[tile]), Turn<P>(qx, eyes.half[tile], q[tile]);
                    dK[tile] = fromLater[i][tile] * *reinterpret_cast<const F4 *>(afters + kChunk * tile + 4 * g);
                    f[tile] += dK[tile] * kf;
                    y[tile] *= -beta * whole;
                    dQ[tile] *= rule.scale * whole;
                    e[tile] += qf * dQ[tile] + kf * y[tile];
                    dK[tile] += y[tile];
                }
                Eights<P>(k[0], k[1], kAll), Eights<P>(q[0], q[1], qAll);
                // dq1 = M11 k1, dq2 = M21 k1 + M22 k2; dk1 = M11' q1 + M21' q2 + N11 k1 + N21' k2,
                // dk2 = M22' q2 + N21 k1 + N22 k2, N11 and N22 with their transposes in them.
                Four m11[kFloatPieces], m21[kFloatPieces], m22[kFloatPieces];
                Four lo[kFloatPieces], hi[kFloatPieces];
                B8 wide[kFloatPieces], turn[kFloatPieces];
                getM(kFirst, m11), getM(kAcross, m21), getM(kSecond, m22);
                dQ[0] = Mfma16(m11, k[0], dQ[0]);
                Eights<kFloatPieces>(m21, m22, wide);
                dQ[1] = Mfma32<kFloatPieces, P>(wide, kAll, dQ[1]);
                Eights<kFloatPieces>(m11, m21, turn);
                Turn<kFloatPieces>(turn, eyes.half[0], lo), Turn<kFloatPieces>(turn, eyes.half[1], hi);
                Eights<kFloatPieces>(lo, hi, wide);
                dK[0] = Mfma32<kFloatPieces, P>(wide, qAll, dK[0]);
                Eights<kFloatPieces>(m22, m22, turn);
                Turn<kFloatPieces>(turn, eyes.half[0], lo);
                dK[1] = Mfma16(lo, q[1], dK[1]);
                getN(kFirst, m11), getN(kAcross, m21), getN(kSecond, m22);
                Eights<kFloatPieces>(m21, m22, wide);
                dK[1] = Mfma32<kFloatPieces, P>(wide, kAll, dK[1]);
                Eights<kFloatPieces>(m21, m21, turn);
                Turn<kFloatPieces>(turn, eyes.half[0], hi);
                Eights<kFloatPieces>(m11, hi, wide);
                dK[0] = Mfma32<kFloatPieces, P>(wide, kAll, dK[0]);

                const Args now = Argument<Args>();
                const int each = now.parted ? rule.heads * now.slices * dk : rule.key_heads * dk;
                const long long to = ((long long)b * time + s0) * each + (now.parted ? h * now.slices + slice : kh) * dk + 16 * t;
#pragma unroll
                for (int tile = 0; tile < 2; tile++)
#pragma unroll
                    for (int r = 0; r < 4; r++) {
                        if (!in(tile, r) || 16 * t + m >= dk) continue;
                        const uint32_t at = 4 * g * each + m;
                        const long long row = to + (kChunk * tile + r) * (long long)each;
                        if (now.parted) {
                            *Lane(static_cast<float *>(now.dQuery) + row, at * sizeof(float)) = dQ[tile][r];
                            *Lane(static_cast<float *>(now.dKey) + row, at * sizeof(float)) = dK[tile][r];
                        } else {
                            *Lane(static_cast<T *>(now.dQuery) + row, at * sizeof(T)) = As<T>(dQ[tile][r]);
                            *Lane(static_cast<T *>(now.dKey) + row, at * sizeof(T)) = As<T>(dK[tile][r]);
                        }
                    }
            }
#pragma unroll
            for (int tile = 0; tile < 2; tile++) {
                F4 eSum, fSum;
#pragma unroll
                for (int r = 0; r < 4; r++) eSum[r] = RowSum(e[tile][r]), fSum[r] = RowSum(f[tile][r]);
                if (m == 0) {
                    *reinterpret_cast<F4 *>(dots + (wave * 4 + 1) * kSegment + kChunk * tile + 4 * g) = eSum;
                    *reinterpret_cast<F4 *>(dots + (wave * 4 + 2) * kSegment + kChunk * tile + 4 * g) = fSum;
                }
            }
            __syncthreads();

            // ---- The gates' gradients, a lane for each step.
            if (wave == Waves - 1) {
                float eAll[2] = {0, 0}, fAll[2] = {0, 0}, bAll[2] = {0, 0}, heldAll = 0;
#pragma unroll
                for (int w = 0; w < Waves; w++) {
#pragma unroll
                    for (int tile = 0; tile < 2; tile++) {
                        bAll[tile] += dots[(w * 4 + 0) * kSegment + kChunk * tile + m];
                        eAll[tile] += dots[(w * 4 + 1) * kSegment + kChunk * tile + m];
                        fAll[tile] += dots[(w * 4 + 2) * kSegment + kChunk * tile + m];
                    }
                    heldAll += dots[(w * 4 + 3) * kSegment];
                }
                const float through = starts ? 0.f : kept * heldAll;
                const auto before = [](float x) { return Dpp<kRowShiftRight + 1>(RowUpTo(x)); };
                float decay[2];
                decay[0] = RowFrom(eAll[0]) + RowSum(eAll[1]) + sums[3 * kChunk + m] + before(sums[6 * kChunk + m]) + before(fAll[0]);
                decay[1] = RowFrom(eAll[1]) + RowFrom(sums[5 * kChunk + m]) + sums[4 * kChunk + m] + RowSum(fAll[0]) + before(fAll[1]);
                bAll[0] += sums[m];
                bAll[1] += sums[kChunk + m] + sums[2 * kChunk + m];
                const Args now = Argument<Args>();
#pragma unroll
                for (int tile = 0; tile < 2; tile++)
                    if (mine(tile) && g == 0) {
                        const long long to = (((long long)b * time + s0 + kChunk * tile + m) * rule.heads + h) * now.slices + slice;
                        Global(now.dDecay)[to] = starts && kChunk * tile + m == low ? 0.f : decay[tile] + through;
                        Global(now.dBeta)[to] = bAll[tile];
                    }
            }
            // What the next part puts down first (betas, matrices) is still read here only by this wavefront
            // (sums, dots), which the next barrier waits for.
        }
    }
    if (rule.d_state) {
        const int rows = dk - 4 * g;
        float *to = static_cast<float *>(rule.d_state) + (long long)head * dk * dv;
        const uint32_t at = (4 * g * dv + column) * sizeof(float);
#pragma unroll
        for (int t = 0; t < KeyTiles; t++)
#pragma unroll
            for (int r = 0; r < 4; r++)
                if (16 * t + r < rows && column < dv) *Lane(to + (16 * t + r) * dv, at) = dS[t][r];
    }
}

// Gradients that several heads or slices share: [row][parts][size] summed over the parts, in their order.
template <class T>
__global__ __launch_bounds__(256) void PartsKernel(const float *parts, T *out, int group, int size, long long count) {
    for (long long i = blockIdx.x * 256ll + threadIdx.x; i < count; i += gridDim.x * 256ll) {
        const long long row = i / size;
        const float *p = parts + row * group * size + (i - row * size);
        float sum = 0;
        for (int n = 0; n < group; n++) sum += p[n * size];
        out[i] = As<T>(sum);
    }
}
template <class T>
void LaunchParts(const float *parts, void *out, int group, int size, long long rows, hipStream_t stream) {
    const long long count = rows * size;
    if (count == 0) return;
    const unsigned blocks = (unsigned)(count < 256ll * 8192 ? (count + 255) / 256 : 8192);
    hipLaunchKernelGGL(PartsKernel<T>, dim3(blocks), dim3(256), 0, stream, parts, static_cast<T *>(out), group, size, count);
}

// Wavefronts of a workgroup, 16 columns each: all of a head's columns, where LDS holds them. Wide workgroups
// find the triangular matrices once and leave no parts to add up: 2,048 heads of 64 steps take, with all 128
// columns against 64 and 64, 400 us against 788 (bfloat16, keys of 128), 302 against 324 (keys of 64), 391
// against 667 (float32), and with 96 columns 279 against 319. Sixteen heads of 256 steps, which leave most of
// the chip idle either way, take 170 us against 166. Floats with keys over 96 do not fit.
int WavesOf(const Rule &r) {
    if (r.value_size <= 32) return 2;
    if (r.value_size <= 64) return 4;
    if (r.value_size <= 96) return 6;
    return r.type == 0 && r.key_size > 96 ? 4 : 8;
}
int SlicesOf(const Rule &r) { return (r.value_size + 16 * WavesOf(r) - 1) / (16 * WavesOf(r)); }
// Floats of the parts of the keys' and queries' gradients, and of the gates'; 0 where there are none.
long long KeyParts(const Rule &r) {
    const bool parted = r.heads * SlicesOf(r) != r.key_heads;
    return parted ? (long long)r.batch * r.time * r.heads * SlicesOf(r) * r.key_size : 0;
}
long long GateParts(const Rule &r) { return SlicesOf(r) > 1 ? (long long)r.batch * r.time * r.heads * SlicesOf(r) : 0; }

template <class T, int KeyTiles>
bool LaunchBackward(const Rule &r, hipStream_t stream) {
    const int slices = SlicesOf(r);
    const long long keyParts = KeyParts(r), gateParts = GateParts(r), steps = (long long)r.batch * r.time;
    float *parts = static_cast<float *>(r.workspace), *gateSums = parts + 2 * keyParts;
    BackwardArgs<T> a{r,
                      ViewOf<const T>(r.query, r.query_strides, r.key_size),
                      ViewOf<const T>(r.key, r.key_strides, r.key_size),
                      ViewOf<const T>(r.value, r.value_strides, r.value_size),
                      ViewOf<const T>(r.d_output, r.d_output_strides, r.value_size),
                      GatesOf(r),
                      keyParts ? parts : r.d_query,
                      keyParts ? parts + keyParts : r.d_key,
                      gateParts ? gateSums : static_cast<float *>(r.d_decay),
                      gateParts ? gateSums + gateParts : static_cast<float *>(r.d_beta),
                      slices,
                      keyParts != 0};
    const bool whole = a.query.whole && a.key.whole && a.value.whole && a.dOutput.whole && Aligned(4 * sizeof(T), r.d_value);
    const auto launch = [&](auto wide, auto packed) {
        constexpr int Waves = decltype(wide)::value;
        const auto kernel = BackwardKernel<T, KeyTiles, Waves, decltype(packed)::value>;
        constexpr int bytes = BackwardShared<KeyTiles, Waves, sizeof(T)>::kFloats * sizeof(float);
        static_assert(bytes <= 160 * 1024, "a head's steps fit a compute unit's LDS");
        if (hipFuncSetAttribute(reinterpret_cast<const void *>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, bytes) !=
            hipSuccess)
            return false;
        hipLaunchKernelGGL(kernel, dim3((unsigned)(r.batch * (long long)r.heads * slices)), dim3(64 * Waves), bytes, stream, a);
        return true;
    };
    const auto width = [&](auto packed) {
        switch (WavesOf(r)) {
            case 2: return launch(std::integral_constant<int, 2>(), packed);
            case 4: return launch(std::integral_constant<int, 4>(), packed);
            case 6: return launch(std::integral_constant<int, 6>(), packed);
            default: return launch(std::integral_constant<int, (sizeof(T) == 4 && KeyTiles > 6 ? 4 : 8)>(), packed);
        }
    };
    const bool set = whole ? width(std::true_type()) : width(std::false_type());
    if (!set) return false;
    if (keyParts) {
        const int group = r.heads / r.key_heads * slices;
        LaunchParts<T>(parts, r.d_query, group, r.key_size, steps * r.key_heads, stream);
        LaunchParts<T>(parts + keyParts, r.d_key, group, r.key_size, steps * r.key_heads, stream);
    }
    if (gateParts) {
        LaunchParts<float>(gateSums, r.d_decay, slices, 1, steps * r.heads, stream);
        LaunchParts<float>(gateSums + gateParts, r.d_beta, slices, 1, steps * r.heads, stream);
    }
    return true;
}

}  // namespace
}  // namespace layers

using namespace layers;

extern "C" __attribute__((visibility("default"))) unsigned long long cuju_delta_rule_workspace(const struct cuju_delta_rule *rule) {
    if (!Fits(rule)) return 0;
    return 2 * (KeyParts(*rule) + GateParts(*rule)) * sizeof(float);
}

extern "C" __attribute__((visibility("default"))) int cuju_delta_rule_backward(const struct cuju_delta_rule *rule, void *stream) {
    if (!Fits(rule)) return -1;
    const Rule &r = *rule;
    if (r.batch == 0) return 0;
    if (r.time > 0 && (!r.query || !r.key || !r.value || !r.decay || !r.beta || !r.d_output || !r.d_query || !r.d_key ||
                       !r.d_value || !r.d_decay || !r.d_beta))
        return Failed("expected inputs and their gradients");
    if (KeyParts(r) + GateParts(r) && !r.workspace) return Failed("expected a workspace");
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
