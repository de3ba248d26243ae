// The arguments of the gated delta rule's kernels, and what the forward and backward kernels share:
// how a chunk of 16 steps is cut at resets, its decays, and its triangular inverse.
#pragma once
#include "../../../include/cuju_amd.h"
#include "common.h"

namespace layers {

constexpr int kChunk = 16;            // steps of a chunk: one tile of the matrix instruction
// Steps between two checkpoints of the memory, which the forward pass keeps for the backward pass.
constexpr int kSegment = 2 * kChunk;
constexpr int kMaxKey = 128, kMaxValue = 128;
// A step whose log decay is below this keeps nothing: the factor is 0 in 32 bits, denormals included.
// Such a step is a reset.
constexpr float kNothingKept = -104.f;

using Rule = cuju_delta_rule;

// One element type's view of a tensor with strides [batch][time][head].
template <class T>
struct View {
    T *p;
    long long batch, time, head;
    bool whole;  // packs of four are aligned, and the last axis is made of them
    __device__ __forceinline__ T *At(int b, int t, int h) const { return Global(p) + b * batch + t * time + h * head; }
};

inline bool Aligned(size_t bytes, const void *p) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }
template <class T>
View<T> ViewOf(const void *p, const long long *strides, int size) {
    View<T> v{static_cast<T *>(const_cast<void *>(p)), strides[0], strides[1], strides[2], false};
    const auto four = [](long long x) { return x % 4 == 0; };
    v.whole = four(strides[0]) && four(strides[1]) && four(strides[2]) && four(size) &&
              Aligned(4 * sizeof(T), p);
    return v;
}

struct Gates {
    const float *decay, *beta;
    const unsigned char *resets;  // or null
    long long decayStrides[3], betaStrides[3], resetStrides[2];
};
inline Gates GatesOf(const Rule &r) {
    Gates g{static_cast<const float *>(r.decay), static_cast<const float *>(r.beta), r.resets, {}, {}, {}};
    for (int i = 0; i < 3; i++) g.decayStrides[i] = r.decay_strides[i], g.betaStrides[i] = r.beta_strides[i];
    for (int i = 0; i < 2; i++) g.resetStrides[i] = r.reset_strides[i];
    return g;
}

// A step's gates, one lane of a row of 16 for each step of a chunk; past the end of time a step that
// keeps everything and writes nothing. What is loaded is looked at only when it is used, so that a load
// ahead of time waits for nothing.
struct StepGates {
    float decay, beta;
    unsigned char cleared;
    __device__ __forceinline__ bool Reset() const { return cleared | (decay < kNothingKept); }
};
__device__ __forceinline__ StepGates LoadGates(const Gates &g, int b, int t, int time, int h) {
    StepGates s{0.f, 0.f, 0};
    if (t < time) {
        s.decay = Global(g.decay)[b * g.decayStrides[0] + t * g.decayStrides[1] + h * g.decayStrides[2]];
        s.beta = Global(g.beta)[b * g.betaStrides[0] + t * g.betaStrides[1] + h * g.betaStrides[2]];
        if (g.resets) s.cleared = Global(g.resets)[b * g.resetStrides[0] + t * g.resetStrides[1]];
    }
    return s;
}

// Log decays are summed in 64 bits (a difference of two long sums keeps its precision) and in base 2,
// the base of the hardware's exponential.
constexpr double kLog2E = 1.4426950408889634;
__device__ __forceinline__ float Exp2(double x) { return __builtin_amdgcn_exp2f((float)x); }

// The inverse of I + A for the strictly lower A of a chunk, in row order, from A in both orders. Blocks of 4 on the
// diagonal are inverted by substitution between the four lanes of a quad (G below); with L the part
// of A below those blocks, I + A = G^-1 (I + N), N = G L, and N^4 = 0, so that
// (I + A)^-1 = (I - N)(I + N N) G. Powers of the whole A would cancel in the sixth digit where keys
// repeat themselves, as they do from one step of a match to the next; the powers of N stay small.
__device__ __forceinline__ F4 UnitLowerInverse(F4 aA, F4 dA, int m, int g) {
    const bool diagonal = g == m / 4;
    F4 aG, dG, dL;
    // Row order: lane m holds row m; row s of a block is final after s steps and is taken off the later ones.
#pragma unroll
    for (int r = 0; r < 4; r++) aG[r] = (m & 3) == r ? 1.f : 0.f;
    const auto takeRow = [&](auto lane) {
        constexpr int s = decltype(lane)::value;
        const float f = aA[s];
#pragma unroll
        for (int r = 0; r <= s; r++) aG[r] -= f * QuadLane<s>(aG[r]);
    };
    takeRow(std::integral_constant<int, 0>());
    takeRow(std::integral_constant<int, 1>());
    takeRow(std::integral_constant<int, 2>());
    // Column order: a lane substitutes down its own column, with A's entries from the quad's lanes.
#pragma unroll
    for (int r = 0; r < 4; r++) dG[r] = (m & 3) == r ? 1.f : 0.f;
    dG[1] -= QuadLane<0>(dA[1]) * dG[0];
    dG[2] -= QuadLane<0>(dA[2]) * dG[0];
    dG[2] -= QuadLane<1>(dA[2]) * dG[1];
    dG[3] -= QuadLane<0>(dA[3]) * dG[0];
    dG[3] -= QuadLane<1>(dA[3]) * dG[1];
    dG[3] -= QuadLane<2>(dA[3]) * dG[2];
#pragma unroll
    for (int r = 0; r < 4; r++) {
        aG[r] = diagonal ? aG[r] : 0.f;
        dG[r] = diagonal ? dG[r] : 0.f;
        dL[r] = g > m / 4 ? dA[r] : 0.f;
    }
    F4 aN = Product(dL, aG);
    const F4 dN = Product(aG, dL);
    F4 aY = Product(dN, aN);
    F4 one;
#pragma unroll
    for (int r = 0; r < 4; r++) one[r] = m == 4 * g + r ? 1.f : 0.f;
    aY += one;
    aN = one - aN;
    const F4 dY = Product(aY, dG);
    return Product(dY, aN);
}

template <class T>
__device__ __forceinline__ Pack<T, 4> Masked(const Pack<T, 4> &x, bool keep) {
    struct Words {
        uint32_t x[sizeof(T)];
    };
    Words r = __builtin_bit_cast(Words, x);
#pragma unroll
    for (int i = 0; i < (int)sizeof(T); i++) r.x[i] = keep ? r.x[i] : 0u;
    return __builtin_bit_cast(Pack<T, 4>, r);
}

// The identity as a right operand for the first or the second half of a pair's eight values: a product
// with it turns that half from row order into column order, exactly.
struct Eyes {
    B8 half[2];
};
__device__ __forceinline__ Eyes EyesOf(int m, int g) {
    Four eye;
#pragma unroll
    for (int j = 0; j < 2; j++)
        eye.x[j] = (4 * g + 2 * j == m ? 0x3f80u : 0u) | (4 * g + 2 * j + 1 == m ? 0x3f800000u : 0u);
    return Eyes{{Eight(eye, Four{}), Eight(Four{}, eye)}};
}
// As floats.
template <int P>
__device__ __forceinline__ F4 Turn(const B8 (&x)[P], B8 eye) {
    F4 sum = {0, 0, 0, 0};
#pragma unroll
    for (int i = P - 1; i >= 0; i--) sum = Mfma32(x[i], eye, sum);
    return sum;
}
// Piece by piece.
template <int P>
__device__ __forceinline__ void Turn(const B8 (&x)[P], B8 eye, Four (&turned)[P]) {
#pragma unroll
    for (int i = 0; i < P; i++) {
        const F4 t = Mfma32(x[i], eye, F4{0, 0, 0, 0});
        const float f[4] = {t[0], t[1], t[2], t[3]};
        Four whole[1];
        Split<1>(f, whole);
        turned[i] = whole[0];
    }
}
template <int P>
__device__ __forceinline__ void Eights(const Four (&lo)[P], const Four (&hi)[P], B8 (&x)[P]) {
#pragma unroll
    for (int i = 0; i < P; i++) x[i] = Eight(lo[i], hi[i]);
}
// The pieces of a lane's eight keys of a pair of tiles.
template <class T>
__device__ __forceinline__ void Pair(const Pack<T, 4> &lo, const Pack<T, 4> &hi, B8 (&x)[kPieces<T>]) {
    Four a[kPieces<T>], b[kPieces<T>];
    Split<T>(lo, a), Split<T>(hi, b);
#pragma unroll
    for (int i = 0; i < kPieces<T>; i++) x[i] = Eight(a[i], b[i]);
}
__device__ __forceinline__ void Pair(F4 lo, F4 hi, B8 (&x)[kFloatPieces]) {
    Four a[kFloatPieces], b[kFloatPieces];
    Split(lo, a), Split(hi, b);
#pragma unroll
    for (int i = 0; i < kFloatPieces; i++) x[i] = Eight(a[i], b[i]);
}

// Whether a call's arguments fit the kernels; the failure is kept otherwise.
inline bool Fits(const Rule *r) {
    if (!r || r->type < 0 || r->type > 2) return Failed("expected a delta rule of the type 0, 1 or 2"), false;
    if (r->batch < 0 || r->time < 0 || r->heads < 1 || r->key_heads < 1 || r->heads % r->key_heads)
        return Failed("expected heads that are a multiple of the key heads"), false;
    // Steps are counted by ints, and a lane's place among the 32 steps of a segment is 32 bits of bytes.
    if (r->time >= (1 << 30) || r->heads >= (1 << 16)) return Failed("expected fewer than 2^30 steps and 2^16 heads"), false;
    // A grid has fewer than 2^32 threads: at most 512 a head.
    if (r->batch * (long long)r->heads >= (1ll << 23)) return Failed("expected fewer than 2^23 heads in the batch"), false;
    if (r->key_size < 1 || r->key_size > kMaxKey || r->value_size < 1 || r->value_size > kMaxValue)
        return Failed("expected key and value sizes from 1 to 128"), false;
    return true;
}

}  // namespace layers
