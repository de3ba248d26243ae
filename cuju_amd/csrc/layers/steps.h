// What the kernels of memories that are played over many steps share: chunks of steps, decays, views of
// tensors with strides, and the pieces of a chunk's inputs as operands of the matrix instruction.
#pragma once
#include "common.h"

namespace layers {

constexpr int kChunk = 16;            // steps of a chunk: one tile of the matrix instruction
constexpr int kMaxKey = 128, kMaxValue = 128;
// A step whose log decay is below this keeps nothing: the factor is 0 in 32 bits, denormals included.
// Such a step is a reset.
constexpr float kNothingKept = -104.f;

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

// Log decays are summed in 64 bits (a difference of two long sums keeps its precision) and in base 2,
// the base of the hardware's exponential.
constexpr double kLog2E = 1.4426950408889634;
__device__ __forceinline__ float Exp2(double x) { return __builtin_amdgcn_exp2f((float)x); }

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

}  // namespace layers
