// What the kernels of memories that are played over many steps share: chunks of steps, decays and views of
// tensors with strides.
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

template <int P>
__device__ __forceinline__ void Eights(const Four (&lo)[P], const Four (&hi)[P], B8 (&x)[P]) {
#pragma unroll
    for (int i = 0; i < P; i++) x[i] = Eight(lo[i], hi[i]);
}

}  // namespace layers
