// What the policy operators' kernels share: element types, loads and stores of four elements, the
// 16x16x4 matrix product in 32 bits with the two ways a 16x16 matrix lies over a wavefront, and sums
// over a row of 16 lanes.
#pragma once
#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>
#include <hip/hip_runtime.h>

#include <cstdint>
#include <string>
#include <type_traits>

namespace eng {
namespace host {
// Keeps `message` as the calling thread's last failure (host/api.cpp).
void KeepError(const std::string &message);
}  // namespace host
}  // namespace eng

namespace layers {

using F4 = __attribute__((ext_vector_type(4))) float;

__device__ __forceinline__ float Float(float x) { return x; }
__device__ __forceinline__ float Float(__hip_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float Float(__half x) { return __half2float(x); }
template <class T>
__device__ __forceinline__ T As(float x);
template <>
__device__ __forceinline__ float As<float>(float x) { return x; }
template <>
__device__ __forceinline__ __hip_bfloat16 As<__hip_bfloat16>(float x) { return __float2bfloat16(x); }
template <>
__device__ __forceinline__ __half As<__half>(float x) { return __float2half(x); }

// An element as the low bits of a word, and element i of those of a word of memory.
template <class T>
__device__ __forceinline__ uint32_t Bits(T x) {
    if constexpr (sizeof(T) == 4) return __builtin_bit_cast(uint32_t, x);
    else return __builtin_bit_cast(uint16_t, x);
}
template <class T>
__device__ __forceinline__ float OfWord(uint32_t word, int i) {
    if constexpr (sizeof(T) == 4) return __uint_as_float(word);
    else if constexpr (std::is_same<T, __hip_bfloat16>::value) return __uint_as_float(i % 2 ? word & 0xffff0000u : word << 16);
    else return __half2float(__builtin_bit_cast(__half, (uint16_t)(i % 2 ? word >> 16 : word)));
}

// N neighbouring elements, moved in one access.
template <class T, int N>
struct alignas(N * sizeof(T)) Pack {
    T x[N];
};

// `N` elements from `p`, the first `valid` of them real and the others zero. `Whole` says that packs of
// the tensor are aligned and never cut by its end, so that all of a pack is real or none.
template <int N, bool Whole, class T>
__device__ __forceinline__ Pack<T, N> Load(const T *p, int valid) {
    Pack<T, N> r{};
    if constexpr (Whole) {
        if (valid > 0) r = *reinterpret_cast<const Pack<T, N> *>(p);
    } else {
#pragma unroll
        for (int i = 0; i < N; i++)
            if (i < valid) r.x[i] = p[i];
    }
    return r;
}
template <int N, bool Whole, class T>
__device__ __forceinline__ void Store(T *p, const Pack<T, N> &v, int valid) {
    if constexpr (Whole) {
        if (valid > 0) *reinterpret_cast<Pack<T, N> *>(p) = v;
    } else {
#pragma unroll
        for (int i = 0; i < N; i++)
            if (i < valid) p[i] = v.x[i];
    }
}

// A value the compiler takes for unknown from here on, so that it does not keep what follows from it
// (a mask for each of many rows) over a long loop.
__device__ __forceinline__ int Opaque(int x) {
    asm volatile("" : "+s"(x));
    return x;
}

// A pointer out of an argument struct, known to be to device memory.
template <class T>
__device__ __forceinline__ T *Global(T *p) { return (T *)(__attribute__((address_space(1))) T *)(uintptr_t)p; }

// `base` (the same in every lane) moved by a lane's `bytes`: the address stays a scalar pair and one
// vector register.
template <class T>
__device__ __forceinline__ T *Lane(T *base, uint32_t bytes) {
    using Byte = typename std::conditional<std::is_const<T>::value, const char, char>::type;
    return Global(reinterpret_cast<T *>(reinterpret_cast<Byte *>(base) + bytes));
}

// What lies in LDS is read again after this rather than kept in registers.
__device__ __forceinline__ void Forget() { asm volatile("" ::: "memory"); }

// The same of a lane's own value, so that what follows from it is not kept over a loop.
__device__ __forceinline__ void Renew(F4 &x) { asm volatile("" : "+v"(x)); }
__device__ __forceinline__ int Renewed(int x) {
    asm volatile("" : "+v"(x));
    return x;
}

// A kernel's only argument, read anew from the arguments' segment: many strides and pointers that are
// each used once in a long loop would not all fit the scalar registers.
template <class X>
__device__ __forceinline__ X Argument() {
    using Word = const __attribute__((address_space(4))) uint32_t;
    static_assert(sizeof(X) % 4 == 0, "whole words");
    Word *p = (Word *)__builtin_amdgcn_kernarg_segment_ptr();
    asm volatile("" : "+s"(p));
    struct Words {
        uint32_t x[sizeof(X) / 4];
    } words;
#pragma unroll
    for (int i = 0; i < (int)(sizeof(X) / 4); i++) words.x[i] = p[i];
    return __builtin_bit_cast(X, words);
}

// A 16x16 matrix M over a wavefront, four values a lane, with m = lane % 16 and g = lane / 16:
//  row order   "a": lane (m, g) holds M[m][4g + r], r = 0..3;
//  column order "d": lane (m, g) holds M[4g + r][m].
// The matrix instruction contracts 4 indices at a time: its left operand gives a lane's row m and
// index g, its right operand index g and column m, its result is in column order. The order of the
// contracted indices is free as long as both operands share it, so step r takes the indices 4g + r,
// and then X in row order times Y in column order needs no movement of data: d(XY) = Product(a(X),
// d(Y)). Since a(M) = d(M transposed), a(XY) = Product(d(Y), a(X)).
__device__ __forceinline__ F4 Mfma(float a, float b, F4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ F4 Product(F4 a, F4 b, F4 c = F4{0, 0, 0, 0}) {
#pragma unroll
    for (int r = 0; r < 4; r++) c = Mfma(a[r], b[r], c);
    return c;
}

// Products in 32 bits on the 16-bit matrix instruction. A float is the exact sum of three bfloat16
// values (its leading 8 bits, the next 8, the last 8), a half of two, so a product of two operands is
// the sum of the instruction's exact products of their pieces, of which those whose orders add up to
// three and more are left out (of two floats 2^-24 of it as a rule and 2^-21 at most): 3 instructions
// for a bfloat16 times a float, 5 for a half, 6 for a float, of 32 contracted indices and 16 cycles each. The same in the 32-bit instruction takes 8 of 32 cycles. An
// infinity has no such pieces: it comes out as a NaN.
using B8 = __attribute__((ext_vector_type(8))) __bf16;
struct Four {  // four bfloat16 values
    uint32_t x[2];
};
template <class T>
constexpr int kPieces = sizeof(T) == 4 ? 3 : std::is_same<T, __half>::value ? 2 : 1;
constexpr int kFloatPieces = 3;

__device__ __forceinline__ B8 Eight(Four lo, Four hi) {
    struct Both {
        Four lo, hi;
    };
    return __builtin_bit_cast(B8, Both{lo, hi});
}
__device__ __forceinline__ F4 Mfma32(B8 a, B8 b, F4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }

template <int Pieces>
__device__ __forceinline__ void Split(const float (&x)[4], Four (&piece)[Pieces]) {
    float rest[4] = {x[0], x[1], x[2], x[3]};
#pragma unroll
    for (int i = 0; i < Pieces; i++)
#pragma unroll
        for (int j = 0; j < 2; j++) {
            const uint32_t lo = __float_as_uint(rest[2 * j]), hi = __float_as_uint(rest[2 * j + 1]);
            piece[i].x[j] = __builtin_amdgcn_perm(hi, lo, 0x07060302);
            if (i + 1 < Pieces) {
                rest[2 * j] -= __uint_as_float(lo & 0xffff0000u);
                rest[2 * j + 1] -= __uint_as_float(hi & 0xffff0000u);
            }
        }
}
__device__ __forceinline__ void Split(F4 x, Four (&piece)[kFloatPieces]) {
    const float f[4] = {x[0], x[1], x[2], x[3]};
    Split<kFloatPieces>(f, piece);
}
// The pieces of four elements as they are in memory.
template <class T>
__device__ __forceinline__ void Split(const Pack<T, 4> &x, Four (&piece)[kPieces<T>]) {
    if constexpr (std::is_same<T, __hip_bfloat16>::value) {
        piece[0] = __builtin_bit_cast(Four, x);
    } else {
        const float f[4] = {Float(x.x[0]), Float(x.x[1]), Float(x.x[2]), Float(x.x[3])};
        Split<kPieces<T>>(f, piece);
    }
}
// The sum over the pieces' products, largest first in neither order: all i + j below three.
template <int A, int B>
__device__ __forceinline__ F4 Mfma32(const B8 (&a)[A], const B8 (&b)[B], F4 c) {
#pragma unroll
    for (int i = A - 1; i >= 0; i--)
#pragma unroll
        for (int j = B - 1; j >= 0; j--)
            if (i + j < 3) c = Mfma32(a[i], b[j], c);
    return c;
}
// A product of only 16 contracted indices, four a lane: two pairs of pieces share an instruction. (The
// instruction for 16 indices does not mix with this one: chained on one accumulator they gave wrong sums.)
template <int A, int B>
__device__ __forceinline__ F4 Mfma16(const Four (&a)[A], const Four (&b)[B], F4 c) {
    Four left{}, right{};
    bool half = false;
#pragma unroll
    for (int i = A - 1; i >= 0; i--)
#pragma unroll
        for (int j = B - 1; j >= 0; j--) {
            if (i + j >= 3) continue;
            if (half) c = Mfma32(Eight(left, a[i]), Eight(right, b[j]), c);
            left = a[i], right = b[j], half = !half;
        }
    return half ? Mfma32(Eight(left, left), Eight(right, Four{}), c) : c;
}

template <int Control>
__device__ __forceinline__ float Dpp(float x) {
    return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), Control, 0xf, 0xf, true));
}
template <int Control>
__device__ __forceinline__ double Dpp(double x) {
    const int lo = __builtin_amdgcn_update_dpp(0, __double2loint(x), Control, 0xf, 0xf, true);
    const int hi = __builtin_amdgcn_update_dpp(0, __double2hiint(x), Control, 0xf, 0xf, true);
    return __hiloint2double(hi, lo);
}
constexpr int kRowShiftRight = 0x110;  // + n: a lane takes the value n lanes below it in its row of 16, else 0
constexpr int kRowShiftLeft = 0x100;   // + n: n lanes above
constexpr int kRowRotate = 0x120;      // + n: rotation within the row
template <int Lane>
__device__ __forceinline__ float QuadLane(float x) {
    return Dpp<Lane * 0x55>(x);
}

// Over a row of 16 lanes: the sum in every lane, the sum up to and with each lane, and from each lane on.
__device__ __forceinline__ float RowSum(float x) {
    x += Dpp<kRowRotate + 8>(x);
    x += Dpp<kRowRotate + 4>(x);
    x += Dpp<kRowRotate + 2>(x);
    x += Dpp<kRowRotate + 1>(x);
    return x;
}
template <class T>
__device__ __forceinline__ T RowUpTo(T x) {
    x += Dpp<kRowShiftRight + 1>(x);
    x += Dpp<kRowShiftRight + 2>(x);
    x += Dpp<kRowShiftRight + 4>(x);
    x += Dpp<kRowShiftRight + 8>(x);
    return x;
}
__device__ __forceinline__ float RowFrom(float x) {
    x += Dpp<kRowShiftLeft + 1>(x);
    x += Dpp<kRowShiftLeft + 2>(x);
    x += Dpp<kRowShiftLeft + 4>(x);
    x += Dpp<kRowShiftLeft + 8>(x);
    return x;
}
__device__ __forceinline__ float WaveSum(float x) {
    x = RowSum(x);
    x += __shfl_xor(x, 16);
    return x + __shfl_xor(x, 32);
}

// The block's place in the work, so that neighbouring pieces of work run on one of the chip's eight
// dies and share its L2: blocks go round the dies one by one.
constexpr unsigned kDies = 8;
__device__ __forceinline__ unsigned Place(unsigned block, unsigned blocks) {
    const unsigned each = blocks / kDies, whole = each * kDies;
    return block < whole ? (block % kDies) * each + block / kDies : block;
}

// Runs `body` with a value of the element type `type` names (0 float, 1 bfloat16, 2 half).
template <class Body>
bool ForType(int type, Body body) {
    switch (type) {
    case 0: body(float()); return true;
    case 1: body(__hip_bfloat16()); return true;
    case 2: body(__half()); return true;
    }
    return false;
}

inline int Failed(const char *what) {
    eng::host::KeepError(what);
    return -1;
}
// The outcome of the launches so far: 0, or -1 with the failure kept.
inline int Launched(const char *what) {
    const hipError_t e = hipGetLastError();
    if (e == hipSuccess) return 0;
    eng::host::KeepError(std::string("hipLaunchKernel: ") + what + ": " + hipGetErrorString(e));
    return -1;
}

}  // namespace layers
