// Norms around a policy's blocks, over rows of up to 8,192 values, and their gradients.
//
//   u = block inner, inner = 1 / sqrt(mean(block^2) + epsilon)    (or u = block, without a norm of its own)
//   b = after act(gate) u
//   h = x + scale b                                               (or h = b, without a stream)
//   y = before e, e = h outer, outer = 1 / sqrt(mean(h^2) + epsilon)
//
// With dh the gradient of h and dy that of y, means over a row and sums over all rows:
//   de = before dy,  dh += outer (de - e mean(de e)),  d_before = sum dy e,  dx = dh;
//   d_scale = sum dh b,  d_after = sum dh scale act(gate) u,  d_gate = dh scale after u act'(gate);
//   du = dh scale after act(gate),  d_block = inner (du - u mean(du u)).
//
// All sums are in 32 bits or more. A row lies in the registers of a part of a wavefront or of a workgroup: every input
// is read once and every output written once, and memory bounds it. With everything, 262,144 rows of 256 in bfloat16 take
// 135 us (0.67 GB, 5.0 TB/s) and their gradients 225 to 233 (1.07 GB, 4.7 TB/s; a copy reaches 4.8). Rows of odd sizes and 16-bit
// rows past 2,048 values reach less: 8,192 rows of 8,192 140 and 274 us (4.8 and 3.9 TB/s), of 8,191 220 and 473.
#include "../../../include/cuju_amd.h"
#include "common.h"

namespace layers {
namespace {

using Rows = cuju_row_norm;
enum Activation { kNone, kSigmoid, kSilu };
constexpr int kMostSize = 8192;
constexpr int kVectors = 3;  // after, scale and before

// The sigmoid of a gate of the type T, and what it leaves of one, each of its own digits: the exponential is of the argument that
// makes it at most one. Of a float both are within 6 x 2^-24 of themselves. For 16-bit gates the hardware's exponential and reciprocal
// do, (|z| + 4) 2^-24 off, at most 2^-17 where a float has digits, beside a rounding of 2^-8 or 2^-11: 1,048,576 rows of 64 in
// bfloat16 take 84 us forward and 131 back, with the float's 132 and 199.
template <class T>
struct Sigmoid {
    float s, rest;
    __device__ __forceinline__ explicit Sigmoid(float z) {
        constexpr bool exact = sizeof(T) == 4;
        const float e = exact ? expf(-fabsf(z)) : __expf(-fabsf(z));
        const float large = exact ? 1.f / (1.f + e) : __builtin_amdgcn_rcpf(1.f + e), small = e * large;
        s = z < 0.f ? small : large, rest = z < 0.f ? large : small;
    }
};
template <class T>
__device__ __forceinline__ float Gate(float z, int activation) {
    if (activation == kNone) return z;
    const float s = sizeof(T) == 4 ? Sigmoid<T>(z).s : __builtin_amdgcn_rcpf(1.f + __expf(-z));
    return activation == kSilu ? z * s : s;
}
template <class T>
__device__ __forceinline__ float GateSlope(float z, int activation) {
    if (activation == kNone) return 1.f;
    const Sigmoid<T> of(z);
    if (activation == kSigmoid) return of.s * of.rest;
    return of.s * fmaf(z, of.rest, 1.f);
}

// A thread's packs of a row: `Lanes` packs side by side, `Packs` such rows of packs after one another. Packs need no
// alignment but their elements'; the last one may be cut by the row's end. They are held as the words of memory, since
// an array of 16-bit elements would take a register for each.
template <class T, int Vector, int Packs, int Lanes>
struct Held {
    static constexpr int kElements = 4 / sizeof(T), kWords = Vector / kElements;
    struct __attribute__((packed, aligned(sizeof(T)))) Loose {
        uint32_t w[kWords];
    };
    uint32_t w[Packs][kWords];
    __device__ __forceinline__ void Load(const T *row, int lane, int size) {
#pragma unroll
        for (int i = 0; i < Packs; i++) {
            const int at = (i * Lanes + lane) * Vector;
            if (at + Vector <= size) {
                const Loose x = *reinterpret_cast<const Loose *>(Global(row) + at);
#pragma unroll
                for (int c = 0; c < kWords; c++) w[i][c] = x.w[c];
            } else {
#pragma unroll
                for (int c = 0; c < kWords; c++) w[i][c] = 0;
                if (at >= size) continue;
#pragma unroll
                for (int c = 0; c < Vector; c++)
                    if (at + c < size) w[i][c / kElements] |= Bits(Global(row)[at + c]) << (16 * (c % kElements));
            }
        }
    }
    __device__ __forceinline__ void Store(T *row, int lane, int size) const {
#pragma unroll
        for (int i = 0; i < Packs; i++) {
            const int at = (i * Lanes + lane) * Vector;
            if (at + Vector <= size) {
                Loose x;
#pragma unroll
                for (int c = 0; c < kWords; c++) x.w[c] = w[i][c];
                *reinterpret_cast<Loose *>(Global(row) + at) = x;
            } else if (at < size) {
#pragma unroll
                for (int c = 0; c < Vector; c++)
                    if (at + c < size) Global(row)[at + c] = As<T>(At(i, c));
            }
        }
    }
    __device__ __forceinline__ float At(int i, int c) const { return OfWord<T>(w[i][c / kElements], c); }
    // The elements of a pack, rounded.
    __device__ __forceinline__ void Set(int i, const float (&x)[Vector]) {
#pragma unroll
        for (int c = 0; c < kWords; c++) {
            w[i][c] = Bits(As<T>(x[c * kElements]));
            if constexpr (kElements == 2) w[i][c] |= Bits(As<T>(x[c * kElements + 1])) << 16;
        }
    }
};
// A vector of the row's columns, held through all rows.
template <int Vector, int Packs, int Lanes>
struct Columns {
    float x[Packs][Vector];
    __device__ __forceinline__ Columns(const void *p, float otherwise, int lane, int size) {
        const float *from = static_cast<const float *>(p);
#pragma unroll
        for (int i = 0; i < Packs; i++)
#pragma unroll
            for (int c = 0; c < Vector; c++) {
                const int at = (i * Lanes + lane) * Vector + c;
                x[i][c] = from && at < size ? from[at] : otherwise;
            }
    }
    __device__ __forceinline__ float At(int i, int c) const { return x[i][c]; }
};
// A thread's sums over its rows, by vector and column: in registers, or in LDS for the largest workgroups, whose threads'
// registers do not hold them too.
template <int Vector, int Packs, int Lanes>
struct Sums {
    static constexpr bool kShared = Lanes >= 1024;
    static constexpr int kBytes = kShared ? kVectors * Packs * Vector * Lanes * (int)sizeof(float) : 0;
    float x[kShared ? 1 : kVectors][kShared ? 1 : Packs][kShared ? 1 : Vector];
    float *shared;
    __device__ __forceinline__ float &At(int v, int i, int c) {
        if constexpr (kShared) return shared[((v * Packs + i) * Vector + c) * Lanes];
        else return x[v][i][c];
    }
    __device__ __forceinline__ void Add(int v, int i, int c, float a, float b) { At(v, i, c) = fmaf(a, b, At(v, i, c)); }
    __device__ __forceinline__ Sums(float *room) : shared(room + threadIdx.x) {
#pragma unroll
        for (int v = 0; v < kVectors; v++)
#pragma unroll
            for (int i = 0; i < Packs; i++)
#pragma unroll
                for (int c = 0; c < Vector; c++) At(v, i, c) = 0.f;
    }
};

// The sum over the threads of a row, in each of them. Rows past a wavefront take `scratch`, two halves of a float for
// each wavefront, used in turn: a wavefront is a sum ahead of another at most.
template <int Lanes>
__device__ __forceinline__ float SumOfRow(float x, float *scratch, int &half) {
    if constexpr (Lanes <= 64) {
#pragma unroll
        for (int d = 1; d < Lanes; d *= 2) x += __shfl_xor(x, d);
    } else {
        constexpr int kWaves = Lanes / 64;
        x = WaveSum(x);
        float *to = scratch + half * kWaves;
        if ((threadIdx.x & 63) == 0) to[threadIdx.x >> 6] = x;
        __syncthreads();
        x = 0;
#pragma unroll
        for (int w = 0; w < kWaves; w++) x += to[w];
        half ^= 1;
    }
    return x;
}

template <int Lanes>
constexpr int kThreads = Lanes <= 64 ? 256 : Lanes;

template <class T>
__device__ __forceinline__ const T *RowOf(const void *p, const long long *strides, long long row, int inner) {
    return static_cast<const T *>(p) + row / inner * strides[0] + row % inner * strides[1];
}

template <class T, int Vector, int Packs, int Lanes, bool Stream>
__global__ __launch_bounds__(kThreads<Lanes>) void ForwardKernel(Rows n) {
    __shared__ float scratch[2 * (Lanes <= 64 ? 1 : Lanes / 64)];
    const int lane = threadIdx.x % Lanes, each = kThreads<Lanes> / Lanes, size = n.size;
    int half = 0;
    const Columns<Vector, Packs, Lanes> after(n.after, 1.f, lane, size);
    const Columns<Vector, Packs, Lanes> scale(n.scales, n.scale, lane, size);
    const Columns<Vector, Packs, Lanes> before(n.before, 1.f, lane, size);
    const float count = 1.f / size;
    for (long long row = (long long)blockIdx.x * each + threadIdx.x / Lanes; row < n.rows; row += (long long)gridDim.x * each) {
        Held<T, Vector, Packs, Lanes> block, gate{}, x{}, out;
        block.Load(RowOf<T>(n.block, n.block_strides, row, n.inner), lane, size);
        if (n.gate) gate.Load(RowOf<T>(n.gate, n.gate_strides, row, n.inner), lane, size);
        if constexpr (Stream) x.Load(RowOf<T>(n.x, n.x_strides, row, n.inner), lane, size);
        float inner = 1.f, outer = 1.f;
        if (n.norm_block) {
            float sum = 0;
#pragma unroll
            for (int i = 0; i < Packs; i++)
#pragma unroll
                for (int c = 0; c < Vector; c++) sum = fmaf(block.At(i, c), block.At(i, c), sum);
            inner = 1.f / sqrtf(fmaf(SumOfRow<Lanes>(sum, scratch, half), count, n.epsilon));
        }
        float h[Packs][Vector], sum = 0;
#pragma unroll
        for (int i = 0; i < Packs; i++)
#pragma unroll
            for (int c = 0; c < Vector; c++) {
                float b = block.At(i, c) * inner * after.At(i, c);
                if (n.gate) b *= Gate<T>(gate.At(i, c), n.activation);
                h[i][c] = Stream ? fmaf(scale.At(i, c), b, x.At(i, c)) : b;
                // Past the row's end all inputs are zeros, and a gate of zero may not be.
                if constexpr (Stream) sum = fmaf(h[i][c], h[i][c], sum);
            }
#pragma unroll
        for (int i = 0; i < Packs; i++) out.Set(i, h[i]);
        out.Store(static_cast<T *>(n.stream) + row * size, lane, size);
        if constexpr (Stream) {
            outer = 1.f / sqrtf(fmaf(SumOfRow<Lanes>(sum, scratch, half), count, n.epsilon));
#pragma unroll
            for (int i = 0; i < Packs; i++) {
#pragma unroll
                for (int c = 0; c < Vector; c++) h[i][c] *= outer * before.At(i, c);
                out.Set(i, h[i]);
            }
            out.Store(static_cast<T *>(n.normed) + row * size, lane, size);
        }
        if (n.stats && lane == 0) {
            float *stats = static_cast<float *>(n.stats) + 2 * row;
            stats[0] = inner, stats[1] = outer;
        }
    }
}

template <class T, int Vector, int Packs, int Lanes, bool Stream>
__global__ __launch_bounds__(kThreads<Lanes>) void BackwardKernel(Rows n, float *parts) {
    constexpr int each = kThreads<Lanes> / Lanes;
    __shared__ float scratch[2 * (Lanes <= 64 ? 1 : Lanes / 64)];
    const int lane = threadIdx.x % Lanes, size = n.size;
    int half = 0;
    const Columns<Vector, Packs, Lanes> after(n.after, 1.f, lane, size);
    const Columns<Vector, Packs, Lanes> scale(n.scales, n.scale, lane, size);
    const Columns<Vector, Packs, Lanes> before(n.before, 1.f, lane, size);
    extern __shared__ float room[];
    Sums<Vector, Packs, Lanes> sums(room);
    const float count = 1.f / size;
    for (long long row = (long long)blockIdx.x * each + threadIdx.x / Lanes; row < n.rows; row += (long long)gridDim.x * each) {
        Held<T, Vector, Packs, Lanes> block, gate{}, x{}, dh{}, dy{}, out;
        block.Load(RowOf<T>(n.block, n.block_strides, row, n.inner), lane, size);
        if (n.d_stream) dh.Load(static_cast<const T *>(n.d_stream) + row * size, lane, size);
        if (n.gate) gate.Load(RowOf<T>(n.gate, n.gate_strides, row, n.inner), lane, size);
        if constexpr (Stream) {
            x.Load(RowOf<T>(n.x, n.x_strides, row, n.inner), lane, size);
            if (n.d_normed) dy.Load(static_cast<const T *>(n.d_normed) + row * size, lane, size);
        }
        const float *stats = static_cast<const float *>(n.stats) + 2 * row;
        const float inner = stats[0], outer = stats[1];
        float factor[Packs][Vector], d[Packs][Vector];
        const auto unit = [&](int i, int c) { return block.At(i, c) * inner; };
        float sum = 0;
#pragma unroll
        for (int i = 0; i < Packs; i++)
#pragma unroll
            for (int c = 0; c < Vector; c++) {
                factor[i][c] = n.gate ? Gate<T>(gate.At(i, c), n.activation) : 1.f;
                d[i][c] = dh.At(i, c);
                if constexpr (Stream) {
                    const float e = outer * fmaf(scale.At(i, c), after.At(i, c) * factor[i][c] * unit(i, c), x.At(i, c));
                    sums.Add(2, i, c, dy.At(i, c), e);
                    sum = fmaf(dy.At(i, c) * before.At(i, c), e, sum);
                }
            }
        if constexpr (Stream) {
            const float mean = SumOfRow<Lanes>(sum, scratch, half) * count;
#pragma unroll
            for (int i = 0; i < Packs; i++) {
#pragma unroll
                for (int c = 0; c < Vector; c++) {
                    const float b = after.At(i, c) * factor[i][c] * unit(i, c), e = outer * fmaf(scale.At(i, c), b, x.At(i, c));
                    d[i][c] = fmaf(outer, fmaf(dy.At(i, c), before.At(i, c), -e * mean), d[i][c]);
                    sums.Add(1, i, c, d[i][c], b);
                }
                out.Set(i, d[i]);
#pragma unroll
                for (int c = 0; c < Vector; c++) d[i][c] *= scale.At(i, c);
            }
            if (n.dx) out.Store(static_cast<T *>(n.dx) + row * size, lane, size);
        }
        sum = 0;
#pragma unroll
        for (int i = 0; i < Packs; i++) {
            float slope[Vector];
#pragma unroll
            for (int c = 0; c < Vector; c++) {
                const float of = d[i][c] * unit(i, c);
                sums.Add(0, i, c, of, factor[i][c]);
                slope[c] = n.gate ? of * after.At(i, c) * GateSlope<T>(gate.At(i, c), n.activation) : 0.f;
                d[i][c] *= after.At(i, c) * factor[i][c];
                sum = fmaf(d[i][c], unit(i, c), sum);
            }
            out.Set(i, slope);
        }
        if (n.d_gate) out.Store(static_cast<T *>(n.d_gate) + row * size, lane, size);
        const float mean = n.norm_block ? SumOfRow<Lanes>(sum, scratch, half) * count : 0.f;
#pragma unroll
        for (int i = 0; i < Packs; i++) {
#pragma unroll
            for (int c = 0; c < Vector; c++) d[i][c] = inner * fmaf(-unit(i, c), mean, d[i][c]);
            out.Set(i, d[i]);
        }
        if (n.d_block) out.Store(static_cast<T *>(n.d_block) + row * size, lane, size);
    }
    if (!parts) return;
    // The workgroup's sums over its rows, one vector after the other.
    __shared__ float shared[each > 1 ? Lanes * Packs * Vector * each : 1];
    void *const outs[kVectors] = {n.d_after, n.d_scales, n.d_before};
#pragma unroll
    for (int v = 0; v < kVectors; v++) {
        if (!outs[v]) continue;
        float *to = parts + ((long long)blockIdx.x * kVectors + v) * size;
        if constexpr (each > 1) {
            __syncthreads();
#pragma unroll
            for (int i = 0; i < Packs; i++)
#pragma unroll
                for (int c = 0; c < Vector; c++)
                    shared[threadIdx.x / Lanes * (Lanes * Packs * Vector) + (i * Lanes + lane) * Vector + c] = sums.At(v, i, c);
            __syncthreads();
            for (int at = threadIdx.x; at < size; at += kThreads<Lanes>) {
                float sum = 0;
                for (int r = 0; r < each; r++) sum += shared[r * (Lanes * Packs * Vector) + at];
                to[at] = sum;
            }
        } else {
#pragma unroll
            for (int i = 0; i < Packs; i++)
#pragma unroll
                for (int c = 0; c < Vector; c++) {
                    const int at = (i * Lanes + lane) * Vector + c;
                    if (at < size) to[at] = sums.At(v, i, c);
                }
        }
    }
}

// The sums of all workgroups, always in the same order: 16 columns and 64 threads for each.
__global__ __launch_bounds__(1024) void PartsKernel(const float *parts, float *after, float *scales, float *before, int size, int blocks) {
    __shared__ double sums[64][17];
    const int column = threadIdx.x % 16, slice = threadIdx.x / 16;
    float *const outs[kVectors] = {after, scales, before};
    float *out = outs[blockIdx.y];
    if (!out) return;
    const int at = blockIdx.x * 16 + column;
    double sum = 0;
    if (at < size) {
        const float *from = parts + (long long)blockIdx.y * size + at;
        const long long step = (long long)kVectors * size;
        int r = slice;
        // Eight loads on the way at a time.
        for (; r + 7 * 64 < blocks; r += 8 * 64) {
            float x[8];
#pragma unroll
            for (int i = 0; i < 8; i++) x[i] = from[(r + i * 64) * step];
#pragma unroll
            for (int i = 0; i < 8; i++) sum += x[i];
        }
        for (; r < blocks; r += 64) sum += from[r * step];
    }
    sums[slice][column] = sum;
    __syncthreads();
    for (int d = 32; d; d /= 2) {
        if (slice < d) sums[slice][column] += sums[slice + d][column];
        __syncthreads();
    }
    if (slice == 0 && at < size) out[at] = (float)sums[0][column];
}

// body(elements of a pack, packs, threads of a row) for rows of `size`.
template <class T, bool Gradients, class Body>
void ForSize(int size, Body body) {
    constexpr int V = 16 / sizeof(T);
    // One pack a thread: two of eight elements are more than the registers of two wavefronts on a SIMD (bfloat16, 65,536
    // rows of 1,024: the gradients 266 us on 128 threads, 366 on 64). Past 512 packs that is the largest workgroup, which
    // the gradients are faster on (8,192 rows of 8,192: 486 against 864 us on 512 threads) and 16-bit outputs slower (204
    // against 166; both with four times the workgroups of now).
    const int packs = (size + V - 1) / V;
    const auto go = [&](auto lanes) { body(std::integral_constant<int, V>(), std::integral_constant<int, 1>(), lanes); };
    if (packs <= 4) go(std::integral_constant<int, 4>());
    else if (packs <= 8) go(std::integral_constant<int, 8>());
    else if (packs <= 16) go(std::integral_constant<int, 16>());
    else if (packs <= 32) go(std::integral_constant<int, 32>());
    else if (packs <= 64) go(std::integral_constant<int, 64>());
    else if (packs <= 128) go(std::integral_constant<int, 128>());
    else if (packs <= 256) go(std::integral_constant<int, 256>());
    else if (packs <= 512) go(std::integral_constant<int, 512>());
    else if (packs <= 1024) {
        if constexpr (Gradients || V == 4) go(std::integral_constant<int, 1024>());
        else body(std::integral_constant<int, V>(), std::integral_constant<int, 2>(), std::integral_constant<int, 512>());
    } else if constexpr (V == 4) body(std::integral_constant<int, V>(), std::integral_constant<int, 2>(), std::integral_constant<int, 1024>());
}
// Workgroups of a launch of rows of packs of V on L threads. 2^18 threads, four wavefronts a SIMD, read few vectors and leave
// few sums: bfloat16, 8,192 rows of 8,192: the gradients 274 us, with 2^19 threads 303, with 2^20 367; 16,384 rows of 4,096:
// 274, 301 and 361. The gradients of rows within a wavefront, whose workgroups leave one sum for all of theirs, and short rows
// that end within a pack, which wait for their last elements, want more wavefronts: 2^18 and 2^19 threads, 262,144 rows of 256
// in bfloat16: 261 and 233 us; 262,144 rows of 65 in float32, forward: 121 and 80 us.
constexpr int kMostBlocks = 1 << 11;
template <int V, int L, bool Gradients>
int Blocks(const Rows &n) {
    constexpr int each = kThreads<L> / L;
    const long long all = (n.rows + each - 1) / each, most = (L <= 64 && (Gradients || n.size % V) ? 1 << 19 : 1 << 18) / kThreads<L>;
    static_assert((1 << 19) / 256 <= kMostBlocks && (1 << 18) / 128 <= kMostBlocks, "as many sums as workgroups");
    return (int)(all < most ? all : most);
}

template <class T>
void Forward(const Rows &n, hipStream_t stream) {
    ForSize<T, false>(n.size, [&](auto vector, auto packs, auto lanes) {
        constexpr int V = decltype(vector)::value, P = decltype(packs)::value, L = decltype(lanes)::value;
        const dim3 grid(Blocks<V, L, false>(n)), threads(kThreads<L>);
        if (n.x) hipLaunchKernelGGL((ForwardKernel<T, V, P, L, true>), grid, threads, 0, stream, n);
        else hipLaunchKernelGGL((ForwardKernel<T, V, P, L, false>), grid, threads, 0, stream, n);
    });
}
template <class T>
int Backward(const Rows &n, hipStream_t stream) {
    bool fits = true;
    const bool summed = n.d_after || n.d_scales || n.d_before;
    float *parts = summed ? static_cast<float *>(n.workspace) : nullptr;
    int blocks = 0;
    ForSize<T, true>(n.size, [&](auto vector, auto packs, auto lanes) {
        constexpr int V = decltype(vector)::value, P = decltype(packs)::value, L = decltype(lanes)::value;
        blocks = Blocks<V, L, true>(n);
        constexpr int bytes = Sums<V, P, L>::kBytes;
        const auto launch = [&](auto kernel) {
            if (bytes && hipFuncSetAttribute(reinterpret_cast<const void *>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, bytes) !=
                             hipSuccess) {
                fits = false;
                return;
            }
            hipLaunchKernelGGL(kernel, dim3(blocks), dim3(kThreads<L>), bytes, stream, n, parts);
        };
        if (n.x) launch(BackwardKernel<T, V, P, L, true>);
        else launch(BackwardKernel<T, V, P, L, false>);
    });
    if (!fits) return Failed("hipFuncSetAttribute: the gradients of norms of rows do not fit the shared memory");
    if (summed)
        hipLaunchKernelGGL(PartsKernel, dim3((n.size + 15) / 16, kVectors), dim3(1024), 0, stream, parts, static_cast<float *>(n.d_after),
                           static_cast<float *>(n.d_scales), static_cast<float *>(n.d_before), n.size, blocks);
    return Launched("the gradients of norms of rows");
}

bool Fits(const Rows *n) {
    if (!n || n->type < 0 || n->type > 2) return Failed("expected a norm of the type 0, 1 or 2"), false;
    if (n->activation < kNone || n->activation > kSilu) return Failed("expected an activation from 0 to 2"), false;
    if (n->rows < 0 || n->inner < 1) return Failed("expected rows"), false;
    if (n->size < 1 || n->size > kMostSize) return Failed("expected rows of 1 to 8192 values"), false;
    return true;
}

}  // namespace
}  // namespace layers

using namespace layers;

extern "C" __attribute__((visibility("default"))) unsigned long long cuju_row_norm_workspace(const struct cuju_row_norm *norm) {
    if (!Fits(norm)) return 0;
    // At least as many workgroups as any launch has: of a row, or fewer.
    return (unsigned long long)(norm->rows < kMostBlocks ? norm->rows : kMostBlocks) * kVectors * norm->size * sizeof(float);
}

extern "C" __attribute__((visibility("default"))) int cuju_row_norm_forward(const struct cuju_row_norm *norm, void *stream) {
    if (!Fits(norm)) return -1;
    const Rows &n = *norm;
    if (n.rows == 0) return 0;
    if (!n.block || !n.stream || (n.x && !n.normed)) return Failed("expected rows and their outputs");
    ForType(n.type, [&](auto x) { Forward<decltype(x)>(n, static_cast<hipStream_t>(stream)); });
    return Launched("norms of rows");
}

extern "C" __attribute__((visibility("default"))) int cuju_row_norm_backward(const struct cuju_row_norm *norm, void *stream) {
    if (!Fits(norm)) return -1;
    const Rows &n = *norm;
    if (n.rows == 0) return 0;
    if (!n.block || !n.stats || (n.d_gate && !n.gate)) return Failed("expected rows, their statistics and a gate for its gradient");
    if ((n.d_after || n.d_scales || n.d_before) && !n.workspace) return Failed("expected a workspace");
    int status = -1;
    ForType(n.type, [&](auto x) { status = Backward<decltype(x)>(n, static_cast<hipStream_t>(stream)); });
    return status;
}
