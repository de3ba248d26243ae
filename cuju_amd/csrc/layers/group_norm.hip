// Group norm with an activation over channels-last maps [batch][pixels][channels], and its gradients.
//
//   xh = (x - mean) inverse, z = weight xh + bias, y = act(z); mean and inverse = 1 / sqrt(variance +
//   epsilon) over the pixels and the group's channels;
//   dz = dy act'(z), d_bias = sum dz, d_weight = sum dz xh over batch and pixels;
//   dx = inverse (weight dz - mean(weight dz) - xh mean(weight dz xh)), means over the group.
//
// All sums are in 32 bits or more. A workgroup that can hold a map (or the channels of some of its
// groups) in registers reads it once: mean, then the squares about the mean, then the output.
// Larger maps are read twice, cut over workgroups, with their sums in a workspace between.
#include "../../../include/cuju_amd.h"
#include "common.h"

namespace layers {
namespace {

using Norm = cuju_group_norm;
enum Activation { kNone, kRelu, kSilu };

__device__ __forceinline__ float Sigmoid(float z) { return __builtin_amdgcn_rcpf(1.f + __expf(-z)); }
__device__ __forceinline__ float Activate(float z, int activation) {
    // A comparison that keeps a NaN.
    if (activation == kRelu) return z < 0.f ? 0.f : z;
    if (activation == kSilu) return z * Sigmoid(z);
    return z;
}
__device__ __forceinline__ float Slope(float z, int activation) {
    if (activation == kRelu) return z > 0.f ? 1.f : 0.f;
    if (activation == kSilu) {
        const float s = Sigmoid(z);
        return s * fmaf(z, 1.f - s, 1.f);
    }
    return 1.f;
}

// How a workgroup lies over the channels it has: `vectors` packs side by side, filled up to `lanes` (a
// power of two, at most a wavefront), and threads / lanes pixels at a time, so that a thread's
// channels never change.
struct Shape {
    int pixels, channels, groups, perGroup;
    int slabs, slabChannels, vectors, lanes;
};

// Sums over the workgroup's pixels of each thread's channel values `v`, into `out` [channels of the slab].
// `scratch` holds [wavefronts][channels of the slab].
template <int Vector>
__device__ __forceinline__ void ChannelSums(float (&v)[Vector], float *scratch, float *out, const Shape &s) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, waves = blockDim.x >> 6;
    const int vector = threadIdx.x & (s.lanes - 1);
    for (int d = s.lanes; d < 64; d *= 2)
#pragma unroll
        for (int i = 0; i < Vector; i++) v[i] += __shfl_xor(v[i], d);
    if (lane < s.lanes && vector < s.vectors)
#pragma unroll
        for (int i = 0; i < Vector; i++) scratch[wave * s.slabChannels + vector * Vector + i] = v[i];
    __syncthreads();
    for (int c = threadIdx.x; c < s.slabChannels; c += blockDim.x) {
        float sum = 0;
        for (int w = 0; w < waves; w++) sum += scratch[w * s.slabChannels + c];
        out[c] = sum;
    }
    __syncthreads();
}
// The groups' sums of a channel array.
__device__ __forceinline__ void GroupSums(const float *channels, float *out, const Shape &s) {
    for (int n = threadIdx.x; n < s.slabChannels / s.perGroup; n += blockDim.x) {
        float sum = 0;
        for (int c = 0; c < s.perGroup; c++) sum += channels[n * s.perGroup + c];
        out[n] = sum;
    }
    __syncthreads();
}

constexpr int kMostSlab = 512;  // channels of a slab: a wavefront of packs of eight

template <class T, int Vector, int Packs, int Threads>
__global__ __launch_bounds__(Threads) void ForwardKernel(const T *x, T *y, const float *weight, const float *bias, float *stats,
                                                         Shape s, float epsilon, int activation) {
    __shared__ float scratch[Threads / 64 * 64 * Vector], channelSums[64 * Vector], means[64 * Vector], squares[64 * Vector];
    const unsigned id = Place(blockIdx.x, gridDim.x);
    const int slab = id % s.slabs;
    const long long n = id / s.slabs;
    const int vector = threadIdx.x & (s.lanes - 1), row = threadIdx.x / s.lanes, rows = Threads / s.lanes;
    const bool mine = vector < s.vectors;
    const int channel = slab * s.slabChannels + vector * Vector;
    const long long base = n * s.pixels * s.channels + channel;
    Pack<T, Vector> v[Packs];
#pragma unroll
    for (int i = 0; i < Packs; i++) {
        const int p = i * rows + row;
        if (mine && p < s.pixels) v[i] = *reinterpret_cast<const Pack<T, Vector> *>(x + base + (long long)p * s.channels);
    }
    float sum[Vector];
#pragma unroll
    for (int c = 0; c < Vector; c++) sum[c] = 0;
#pragma unroll
    for (int i = 0; i < Packs; i++)
        if (mine && i * rows + row < s.pixels)
#pragma unroll
            for (int c = 0; c < Vector; c++) sum[c] += Float(v[i].x[c]);
    ChannelSums<Vector>(sum, scratch, channelSums, s);
    GroupSums(channelSums, means, s);
    const float count = 1.f / ((float)s.pixels * s.perGroup);
    float mean[Vector];
#pragma unroll
    for (int c = 0; c < Vector; c++) {
        mean[c] = mine ? means[(vector * Vector + c) / s.perGroup] * count : 0.f;
        sum[c] = 0;
    }
#pragma unroll
    for (int i = 0; i < Packs; i++)
        if (mine && i * rows + row < s.pixels)
#pragma unroll
            for (int c = 0; c < Vector; c++) {
                const float d = Float(v[i].x[c]) - mean[c];
                sum[c] = fmaf(d, d, sum[c]);
            }
    ChannelSums<Vector>(sum, scratch, channelSums, s);
    GroupSums(channelSums, squares, s);
    const int slabGroups = s.slabChannels / s.perGroup;
    if (stats)
        for (int i = threadIdx.x; i < slabGroups; i += Threads) {
            float *to = stats + (n * s.groups + slab * slabGroups + i) * 2;
            to[0] = means[i] * count;
            to[1] = 1.f / sqrtf(squares[i] * count + epsilon);
        }
    float scale[Vector], shift[Vector];
#pragma unroll
    for (int c = 0; c < Vector; c++) {
        scale[c] = 0, shift[c] = 0;
        if (!mine) continue;
        scale[c] = 1.f / sqrtf(squares[(vector * Vector + c) / s.perGroup] * count + epsilon);
        if (weight) scale[c] *= weight[channel + c];
        if (bias) shift[c] = bias[channel + c];
    }
#pragma unroll
    for (int i = 0; i < Packs; i++) {
        const int p = i * rows + row;
        if (!mine || p >= s.pixels) continue;
        Pack<T, Vector> out;
#pragma unroll
        for (int c = 0; c < Vector; c++)
            out.x[c] = As<T>(Activate(fmaf(Float(v[i].x[c]) - mean[c], scale[c], shift[c]), activation));
        *reinterpret_cast<Pack<T, Vector> *>(y + base + (long long)p * s.channels) = out;
    }
}

template <class T, int Vector, int Packs, int Threads>
__global__ __launch_bounds__(Threads) void BackwardKernel(const T *x, const T *dy, T *dx, const float *weight,
                                                          const float *bias, const float *stats, float *parts, Shape s,
                                                          int activation) {
    __shared__ float scratch[Threads / 64 * 64 * Vector], biasSums[64 * Vector], weightSums[64 * Vector];
    __shared__ float channelMeans[64 * Vector], first[64 * Vector], second[64 * Vector];
    const unsigned id = Place(blockIdx.x, gridDim.x);
    const int slab = id % s.slabs;
    const long long n = id / s.slabs;
    const int vector = threadIdx.x & (s.lanes - 1), row = threadIdx.x / s.lanes, rows = Threads / s.lanes;
    const bool mine = vector < s.vectors;
    const int channel = slab * s.slabChannels + vector * Vector;
    const long long base = n * s.pixels * s.channels + channel;
    Pack<T, Vector> v[Packs], d[Packs];
#pragma unroll
    for (int i = 0; i < Packs; i++) {
        const int p = i * rows + row;
        if (mine && p < s.pixels) {
            v[i] = *reinterpret_cast<const Pack<T, Vector> *>(x + base + (long long)p * s.channels);
            d[i] = *reinterpret_cast<const Pack<T, Vector> *>(dy + base + (long long)p * s.channels);
        }
    }
    float mean[Vector], inverse[Vector], w[Vector], shift[Vector], sumB[Vector], sumW[Vector];
#pragma unroll
    for (int c = 0; c < Vector; c++) {
        mean[c] = inverse[c] = shift[c] = sumB[c] = sumW[c] = 0, w[c] = 1;
        if (!mine) continue;
        const float *from = stats + (n * s.groups + (channel + c) / s.perGroup) * 2;
        mean[c] = from[0], inverse[c] = from[1];
        if (weight) w[c] = weight[channel + c];
        if (bias) shift[c] = bias[channel + c];
    }
#pragma unroll
    for (int i = 0; i < Packs; i++)
        if (mine && i * rows + row < s.pixels)
#pragma unroll
            for (int c = 0; c < Vector; c++) {
                const float xh = (Float(v[i].x[c]) - mean[c]) * inverse[c];
                const float dz = Float(d[i].x[c]) * Slope(fmaf(w[c], xh, shift[c]), activation);
                sumB[c] += dz;
                sumW[c] = fmaf(dz, xh, sumW[c]);
            }
    ChannelSums<Vector>(sumB, scratch, biasSums, s);
    ChannelSums<Vector>(sumW, scratch, weightSums, s);
    for (int c = threadIdx.x; c < s.slabChannels; c += Threads) {
        const int at = slab * s.slabChannels + c;
        parts[(n * 2 + 0) * s.channels + at] = weightSums[c];
        parts[(n * 2 + 1) * s.channels + at] = biasSums[c];
        const float each = weight ? weight[at] : 1.f;
        biasSums[c] *= each, weightSums[c] *= each;
    }
    __syncthreads();
    GroupSums(biasSums, first, s);
    GroupSums(weightSums, second, s);
    const float count = 1.f / ((float)s.pixels * s.perGroup);
    float m1[Vector], m2[Vector];
#pragma unroll
    for (int c = 0; c < Vector; c++) {
        m1[c] = mine ? first[(vector * Vector + c) / s.perGroup] * count : 0.f;
        m2[c] = mine ? second[(vector * Vector + c) / s.perGroup] * count : 0.f;
    }
#pragma unroll
    for (int i = 0; i < Packs; i++) {
        const int p = i * rows + row;
        if (!mine || p >= s.pixels) continue;
        Pack<T, Vector> out;
#pragma unroll
        for (int c = 0; c < Vector; c++) {
            const float xh = (Float(v[i].x[c]) - mean[c]) * inverse[c];
            const float dz = Float(d[i].x[c]) * Slope(fmaf(w[c], xh, shift[c]), activation);
            out.x[c] = As<T>(inverse[c] * (fmaf(w[c], dz, -m1[c]) - xh * m2[c]));
        }
        *reinterpret_cast<Pack<T, Vector> *>(dx + base + (long long)p * s.channels) = out;
    }
}

// ------------------------------------------------------------- maps that no workgroup's registers hold

constexpr int kSplitThreads = 256;

// A workgroup's part: a slab of a map, and cut `blockIdx.y` of its pixels.
struct Cut {
    int vector, first, step, end, slab, channel, channels;
    long long map;
    bool mine;
    __device__ Cut(const Shape &s, int Vector) {
        vector = threadIdx.x & (s.lanes - 1);
        slab = blockIdx.x % s.slabs * s.slabChannels;
        map = blockIdx.x / s.slabs;
        channel = slab + vector * Vector;
        channels = min(s.slabChannels, s.channels - slab);
        mine = vector * Vector < channels;
        const int each = (s.pixels + gridDim.y - 1) / gridDim.y;
        step = kSplitThreads / s.lanes;
        first = blockIdx.y * each + threadIdx.x / s.lanes;
        end = min(s.pixels, (int)(blockIdx.y + 1) * each);
    }
};

// Each channel's sum and sum of squares about its value at the first pixel: [map][cut][2][channels].
template <class T, int Vector>
__global__ __launch_bounds__(kSplitThreads) void SumsKernel(const T *x, float *parts, Shape s) {
    __shared__ float scratch[kSplitThreads * Vector], out[64 * Vector];
    const Cut cut(s, Vector);
    const T *at = x + cut.map * s.pixels * s.channels + cut.channel;
    float about[Vector], sum[Vector], square[Vector];
#pragma unroll
    for (int c = 0; c < Vector; c++) about[c] = cut.mine ? Float(at[c]) : 0.f, sum[c] = square[c] = 0;
    if (cut.mine)
        for (int p = cut.first; p < cut.end; p += cut.step) {
            const auto v = *reinterpret_cast<const Pack<T, Vector> *>(at + (long long)p * s.channels);
#pragma unroll
            for (int c = 0; c < Vector; c++) {
                const float d = Float(v.x[c]) - about[c];
                sum[c] += d;
                square[c] = fmaf(d, d, square[c]);
            }
        }
    Shape slab = s;
    slab.vectors = cut.channels / Vector;
    float *to = parts + (cut.map * gridDim.y + blockIdx.y) * 2 * s.channels + cut.slab;
    for (int k = 0; k < 2; k++) {
        ChannelSums<Vector>(k ? square : sum, scratch, out, slab);
        for (int c = threadIdx.x; c < cut.channels; c += kSplitThreads) to[k * s.channels + c] = out[c];
        __syncthreads();
    }
}
// A wavefront a group: its mean and inverse deviation, from the cuts' sums, in 64 bits.
template <class T>
__global__ __launch_bounds__(64) void StatsKernel(const T *x, const float *parts, float *stats, Shape s, int cuts, float epsilon) {
    const int group = blockIdx.x % s.groups;
    const long long n = blockIdx.x / s.groups;
    const auto sumOver = [&](auto value) {
        double total = 0;
        for (int i = threadIdx.x; i < s.perGroup; i += 64) total += value(group * s.perGroup + i);
        for (int d = 1; d < 64; d *= 2) total += __shfl_xor(total, d);
        return total;
    };
    const auto part = [&](int k, int c) {
        double total = 0;
        for (int i = 0; i < cuts; i++) total += parts[((n * cuts + i) * 2 + k) * s.channels + c];
        return total;
    };
    const T *first = x + n * s.pixels * s.channels;
    const double count = (double)s.pixels * s.perGroup;
    const double mean = sumOver([&](int c) { return part(0, c) + (double)s.pixels * Float(first[c]); }) / count;
    const double squares = sumOver([&](int c) {
        const double off = mean - Float(first[c]);
        return part(1, c) - 2 * off * part(0, c) + s.pixels * off * off;
    });
    if (threadIdx.x == 0) {
        float *to = stats + (n * s.groups + group) * 2;
        to[0] = (float)mean;
        to[1] = (float)(1.0 / sqrt(fmax(squares, 0.0) / count + epsilon));
    }
}
template <class T, int Vector>
__global__ __launch_bounds__(kSplitThreads) void ApplyKernel(const T *x, T *y, const float *weight, const float *bias,
                                                             const float *stats, Shape s, int activation) {
    const Cut cut(s, Vector);
    if (!cut.mine) return;
    const long long n = cut.map, base = n * s.pixels * s.channels + cut.channel;
    float mean[Vector], scale[Vector], shift[Vector];
#pragma unroll
    for (int c = 0; c < Vector; c++) {
        const float *from = stats + (n * s.groups + (cut.channel + c) / s.perGroup) * 2;
        mean[c] = from[0];
        scale[c] = from[1] * (weight ? weight[cut.channel + c] : 1.f);
        shift[c] = bias ? bias[cut.channel + c] : 0.f;
    }
    for (int p = cut.first; p < cut.end; p += cut.step) {
        const auto v = *reinterpret_cast<const Pack<T, Vector> *>(x + base + (long long)p * s.channels);
        Pack<T, Vector> out;
#pragma unroll
        for (int c = 0; c < Vector; c++)
            out.x[c] = As<T>(Activate(fmaf(Float(v.x[c]) - mean[c], scale[c], shift[c]), activation));
        *reinterpret_cast<Pack<T, Vector> *>(y + base + (long long)p * s.channels) = out;
    }
}
// The gradients' channel sums: [map][cut][2][channels], of dz xh and of dz.
template <class T, int Vector>
__global__ __launch_bounds__(kSplitThreads) void GradientSumsKernel(const T *x, const T *dy, const float *weight,
                                                                    const float *bias, const float *stats, float *parts,
                                                                    Shape s, int activation) {
    __shared__ float scratch[kSplitThreads * Vector], out[64 * Vector];
    const Cut cut(s, Vector);
    const long long n = cut.map, base = n * s.pixels * s.channels + cut.channel;
    float mean[Vector], inverse[Vector], w[Vector], shift[Vector], sumB[Vector], sumW[Vector];
#pragma unroll
    for (int c = 0; c < Vector; c++) {
        sumB[c] = sumW[c] = mean[c] = inverse[c] = shift[c] = 0, w[c] = 1;
        if (!cut.mine) continue;
        const float *from = stats + (n * s.groups + (cut.channel + c) / s.perGroup) * 2;
        mean[c] = from[0], inverse[c] = from[1];
        if (weight) w[c] = weight[cut.channel + c];
        if (bias) shift[c] = bias[cut.channel + c];
    }
    if (cut.mine)
        for (int p = cut.first; p < cut.end; p += cut.step) {
            const auto v = *reinterpret_cast<const Pack<T, Vector> *>(x + base + (long long)p * s.channels);
            const auto d = *reinterpret_cast<const Pack<T, Vector> *>(dy + base + (long long)p * s.channels);
#pragma unroll
            for (int c = 0; c < Vector; c++) {
                const float xh = (Float(v.x[c]) - mean[c]) * inverse[c];
                const float dz = Float(d.x[c]) * Slope(fmaf(w[c], xh, shift[c]), activation);
                sumB[c] += dz;
                sumW[c] = fmaf(dz, xh, sumW[c]);
            }
        }
    Shape slab = s;
    slab.vectors = cut.channels / Vector;
    float *to = parts + (n * gridDim.y + blockIdx.y) * 2 * s.channels + cut.slab;
    for (int k = 0; k < 2; k++) {
        ChannelSums<Vector>(k ? sumB : sumW, scratch, out, slab);
        for (int c = threadIdx.x; c < cut.channels; c += kSplitThreads) to[k * s.channels + c] = out[c];
        __syncthreads();
    }
}
// A wavefront a group: the means of weight dz and weight dz xh, [map][group][2].
__global__ __launch_bounds__(64) void GradientMeansKernel(const float *parts, const float *weight, float *means, Shape s,
                                                          int cuts) {
    const int group = blockIdx.x % s.groups;
    const long long n = blockIdx.x / s.groups;
    for (int k = 0; k < 2; k++) {
        double total = 0;
        for (int i = threadIdx.x; i < s.perGroup; i += 64) {
            const int c = group * s.perGroup + i;
            double sum = 0;
            for (int j = 0; j < cuts; j++) sum += parts[((n * cuts + j) * 2 + k) * s.channels + c];
            total += weight ? sum * weight[c] : sum;
        }
        for (int d = 1; d < 64; d *= 2) total += __shfl_xor(total, d);
        if (threadIdx.x == 0) means[(n * s.groups + group) * 2 + k] = (float)(total / ((double)s.pixels * s.perGroup));
    }
}
template <class T, int Vector>
__global__ __launch_bounds__(kSplitThreads) void GradientKernel(const T *x, const T *dy, T *dx, const float *weight,
                                                                const float *bias, const float *stats, const float *means,
                                                                Shape s, int activation) {
    const Cut cut(s, Vector);
    if (!cut.mine) return;
    const long long n = cut.map, base = n * s.pixels * s.channels + cut.channel;
    float mean[Vector], inverse[Vector], w[Vector], shift[Vector], m1[Vector], m2[Vector];
#pragma unroll
    for (int c = 0; c < Vector; c++) {
        const long long at = (n * s.groups + (cut.channel + c) / s.perGroup) * 2;
        mean[c] = stats[at], inverse[c] = stats[at + 1];
        m2[c] = means[at], m1[c] = means[at + 1];
        w[c] = weight ? weight[cut.channel + c] : 1.f;
        shift[c] = bias ? bias[cut.channel + c] : 0.f;
    }
    for (int p = cut.first; p < cut.end; p += cut.step) {
        const auto v = *reinterpret_cast<const Pack<T, Vector> *>(x + base + (long long)p * s.channels);
        const auto d = *reinterpret_cast<const Pack<T, Vector> *>(dy + base + (long long)p * s.channels);
        Pack<T, Vector> out;
#pragma unroll
        for (int c = 0; c < Vector; c++) {
            const float xh = (Float(v.x[c]) - mean[c]) * inverse[c];
            const float dz = Float(d.x[c]) * Slope(fmaf(w[c], xh, shift[c]), activation);
            out.x[c] = As<T>(inverse[c] * (fmaf(w[c], dz, -m1[c]) - xh * m2[c]));
        }
        *reinterpret_cast<Pack<T, Vector> *>(dx + base + (long long)p * s.channels) = out;
    }
}

// The sums over maps (and cuts) of [rows][2][channels], 64 columns a workgroup of 16 rows at a time.
__global__ __launch_bounds__(1024) void ColumnsKernel(const float *parts, float *dWeight, float *dBias, long long rows,
                                                      int channels) {
    __shared__ float sums[16][64];
    const int column = blockIdx.x * 64 + (threadIdx.x & 63), slot = threadIdx.x >> 6;
    float sum = 0;
    if (column < 2 * channels)
        for (long long i = slot; i < rows; i += 16) sum += parts[i * 2 * channels + column];
    sums[slot][threadIdx.x & 63] = sum;
    __syncthreads();
    if (slot == 0 && column < 2 * channels) {
        for (int i = 1; i < 16; i++) sum += sums[i][threadIdx.x];
        float *to = column < channels ? dWeight : dBias;
        if (to) to[column < channels ? column : column - channels] = sum;
    }
}

// --------------------------------------------------------------------------------------------- rules

int PowerOfTwo(int x) {
    int p = 1;
    while (p < x) p *= 2;
    return p;
}
Shape SlabsOf(const Norm &n, int slabs, int vector) {
    Shape s{n.pixels, n.channels, n.groups, n.channels / n.groups, slabs, n.channels / slabs, 0, 0};
    s.vectors = s.slabChannels / vector;
    s.lanes = PowerOfTwo(s.vectors);
    return s;
}
// The largest pack of elements that the channels and the tensors' alignment allow, in elements.
int VectorOf(const Norm &n) {
    const int size = n.type == 0 ? 4 : 2;
    uintptr_t all = reinterpret_cast<uintptr_t>(n.x) | reinterpret_cast<uintptr_t>(n.y) |
                    reinterpret_cast<uintptr_t>(n.dy) | reinterpret_cast<uintptr_t>(n.dx);
    int vector = 16 / size;
    while (vector > 1 && (n.channels % vector || all % (vector * size))) vector /= 2;
    return vector;
}
// The first count of slabs (each of whole groups and whole packs) whose pixels fit `packs` packs of
// each of `threads` threads; 0 if none does.
int SlabsFor(const Norm &n, int vector, int packs, int threads) {
    for (int slabs = 1; slabs <= n.groups; slabs++) {
        if (n.groups % slabs || n.channels / slabs % vector) continue;
        const Shape s = SlabsOf(n, slabs, vector);
        if (s.lanes <= 64 && s.pixels <= (long long)packs * (threads / s.lanes)) return slabs;
    }
    return 0;
}
// Maps past the registers: channels in slabs of at most a wavefront of packs, pixels cut so that about
// 2,048 workgroups run, at least 64 KB each.
Shape SplitShape(const Norm &n, int vector) {
    Shape s{n.pixels, n.channels, n.groups, n.channels / n.groups, 1, n.channels, 0, 0};
    s.slabChannels = n.channels < 64 * vector ? n.channels : 64 * vector;
    s.slabs = (n.channels + s.slabChannels - 1) / s.slabChannels;
    s.vectors = s.slabChannels / vector;
    s.lanes = PowerOfTwo(s.vectors);
    return s;
}
int CutsOf(const Norm &n) {
    const long long bytes = (long long)n.pixels * n.channels * (n.type == 0 ? 4 : 2);
    long long cuts = bytes / 65536;
    const long long wanted = (2048 + n.batch - 1) / (n.batch > 0 ? n.batch : 1);
    if (cuts > wanted) cuts = wanted;
    return (int)(cuts < 1 ? 1 : cuts > 1024 ? 1024 : cuts);
}

template <class Body>
void ForVector(int vector, Body body) {
    switch (vector) {
    case 8: body(std::integral_constant<int, 8>()); break;
    case 4: body(std::integral_constant<int, 4>()); break;
    case 2: body(std::integral_constant<int, 2>()); break;
    default: body(std::integral_constant<int, 1>()); break;
    }
}

template <class T>
void Forward(const Norm &n, hipStream_t stream) {
    const int vector = VectorOf(n);
    const T *x = static_cast<const T *>(n.x);
    T *y = static_cast<T *>(n.y);
    const float *weight = static_cast<const float *>(n.weight), *bias = static_cast<const float *>(n.bias);
    float *stats = static_cast<float *>(n.stats), *work = static_cast<float *>(n.workspace);
    ForVector(vector, [&](auto wide) {
        constexpr int V = decltype(wide)::value;
        if constexpr (V * sizeof(T) <= 16) {
            const auto resident = [&](auto kernel, int slabs, int threads) {
                hipLaunchKernelGGL(kernel, dim3((unsigned)((long long)n.batch * slabs)), dim3(threads), 0, stream, x, y,
                                   weight, bias, stats, SlabsOf(n, slabs, V), n.epsilon, n.activation);
            };
            if (SlabsFor(n, V, 4, 256) == 1) return resident(ForwardKernel<T, V, 4, 256>, 1, 256);
            if (SlabsFor(n, V, 8, 512) == 1) return resident(ForwardKernel<T, V, 8, 512>, 1, 512);
            if (const int slabs = SlabsFor(n, V, 14, 1024)) return resident(ForwardKernel<T, V, 14, 1024>, slabs, 1024);
            const Shape s = SplitShape(n, V);
            const int cuts = CutsOf(n);
            const dim3 grid((unsigned)((long long)s.slabs * n.batch), cuts);
            hipLaunchKernelGGL((SumsKernel<T, V>), grid, dim3(kSplitThreads), 0, stream, x, work, s);
            hipLaunchKernelGGL(StatsKernel<T>, dim3((unsigned)((long long)n.groups * n.batch)), dim3(64), 0, stream, x, work, stats, s, cuts, n.epsilon);
            hipLaunchKernelGGL((ApplyKernel<T, V>), grid, dim3(kSplitThreads), 0, stream, x, y, weight, bias, stats, s,
                               n.activation);
        }
    });
}

template <class T>
void Backward(const Norm &n, hipStream_t stream) {
    const int vector = VectorOf(n);
    const T *x = static_cast<const T *>(n.x), *dy = static_cast<const T *>(n.dy);
    T *dx = static_cast<T *>(n.dx);
    const float *weight = static_cast<const float *>(n.weight), *bias = static_cast<const float *>(n.bias);
    const float *stats = static_cast<const float *>(n.stats);
    float *parts = static_cast<float *>(n.workspace);
    long long rows = n.batch;
    ForVector(vector, [&](auto wide) {
        constexpr int V = decltype(wide)::value;
        if constexpr (V * sizeof(T) <= 16) {
            const auto resident = [&](auto kernel, int slabs, int threads) {
                hipLaunchKernelGGL(kernel, dim3((unsigned)((long long)n.batch * slabs)), dim3(threads), 0, stream, x, dy, dx,
                                   weight, bias, stats, parts, SlabsOf(n, slabs, V), n.activation);
            };
            if (SlabsFor(n, V, 4, 256) == 1) return resident(BackwardKernel<T, V, 4, 256>, 1, 256);
            if (const int slabs = SlabsFor(n, V, 14, 512)) return resident(BackwardKernel<T, V, 14, 512>, slabs, 512);
            const Shape s = SplitShape(n, V);
            const int cuts = CutsOf(n);
            rows = (long long)n.batch * cuts;
            float *means = parts + rows * 2 * n.channels;
            const dim3 grid((unsigned)((long long)s.slabs * n.batch), cuts);
            hipLaunchKernelGGL((GradientSumsKernel<T, V>), grid, dim3(kSplitThreads), 0, stream, x, dy, weight, bias, stats,
                               parts, s, n.activation);
            hipLaunchKernelGGL(GradientMeansKernel, dim3((unsigned)((long long)n.groups * n.batch)), dim3(64), 0, stream, parts, weight, means, s, cuts);
            hipLaunchKernelGGL((GradientKernel<T, V>), grid, dim3(kSplitThreads), 0, stream, x, dy, dx, weight, bias, stats,
                               means, s, n.activation);
        }
    });
    if (n.d_weight || n.d_bias)
        hipLaunchKernelGGL(ColumnsKernel, dim3((2 * n.channels + 63) / 64), dim3(1024), 0, stream, parts,
                           static_cast<float *>(n.d_weight), static_cast<float *>(n.d_bias), rows, n.channels);
}

bool Fits(const Norm *n) {
    if (!n || n->type < 0 || n->type > 2) return Failed("expected a group norm of the type 0, 1 or 2"), false;
    if (n->activation < kNone || n->activation > kSilu) return Failed("expected an activation from 0 to 2"), false;
    if (n->batch < 0 || n->pixels < 0 || n->channels < 1 || n->groups < 1 || n->channels % n->groups)
        return Failed("expected channels that are a multiple of the groups"), false;
    // A grid has fewer than 2^32 threads: at most 1,024 a workgroup, and 64 a group of a map.
    if ((long long)n->batch * n->groups >= (1ll << 22)) return Failed("expected fewer than 2^22 groups in the batch"), false;
    return true;
}

}  // namespace
}  // namespace layers

using namespace layers;

extern "C" __attribute__((visibility("default"))) unsigned long long cuju_group_norm_workspace(const struct cuju_group_norm *norm) {
    if (!Fits(norm)) return 0;
    const Norm &n = *norm;
    return ((unsigned long long)n.batch * CutsOf(n) * 2 * n.channels + 2ull * n.batch * n.groups) * sizeof(float);
}

extern "C" __attribute__((visibility("default"))) int cuju_group_norm_forward(const struct cuju_group_norm *norm, void *stream) {
    if (!Fits(norm)) return -1;
    const Norm &n = *norm;
    if (n.batch == 0 || n.pixels == 0) return 0;
    if (!n.x || !n.y || !n.stats || !n.workspace) return Failed("expected a map, its output, statistics and workspace");
    ForType(n.type, [&](auto x) { Forward<decltype(x)>(n, static_cast<hipStream_t>(stream)); });
    return Launched("group norm");
}

extern "C" __attribute__((visibility("default"))) int cuju_group_norm_backward(const struct cuju_group_norm *norm, void *stream) {
    if (!Fits(norm)) return -1;
    const Norm &n = *norm;
    if (n.batch == 0 || n.pixels == 0) return 0;
    if (!n.x || !n.dy || !n.dx || !n.stats || !n.workspace)
        return Failed("expected a map, its gradients, statistics and workspace");
    ForType(n.type, [&](auto x) { Backward<decltype(x)>(n, static_cast<hipStream_t>(stream)); });
    return Launched("the gradients of group norm");
}
