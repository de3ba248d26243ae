// Group norm with an activation over channels-last maps [batch][pixels][channels], and its gradients.
//
//   xh = (x - mean) inverse, z = weight xh + bias, y = act(z); mean and inverse = 1 / sqrt(variance +
//   epsilon) over the pixels and the group's channels;
//   dz = dy act'(z), d_bias = sum dz, d_weight = sum dz xh over batch and pixels;
//   dx = inverse (weight dz - mean(weight dz) - xh mean(weight dz xh)), means over the group.
//
// All sums are in 32 bits or more. A workgroup that can hold a map (or the channels of some of its
// groups) in registers reads it once: mean, then the squares about the mean, then the output.
// Larger maps are read twice, cut over workgroups, with their sums in a workspace between. Both are bound
// by memory: 600 bfloat16 maps of 432 KB, read twice and written once, 796 MB, take 165 us, 4.8 TB/s; 600
// of 216 KB 76 us and their gradients, 663 MB, 148 us, 4.5 TB/s.
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
template <int Vector, class Sum>
__device__ __forceinline__ void ChannelSums(Sum (&v)[Vector], Sum *scratch, Sum *out, const Shape &s) {
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
        Sum sum = 0;
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

// The workgroup's packs: thread by thread, `Packs` rows of threads one after the other. A pack past the
// map's end is a copy of the first pixel, so that all loads are alike; what is made of it is left out.
template <class T, int Vector, int Packs>
struct Held {
    Pack<T, Vector> x[Packs];
    __device__ __forceinline__ void Load(const T *from, const Shape &s, int row, int rows, bool mine) {
        const T *p = from + (long long)row * s.channels;
        const long long step = (long long)rows * s.channels;
#pragma unroll
        for (int i = 0; i < Packs; i++, p += step) {
            // Whole rows of threads first, without a comparison of their own.
            if ((i + 1) * rows <= s.pixels) {
                if (mine) x[i] = *reinterpret_cast<const Pack<T, Vector> *>(p);
            } else if (i * rows < s.pixels) {
                if (mine) x[i] = *reinterpret_cast<const Pack<T, Vector> *>(i * rows + row < s.pixels ? p : from);
            }
        }
    }
};
// The packs' body, for each that the map has: body(i, whether this thread's is past the end).
template <int Packs, class Body>
__device__ __forceinline__ void ForPacks(const Shape &s, int row, int rows, Body body) {
#pragma unroll
    for (int i = 0; i < Packs; i++)
        if (i * rows < s.pixels) body(i, i * rows + row >= s.pixels);
}

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
    Held<T, Vector, Packs> held{};
    held.Load(x + base, s, row, rows, mine);
    const float count = 1.f / ((float)s.pixels * s.perGroup);
    float mean[Vector], sum[Vector];
#pragma unroll
    for (int c = 0; c < Vector; c++) sum[c] = 0;
    ForPacks<Packs>(s, row, rows, [&](int i, bool past) {
#pragma unroll
        for (int c = 0; c < Vector; c++) sum[c] += past ? 0.f : Float(held.x[i].x[c]);
    });
    ChannelSums<Vector>(sum, scratch, channelSums, s);
    GroupSums(channelSums, means, s);
#pragma unroll
    for (int c = 0; c < Vector; c++) {
        mean[c] = mine ? means[(vector * Vector + c) / s.perGroup] * count : 0.f;
        sum[c] = 0;
    }
    ForPacks<Packs>(s, row, rows, [&](int i, bool past) {
#pragma unroll
        for (int c = 0; c < Vector; c++) {
            const float d = past ? 0.f : Float(held.x[i].x[c]) - mean[c];
            sum[c] = fmaf(d, d, sum[c]);
        }
    });
    ChannelSums<Vector>(sum, scratch, channelSums, s);
    GroupSums(channelSums, squares, s);
    const int slabGroups = s.slabChannels / s.perGroup;
    if (stats)
        for (int i = threadIdx.x; i < slabGroups; i += Threads) {
            float *to = stats + (n * s.groups + slab * slabGroups + i) * 2;
            to[0] = means[i] * count;
            to[1] = 1.f / sqrtf(squares[i] * count + epsilon);
        }
    if (!mine) return;
    float scale[Vector], shift[Vector];
#pragma unroll
    for (int c = 0; c < Vector; c++) {
        scale[c] = 1.f / sqrtf(squares[(vector * Vector + c) / s.perGroup] * count + epsilon);
        shift[c] = bias ? bias[channel + c] : 0.f;
        if (weight) scale[c] *= weight[channel + c];
    }
    T *to = y + base + (long long)row * s.channels;
    const long long step = (long long)rows * s.channels;
    ForPacks<Packs>(s, row, rows, [&](int i, bool past) {
        Pack<T, Vector> out;
#pragma unroll
        for (int c = 0; c < Vector; c++)
            out.x[c] = As<T>(Activate(fmaf(Float(held.x[i].x[c]) - mean[c], scale[c], shift[c]), activation));
        if (!past) *reinterpret_cast<Pack<T, Vector> *>(to + i * step) = out;
    });
}

template <class T, int Vector, int Packs, int Threads>
__global__ __launch_bounds__(Threads) void BackwardKernel(const T *x, const T *dy, T *dx, const float *weight,
                                                          const float *bias, const float *stats, float *parts, Shape s,
                                                          int activation) {
    __shared__ float scratch[Threads / 64 * 64 * Vector], biasSums[64 * Vector], weightSums[64 * Vector];
    __shared__ float first[64 * Vector], second[64 * Vector];
    const unsigned id = Place(blockIdx.x, gridDim.x);
    const int slab = id % s.slabs;
    const long long n = id / s.slabs;
    const int vector = threadIdx.x & (s.lanes - 1), row = threadIdx.x / s.lanes, rows = Threads / s.lanes;
    const bool mine = vector < s.vectors;
    const int channel = slab * s.slabChannels + vector * Vector;
    const long long base = n * s.pixels * s.channels + channel;
    Held<T, Vector, Packs> v{}, d{};
    v.Load(x + base, s, row, rows, mine);
    d.Load(dy + base, s, row, rows, mine);
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
    ForPacks<Packs>(s, row, rows, [&](int i, bool past) {
#pragma unroll
        for (int c = 0; c < Vector; c++) {
            const float xh = (Float(v.x[i].x[c]) - mean[c]) * inverse[c];
            const float dz = past ? 0.f : Float(d.x[i].x[c]) * Slope(fmaf(w[c], xh, shift[c]), activation);
            sumB[c] += dz;
            sumW[c] = fmaf(dz, xh, sumW[c]);
        }
    });
    ChannelSums<Vector>(sumB, scratch, biasSums, s);
    ChannelSums<Vector>(sumW, scratch, weightSums, s);
    for (int c = threadIdx.x; c < s.slabChannels; c += Threads) {
        const int at = slab * s.slabChannels + c;
        if (parts) {
            parts[(n * 2 + 0) * s.channels + at] = weightSums[c];
            parts[(n * 2 + 1) * s.channels + at] = biasSums[c];
        }
        const float each = weight ? weight[at] : 1.f;
        biasSums[c] *= each, weightSums[c] *= each;
    }
    __syncthreads();
    GroupSums(biasSums, first, s);
    GroupSums(weightSums, second, s);
    if (!mine) return;
    const float count = 1.f / ((float)s.pixels * s.perGroup);
    float m1[Vector], m2[Vector];
#pragma unroll
    for (int c = 0; c < Vector; c++) {
        m1[c] = first[(vector * Vector + c) / s.perGroup] * count;
        m2[c] = second[(vector * Vector + c) / s.perGroup] * count;
    }
    T *to = dx + base + (long long)row * s.channels;
    const long long step = (long long)rows * s.channels;
    ForPacks<Packs>(s, row, rows, [&](int i, bool past) {
        Pack<T, Vector> out;
#pragma unroll
        for (int c = 0; c < Vector; c++) {
            const float xh = (Float(v.x[i].x[c]) - mean[c]) * inverse[c];
            const float dz = Float(d.x[i].x[c]) * Slope(fmaf(w[c], xh, shift[c]), activation);
            out.x[c] = As<T>(inverse[c] * (fmaf(w[c], dz, -m1[c]) - xh * m2[c]));
        }
        if (!past) *reinterpret_cast<Pack<T, Vector> *>(to + i * step) = out;
    });
}

// ------------------------------------------------------------- maps that no workgroup's registers hold

constexpr int kSplitThreads = 256;

// A workgroup's part: a slab of a map, and a cut of its pixels. The second reading goes backwards, from what
// the first read last and the last-level cache still holds: 600 bfloat16 maps of 432 KB 168 us against 179, their
// gradients 291 against 305; 4,096 maps of 54 KB 129 against 136, 225 against 244.
struct Cut {
    int vector, first, step, end, slab, channel, channels;
    long long map;
    bool mine;
    __device__ Cut(const Shape &s, int Vector, bool backwards) {
        const unsigned place = backwards ? gridDim.x - 1 - blockIdx.x : blockIdx.x;
        const int cut = backwards ? gridDim.y - 1 - blockIdx.y : blockIdx.y;
        vector = threadIdx.x & (s.lanes - 1);
        slab = place % s.slabs * s.slabChannels;
        map = place / s.slabs;
        channel = slab + vector * Vector;
        channels = min(s.slabChannels, s.channels - slab);
        mine = vector * Vector < channels;
        const int each = (s.pixels + gridDim.y - 1) / gridDim.y;
        step = kSplitThreads / s.lanes;
        first = cut * each + threadIdx.x / s.lanes;
        end = min(s.pixels, (cut + 1) * each);
    }
};

// A cut's pixels, four of a thread's at a time, so that their loads are on the way together: load(n, p)
// for each, then body(n, p).
constexpr int kAhead = 4;
template <class Load, class Body>
__device__ __forceinline__ void ForPixels(const Cut &cut, Load load, Body body) {
    int p = cut.first;
    for (; p + (kAhead - 1) * cut.step < cut.end; p += kAhead * cut.step) {
#pragma unroll
        for (int n = 0; n < kAhead; n++) load(n, p + n * cut.step);
#pragma unroll
        for (int n = 0; n < kAhead; n++) body(n, p + n * cut.step);
    }
    for (; p < cut.end; p += cut.step) load(0, p), body(0, p);
}

// Pixels of a cut.
__device__ __forceinline__ int PixelsOf(const Shape &s, int cuts, int cut) {
    const int each = (s.pixels + cuts - 1) / cuts;
    return max(0, min(s.pixels, (cut + 1) * each) - cut * each);
}

// Each channel's mean over a cut, and the squares about it: [map][cut][2][channels]. The sums are in 64 bits, so
// that the squares lose nothing where values lie far from zero or a few lie far from the rest; the squares about a
// cut's own mean are then sums of nothing below zero, which 32 bits hold.
template <class T, int Vector>
__global__ __launch_bounds__(kSplitThreads) void SumsKernel(const T *x, float *parts, Shape s) {
    __shared__ double scratch[kSplitThreads * Vector], sums[64 * Vector], squares[64 * Vector];
    const Cut cut(s, Vector, false);
    const T *at = x + cut.map * s.pixels * s.channels + cut.channel;
    double sum[Vector], square[Vector];
#pragma unroll
    for (int c = 0; c < Vector; c++) sum[c] = square[c] = 0;
    Pack<T, Vector> v[kAhead];
    if (cut.mine)
        ForPixels(cut, [&](int n, int p) { v[n] = *reinterpret_cast<const Pack<T, Vector> *>(at + (long long)p * s.channels); },
                  [&](int n, int) {
#pragma unroll
                      for (int c = 0; c < Vector; c++) {
                          const double d = Float(v[n].x[c]);
                          sum[c] += d;
                          square[c] = fma(d, d, square[c]);
                      }
                  });
    Shape slab = s;
    slab.vectors = cut.channels / Vector;
    slab.slabChannels = cut.channels;
    ChannelSums<Vector>(sum, scratch, sums, slab);
    ChannelSums<Vector>(square, scratch, squares, slab);
    const int count = PixelsOf(s, gridDim.y, blockIdx.y);
    float *to = parts + (cut.map * gridDim.y + blockIdx.y) * 2 * s.channels + cut.slab;
    for (int c = threadIdx.x; c < cut.channels; c += kSplitThreads) {
        const double mean = count ? sums[c] / count : 0.0, about = squares[c] - sums[c] * mean;
        to[c] = (float)mean;
        // A comparison that keeps a NaN.
        to[s.channels + c] = about < 0.0 ? 0.f : (float)about;
    }
}
// A sum of `value(channel, cut)` over a group's channels and all cuts, the same in every lane of a
// wavefront.
template <class Value>
__device__ __forceinline__ double GroupSum(const Shape &s, int group, int cuts, Value value) {
    double total = 0;
    for (int i = threadIdx.x & 63; i < s.perGroup * cuts; i += 64) total += value(group * s.perGroup + i % s.perGroup, i / s.perGroup);
    for (int d = 1; d < 64; d *= 2) total += __shfl_xor(total, d);
    return total;
}
__device__ __forceinline__ double PartOf(const float *parts, const Shape &s, long long n, int cuts, int cut, int k, int c) {
    return parts[((n * cuts + cut) * 2 + k) * s.channels + c];
}
// A group's mean and inverse deviation from the cuts' means and squares, in 64 bits, by a wavefront. An infinity
// leaves its group neither: the squares are NaN.
__device__ __forceinline__ float2 StatsOf(const float *parts, const Shape &s, long long n, int group, int cuts, float epsilon) {
    const double count = (double)s.pixels * s.perGroup;
    const double mean = GroupSum(s, group, cuts, [&](int c, int cut) {
                            return PixelsOf(s, cuts, cut) * PartOf(parts, s, n, cuts, cut, 0, c);
                        }) / count;
    const double squares = GroupSum(s, group, cuts, [&](int c, int cut) {
        const double off = PartOf(parts, s, n, cuts, cut, 0, c) - mean;
        return fma(PixelsOf(s, cuts, cut) * off, off, PartOf(parts, s, n, cuts, cut, 1, c));
    });
    return float2{(float)mean, (float)(1.0 / sqrt(squares / count + epsilon))};
}
// The means of weight dz and of weight dz xh over a group, by a wavefront.
__device__ __forceinline__ float2 MeansOf(const float *parts, const float *weight, const Shape &s, long long n, int group,
                                          int cuts) {
    float2 means;
    const double count = (double)s.pixels * s.perGroup;
    for (int k = 0; k < 2; k++) {
        const double total = GroupSum(s, group, cuts, [&](int c, int cut) {
            const double sum = PartOf(parts, s, n, cuts, cut, k, c);
            return weight ? sum * weight[c] : sum;
        });
        (k ? means.x : means.y) = (float)(total / count);
    }
    return means;
}
// Slabs of whole groups, up to this many, find their groups' statistics themselves; others have a
// kernel of a wavefront a group for it.
constexpr int kMostGroups = 128;
__global__ __launch_bounds__(64) void StatsKernel(const float *parts, float2 *stats, Shape s, long long count, int cuts, float epsilon) {
    for (long long i = blockIdx.x; i < count; i += gridDim.x) {
        const float2 found = StatsOf(parts, s, i / s.groups, i % s.groups, cuts, epsilon);
        if (threadIdx.x == 0) stats[i] = found;
    }
}
__global__ __launch_bounds__(64) void MeansKernel(const float *parts, const float *weight, float2 *means, Shape s, long long count,
                                                  int cuts) {
    for (long long i = blockIdx.x; i < count; i += gridDim.x) {
        const float2 found = MeansOf(parts, weight, s, i / s.groups, i % s.groups, cuts);
        if (threadIdx.x == 0) means[i] = found;
    }
}
// Their grid: a workgroup a group, up to a number far past what the chip holds at once.
dim3 GroupGrid(const Norm &n) {
    const long long groups = (long long)n.batch * n.groups;
    return dim3((unsigned)(groups < (1 << 20) ? groups : 1 << 20));
}

template <class T, int Vector>
__global__ __launch_bounds__(kSplitThreads) void ApplyKernel(const T *x, T *y, const float *weight, const float *bias,
                                                             const float *parts, float2 *stats, Shape s, float epsilon,
                                                             int activation) {
    __shared__ float2 found[kMostGroups];
    const Cut cut(s, Vector, true);
    const long long n = cut.map, base = n * s.pixels * s.channels + cut.channel;
    const int firstGroup = cut.slab / s.perGroup;
    if (parts) {
        for (int i = threadIdx.x >> 6; i < cut.channels / s.perGroup; i += kSplitThreads / 64) {
            const float2 each = StatsOf(parts, s, n, firstGroup + i, gridDim.y, epsilon);
            if ((threadIdx.x & 63) == 0) {
                found[i] = each;
                if (blockIdx.y == 0) stats[n * s.groups + firstGroup + i] = each;
            }
        }
        __syncthreads();
    }
    if (!cut.mine) return;
    float mean[Vector], scale[Vector], shift[Vector];
#pragma unroll
    for (int c = 0; c < Vector; c++) {
        const int group = (cut.channel + c) / s.perGroup;
        const float2 each = parts ? found[group - firstGroup] : stats[n * s.groups + group];
        mean[c] = each.x;
        scale[c] = each.y * (weight ? weight[cut.channel + c] : 1.f);
        shift[c] = bias ? bias[cut.channel + c] : 0.f;
    }
    Pack<T, Vector> v[kAhead];
    ForPixels(cut, [&](int n, int p) { v[n] = *reinterpret_cast<const Pack<T, Vector> *>(x + base + (long long)p * s.channels); },
              [&](int n, int p) {
                  Pack<T, Vector> out;
#pragma unroll
                  for (int c = 0; c < Vector; c++)
                      out.x[c] = As<T>(Activate(fmaf(Float(v[n].x[c]) - mean[c], scale[c], shift[c]), activation));
                  *reinterpret_cast<Pack<T, Vector> *>(y + base + (long long)p * s.channels) = out;
              });
}
// The gradients' channel sums: [map][cut][2][channels], of dz xh and of dz.
template <class T, int Vector>
__global__ __launch_bounds__(kSplitThreads) void GradientSumsKernel(const T *x, const T *dy, const float *weight,
                                                                    const float *bias, const float *stats, float *parts,
                                                                    Shape s, int activation) {
    __shared__ float scratch[kSplitThreads * Vector], out[64 * Vector];
    const Cut cut(s, Vector, false);
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
    Pack<T, Vector> v[kAhead], d[kAhead];
    const auto load = [&](int n, int p) {
        v[n] = *reinterpret_cast<const Pack<T, Vector> *>(x + base + (long long)p * s.channels);
        d[n] = *reinterpret_cast<const Pack<T, Vector> *>(dy + base + (long long)p * s.channels);
    };
    if (cut.mine)
        ForPixels(cut, load, [&](int n, int) {
#pragma unroll
            for (int c = 0; c < Vector; c++) {
                const float xh = (Float(v[n].x[c]) - mean[c]) * inverse[c];
                const float dz = Float(d[n].x[c]) * Slope(fmaf(w[c], xh, shift[c]), activation);
                sumB[c] += dz;
                sumW[c] = fmaf(dz, xh, sumW[c]);
            }
        });
    Shape slab = s;
    slab.vectors = cut.channels / Vector;
    float *to = parts + (n * gridDim.y + blockIdx.y) * 2 * s.channels + cut.slab;
    for (int k = 0; k < 2; k++) {
        ChannelSums<Vector>(k ? sumB : sumW, scratch, out, slab);
        for (int c = threadIdx.x; c < cut.channels; c += kSplitThreads) to[k * s.channels + c] = out[c];
        __syncthreads();
    }
}
template <class T, int Vector>
__global__ __launch_bounds__(kSplitThreads) void GradientKernel(const T *x, const T *dy, T *dx, const float *weight,
                                                                const float *bias, const float2 *stats, const float *parts,
                                                                const float2 *means, Shape s, int activation) {
    __shared__ float2 found[kMostGroups];
    const Cut cut(s, Vector, true);
    const long long n = cut.map, base = n * s.pixels * s.channels + cut.channel;
    const int firstGroup = cut.slab / s.perGroup;
    if (parts) {
        for (int i = threadIdx.x >> 6; i < cut.channels / s.perGroup; i += kSplitThreads / 64) {
            const float2 each = MeansOf(parts, weight, s, n, firstGroup + i, gridDim.y);
            if ((threadIdx.x & 63) == 0) found[i] = each;
        }
        __syncthreads();
    }
    if (!cut.mine) return;
    float mean[Vector], inverse[Vector], w[Vector], shift[Vector], m1[Vector], m2[Vector];
#pragma unroll
    for (int c = 0; c < Vector; c++) {
        const int group = (cut.channel + c) / s.perGroup;
        const float2 each = stats[n * s.groups + group];
        const float2 over = parts ? found[group - firstGroup] : means[n * s.groups + group];
        mean[c] = each.x, inverse[c] = each.y;
        m1[c] = over.x, m2[c] = over.y;
        w[c] = weight ? weight[cut.channel + c] : 1.f;
        shift[c] = bias ? bias[cut.channel + c] : 0.f;
    }
    Pack<T, Vector> v[kAhead], d[kAhead];
    const auto load = [&](int n, int p) {
        v[n] = *reinterpret_cast<const Pack<T, Vector> *>(x + base + (long long)p * s.channels);
        d[n] = *reinterpret_cast<const Pack<T, Vector> *>(dy + base + (long long)p * s.channels);
    };
    ForPixels(cut, load, [&](int n, int p) {
        Pack<T, Vector> out;
#pragma unroll
        for (int c = 0; c < Vector; c++) {
            const float xh = (Float(v[n].x[c]) - mean[c]) * inverse[c];
            const float dz = Float(d[n].x[c]) * Slope(fmaf(w[c], xh, shift[c]), activation);
            out.x[c] = As<T>(inverse[c] * (fmaf(w[c], dz, -m1[c]) - xh * m2[c]));
        }
        *reinterpret_cast<Pack<T, Vector> *>(dx + base + (long long)p * s.channels) = out;
    });
}

// The sums over maps (and cuts) of [rows][2][channels]: 16 columns a workgroup, 64 rows at a time.
__global__ __launch_bounds__(1024) void ColumnsKernel(const float *parts, float *dWeight, float *dBias, long long rows,
                                                      int channels) {
    __shared__ float sums[64][16];
    const int column = blockIdx.x * 16 + (threadIdx.x & 15), slot = threadIdx.x >> 4;
    float sum = 0;
    if (column < 2 * channels) {
        const float *at = parts + column;
        long long i = slot;
        for (; i + 3 * 64 < rows; i += 4 * 64) {
            float x[4];
#pragma unroll
            for (int n = 0; n < 4; n++) x[n] = at[(i + n * 64) * 2 * channels];
            sum += (x[0] + x[1]) + (x[2] + x[3]);
        }
        for (; i < rows; i += 64) sum += at[i * 2 * channels];
    }
    sums[slot][threadIdx.x & 15] = sum;
    for (int half = 32; half > 0; half /= 2) {
        __syncthreads();
        if (slot < half) sums[slot][threadIdx.x & 15] += sums[slot + half][threadIdx.x & 15];
    }
    if (slot == 0 && column < 2 * channels) {
        float *to = column < channels ? dWeight : dBias;
        if (to) to[column < channels ? column : column - channels] = sums[0][threadIdx.x];
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
// The largest pack of elements that the channels and the tensors' alignment allow, in elements, up to
// four: with eight, a thread's sums, scales and shifts of as many channels halve the wavefronts on a
// SIMD (600 bfloat16 maps of 216 KB: the gradients 147 us with eight, 140 with four; 64 maps of 432 KB
// 55 and 43).
int VectorOf(const Norm &n) {
    const int size = n.type == 0 ? 4 : 2;
    uintptr_t all = reinterpret_cast<uintptr_t>(n.x) | reinterpret_cast<uintptr_t>(n.y) |
                    reinterpret_cast<uintptr_t>(n.dy) | reinterpret_cast<uintptr_t>(n.dx);
    int vector = 4;
    while (vector > 1 && (n.channels % vector || all % (vector * size))) vector /= 2;
    return vector;
}
// The first count of slabs up to `most` (each of whole groups and whole packs) whose pixels fit `packs` packs
// of each of `threads` threads; 0 if none does.
//
// Which maps a workgroup holds (us, held against cut, forward; then the gradients):
//  - up to 16 KB, 256 threads: 4,000 bfloat16 maps of 16 KB 38 against 47; 63 against 75;
//  - floats up to 224 KB (112 KB with their gradient) in one or two slabs, 512 threads: 4,000 maps of
//    108 KB 187 against 269; 325 against 436. In four slabs, 600 maps of 432 KB, 171 against 166.
//  - 16-bit maps past 16 KB are cut: a pack of four is 8 bytes there, and 4,000 maps of 32 KB took 100
//    against 68; 149 against 133.
int SlabsFor(const Norm &n, int vector, int packs, int threads, int most) {
    for (int slabs = 1; slabs <= most; slabs++) {
        if (n.groups % slabs || n.channels / slabs % vector) continue;
        const Shape s = SlabsOf(n, slabs, vector);
        if (s.lanes <= 64 && s.pixels <= (long long)packs * (threads / s.lanes)) return slabs;
    }
    return 0;
}
// Other maps: channels in slabs of at most a wavefront of packs, of whole groups where they have it.
Shape SplitShape(const Norm &n, int vector) {
    Shape s{n.pixels, n.channels, n.groups, n.channels / n.groups, 1, n.channels, 0, 0};
    if (n.channels > 64 * vector) {
        int whole = s.perGroup;
        while (whole % vector) whole += s.perGroup;
        s.slabChannels = whole <= 64 * vector ? 64 * vector / whole * whole : 64 * vector;
    }
    s.slabs = (n.channels + s.slabChannels - 1) / s.slabChannels;
    s.vectors = s.slabChannels / vector;
    s.lanes = PowerOfTwo(s.vectors);
    return s;
}
bool FindsItself(const Shape &s) { return s.slabChannels % s.perGroup == 0 && s.slabChannels / s.perGroup <= kMostGroups; }
// Pixels are cut so that about 2,048 workgroups run, with at least 16 KB each.
int CutsOf(const Norm &n) {
    const long long bytes = (long long)n.pixels * n.channels * (n.type == 0 ? 4 : 2);
    long long cuts = n.batch > 0 ? 2048 / n.batch : 1;
    if (cuts > bytes / 16384) cuts = bytes / 16384;
    return (int)(cuts < 1 ? 1 : cuts > 64 ? 64 : cuts);
}

// Packs of `bytes` of a thread's registers.
template <class T, int Vector>
constexpr int Packs(int bytes) {
    return bytes / (Vector * (int)sizeof(T)) < bytes / 8 ? bytes / (Vector * (int)sizeof(T)) : bytes / 8;
}

template <class Body>
void ForVector(int vector, Body body) {
    switch (vector) {
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
        const auto resident = [&](auto kernel, int slabs, int threads) {
            hipLaunchKernelGGL(kernel, dim3((unsigned)((long long)n.batch * slabs)), dim3(threads), 0, stream, x, y,
                               weight, bias, stats, SlabsOf(n, slabs, V), n.epsilon, n.activation);
        };
        if (SlabsFor(n, V, Packs<T, V>(64), 256, 1)) return resident(ForwardKernel<T, V, Packs<T, V>(64), 256>, 1, 256);
        if constexpr (sizeof(T) == 4)
            if (const int slabs = SlabsFor(n, V, Packs<T, V>(224), 512, 2))
                return resident(ForwardKernel<T, V, Packs<T, V>(224), 512>, slabs, 512);
        const Shape s = SplitShape(n, V);
        const int cuts = CutsOf(n);
        const dim3 grid((unsigned)((long long)s.slabs * n.batch), cuts);
        hipLaunchKernelGGL((SumsKernel<T, V>), grid, dim3(kSplitThreads), 0, stream, x, work, s);
        float2 *found = reinterpret_cast<float2 *>(stats);
        if (!FindsItself(s))
            hipLaunchKernelGGL(StatsKernel, GroupGrid(n), dim3(64), 0, stream, work, found, s, (long long)n.batch * n.groups,
                               cuts, n.epsilon);
        hipLaunchKernelGGL((ApplyKernel<T, V>), grid, dim3(kSplitThreads), 0, stream, x, y, weight, bias,
                           FindsItself(s) ? work : nullptr, found, s, n.epsilon, n.activation);
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
    const bool summed = n.d_weight || n.d_bias;
    long long rows = n.batch;
    ForVector(vector, [&](auto wide) {
        constexpr int V = decltype(wide)::value;
        const auto resident = [&](auto kernel, int slabs, int threads) {
            hipLaunchKernelGGL(kernel, dim3((unsigned)((long long)n.batch * slabs)), dim3(threads), 0, stream, x, dy, dx,
                               weight, bias, stats, summed ? parts : nullptr, SlabsOf(n, slabs, V), n.activation);
        };
        if (SlabsFor(n, V, Packs<T, V>(64), 256, 1)) return resident(BackwardKernel<T, V, Packs<T, V>(64), 256>, 1, 256);
        if constexpr (sizeof(T) == 4)
            if (const int slabs = SlabsFor(n, V, Packs<T, V>(112), 512, 2))
                return resident(BackwardKernel<T, V, Packs<T, V>(112), 512>, slabs, 512);
        const Shape s = SplitShape(n, V);
        const int cuts = CutsOf(n);
        rows = (long long)n.batch * cuts;
        float2 *means = reinterpret_cast<float2 *>(parts + rows * 2 * n.channels);
        const dim3 grid((unsigned)((long long)s.slabs * n.batch), cuts);
        hipLaunchKernelGGL((GradientSumsKernel<T, V>), grid, dim3(kSplitThreads), 0, stream, x, dy, weight, bias, stats,
                           parts, s, n.activation);
        if (!FindsItself(s))
            hipLaunchKernelGGL(MeansKernel, GroupGrid(n), dim3(64), 0, stream, parts, weight, means, s,
                               (long long)n.batch * n.groups, cuts);
        hipLaunchKernelGGL((GradientKernel<T, V>), grid, dim3(kSplitThreads), 0, stream, x, dy, dx, weight, bias,
                           reinterpret_cast<const float2 *>(stats), FindsItself(s) ? parts : nullptr, means, s, n.activation);
    });
    if (summed)
        hipLaunchKernelGGL(ColumnsKernel, dim3((2 * n.channels + 15) / 16), dim3(1024), 0, stream, parts,
                           static_cast<float *>(n.d_weight), static_cast<float *>(n.d_bias), rows, n.channels);
}

bool Fits(const Norm *n) {
    if (!n || n->type < 0 || n->type > 2) return Failed("expected a group norm of the type 0, 1 or 2"), false;
    if (n->activation < kNone || n->activation > kSilu) return Failed("expected an activation from 0 to 2"), false;
    if (n->batch < 0 || n->pixels < 0 || n->channels < 1 || n->groups < 1 || n->channels % n->groups)
        return Failed("expected channels that are a multiple of the groups"), false;
    // Places within a map are ints, and a grid has fewer than 2^32 threads: at most 512 for each of two slabs
    // of a map, 256 for each slab of a map that is cut (of 33 channels and more), 128 for each channel of a map.
    if ((long long)n->pixels * n->channels >= (1ll << 30) || n->channels >= (1 << 24))
        return Failed("expected fewer than 2^30 values and 2^24 channels in a map"), false;
    if (n->batch >= (1 << 22) || (long long)n->batch * n->channels >= (1ll << 29))
        return Failed("expected fewer than 2^22 maps and 2^29 channels in the batch"), false;
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
