// Gradients clipped by their global norm: n = sqrt(sum g^2) over all values of all tensors, and g *= min(1, most / (n + epsilon)).
//
// Squares are summed in 64 bits, so that no value of 32 bits is too large or too small, in an order that is always the
// same. Two kernels: the sums of squares by workgroup, and the factor, which each workgroup finds again from those sums,
// with the scaling. Where the factor is 1 nothing is written. Memory bounds it: 1.9 GB of gradients take 350 to 370 us to read
// (5.3 TB/s) and 700 to 710 to scale in place (5.4 TB/s, of 5.9).
#include "../../../include/cuju_amd.h"
#include "common.h"

#include <algorithm>
#include <cmath>
#include <exception>
#include <limits>
#include <utility>
#include <vector>

namespace layers {
namespace {

using Gradients = cuju_gradients;

// The tensors of a launch lie in the kernel's arguments, cut into tiles of kTile bytes each. Small tiles spread a small
// policy's gradients over the chip, large ones have fewer searches for their tensor and loads in a row. Measured for
// float tensors of 1, 8, 32 and 2,000 MB in all: tiles of 8 KB 8.5, 16.5, 35.8 and 2,133 us, of 32 KB 7.7, 12.1, 21.8 and
// 1,105, of 128 KB 9.2, 16.5, 21.0 and 1,086. Of 512, 1,024 and 2,048 workgroups none is faster.
constexpr int kTensors = 128, kThreads = 256, kMostBlocks = 1024, kUnroll = 4, kTile = 32 << 10;
struct Table {
    void *data[kTensors];
    long long size[kTensors];
    int tiles[kTensors + 1];  // before each tensor
    unsigned char type[kTensors];
    int count;
};

template <class T, int N>
struct __attribute__((packed, aligned(sizeof(T)))) Loose {
    T x[N];
};

__device__ __forceinline__ double BlockSum(double x) {
    __shared__ double sums[kThreads / 64];
#pragma unroll
    for (int d = 1; d < 64; d *= 2) x += __shfl_xor(x, d);
    if ((threadIdx.x & 63) == 0) sums[threadIdx.x >> 6] = x;
    __syncthreads();
    x = 0;
#pragma unroll
    for (int w = 0; w < kThreads / 64; w++) x += sums[w];
    return x;
}

// body(pointer to the first value of a tile, its values) with the tensor's element type, for the tiles of this workgroup.
template <class Body>
__device__ __forceinline__ void ForTiles(const Table &table, bool backwards, Body body) {
    const int tiles = table.tiles[table.count];
    for (int place = blockIdx.x; place < tiles; place += gridDim.x) {
        const int n = backwards ? tiles - 1 - place : place;
        int low = 0, high = table.count;
        while (high - low > 1) {
            const int middle = (low + high) / 2;
            if (table.tiles[middle] <= n) low = middle;
            else high = middle;
        }
        const auto tile = [&](auto element) {
            using T = decltype(element);
            const long long values = kTile / sizeof(T), first = (n - table.tiles[low]) * values;
            body(Global(static_cast<T *>(table.data[low])) + first, (int)min(values, table.size[low] - first));
        };
        if (table.type[low] == 0) tile(float());
        else if (table.type[low] == 1) tile(__hip_bfloat16());
        else tile(__half());
    }
}

__global__ __launch_bounds__(kThreads) void SquaresKernel(Table table, double *sums) {
    double sum = 0;
    ForTiles(table, false, [&](auto *data, int values) {
        using T = std::remove_reference_t<decltype(*data)>;
        constexpr int N = 16 / sizeof(T);
        int at = threadIdx.x * N;
        for (; at + (kUnroll - 1) * kThreads * N + N <= values; at += kUnroll * kThreads * N) {
            Loose<T, N> x[kUnroll];
#pragma unroll
            for (int i = 0; i < kUnroll; i++) x[i] = *reinterpret_cast<const Loose<T, N> *>(data + at + i * kThreads * N);
#pragma unroll
            for (int i = 0; i < kUnroll; i++)
#pragma unroll
                for (int c = 0; c < N; c++) {
                    const double v = Float(x[i].x[c]);
                    sum = fma(v, v, sum);
                }
        }
        for (; at < values; at += kThreads * N)
            for (int c = 0; c < N; c++)
                if (at + c < values) {
                    const double v = Float(data[at + c]);
                    sum = fma(v, v, sum);
                }
    });
    sum = BlockSum(sum);
    if (threadIdx.x == 0) sums[blockIdx.x] = sum;
}

__device__ __forceinline__ double NormOf(const double *sums, int count) {
    double sum = 0;
    for (int i = threadIdx.x; i < count; i += kThreads) sum += sums[i];
    return sqrt(BlockSum(sum));
}

__global__ __launch_bounds__(kThreads) void NormKernel(const double *sums, int count, float *norm) {
    const double n = NormOf(sums, count);
    if (threadIdx.x == 0) *norm = (float)n;
}

__global__ __launch_bounds__(kThreads) void ClipKernel(Table table, const double *sums, int count, double most, double epsilon, float *norm) {
    const double n = NormOf(sums, count);
    if (norm && blockIdx.x == 0 && threadIdx.x == 0) *norm = (float)n;
    const double whole = most / (n + epsilon);
    // A comparison that keeps a NaN.
    if ((float)whole >= 1.f) return;
    // A factor that a float has no digits for is taken in two steps.
    const float factor = whole < 0x1p-100 ? 0x1p-100f : (float)whole, rest = whole < 0x1p-100 ? (float)(whole * 0x1p100) : 1.f;
    // Backwards, from what the first kernel read last and the last-level cache still holds.
    ForTiles(table, true, [&](auto *data, int values) {
        using T = std::remove_reference_t<decltype(*data)>;
        constexpr int N = 16 / sizeof(T);
        int at = threadIdx.x * N;
        for (; at + (kUnroll - 1) * kThreads * N + N <= values; at += kUnroll * kThreads * N) {
            Loose<T, N> x[kUnroll];
#pragma unroll
            for (int i = 0; i < kUnroll; i++) x[i] = *reinterpret_cast<const Loose<T, N> *>(data + at + i * kThreads * N);
#pragma unroll
            for (int i = 0; i < kUnroll; i++) {
#pragma unroll
                for (int c = 0; c < N; c++) x[i].x[c] = As<T>(Float(x[i].x[c]) * factor * rest);
                *reinterpret_cast<Loose<T, N> *>(data + at + i * kThreads * N) = x[i];
            }
        }
        for (; at < values; at += kThreads * N)
            for (int c = 0; c < N; c++)
                if (at + c < values) data[at + c] = As<T>(Float(data[at + c]) * factor * rest);
    });
}

int SizeOf(long long type) { return type == 0 ? 4 : 2; }
// body(table, workgroups) for each launch; tensors without values are left out. A launch has fewer than 2^30 tiles.
template <class Body>
void ForTables(const Gradients &g, Body body) {
    Table table{};
    const auto launch = [&] {
        if (!table.count) return;
        body(table, std::min(table.tiles[table.count], kMostBlocks));
        table.count = 0;
    };
    for (long long i = 0; i < g.count; i++) {
        const cuju_gradient &each = g.gradients[i];
        const long long most = (1ll << 28) * (kTile / SizeOf(each.type));
        // A tensor of more tiles than a launch has is cut.
        for (long long first = 0; first < each.size; first += most) {
            const long long size = std::min(most, each.size - first), tiles = (size * SizeOf(each.type) + kTile - 1) / kTile;
            if (table.count == kTensors || (table.count && table.tiles[table.count] + tiles > (1ll << 29))) launch();
            const int at = table.count++;
            table.data[at] = static_cast<char *>(each.data) + first * SizeOf(each.type), table.size[at] = size;
            table.type[at] = (unsigned char)each.type;
            table.tiles[at + 1] = table.tiles[at] + (int)tiles;
        }
    }
    launch();
}

bool Fits(const Gradients *g) {
    if (!g || g->count < 0 || (g->count > 0 && !g->gradients)) return Failed("expected gradients"), false;
    if (!(g->most >= 0) || !(g->epsilon >= 0)) return Failed("expected a norm and an epsilon of at least 0"), false;
    for (long long i = 0; i < g->count; i++) {
        const cuju_gradient &each = g->gradients[i];
        if (each.type < 0 || each.type > 2) return Failed("expected gradients of the type 0, 1 or 2"), false;
        if (each.size < 0 || each.size >= (1ll << 44)) return Failed("expected gradients of 0 to 2^44 values"), false;
        if (each.size && !each.data) return Failed("expected the data of every gradient"), false;
    }
    return true;
}
// Whether two tensors share memory: one of them would be scaled twice, and by two workgroups at a time.
bool Overlaps(const Gradients &g) {
    std::vector<std::pair<uintptr_t, uintptr_t>> ranges;
    ranges.reserve(g.count);
    for (long long i = 0; i < g.count; i++) {
        const uintptr_t first = reinterpret_cast<uintptr_t>(g.gradients[i].data);
        if (g.gradients[i].size) ranges.emplace_back(first, first + g.gradients[i].size * SizeOf(g.gradients[i].type));
    }
    std::sort(ranges.begin(), ranges.end());
    for (size_t i = 1; i < ranges.size(); i++)
        if (ranges[i].first < ranges[i - 1].second) return true;
    return false;
}

int Clip(const Gradients &g, hipStream_t stream) {
    if (Overlaps(g)) return Failed("expected gradients that do not overlap");
    double *sums = static_cast<double *>(g.workspace);
    int count = 0;
    ForTables(g, [&](const Table &table, int blocks) {
        hipLaunchKernelGGL(SquaresKernel, dim3(blocks), dim3(kThreads), 0, stream, table, sums + count);
        count += blocks;
    });
    float *norm = static_cast<float *>(g.norm);
    if (count == 0 || g.most == std::numeric_limits<double>::infinity()) {
        hipLaunchKernelGGL(NormKernel, dim3(1), dim3(kThreads), 0, stream, sums, count, norm);
        return Launched("the norm of gradients");
    }
    ForTables(g, [&](const Table &table, int blocks) {
        hipLaunchKernelGGL(ClipKernel, dim3(blocks), dim3(kThreads), 0, stream, table, sums, count, g.most, g.epsilon, norm);
        norm = nullptr;
    });
    return Launched("clipped gradients");
}

// No C++ exception leaves the library.
template <class Body>
auto Guarded(Body body, decltype(body()) otherwise) -> decltype(body()) {
    try {
        return body();
    } catch (const std::exception &e) {
        Failed(e.what());
        return otherwise;
    }
}

}  // namespace
}  // namespace layers

using namespace layers;

extern "C" __attribute__((visibility("default"))) unsigned long long cuju_clip_gradients_workspace(const struct cuju_gradients *gradients) {
    if (!Fits(gradients)) return 0;
    unsigned long long blocks = 0;
    ForTables(*gradients, [&](const Table &, int count) { blocks += count; });
    return blocks * sizeof(double);
}

extern "C" __attribute__((visibility("default"))) int cuju_clip_gradients(const struct cuju_gradients *gradients, void *stream) {
    if (!Fits(gradients)) return -1;
    const Gradients &g = *gradients;
    if (!g.norm) return Failed("expected a place for the norm");
    if (cuju_clip_gradients_workspace(gradients) && !g.workspace) return Failed("expected a workspace");
    return Guarded([&] { return Clip(g, static_cast<hipStream_t>(stream)); }, -1);
}
