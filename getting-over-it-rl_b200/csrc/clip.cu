// Gradient clipping by the global norm over many tensors (goib2d_clip_grads): norm = sqrt(sum of squares of every
// element of every tensor), then every element times min(1, max_norm / (norm + 1e-6)).
//
// Bound by the bytes: each element read and written once where the SMs can hold it in between. One launch: a block of
// an SM sums the squares of its tiles of 16 KB and keeps the first kKept of them in shared memory (28 MB on all SMs), the
// grid meets, and every block scales what it kept and then its other tiles, the last read first, which the L2 cache still
// holds some 100 MB of. The tensor table travels in the launch's parameters: a call makes no copy and keeps nothing.
// Squares are summed in float32 over a thread's 16 bytes, and from there on in float64; where such a sum leaves the
// range in which float32 carries it, in float64 from the squares on. Every block's sum goes to its own place and every
// block adds all of them in one order: the same inputs give the same bits. 63 M weights in
// bfloat16 and float32 (253 MB read and written once): 64 us from a cold L2, 54 from a warm one, 4.0 and 4.7 TB/s; where there is nothing
// to scale 37 and 31. 205 k: 6.4 us, the launch and the meeting. A block's tiles are neighbours, so that most batches of them
// lie in one tensor and need one branch and no bookkeeping a piece: with tiles a grid apart, 72 and 70 us, at 2.4 times the instructions.
#include <cooperative_groups.h>

#include "policy.cuh"

namespace gb {
namespace {

constexpr int kThreads = 1024;
constexpr int kBytes = kThreads * 16;  // of a tile
constexpr int kKept = 12;              // tiles of a block that stay in shared memory, whole batches
constexpr int kBatch = 4;              // tiles whose loads are in flight together
constexpr int kSms = 148;
constexpr int kMost = 1024;            // tensors of a launch: 20 KB of its 32 KB of parameters

enum { kSum = 1, kScale = 2 };

template <int N>
struct Table {
    int32_t n, mode;
    int32_t first, sums;               // where this launch's partial sums go; how many there are in all
    float max_norm;
    float *norm;
    double *part;
    void *ptr[N];
    int32_t end[N];                    // (tiles up to and with this tensor) << 1 | bfloat16
    int64_t numel[N];
};

// A thread's 16 bytes of a tile. Aligned tensors: neighbouring elements; others: elements kThreads apart. `left`: elements
// of the tensor from its first one on (many, where the tile is whole).
struct Piece {
    char *p;
    int64_t left;
    bool half, wide;
};

// The tensor that the last tile asked for is of: tiles lo to hi - 1.
template <int N>
struct Cursor {
    const Table<N> &T;
    int i = 0, lo = 0, hi;
    char *base;
    bool half, wide;
    __device__ __forceinline__ void tensor() {
        lo = i ? T.end[i - 1] >> 1 : 0, hi = T.end[i] >> 1, half = T.end[i] & 1, wide = (uintptr_t)T.ptr[i] % 16 == 0;
        base = (char *)T.ptr[i] + threadIdx.x * (wide ? 16 : half ? 2 : 4);
    }
    __device__ __forceinline__ explicit Cursor(const Table<N> &T) : T(T) { tensor(); }
    __device__ __forceinline__ void to(int t) {
        if (t < lo || t >= hi) {
            while (t >= T.end[i] >> 1) ++i;
            while (i > 0 && t < T.end[i - 1] >> 1) --i;
            tensor();
        }
    }
    // The thread's 16 bytes of tile t where it and the kBatch - 1 behind it are whole tiles of one aligned tensor, else NULL.
    __device__ __forceinline__ uint4 *batch(int t) {
        to(t);
        return wide && t + kBatch < hi ? (uint4 *)(base + (int64_t)(t - lo) * kBytes) : nullptr;
    }
    __device__ __forceinline__ Piece at(int t) {
        to(t);
        Piece x{base + (int64_t)(t - lo) * kBytes, 1 << 30, half, wide};
        if (t + 1 == hi) {
            const int size = half ? 2 : 4;
            x.left = T.numel[i] - (int64_t)(t - lo) * (kBytes / size) - threadIdx.x * (wide ? 16 / size : 1);
        }
        return x;
    }
};

__device__ __forceinline__ uint4 load(const Piece &x) {
    const int n = x.half ? 8 : 4;
    if (x.wide && x.left >= n) return *(const uint4 *)x.p;
    uint32_t v[4] = {};
    const int64_t step = x.wide ? 1 : kThreads;
    if (x.half) {
#pragma unroll
        for (int e = 0; e < 8; ++e)
            if (e * step < x.left) v[e / 2] |= (uint32_t)((const uint16_t *)x.p)[e * step] << e % 2 * 16;
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (e * step < x.left) v[e] = ((const uint32_t *)x.p)[e * step];
    }
    return make_uint4(v[0], v[1], v[2], v[3]);
}

__device__ __forceinline__ void store(const Piece &x, uint4 y) {
    const int n = x.half ? 8 : 4;
    if (x.wide && x.left >= n) {
        __stcs((uint4 *)x.p, y);
        return;
    }
    const uint32_t v[4] = {y.x, y.y, y.z, y.w};
    const int64_t step = x.wide ? 1 : kThreads;
    if (x.half) {
#pragma unroll
        for (int e = 0; e < 8; ++e)
            if (e * step < x.left) ((uint16_t *)x.p)[e * step] = (uint16_t)(v[e / 2] >> e % 2 * 16);
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (e * step < x.left) ((uint32_t *)x.p)[e * step] = v[e];
    }
}

__device__ __forceinline__ void values(float (&f)[8], uint4 y, bool half) {
    const uint32_t v[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        f[e] = __uint_as_float(half ? v[e] << 16 : v[e]);
        f[4 + e] = half ? __uint_as_float(v[e] & 0xffff0000u) : 0.0f;
    }
}

__device__ __forceinline__ double squares(uint4 y, bool half) {
    float f[8], s = 0.0f;
    values(f, y, half);
#pragma unroll
    for (int e = 0; e < 8; ++e) s = fmaf(f[e], f[e], s);
    if (s >= 1e-20f && s <= 1e30f) return s;
    double d = 0.0;
#pragma unroll
    for (int e = 0; e < 8; ++e) d += (double)f[e] * f[e];
    return d;
}

__device__ __forceinline__ uint4 scaled(uint4 y, bool half, float c) {
    float f[8];
    values(f, y, half);
    uint32_t v[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        if (half) {
            const __nv_bfloat162 b = __floats2bfloat162_rn(f[e] * c, f[4 + e] * c);
            v[e] = *(const uint32_t *)&b;
        } else {
            v[e] = __float_as_uint(f[e] * c);
        }
    }
    return make_uint4(v[0], v[1], v[2], v[3]);
}

__device__ __forceinline__ double block_sum(double x) {
    __shared__ double warp[kThreads / 32];
    __syncthreads();
    for (int o = 16; o > 0; o >>= 1) x += __shfl_xor_sync(~0u, x, o);
    if (threadIdx.x % 32 == 0) warp[threadIdx.x / 32] = x;
    __syncthreads();
    x = warp[threadIdx.x % 32];
    for (int o = 16; o > 0; o >>= 1) x += __shfl_xor_sync(~0u, x, o);
    return x;
}

template <int N>
__global__ void __launch_bounds__(kThreads) goib2d_clip_kernel(const __grid_constant__ Table<N> T) {
    extern __shared__ uint4 kept[];
    const int tiles = T.n ? T.end[T.n - 1] >> 1 : 0;
    const int first = (int)((int64_t)blockIdx.x * tiles / gridDim.x);  // the block's tiles, neighbours
    const int mine = (int)((int64_t)(blockIdx.x + 1) * tiles / gridDim.x) - first;
    Cursor<N> cursor(T);
    if (T.mode & kSum) {
        double sum = 0.0;
        for (int k = 0; k < mine; k += kBatch) {
            uint4 y[kBatch];
            const uint4 *p = k + kBatch <= mine ? cursor.batch(first + k) : nullptr;
            if (p) {
                if (k < kKept)
#pragma unroll
                    for (int e = 0; e < kBatch; ++e) y[e] = __ldcs(p + e * kThreads);
                else
#pragma unroll
                    for (int e = 0; e < kBatch; ++e) y[e] = p[e * kThreads];
                if (cursor.half)
#pragma unroll
                    for (int e = 0; e < kBatch; ++e) sum += squares(y[e], true);
                else
#pragma unroll
                    for (int e = 0; e < kBatch; ++e) sum += squares(y[e], false);
            } else {
                bool half[kBatch];
#pragma unroll
                for (int e = 0; e < kBatch; ++e) {
                    y[e] = make_uint4(0, 0, 0, 0), half[e] = false;
                    if (k + e < mine) {
                        const Piece x = cursor.at(first + k + e);
                        y[e] = load(x), half[e] = x.half;
                    }
                }
#pragma unroll
                for (int e = 0; e < kBatch; ++e) sum += squares(y[e], half[e]);
            }
            if (k < kKept)
#pragma unroll
                for (int e = 0; e < kBatch; ++e) kept[(k + e) * kThreads + threadIdx.x] = y[e];
        }
        sum = block_sum(sum);
        if (threadIdx.x == 0) T.part[T.first + blockIdx.x] = sum;
        if (!(T.mode & kScale)) return;
        cooperative_groups::this_grid().sync();
    }
    double sum = 0.0;
    for (int j = threadIdx.x; j < T.sums; j += kThreads) sum += T.part[j];
    const float norm = (float)sqrt(block_sum(sum));
    if (T.norm && blockIdx.x == 0 && threadIdx.x == 0) *T.norm = norm;
    const float c = T.max_norm / (norm + 1e-6f);
    if (c >= 1.0f) return;  // NaN goes on: every element becomes NaN
    const int held = T.mode & kSum ? (mine < kKept ? mine : kKept) : 0;
    for (int k = mine; k > 0;) {
        const bool here = k <= held;
        const int n = k - (here ? 0 : held) < kBatch ? k - (here ? 0 : held) : kBatch;
        k -= n;
        uint4 *const p = n == kBatch ? cursor.batch(first + k) : nullptr;
        uint4 y[kBatch];
        if (p) {
#pragma unroll
            for (int e = 0; e < kBatch; ++e) y[e] = here ? kept[(k + e) * kThreads + threadIdx.x] : p[e * kThreads];
            if (cursor.half)
#pragma unroll
                for (int e = 0; e < kBatch; ++e) __stcs(p + e * kThreads, scaled(y[e], true, c));
            else
#pragma unroll
                for (int e = 0; e < kBatch; ++e) __stcs(p + e * kThreads, scaled(y[e], false, c));
        } else {
            for (int e = 0; e < n; ++e) {
                const Piece x = cursor.at(first + k + e);
                store(x, scaled(here ? kept[(k + e) * kThreads + threadIdx.x] : load(x), x.half, c));
            }
        }
    }
}

int launches(int32_t n) { return n ? (n + kMost - 1) / kMost : 1; }

template <int N>
cudaError_t clip_tables(const goib2d_grad *grads, int32_t n, float max_norm, float *norm, double *part, cudaStream_t s) {
    const size_t smem = (size_t)kKept * kBytes;
    cudaError_t e = cudaFuncSetAttribute(goib2d_clip_kernel<N>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    if (e != cudaSuccess) return e;
    int sms = 0, dev = 0;
    if ((e = cudaGetDevice(&dev)) != cudaSuccess) return e;
    if ((e = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev)) != cudaSuccess) return e;
    sms = sms < kSms ? sms : kSms;
    Table<N> T;
    T.max_norm = max_norm, T.part = part, T.first = 0;
    const bool one = n <= N;
    for (int mode = one ? kSum | kScale : kSum; mode <= (kSum | kScale); mode = mode == kSum ? kScale : 4) {
        if (mode == kScale) T.sums = T.first;
        T.mode = mode, T.norm = mode & kScale ? norm : nullptr;
        for (int32_t from = 0; from == 0 || from < n; from += N) {
            T.n = n - from < N ? n - from : N;
            int64_t tiles = 0;
            for (int i = 0; i < T.n; ++i) {
                const goib2d_grad &g = grads[from + i];
                const int64_t elements = kBytes / (g.dtype == GOIB2D_BFLOAT16 ? 2 : 4);
                tiles += (g.numel + elements - 1) / elements;
                T.ptr[i] = g.data, T.numel[i] = g.numel;
                T.end[i] = (int32_t)(tiles << 1) | (g.dtype == GOIB2D_BFLOAT16);
            }
            const int blocks = tiles < sms ? (tiles ? (int)tiles : 1) : sms;
            if (one) T.sums = blocks;
            void *args[] = {&T};
            e = cudaLaunchCooperativeKernel((const void *)goib2d_clip_kernel<N>, dim3(blocks), dim3(kThreads), args, smem, s);
            if (e != cudaSuccess) return e;
            if (mode == kSum) T.first += blocks;
            T.norm = nullptr;
        }
    }
    return cudaSuccess;
}

}  // namespace

int64_t clip_workspace_bytes(const goib2d_grad *, int32_t n) { return (int64_t)sizeof(double) * kSms * launches(n); }

cudaError_t launch_clip(const goib2d_grad *grads, int32_t n, float max_norm, float *norm, void *workspace,
                        cudaStream_t s) {
    // the table is copied with the launch: a small one for few tensors
    return n <= 64 ? clip_tables<64>(grads, n, max_norm, norm, (double *)workspace, s)
                   : clip_tables<kMost>(grads, n, max_norm, norm, (double *)workspace, s);
}

}  // namespace gb
