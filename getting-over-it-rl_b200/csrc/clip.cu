// Gradient clipping by the global norm over many tensors (goib2d_clip_grads): norm = sqrt(sum of squares of every
// element of every tensor), then every element times min(1, max_norm / (norm + 1e-6)).
//
// The tensor table travels in the launch's parameters, so a call makes no copy and keeps nothing. Squares are summed
// in float64: no overflow or underflow of a square in float32's range, and 5.8 conversions and multiply-adds per clock and SM at the
// full HBM rate are far below what the SM does. Every block's sum goes to its own place and every block adds all of them in
// one order: the same inputs give the same bits.
#include "policy.cuh"

namespace gb {
namespace {

constexpr int kTable = 1024;        // tensors per launch: 24 KB of the 32 KB of launch parameters
constexpr int kTile = 4096;         // elements of one block's turn
constexpr int kThreads = 256;
constexpr int kBlocks = 148 * 4;    // partial sums per launch

struct Table {
    int32_t n;                      // tensors
    int32_t first;                  // where this launch's partial sums go
    int32_t sums;                   // partial sums of all launches (clip)
    float max_norm;
    float *norm;
    double *part;
    void *ptr[kTable];
    int64_t end[kTable];            // (tiles up to and with this tensor) << 1 | bfloat16
    int64_t numel[kTable];
};

// The tensor of tile t, and the tile's place in it.
__device__ __forceinline__ int find(const Table &T, int64_t t, int64_t &at) {
    int lo = 0, hi = T.n - 1;
    while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (t < (T.end[mid] >> 1)) hi = mid;
        else lo = mid + 1;
    }
    at = (t - (lo ? T.end[lo - 1] >> 1 : 0)) * kTile;
    return lo;
}

__device__ __forceinline__ double block_sum(double x) {
    __shared__ double warp[kThreads / 32];
    for (int o = 16; o > 0; o >>= 1) x += __shfl_xor_sync(~0u, x, o);
    if (threadIdx.x % 32 == 0) warp[threadIdx.x / 32] = x;
    __syncthreads();
    x = 0.0;
    for (int i = 0; i < kThreads / 32; ++i) x += warp[i];
    return x;
}

__global__ void __launch_bounds__(kThreads) goib2d_grad_norm_kernel(const __grid_constant__ Table T) {
    const int64_t tiles = T.end[T.n - 1] >> 1;
    double sum = 0.0;
    for (int64_t t = blockIdx.x; t < tiles; t += gridDim.x) {
        int64_t at;
        const int i = find(T, t, at);
        const int64_t stop = at + kTile < T.numel[i] ? at + kTile : T.numel[i];
        if (T.end[i] & 1) {
            const __nv_bfloat16 *x = (const __nv_bfloat16 *)T.ptr[i];
            for (int64_t j = at + threadIdx.x; j < stop; j += kThreads) {
                const double y = __bfloat162float(x[j]);
                sum += y * y;
            }
        } else {
            const float *x = (const float *)T.ptr[i];
            for (int64_t j = at + threadIdx.x; j < stop; j += kThreads) {
                const double y = x[j];
                sum += y * y;
            }
        }
    }
    sum = block_sum(sum);
    if (threadIdx.x == 0) T.part[T.first + blockIdx.x] = sum;
}

__global__ void __launch_bounds__(kThreads) goib2d_grad_clip_kernel(const __grid_constant__ Table T) {
    double sum = 0.0;
    for (int i = threadIdx.x; i < T.sums; i += kThreads) sum += T.part[i];
    const float norm = (float)sqrt(block_sum(sum));
    if (T.norm && blockIdx.x == 0 && threadIdx.x == 0) *T.norm = norm;
    const float c = T.max_norm / (norm + 1e-6f);
    if (c >= 1.0f || T.n == 0) return;  // NaN goes on: every element becomes NaN
    const int64_t tiles = T.end[T.n - 1] >> 1;
    for (int64_t t = blockIdx.x; t < tiles; t += gridDim.x) {
        int64_t at;
        const int i = find(T, t, at);
        const int64_t stop = at + kTile < T.numel[i] ? at + kTile : T.numel[i];
        if (T.end[i] & 1) {
            __nv_bfloat16 *x = (__nv_bfloat16 *)T.ptr[i];
            for (int64_t j = at + threadIdx.x; j < stop; j += kThreads)
                x[j] = __float2bfloat16_rn(__bfloat162float(x[j]) * c);
        } else {
            float *x = (float *)T.ptr[i];
            for (int64_t j = at + threadIdx.x; j < stop; j += kThreads) x[j] *= c;
        }
    }
}

int launches(int32_t n) { return n ? (n + kTable - 1) / kTable : 1; }

}  // namespace

int64_t clip_workspace_bytes(const goib2d_grad *, int32_t n) { return (int64_t)sizeof(double) * kBlocks * launches(n); }

cudaError_t launch_clip(const goib2d_grad *grads, int32_t n, float max_norm, float *norm, void *workspace,
                        cudaStream_t s) {
    Table T;
    T.max_norm = max_norm, T.part = (double *)workspace;
    for (int pass = 0; pass < 2; ++pass) {
        T.sums = pass ? T.first : 0;
        T.first = 0, T.norm = pass ? norm : nullptr;
        for (int32_t from = 0; from == 0 || from < n; from += kTable) {
            T.n = n - from < kTable ? n - from : kTable;
            int64_t tiles = 0;
            for (int i = 0; i < T.n; ++i) {
                const goib2d_grad &g = grads[from + i];
                tiles += (g.numel + kTile - 1) / kTile;
                T.ptr[i] = g.data, T.numel[i] = g.numel;
                T.end[i] = tiles << 1 | (g.dtype == GOIB2D_BFLOAT16);
            }
            const int blocks = tiles < kBlocks ? (tiles ? (int)tiles : 1) : kBlocks;
            if (!pass) {
                if (tiles) goib2d_grad_norm_kernel<<<blocks, kThreads, 0, s>>>(T);
                T.first += tiles ? blocks : 0;
            } else {
                if (tiles || T.norm) goib2d_grad_clip_kernel<<<blocks, kThreads, 0, s>>>(T);
                T.norm = nullptr;
            }
            const cudaError_t e = cudaGetLastError();
            if (e != cudaSuccess) return e;
        }
    }
    return cudaSuccess;
}

}  // namespace gb
