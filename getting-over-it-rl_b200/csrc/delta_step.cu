// The gated delta rule, one token per world (goib2d_delta_step).
#include "delta.cuh"
#include "delta_step.h"
#include "mma.cuh"

namespace gb {
namespace {

// Bound by the state's bytes: 8 K V per (world, head), each read and written once and kept in registers between. A
// thread holds four columns of some rows; x runs over the columns, y over the row groups, z over the heads of a block.
// Both products with the state come from one pass, S'^T k = a (S^T k) and S^T q = a (S^T q) + (k.q) u, summed over the row
// groups in shared memory, where k and q lie as float32 pairs.

// Rows of whole 16-byte pieces: a thread's columns are neighbours, read and written 16 bytes at a time.
constexpr int kRows = 16;  // of a thread. 8: 100 us, 16: 89 us, 32: 125 us for 4096 worlds x 4 heads of 64 x 64
template <class T>
__global__ void __launch_bounds__(512) goib2d_delta_step_kernel(const __grid_constant__ goib2d_delta_desc d) {
    extern __shared__ __align__(16) float sm[];
    const int K = d.key_dim, V = d.value_dim, RY = blockDim.y, Z = blockDim.z, y = threadIdx.y, z = threadIdx.z;
    const int c = threadIdx.x * 4;
    const StepShared at(K, V, RY, Z);
    float2 *kq = (float2 *)(sm + at.pairs) + z * K;
    float *part = sm + at.sums + z * RY * 2 * V + c, *dots = sm + at.dots + z * RY;
    const uint32_t nh = blockIdx.x * Z + z;
    const bool live = nh < (uint32_t)(d.n_worlds * d.heads);
    const int64_t n = live ? nh / (uint32_t)d.heads : 0;
    const int h = live ? (int)(nh - (uint32_t)n * d.heads) : 0, hk = h / (d.heads / d.key_heads);
    const T *k = row<T>(d.k, d.k_stride, n, 0, hk), *q = row<T>(d.q, d.q_stride, n, 0, hk);
    for (int i = y * blockDim.x + threadIdx.x; i < K; i += blockDim.x * RY)
        kq[i] = live ? make_float2(to_float(k[i]), to_float(q[i])) : make_float2(0.0f, 0.0f);
    const T *v = row<T>(d.v, d.v_stride, n, 0, h) + c;
    float u[4], b = 0.0f, a = 0.0f;
    bool fresh = !live || (d.reset && d.reset[n * d.reset_stride[0]]);
#pragma unroll
    for (int j = 0; j < 4; ++j) u[j] = live ? to_float(v[j]) : 0.0f;
    if (live) {
        b = to_float(*row<T>(d.beta, d.beta_stride, n, 0, h));
        a = expf(to_float(*row<T>(d.g, d.g_stride, n, 0, h)));
    }
    float S[kRows][4];
    const float *in = d.state_in + (live ? (int64_t)nh * K * V : 0) + c;
#pragma unroll
    for (int i = 0; i < kRows; ++i) {
        const int r = y + i * RY;
        // This launch usually writes the same memory: no read-only loads. Heads of 64 x 64, us with those, these and plain
        // ones: 4096 x 4 in bfloat16 88.9, 88.1, 91.1; 65536 374, 381, 383.
        const float4 e = live && r < K ? __ldcs((const float4 *)(in + r * V)) : make_float4(0, 0, 0, 0);
        S[i][0] = e.x, S[i][1] = e.y, S[i][2] = e.z, S[i][3] = e.w;
    }
    __syncthreads();
    a = fresh ? 0.0f : a;
#pragma unroll
    for (int i = 0; i < kRows; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) S[i][j] = a == 0.0f ? 0.0f : S[i][j];
    float pk[4] = {}, pq[4] = {}, dot = 0.0f;
#pragma unroll
    for (int i = 0; i < kRows; ++i) {
        const int r = y + i * RY;
        const float2 e = r < K ? kq[r] : make_float2(0.0f, 0.0f);
        dot += e.x * e.y;
#pragma unroll
        for (int j = 0; j < 4; ++j) pk[j] += S[i][j] * e.x, pq[j] += S[i][j] * e.y;
    }
    *(float4 *)(part + y * 2 * V) = make_float4(pk[0], pk[1], pk[2], pk[3]);
    *(float4 *)(part + y * 2 * V + V) = make_float4(pq[0], pq[1], pq[2], pq[3]);
    if (threadIdx.x == 0) dots[y] = dot;
    __syncthreads();
    if (!live) return;
#pragma unroll
    for (int j = 0; j < 4; ++j) pk[j] = pq[j] = 0.0f;
    dot = 0.0f;
    for (int i = 0; i < RY; ++i) {
        const float4 e = *(const float4 *)(part + i * 2 * V), f = *(const float4 *)(part + i * 2 * V + V);
        pk[0] += e.x, pk[1] += e.y, pk[2] += e.z, pk[3] += e.w;
        pq[0] += f.x, pq[1] += f.y, pq[2] += f.z, pq[3] += f.w;
        dot += dots[i];
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) u[j] = b * (u[j] - a * pk[j]);
    if (y == 0) {
        T *o = row<T>(d.out, d.out_stride, n, 0, h) + c;
#pragma unroll
        for (int j = 0; j < 4; ++j) o[j] = from_float<T>(d.scale * (a * pq[j] + dot * u[j]));
    }
    float *to = d.state_out + (int64_t)nh * K * V + c;
#pragma unroll
    for (int i = 0; i < kRows; ++i) {
        const int r = y + i * RY;
        if (r >= K) break;
        const float e = kq[r].x;
        __stcs((float4 *)(to + r * V),
               make_float4(a * S[i][0] + e * u[0], a * S[i][1] + e * u[1], a * S[i][2] + e * u[2], a * S[i][3] + e * u[3]));
    }
}

// Other rows: the block's heads, one behind the other in memory, come through shared memory as one piece, by 16-byte
// copies where every head's piece is whole (WIDE), else by 4-byte ones, and leave it so. A thread's columns lie X apart:
// neighbouring threads read neighbouring words.
constexpr int kFlatRows = 8;  // 4: 63 us, 8: 40 us, 16: 52 us for 1023 worlds x 6 heads of 40 x 71
template <class T, bool WIDE>
__global__ void __launch_bounds__(1024) goib2d_delta_step_flat_kernel(const __grid_constant__ goib2d_delta_desc d) {
    extern __shared__ __align__(16) float sm[];
    const int K = d.key_dim, V = d.value_dim, X = blockDim.x, RY = blockDim.y, Z = blockDim.z;
    const int x = threadIdx.x, y = threadIdx.y, z = threadIdx.z;
    float *base = sm + (Z * K * V + 3) / 4 * 4;
    float2 *kq = (float2 *)base + z * K;
    float *part = base + 2 * Z * K + z * RY * 8 * X + x, *dots = base + 2 * Z * (K + RY * 4 * X) + z * RY;
    const uint32_t heads = (uint32_t)(d.n_worlds * d.heads), first = blockIdx.x * Z, nh = first + z;
    const bool live = nh < heads;
    const int64_t n = live ? nh / (uint32_t)d.heads : 0;
    const int h = live ? (int)(nh - (uint32_t)n * d.heads) : 0, hk = h / (d.heads / d.key_heads);
    const int held = (int)(heads - first < (uint32_t)Z ? heads - first : Z) * K * V;  // floats of the block
    const int tid = (z * RY + y) * X + x, threads = X * RY * Z;
    const float *in = d.state_in + (int64_t)first * K * V;
    if constexpr (WIDE)
        for (int i = tid * 4; i < held; i += threads * 4) cp_async<16>(sm + i, in + i);
    else
        for (int i = tid; i < held; i += threads) cp_async<4>(sm + i, in + i);
    cp_commit();
    const T *k = row<T>(d.k, d.k_stride, n, 0, hk), *q = row<T>(d.q, d.q_stride, n, 0, hk);
    for (int i = y * X + x; i < K; i += X * RY)
        kq[i] = live ? make_float2(to_float(k[i]), to_float(q[i])) : make_float2(0.0f, 0.0f);
    const T *v = row<T>(d.v, d.v_stride, n, 0, h);
    float u[4], b = 0.0f, a = 0.0f;
#pragma unroll
    for (int j = 0; j < 4; ++j) u[j] = live && x + j * X < V ? to_float(v[x + j * X]) : 0.0f;
    if (live) b = to_float(*row<T>(d.beta, d.beta_stride, n, 0, h)), a = decay_at<T>(d, n, 0, h);
    cp_wait<0>();
    __syncthreads();
    float S[kFlatRows][4], pk[4] = {}, pq[4] = {}, dot = 0.0f;
    float *mine = sm + z * K * V + x;
#pragma unroll
    for (int i = 0; i < kFlatRows; ++i) {
        const int r = y + i * RY;
        const float2 e = r < K ? kq[r] : make_float2(0.0f, 0.0f);
        dot += e.x * e.y;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            // the old state may hold anything where a is 0
            S[i][j] = live && a != 0.0f && r < K && x + j * X < V ? mine[r * V + j * X] : 0.0f;
            pk[j] += S[i][j] * e.x, pq[j] += S[i][j] * e.y;
        }
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) part[(y * 8 + j) * X] = pk[j], part[(y * 8 + 4 + j) * X] = pq[j];
    if (x == 0) dots[y] = dot;
    __syncthreads();
#pragma unroll
    for (int j = 0; j < 4; ++j) pk[j] = pq[j] = 0.0f;
    dot = 0.0f;
    for (int i = 0; i < RY; ++i) {
#pragma unroll
        for (int j = 0; j < 4; ++j) pk[j] += part[(i * 8 + j) * X], pq[j] += part[(i * 8 + 4 + j) * X];
        dot += dots[i];
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) u[j] = b * (u[j] - a * pk[j]);
    if (y == 0 && live) {
        T *o = row<T>(d.out, d.out_stride, n, 0, h);
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (x + j * X < V) o[x + j * X] = from_float<T>(d.scale * (a * pq[j] + dot * u[j]));
    }
#pragma unroll
    for (int i = 0; i < kFlatRows; ++i) {
        const int r = y + i * RY;
        if (r >= K) break;
        const float e = kq[r].x;
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (x + j * X < V) mine[r * V + j * X] = a * S[i][j] + e * u[j];
    }
    __syncthreads();
    float *to = d.state_out + (int64_t)first * K * V;
    if constexpr (WIDE)
        for (int i = tid * 4; i < held; i += threads * 4) __stcs((float4 *)(to + i), *(const float4 *)(sm + i));
    else
        for (int i = tid; i < held; i += threads) __stcs(to + i, sm[i]);
}

struct Shape : StepShape {
    Shape(const goib2d_delta_desc &d, int rows) : StepShape(d.key_dim, d.value_dim, rows) {}
    unsigned blocks(const goib2d_delta_desc &d) const { return (unsigned)((d.n_worlds * d.heads + z - 1) / z); }
    size_t bytes(const goib2d_delta_desc &d) const { return sizeof(float) * StepShared(d.key_dim, 4 * x, y, z).end; }
};

template <class T, bool WIDE>
cudaError_t step_flat(const goib2d_delta_desc &d, cudaStream_t s) {
    const Shape b(d, kFlatRows);
    const size_t smem = sizeof(float) * ((size_t)(b.z * d.key_dim * d.value_dim + 3) / 4 * 4) + b.bytes(d);
    cudaError_t e = allow_smem(goib2d_delta_step_flat_kernel<T, WIDE>, smem);
    if (e != cudaSuccess) return e;
    goib2d_delta_step_flat_kernel<T, WIDE><<<b.blocks(d), dim3(b.x, b.y, b.z), smem, s>>>(d);
    return cudaGetLastError();
}

template <class T>
cudaError_t step_typed(const goib2d_delta_desc &d, cudaStream_t s) {
    const bool aligned = (uintptr_t)d.state_in % 16 == 0 && (uintptr_t)d.state_out % 16 == 0;
    if (!aligned || d.value_dim % 4)
        return aligned && d.key_dim * d.value_dim % 4 == 0 ? step_flat<T, true>(d, s) : step_flat<T, false>(d, s);
    const Shape b(d, kRows);
    goib2d_delta_step_kernel<T><<<b.blocks(d), dim3(b.x, b.y, b.z), b.bytes(d), s>>>(d);
    return cudaGetLastError();
}

}  // namespace

cudaError_t launch_delta_step(const goib2d_delta_desc &d, cudaStream_t s) {
    return d.dtype == GOIB2D_BFLOAT16 ? step_typed<__nv_bfloat16>(d, s) : step_typed<float>(d, s);
}

}  // namespace gb
