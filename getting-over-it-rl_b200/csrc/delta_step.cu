// The gated delta rule, one token per world (goib2d_delta_step).
#include "delta.cuh"

namespace gb {
namespace {

// ---- one token per world
//
// Bound by the state's bytes: 8 K V per (world, head), each read and written once, from registers. A thread holds VEC
// neighbouring columns (16-byte accesses where V allows them) of up to ROWS rows; x runs over the columns, y over the
// row groups, z over the heads of a block. Both products with the state come from one pass, S'^T k = a (S^T k) and
// S^T q = a (S^T q) + (k.q) u, summed over the row groups in shared memory.
template <class T, int VEC, int ROWS>
__global__ void __launch_bounds__(256) goib2d_delta_step_kernel(const __grid_constant__ goib2d_delta_desc d) {
    extern __shared__ float part[];  // [z][y][2 V + 1]
    const int K = d.key_dim, V = d.value_dim, RY = blockDim.y;
    const int64_t nh = (int64_t)blockIdx.x * blockDim.z + threadIdx.z;
    const bool live = nh < d.n_worlds * d.heads;
    const int64_t n = live ? nh / d.heads : 0;
    const int h = live ? (int)(nh - n * d.heads) : 0, hk = h / (d.heads / d.key_heads);
    const int c = threadIdx.x * VEC;
    const float a = live ? decay_at<T>(d, n, 0, h) : 0.0f;
    const float *in = d.state_in + (live ? nh * K * V : 0) + c;
    const T *k = row<T>(d.k, d.k_stride, n, 0, hk), *q = row<T>(d.q, d.q_stride, n, 0, hk);
    float S[ROWS][VEC], kr[ROWS], pk[VEC] = {}, pq[VEC] = {}, kq = 0.0f;
#pragma unroll
    for (int i = 0; i < ROWS; ++i) {
        const int r = threadIdx.y + i * RY;
#pragma unroll
        for (int j = 0; j < VEC; ++j) S[i][j] = 0.0f;
        if (live && r < K && a != 0.0f) {
            if constexpr (VEC == 4) {
                const float4 x = *(const float4 *)(in + (int64_t)r * V);
                S[i][0] = x.x, S[i][1] = x.y, S[i][2] = x.z, S[i][3] = x.w;
            } else {
                S[i][0] = in[(int64_t)r * V];
            }
        }
    }
#pragma unroll
    for (int i = 0; i < ROWS; ++i) {
        const int r = threadIdx.y + i * RY;
        const bool has = live && r < K;
        kr[i] = has ? to_float(k[r]) : 0.0f;
        const float qr = has ? to_float(q[r]) : 0.0f;
        kq += kr[i] * qr;
#pragma unroll
        for (int j = 0; j < VEC; ++j) pk[j] += S[i][j] * kr[i], pq[j] += S[i][j] * qr;
    }
    float *mine = part + (threadIdx.z * RY + threadIdx.y) * (2 * V + 1);
#pragma unroll
    for (int j = 0; j < VEC; ++j) mine[c + j] = pk[j], mine[V + c + j] = pq[j];
    if (threadIdx.x == 0) mine[2 * V] = kq;
    __syncthreads();
    if (!live) return;
    kq = 0.0f;
#pragma unroll
    for (int j = 0; j < VEC; ++j) pk[j] = pq[j] = 0.0f;
    for (int y = 0; y < RY; ++y) {
        const float *p = part + (threadIdx.z * RY + y) * (2 * V + 1);
#pragma unroll
        for (int j = 0; j < VEC; ++j) pk[j] += p[c + j], pq[j] += p[V + c + j];
        kq += p[2 * V];
    }
    const T *v = row<T>(d.v, d.v_stride, n, 0, h) + c;
    const float b = to_float(*row<T>(d.beta, d.beta_stride, n, 0, h));
    float u[VEC];
#pragma unroll
    for (int j = 0; j < VEC; ++j) u[j] = b * (to_float(v[j]) - a * pk[j]);
    if (threadIdx.y == 0) {
        T *o = row<T>(d.out, d.out_stride, n, 0, h) + c;
#pragma unroll
        for (int j = 0; j < VEC; ++j) o[j] = from_float<T>(d.scale * (a * pq[j] + kq * u[j]));
    }
    float *to = d.state_out + nh * K * V + c;
#pragma unroll
    for (int i = 0; i < ROWS; ++i) {
        const int r = threadIdx.y + i * RY;
        if (r >= K) break;
        if constexpr (VEC == 4) {
            *(float4 *)(to + (int64_t)r * V) = make_float4(a * S[i][0] + kr[i] * u[0], a * S[i][1] + kr[i] * u[1],
                                                           a * S[i][2] + kr[i] * u[2], a * S[i][3] + kr[i] * u[3]);
        } else {
            to[(int64_t)r * V] = a * S[i][0] + kr[i] * u[0];
        }
    }
}

template <class T, int VEC, int ROWS>
cudaError_t step_of(const goib2d_delta_desc &d, cudaStream_t s) {
    const int x = d.value_dim / VEC, y = (d.key_dim + ROWS - 1) / ROWS;
    int z = 128 / (x * y);
    z = z < 1 ? 1 : z > 64 ? 64 : z;
    const int64_t blocks = (d.n_worlds * d.heads + z - 1) / z;
    const size_t smem = sizeof(float) * (size_t)z * y * (2 * d.value_dim + 1);
    goib2d_delta_step_kernel<T, VEC, ROWS><<<(unsigned)blocks, dim3(x, y, z), smem, s>>>(d);
    return cudaGetLastError();
}

template <class T>
cudaError_t step_typed(const goib2d_delta_desc &d, cudaStream_t s) {
    const bool wide = d.value_dim % 4 == 0 && (uintptr_t)d.state_in % 16 == 0 && (uintptr_t)d.state_out % 16 == 0;
    if (wide) return step_of<T, 4, 16>(d, s);
    return d.value_dim <= 32 ? step_of<T, 1, 16>(d, s) : step_of<T, 1, 64>(d, s);
}

}  // namespace

cudaError_t launch_delta_step(const goib2d_delta_desc &d, cudaStream_t s) {
    return d.dtype == GOIB2D_BFLOAT16 ? step_typed<__nv_bfloat16>(d, s) : step_typed<float>(d, s);
}

}  // namespace gb
