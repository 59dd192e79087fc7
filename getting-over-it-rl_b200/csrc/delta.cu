// The gated delta rule, a policy's memory per world (goib2d_delta_*): each (world, head) holds a matrix S [K][V] in
// float32. Token t with decay a = exp(g), key k, value v, query q, write strength b:
//     S' = a S,  r = v - S'^T k,  u = b r,  S = S' + k u^T,  o = scale S^T q.
// A token whose reset flag is set, or whose decay is 0 in float32, starts from S' = 0 without reading the old state
// (so what the old state held, infinities included, does not matter).
#include "policy.cuh"

namespace gb {
namespace {

__device__ __forceinline__ float to_float(float x) { return x; }
__device__ __forceinline__ float to_float(__nv_bfloat16 x) { return __bfloat162float(x); }
template <class T>
__device__ __forceinline__ T from_float(float x);
template <>
__device__ __forceinline__ float from_float<float>(float x) { return x; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }

// A strided (world, step, head, channel) tensor's row at (n, t, h); channels are contiguous.
template <class T>
__device__ __forceinline__ const T *row(const void *p, const int64_t *s, int64_t n, int64_t t, int h) {
    return (const T *)p + n * s[0] + t * s[1] + h * s[2];
}
template <class T>
__device__ __forceinline__ T *row(void *p, const int64_t *s, int64_t n, int64_t t, int h) {
    return (T *)p + n * s[0] + t * s[1] + h * s[2];
}

// The decay of token t, 0 where the state starts afresh.
template <class T>
__device__ __forceinline__ float decay_at(const goib2d_delta_desc &d, int64_t n, int64_t t, int h) {
    if (d.reset && d.reset[n * d.reset_stride[0] + t * d.reset_stride[1]]) return 0.0f;
    return expf(to_float(*row<T>(d.g, d.g_stride, n, t, h)));
}

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

// ---- rollouts: the recurrence token by token, a column of S per thread in shared memory

template <class T>
__global__ void __launch_bounds__(128) goib2d_delta_forward_kernel(const __grid_constant__ goib2d_delta_desc d,
                                                                   float *saved) {
    extern __shared__ float sm[];
    const int K = d.key_dim, V = d.value_dim, c = threadIdx.x;
    float *S = sm, *kq = sm + K * V;  // S [K][V]; k and q of the token
    const int64_t nh = blockIdx.x, n = nh / d.heads;
    const int h = (int)(nh - n * d.heads), hk = h / (d.heads / d.key_heads);
    if (c < V)
        for (int i = 0; i < K; ++i) S[i * V + c] = d.state_in ? d.state_in[(nh * K + i) * V + c] : 0.0f;
    for (int64_t t = 0; t < d.n_steps; ++t) {
        __syncthreads();
        for (int i = c; i < K; i += blockDim.x) {
            kq[i] = to_float(row<T>(d.k, d.k_stride, n, t, hk)[i]);
            kq[K + i] = to_float(row<T>(d.q, d.q_stride, n, t, hk)[i]);
        }
        __syncthreads();
        if (c >= V) continue;
        const float a = decay_at<T>(d, n, t, h), b = to_float(*row<T>(d.beta, d.beta_stride, n, t, h));
        float dot = 0.0f, o = 0.0f;
        for (int i = 0; i < K; ++i) {
            const float x = a == 0.0f ? 0.0f : a * S[i * V + c];
            S[i * V + c] = x;
            dot += x * kq[i];
        }
        const float r = to_float(row<T>(d.v, d.v_stride, n, t, h)[c]) - dot, u = b * r;
        for (int i = 0; i < K; ++i) {
            const float x = S[i * V + c] + kq[i] * u;
            S[i * V + c] = x;
            o += x * kq[K + i];
        }
        row<T>(d.out, d.out_stride, n, t, h)[c] = from_float<T>(d.scale * o);
        if (saved) saved[((n * d.n_steps + t) * d.heads + h) * V + c] = r;
    }
    if (c < V)
        for (int i = 0; i < K; ++i) d.state_out[(nh * K + i) * V + c] = S[i * V + c];
}

__device__ float block_sum(float x, float *tmp) {  // of 128 threads, the same order every time
    __syncthreads();
    tmp[threadIdx.x] = x;
    __syncthreads();
    for (int w = 64; w > 0; w >>= 1) {
        if (threadIdx.x < w) tmp[threadIdx.x] += tmp[threadIdx.x + w];
        __syncthreads();
    }
    return tmp[0];
}

struct BackParams {
    goib2d_delta_desc d;
    goib2d_delta_grads gr;
    const float *r;          // [n][t][h][V]
    float *dv, *dq, *dk;     // [n][t][h][V], [n][t][h][K]: per value head
    float *dG;               // [n][t][h]
    float *end;              // [n][h]: <S, dS> after the last token
};

// dS backwards: dv, dbeta, and the write part of dk
template <class T>
__global__ void __launch_bounds__(128) goib2d_delta_back_state_kernel(const __grid_constant__ BackParams p) {
    extern __shared__ float sm[];
    const goib2d_delta_desc &d = p.d;
    const int K = d.key_dim, V = d.value_dim, c = threadIdx.x, W = V + 1;
    float *dS = sm, *kq = dS + K * W, *us = kq + 2 * K, *tmp = us + V;
    const int64_t nh = blockIdx.x, n = nh / d.heads;
    const int h = (int)(nh - n * d.heads), hk = h / (d.heads / d.key_heads);
    float end = 0.0f;
    for (int i = 0; i < K; ++i)
        if (c < V) {
            const float x = p.gr.dstate_out ? p.gr.dstate_out[(nh * K + i) * V + c] : 0.0f;
            dS[i * W + c] = x;
            if (p.gr.dstate_out) end += x * d.state_out[(nh * K + i) * V + c];
        }
    end = block_sum(end, tmp);
    if (c == 0) p.end[nh] = end;
    for (int64_t t = d.n_steps - 1; t >= 0; --t) {
        const int64_t at = (n * d.n_steps + t) * d.heads + h;
        __syncthreads();
        for (int i = c; i < K; i += blockDim.x) {
            kq[i] = to_float(row<T>(d.k, d.k_stride, n, t, hk)[i]);
            kq[K + i] = to_float(row<T>(d.q, d.q_stride, n, t, hk)[i]);
        }
        __syncthreads();
        const float a = decay_at<T>(d, n, t, h), b = to_float(*row<T>(d.beta, d.beta_stride, n, t, h));
        float du = 0.0f, r = 0.0f;
        if (c < V) {
            const float o = p.gr.dout ? d.scale * to_float(row<T>(p.gr.dout, p.gr.dout_stride, n, t, h)[c]) : 0.0f;
            for (int i = 0; i < K; ++i) {
                const float x = dS[i * W + c] + kq[K + i] * o;
                dS[i * W + c] = x;
                du += x * kq[i];
            }
            r = p.r[at * V + c];
            us[c] = b * r;
            p.dv[at * V + c] = b * du;
            row<T>(p.gr.dv, p.gr.dv_stride, n, t, h)[c] = from_float<T>(b * du);
        }
        const float db = block_sum(du * r, tmp);
        if (c == 0) *row<T>(p.gr.dbeta, p.gr.dbeta_stride, n, t, h) = from_float<T>(db);
        if (c < K) {
            float x = 0.0f;
            for (int j = 0; j < V; ++j) x += dS[c * W + j] * us[j];
            p.dk[at * K + c] = x;
        }
        __syncthreads();
        if (c < V)
            for (int i = 0; i < K; ++i) dS[i * W + c] = a == 0.0f ? 0.0f : a * (dS[i * W + c] - kq[i] * b * du);
    }
    if (c < V && p.gr.dstate_in)
        for (int i = 0; i < K; ++i) p.gr.dstate_in[(nh * K + i) * V + c] = dS[i * W + c];
}

// S forwards again: dq, the read part of dk, and what the decays get from each token
template <class T>
__global__ void __launch_bounds__(128) goib2d_delta_back_token_kernel(const __grid_constant__ BackParams p) {
    extern __shared__ float sm[];
    const goib2d_delta_desc &d = p.d;
    const int K = d.key_dim, V = d.value_dim, c = threadIdx.x, W = V + 1;
    float *S = sm, *kq = S + K * W, *dvs = kq + 2 * K, *dos = dvs + V, *tmp = dos + V;
    const int64_t nh = blockIdx.x, n = nh / d.heads;
    const int h = (int)(nh - n * d.heads), hk = h / (d.heads / d.key_heads);
    for (int i = 0; i < K; ++i)
        if (c < V) S[i * W + c] = d.state_in ? d.state_in[(nh * K + i) * V + c] : 0.0f;
    for (int64_t t = 0; t < d.n_steps; ++t) {
        const int64_t at = (n * d.n_steps + t) * d.heads + h;
        __syncthreads();
        for (int i = c; i < K; i += blockDim.x) {
            kq[i] = to_float(row<T>(d.k, d.k_stride, n, t, hk)[i]);
            kq[K + i] = to_float(row<T>(d.q, d.q_stride, n, t, hk)[i]);
        }
        const float a = decay_at<T>(d, n, t, h), b = to_float(*row<T>(d.beta, d.beta_stride, n, t, h));
        if (c < V) {
            dvs[c] = p.dv[at * V + c];
            dos[c] = p.gr.dout ? d.scale * to_float(row<T>(p.gr.dout, p.gr.dout_stride, n, t, h)[c]) : 0.0f;
            for (int i = 0; i < K; ++i) S[i * W + c] = a == 0.0f ? 0.0f : a * S[i * W + c];
        }
        __syncthreads();
        float read = 0.0f;
        if (c < K)
            for (int j = 0; j < V; ++j) read -= S[c * W + j] * dvs[j];
        __syncthreads();
        if (c < V) {
            const float u = b * p.r[at * V + c];
            for (int i = 0; i < K; ++i) S[i * W + c] += kq[i] * u;
        }
        __syncthreads();
        float dG = 0.0f;
        if (c < K) {
            float x = 0.0f;
            for (int j = 0; j < V; ++j) x += S[c * W + j] * dos[j];
            const float write = p.dk[at * K + c];
            p.dq[at * K + c] = x;
            p.dk[at * K + c] = read + write;
            dG = kq[K + c] * x + kq[c] * (read - write);
        }
        dG = block_sum(dG, tmp);
        if (c == 0) p.dG[at] = dG;
    }
}

// dg: the sum of dG from a token to its segment's end (a reset ends the segment before it)
template <class T>
__global__ void goib2d_delta_back_decay_kernel(const __grid_constant__ BackParams p) {
    const goib2d_delta_desc &d = p.d;
    const int64_t nh = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
    if (nh >= d.n_worlds * d.heads) return;
    const int64_t n = nh / d.heads;
    const int h = (int)(nh - n * d.heads);
    double sum = p.end[nh];
    for (int64_t t = d.n_steps - 1; t >= 0; --t) {
        sum += p.dG[(n * d.n_steps + t) * d.heads + h];
        if (decay_at<T>(d, n, t, h) == 0.0f) sum = 0.0;
        *row<T>(p.gr.dg, p.gr.dg_stride, n, t, h) = from_float<T>((float)sum);
    }
}

// dq and dk: summed over the value heads that share a key head, in head order
template <class T>
__global__ void goib2d_delta_back_heads_kernel(const __grid_constant__ BackParams p) {
    const goib2d_delta_desc &d = p.d;
    const int K = d.key_dim, group = d.heads / d.key_heads;
    const int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
    if (i >= d.n_worlds * d.n_steps * d.key_heads * K) return;
    const int c = (int)(i % K), hk = (int)(i / K % d.key_heads);
    const int64_t t = i / K / d.key_heads % d.n_steps, n = i / K / d.key_heads / d.n_steps;
    float q = 0.0f, k = 0.0f;
    for (int j = 0; j < group; ++j) {
        const int64_t at = ((n * d.n_steps + t) * d.heads + hk * group + j) * K + c;
        q += p.dq[at], k += p.dk[at];
    }
    row<T>(p.gr.dq, p.gr.dq_stride, n, t, hk)[c] = from_float<T>(q);
    row<T>(p.gr.dk, p.gr.dk_stride, n, t, hk)[c] = from_float<T>(k);
}

template <class F>
cudaError_t allow_smem(F *f, size_t bytes) {
    return bytes <= 48 << 10 ? cudaSuccess
                             : cudaFuncSetAttribute(f, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
}

template <class T>
cudaError_t forward_typed(const goib2d_delta_desc &d, void *saved, cudaStream_t s) {
    const size_t smem = sizeof(float) * ((size_t)d.key_dim * d.value_dim + 2 * d.key_dim);
    cudaError_t e = allow_smem(goib2d_delta_forward_kernel<T>, smem);
    if (e != cudaSuccess) return e;
    goib2d_delta_forward_kernel<T><<<(unsigned)(d.n_worlds * d.heads), 128, smem, s>>>(d, (float *)saved);
    return cudaGetLastError();
}

template <class T>
cudaError_t backward_typed(const goib2d_delta_desc &d, const goib2d_delta_grads &gr, const void *saved, void *ws,
                           cudaStream_t s) {
    const int64_t nh = d.n_worlds * d.heads, tokens = nh * d.n_steps;
    BackParams p{d, gr, (const float *)saved};
    p.dv = (float *)ws, p.dq = p.dv + tokens * d.value_dim, p.dk = p.dq + tokens * d.key_dim;
    p.dG = p.dk + tokens * d.key_dim, p.end = p.dG + tokens;
    const size_t smem = sizeof(float) * ((size_t)d.key_dim * (d.value_dim + 1) + 2 * d.key_dim + 2 * d.value_dim + 128);
    cudaError_t e = allow_smem(goib2d_delta_back_state_kernel<T>, smem);
    if (e == cudaSuccess) e = allow_smem(goib2d_delta_back_token_kernel<T>, smem);
    if (e != cudaSuccess) return e;
    goib2d_delta_back_state_kernel<T><<<(unsigned)nh, 128, smem, s>>>(p);
    goib2d_delta_back_token_kernel<T><<<(unsigned)nh, 128, smem, s>>>(p);
    goib2d_delta_back_decay_kernel<T><<<(unsigned)((nh + 127) / 128), 128, 0, s>>>(p);
    const int64_t items = d.n_worlds * d.n_steps * d.key_heads * d.key_dim;
    if (items) goib2d_delta_back_heads_kernel<T><<<(unsigned)((items + 255) / 256), 256, 0, s>>>(p);
    return cudaGetLastError();
}

}  // namespace

int64_t delta_saved_bytes(const goib2d_delta_desc &d) {
    return 4 * d.n_worlds * d.n_steps * d.heads * d.value_dim;
}

int64_t delta_workspace_bytes(const goib2d_delta_desc &d) {
    const int64_t nh = d.n_worlds * d.heads;
    return 4 * (nh * d.n_steps * ((int64_t)d.value_dim + 2 * d.key_dim + 1) + nh);
}

cudaError_t launch_delta_step(const goib2d_delta_desc &d, cudaStream_t s) {
    return d.dtype == GOIB2D_BFLOAT16 ? step_typed<__nv_bfloat16>(d, s) : step_typed<float>(d, s);
}

cudaError_t launch_delta_forward(const goib2d_delta_desc &d, void *saved, cudaStream_t s) {
    return d.dtype == GOIB2D_BFLOAT16 ? forward_typed<__nv_bfloat16>(d, saved, s) : forward_typed<float>(d, saved, s);
}

cudaError_t launch_delta_backward(const goib2d_delta_desc &d, const goib2d_delta_grads &gr, const void *saved,
                                  void *workspace, cudaStream_t s) {
    return d.dtype == GOIB2D_BFLOAT16 ? backward_typed<__nv_bfloat16>(d, gr, saved, workspace, s)
                                      : backward_typed<float>(d, gr, saved, workspace, s);
}

}  // namespace gb
