// What the kernels of the gated delta rule share (delta_step.cu, delta_forward.cu, delta_backward.cu): each (world, head)
// holds a matrix S [K][V] in float32. Token t with decay a = exp(g), key k, value v, query q, write strength b:
//     S' = a S,  r = v - S'^T k,  u = b r,  S = S' + k u^T,  o = scale S^T q.
// A token whose reset flag is set, or whose decay is 0 in float32, starts from S' = 0 without reading the old state
// (so what the old state held, infinities included, does not matter).
#pragma once
#include "policy.cuh"

namespace gb {

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

// The largest piece, of 16, 8 or 4 bytes, that the rows of a strided tensor and their starts are whole multiples of; 0:
// none (bfloat16 rows of odd places). n0, n1, n2: how many worlds, steps and heads there are.
inline int rows_grain(const void *p, const int64_t (&s)[3], int64_t n0, int64_t n1, int64_t n2, int cols, int size) {
    for (int bytes = 16; bytes >= 4; bytes /= 2) {
        const int64_t e = bytes / size;
        if ((uintptr_t)p % bytes == 0 && cols % e == 0 && (n0 == 1 || s[0] % e == 0) && (n1 == 1 || s[1] % e == 0) &&
            (n2 == 1 || s[2] % e == 0))
            return bytes;
    }
    return 0;
}
inline int dense_grain(int cols, int size) {  // of dense rows from an aligned start on
    return cols * size % 16 == 0 ? 16 : cols * size % 8 == 0 ? 8 : cols * size % 4 == 0 ? 4 : 0;
}

// Gradients whose products run in full precision (mma.cuh, Full): those of float32 inputs, and those of few tokens in
// bfloat16. A gradient such as dg or db is a sum that may cancel; over many tokens the rounding of bfloat16 operands
// (2^-9) averages out to 2^-9 of their norm, over a few it need not. Largest error of a gradient (of its norm) over six
// draws, rounded / full, where rounding the result alone gives 1.7e-3: 1 token of 64 x 64 2.0e-2 / 3.7e-3, 16 tokens
// 4.5e-3 / 2.2e-3, 256 tokens 3.1e-3 / 1.9e-3, 4096 tokens 2.9e-3 / 1.7e-3; of 1 x 1 at 16 tokens 6.2e-3 / 2.4e-3 and at
// 2048 8.5e-3 / 1.7e-3. So a world's gradients may differ by this much with the number of tokens beside its own. The
// price, us of a training step: 64 x 16 steps x 2 heads of 64 x 64 68 for either (the host's), 1 x 1024 x 4 heads 178 /
// 354, 1 x 4096 of 128 x 128 799 / 2041.
inline bool delta_full(const goib2d_delta_desc &d) {
    return d.dtype == GOIB2D_FLOAT32 || d.n_worlds * d.n_steps * d.heads <= 4096;
}

// What goib2d_delta_forward keeps for goib2d_delta_backward: r [n][h][t][V], and S at every keep-th token, as its S^T
// [n][h][t / keep][V up to 16s][padded keys]. In float32 for gradients in full products (delta_full). Otherwise in
// bfloat16, which the products would round them to anyway: half of what is written and read again (for 4096 worlds x 64
// steps x 4 heads of 64 x 64 in all 0.27 GB).
struct Saved {
    int64_t r, states, bytes;   // bytes: both
    int32_t keep, tiles_v, tiles_k, size;
};
inline int padded_keys(int K) { return K <= 32 ? 32 : K <= 64 ? 64 : 128; }
inline Saved delta_saved(const goib2d_delta_desc &d) {
    const int64_t nh = d.n_worlds * d.heads;
    Saved s;
    s.size = delta_full(d) ? 4 : 2;
    // spans of 64 tokens; of 32 where 64 tokens of float32 with their state do not fit in shared memory
    s.keep = s.size == 2 || (d.key_dim <= 64 && d.value_dim <= 64) ? 64 : 32;
    s.tiles_v = (d.value_dim + 15) / 16, s.tiles_k = padded_keys(d.key_dim) / 16;
    s.r = (nh * d.n_steps * d.value_dim * s.size + 15) / 16 * 16;
    s.states = nh * ((d.n_steps + s.keep - 1) / s.keep) * s.tiles_v * s.tiles_k * 256 * s.size;
    s.bytes = s.r + s.states;
    return s;
}

// How the columns of V are shared out in the passes over rollouts: a block takes 64 columns of one (world, head). With
// many, by warps of 32 columns that do everything in turn. Ahead (delta_chunk.cuh), by warps of 16 and two more that
// prepare: where all blocks run at once that way, at 168 registers a thread, and at more than 64 key channels (64
// accumulators a thread with 16 columns). With fewer blocks than SMs, blocks of fewer warps, down to one, for up to
// 100 of them, and 232 registers, which leave an SM one block. Measured, many / ahead, us:
//   rollouts of 256 steps, 64 x 64 bfloat16: 148 (world, head)s 46 / 23, 296: 46 / 27, 444: 57 / 50 (16 steps: 8.4 / 8.8),
//   4096 worlds x 4: 404 / 458; float32: 296 of 256 steps 92 / 59, 444 of 16: 10.5 / 13.1;
//   32 x 32 float32 (three blocks an SM): 444 of 16 steps 6.2 / 5.8, 512: 6.4 / 9.3;
//   128 x 128, training, 64 steps: 1024 x 4 bfloat16 1311 / 1261, 512 x 4 float32 1931 / 1817;
//   128 x 128 bfloat16, training, 37 (world, head)s of 512 steps: 206 at 168 registers, 173 at 232.
// At 444 (world, head)s of 64 x 64 either may win by the number of steps (57 / 50, but 8.4 / 8.8 and 10.5 / 13.1): they are
// the first that do not run at once ahead, and the rule goes by that alone.
struct Split {
    int MT, warps, blocks;
    int ahead;  // 0: no; 1: one block to an SM; 2: more
    explicit Split(const goib2d_delta_desc &d) {
        const int64_t nh = d.n_worlds * d.heads;
        const int tiles = (d.value_dim + 15) / 16, most = tiles < 4 ? tiles : 4;
        const int at_once = 148 * (65536 / (168 * 32 * (most + 2)));
        ahead = d.key_dim > 64 || nh * ((tiles + 3) / 4) <= at_once ? 2 : 0;
        MT = ahead || tiles == 1 ? 1 : 2;
        const int all = (tiles + MT - 1) / MT;
        warps = all < 4 / MT ? all : 4 / MT;
        if (ahead)
            while (warps > 1 && nh * ((all + warps - 1) / warps) < 100) warps = (warps + 1) / 2;
        blocks = (all + warps - 1) / warps;
        if (ahead && nh * blocks <= 148) ahead = 1;
    }
};

// Allow a kernel `bytes` of dynamic shared memory, and the SM's largest share of it for its blocks. The 48 KB that need no
// leave count what the kernel declares itself, too (10 KB at most here).
template <class F>
cudaError_t allow_smem(F *f, size_t bytes) {
    cudaError_t e = cudaFuncSetAttribute(f, cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxShared);
    if (e == cudaSuccess && bytes > 38 << 10)
        e = cudaFuncSetAttribute(f, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
    return e;
}

}  // namespace gb
