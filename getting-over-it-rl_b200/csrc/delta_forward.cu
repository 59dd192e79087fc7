// The gated delta rule over rollouts (goib2d_delta_forward), in chunks of 16 tokens (delta_chunk.cuh).
//
// One block per (world, head); each warp owns MT * 16 columns of S, as the transposed accumulators S^T [V][K] of its
// matrix products, for the whole rollout: q, k, v are read once, o written once, and the state never leaves the
// registers. A chunk's products chain without shared memory: S^T is the A operand of S^T K^T and S^T Q^T, their
// result (V - a Y)^T that of (..) Z^T, its result u^T that of u^T P^T and of the update u^T K. Tiles of two chunks are
// loaded ahead by asynchronous copies while the warps solve the current one; the warps share out the chunks' Z and P.
#include "delta_chunk.cuh"

namespace gb {
namespace {

struct Forward {
    goib2d_delta_desc d;
    void *r;          // [n][h][t][V], or NULL
    void *kept;       // S at the start of every span (Saved), or NULL
    int32_t keep;     // tokens of a span
    int32_t tiles_v;  // 16-column tiles of V
    bool wide_q, wide_k, wide_v, wide_o, wide_r;
};

template <class P, int KP, int MT>
struct Layout {
    static constexpr int pitch = KP + 8, E = sizeof(typename P::E);
    __host__ __device__ static int v_pitch(int warps) { return warps * 16 * MT + (E == 2 ? 8 : 4); }
    __host__ __device__ static int stage(int warps) { return kTile<P> * (2 * pitch + v_pitch(warps)) * E; }
    __host__ __device__ static int bytes(int warps) { return 2 * stage(warps) + kTile<P> / kChunk * (int)sizeof(Chunk<P>); }
};

// A chunk that holds infinities or NaN, token by token: within the products a token meets every other one, if only as 0
// times it, which these values pass. S: the warp's accumulators, in memory.
template <class T, class P, int KP, int MT>
__device__ __noinline__ void odd_chunk(const Forward &f, float *S, const typename P::E *Q, const typename P::E *K,
                                       const typename P::E *V, int vp, int64_t n, int h, int64_t at, int v0, int lane) {
    const goib2d_delta_desc &d = f.d;
    const int g = lane >> 2, t = lane & 3, tokens = (int)(d.n_steps - at < kChunk ? d.n_steps - at : kChunk);
    for (int i = 0; i < tokens; ++i) {
        const Gate gate = load_gate<T>(d, n, at + i, h);
        const float a = gate.fresh ? 0.0f : expf(gate.g);
        for (int m = 0; m < 2 * MT; ++m) {  // the thread's rows
            float *s = S + (m >> 1) * (KP / 8) * 4 + (m & 1) * 2;
            const int v = v0 + 16 * (m >> 1) + 8 * (m & 1) + g;
            float sk = 0.0f, sq = 0.0f, kq = 0.0f;
            for (int j = 0; j < KP / 8; ++j)
                for (int e = 0; e < 2; ++e) {
                    float &x = s[4 * j + e];
                    const float k = to_float(K[i * (KP + 8) + 8 * j + 2 * t + e]), q = to_float(Q[i * (KP + 8) + 8 * j + 2 * t + e]);
                    x = gate.fresh ? 0.0f : a * x;
                    sk += x * k, sq += x * q, kq += k * q;
                }
            for (int o = 1; o < 4; o *= 2)
                sk += __shfl_xor_sync(~0u, sk, o), sq += __shfl_xor_sync(~0u, sq, o), kq += __shfl_xor_sync(~0u, kq, o);
            const float r = to_float(V[i * vp + v]) - sk, u = gate.b * r;
            for (int j = 0; j < KP / 8; ++j)
                for (int e = 0; e < 2; ++e) s[4 * j + e] += to_float(K[i * (KP + 8) + 8 * j + 2 * t + e]) * u;
            if (t == 0 && v < d.value_dim) {
                row<T>(d.out, d.out_stride, n, at + i, h)[v] = from_float<T>(d.scale * (sq + kq * u));
                if (f.r)
                    ((typename P::E *)f.r)[((n * d.heads + h) * d.n_steps + at + i) * d.value_dim + v] =
                        from_float<typename P::E>(r);
            }
        }
    }
}

template <class T, class P, int KP, int MT>
__global__ void __launch_bounds__(MT == 2 ? 128 : 256, MT == 2 && KP <= 64 ? 3 : 1) goib2d_delta_forward_kernel(const __grid_constant__ Forward f) {
    using L = Layout<P, KP, MT>;
    using E = typename P::E;
    constexpr int KT = KP / 16, TILE = kTile<P>;
    constexpr bool half = sizeof(E) == 2;
    extern __shared__ __align__(16) char sm[];
    const goib2d_delta_desc &d = f.d;
    const int K = d.key_dim, V = d.value_dim, threads = blockDim.x, warps = threads / 32;
    const int tid = threadIdx.x, w = tid / 32, lane = tid % 32, t = lane & 3;
    const int64_t nh = blockIdx.x, n = nh / d.heads, steps = d.n_steps;
    const int h = (int)(nh - n * d.heads), hk = h / (d.heads / d.key_heads);
    const int stage = L::stage(warps), vp = L::v_pitch(warps), v0 = w * 16 * MT;
    Chunk<P> *chunks = (Chunk<P> *)(sm + 2 * stage);

    float S[MT][KP / 8][4];  // S^T: rows v, columns k
    load_state<MT, KP>(S, d.state_in ? d.state_in + nh * K * V : nullptr, K, V, v0, lane);

    const T *q0 = row<T>(d.q, d.q_stride, n, 0, hk), *k0 = row<T>(d.k, d.k_stride, n, 0, hk);
    const T *v_0 = row<T>(d.v, d.v_stride, n, 0, h);
    auto load = [&](int64_t tile) {
        E *Q = (E *)(sm + (int)(tile & 1) * stage), *Kb = Q + TILE * L::pitch, *Vb = Kb + TILE * L::pitch;
        const int64_t at = tile * TILE;
        const int left = (int)(steps - at < TILE ? steps - at : TILE);
        load_rows(Q, L::pitch, q0 + at * d.q_stride[1], d.q_stride[1], left, TILE, K, KP, f.wide_q, tid, threads);
        load_rows(Kb, L::pitch, k0 + at * d.k_stride[1], d.k_stride[1], left, TILE, K, KP, f.wide_k, tid, threads);
        load_rows(Vb, vp, v_0 + at * d.v_stride[1], d.v_stride[1], left, TILE, V, warps * 16 * MT, f.wide_v, tid, threads);
        cp_commit();
    };
    const int64_t tiles = (steps + TILE - 1) / TILE;
    if (tiles) load(0);
    Gate gate[TILE / kChunk];
    auto gates = [&](int64_t tile) {
#pragma unroll
        for (int s = 0; s < TILE / kChunk; ++s)
            if ((tile * (TILE / kChunk) + s) % warps == w) gate[s] = load_gate<T>(d, n, tile * TILE + s * kChunk + (lane & 15), h);
    };
    gates(0);
    for (int64_t tile = 0; tile < tiles; ++tile) {
        const E *Q = (const E *)(sm + (int)(tile & 1) * stage), *Kb = Q + TILE * L::pitch;
        E *Vb = (E *)(Kb + TILE * L::pitch);
        cp_wait<0>();
        __syncthreads();
        if (tile + 1 < tiles) load(tile + 1);
#pragma unroll
        for (int s = 0; s < TILE / kChunk; ++s)
            if ((tile * (TILE / kChunk) + s) % warps == w)
                prepare<P, KP, false>(chunks[s], Q + s * kChunk * L::pitch, Kb + s * kChunk * L::pitch, L::pitch, gate[s],
                                      d.scale, lane);
        if (tile + 1 < tiles) gates(tile + 1);
        __syncthreads();
        if (f.kept && tile * TILE % f.keep == 0) {
            const int64_t at = nh * ((steps + f.keep - 1) / f.keep) + tile * TILE / f.keep;
#pragma unroll
            for (int m = 0; m < MT; ++m)
                if (w * MT + m < f.tiles_v) keep_state<KT>((E *)f.kept + (at * f.tiles_v + w * MT + m) * 16 * KP, S[m], lane);
        }
#pragma unroll 1
        for (int s = 0; s < TILE / kChunk; ++s) {
            const int64_t at = tile * TILE + s * kChunk;
            if (at >= steps) break;
            const Chunk<P> &c = chunks[s];
            const E *Qs = Q + s * kChunk * L::pitch, *Ks = Kb + s * kChunk * L::pitch;
            E *Vs = Vb + s * kChunk * vp;
            const uint32_t tokens = steps - at < kChunk ? (1u << (steps - at)) - 1 : 0xffffu;
            float Y[MT][2][4] = {}, O[MT][2][4] = {};
#pragma unroll
            for (int j = 0; j < KT; ++j) {
                const typename P::B1 kb = P::n_rows(Ks, L::pitch, 0, 16 * j, lane), qb = P::n_rows(Qs, L::pitch, 0, 16 * j, lane);
#pragma unroll
                for (int m = 0; m < MT; ++m) {
                    const typename P::A2 a = P::exact(S[m][2 * j], S[m][2 * j + 1]);
                    P::mul(Y[m][0], Y[m][1], a, kb);
                    P::mul(O[m][0], O[m][1], P::first(a), qb);  // Half: o is rounded to bfloat16, S once before it
                }
            }
            const typename P::B2 z = c.z.k_rows(lane);
            float bad = 0.0f;
#pragma unroll
            for (int m = 0; m < MT; ++m) {
                float x[2][4];
                P::values_t(x, Vs, vp, 0, v0 + 16 * m, lane);
#pragma unroll
                for (int j = 0; j < 2; ++j)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const int i = j * 8 + 2 * t + (e & 1);
                        x[j][e] -= c.a[i] * Y[m][j][e];
                        O[m][j][e] *= c.sa[i];
                        Y[m][j][e] = 0.0f;
                    }
                P::mul(Y[m][0], Y[m][1], P::exact(x[0], x[1]), z);  // r
#pragma unroll
                for (int j = 0; j < 2; ++j)
#pragma unroll
                    for (int e = 0; e < 4; ++e) bad = fmaf(0.0f, Y[m][j][e], bad);
            }
            if (__any_sync(~0u, c.odd || bad != 0.0f)) {
                float s[MT * (KP / 8) * 4];
#pragma unroll
                for (int i = 0; i < MT * (KP / 8) * 4; ++i) s[i] = S[i / (KP / 2)][i / 4 % (KP / 8)][i % 4];
                odd_chunk<T, P, KP, MT>(f, s, Qs, Ks, Vs, vp, n, h, at, v0, lane);
#pragma unroll
                for (int i = 0; i < MT * (KP / 8) * 4; ++i) S[i / (KP / 2)][i / 4 % (KP / 8)][i % 4] = s[i];
                continue;
            }
            if (f.r) {
                E *to = (E *)f.r + (nh * steps + at) * V;
                if (half)
                    store_rows<MT>((bf16 *)to, V, tokens, v0, V, f.wide_r, (bf16 *)Vs, vp, Y, lane);
                else
#pragma unroll
                    for (int m = 0; m < MT; ++m) store_direct<E>(to, V, tokens, v0 + 16 * m, V, Y[m], lane);
            }
            typename P::A2 u[MT];
            {
                const typename P::B1 p = c.p.n_rows1(lane);
#pragma unroll
                for (int m = 0; m < MT; ++m) {
                    P::mul(O[m][0], O[m][1], P::rounded(Y[m][0], Y[m][1]), p);
#pragma unroll
                    for (int j = 0; j < 2; ++j)
#pragma unroll
                        for (int e = 0; e < 4; ++e) Y[m][j][e] *= c.bd[j * 8 + 2 * t + (e & 1)];
                    u[m] = P::exact(Y[m][0], Y[m][1]);
                }
            }
            T *to = row<T>(d.out, d.out_stride, n, at, h);
            if (half)
                store_rows<MT>((bf16 *)to, d.out_stride[1], tokens, v0, V, f.wide_o, (bf16 *)Vs, vp, O, lane);
            else
#pragma unroll
                for (int m = 0; m < MT; ++m) store_direct<T>(to, d.out_stride[1], tokens, v0 + 16 * m, V, O[m], lane);
            const float a_end = c.a_end;
#pragma unroll
            for (int j = 0; j < KT; ++j) {
                const typename P::B1 kb = P::k_rows(Ks, L::pitch, 0, 16 * j, lane);
#pragma unroll
                for (int m = 0; m < MT; ++m) {
                    float(&c0)[4] = S[m][2 * j], (&c1)[4] = S[m][2 * j + 1];
#pragma unroll
                    for (int e = 0; e < 4; ++e) c0[e] *= a_end, c1[e] *= a_end;
                    P::mul(c0, c1, u[m], kb);
                }
            }
        }
    }
    store_state<MT, KP>(d.state_out + nh * K * V, S, K, V, v0, lane);
}

template <class T, class P, int KP, int MT>
cudaError_t forward_of(const Forward &f, cudaStream_t s) {
    const int warps = (f.d.value_dim + 16 * MT - 1) / (16 * MT);
    const size_t smem = Layout<P, KP, MT>::bytes(warps);
    cudaError_t e = allow_smem(goib2d_delta_forward_kernel<T, P, KP, MT>, smem);
    if (e != cudaSuccess) return e;
    goib2d_delta_forward_kernel<T, P, KP, MT><<<(unsigned)(f.d.n_worlds * f.d.heads), 32 * warps, smem, s>>>(f);
    return cudaGetLastError();
}

template <class T, class P, int KP>
cudaError_t forward_wide(const Forward &f, cudaStream_t s) {
    return f.d.value_dim <= 16 ? forward_of<T, P, KP, 1>(f, s) : forward_of<T, P, KP, 2>(f, s);
}

template <class T, class P>
cudaError_t forward_typed(const goib2d_delta_desc &d, void *saved, cudaStream_t s) {
    Forward f{d};
    const Saved at = delta_saved(d);
    f.r = saved, f.kept = saved ? (char *)saved + at.r : nullptr, f.keep = at.keep, f.tiles_v = at.tiles_v;
    const int V = d.value_dim, z = sizeof(T);
    f.wide_q = rows_aligned(d.q, d.q_stride, d.n_worlds, d.n_steps, d.key_heads, d.key_dim, z);
    f.wide_k = rows_aligned(d.k, d.k_stride, d.n_worlds, d.n_steps, d.key_heads, d.key_dim, z);
    f.wide_v = rows_aligned(d.v, d.v_stride, d.n_worlds, d.n_steps, d.heads, V, z);
    f.wide_o = rows_aligned(d.out, d.out_stride, d.n_worlds, d.n_steps, d.heads, V, z);
    f.wide_r = V % 8 == 0;
    switch (padded_keys(d.key_dim)) {
        case 16: return forward_wide<T, P, 16>(f, s);
        case 32: return forward_wide<T, P, 32>(f, s);
        case 64: return forward_wide<T, P, 64>(f, s);
        default: return forward_wide<T, P, 128>(f, s);
    }
}

}  // namespace

int64_t delta_saved_bytes(const goib2d_delta_desc &d) { return delta_saved(d).bytes; }

cudaError_t launch_delta_forward(const goib2d_delta_desc &d, void *saved, cudaStream_t s) {
    if (d.dtype == GOIB2D_FLOAT32) return forward_typed<float, Full>(d, saved, s);
    return saved && delta_full(d) ? forward_typed<bf16, Full>(d, saved, s) : forward_typed<bf16, Half>(d, saved, s);
}

}  // namespace gb
