// The gated delta rule over rollouts (goib2d_delta_forward), in chunks of 16 tokens (delta_chunk.cuh).
//
// A block takes some columns of V of one (world, head); a warp owns MT * 16 of them, as the transposed accumulators S^T
// [V][K] of its matrix products, for the whole rollout: v is read once, o written once, and the state never leaves the
// registers. A chunk's products chain without shared memory: S^T is the A operand of S^T K^T and S^T Q^T, their result
// (V - a Y)^T that of (..) Z^T, its result r^T that of r^T P^T and of the update u^T K.
//
// 4096 worlds x 64 steps x 4 heads of 64 x 64, bfloat16: 403 us, 2.7 TB/s of inputs, outputs and states; 47 % of the issue
// slots at 12 warps an SM, bound by the instructions between the products (about 13 of 14 are no products) and their
// latencies. 8 x 8192 x 4 of 128 x 128: 732 us, 1.4 us a chunk, bound by the chain of a chunk's products.
#include "delta_chunk.cuh"

namespace gb {
namespace {

struct Forward {
    goib2d_delta_desc d;
    void *r;          // [n][h][t][V], or NULL
    void *kept;       // S at the start of every span (Saved), or NULL
    int32_t keep;     // tokens of a span
    int32_t tiles_v;  // 16-column tiles of V
    int grain_q, grain_k, grain_v;  // rows_grain
    bool wide_o, wide_r;                     // rows of 16-byte pieces
};

template <class P, int KP, int MT, bool AHEAD>
struct Layout {
    using E = typename P::E;
    static constexpr int pitch = KP + 8, slots = AHEAD ? 4 : 2, chunks = AHEAD ? 2 : kTile<P> / kChunk;
    static constexpr int rows = AHEAD ? kChunk : kTile<P>;  // of a slot
    __host__ __device__ static int v_pitch(int warps) { return warps * 16 * MT + (sizeof(E) == 2 ? 8 : 4); }
    __host__ __device__ static int slot(int warps) { return rows * (2 * pitch + v_pitch(warps)) * (int)sizeof(E); }
    __host__ __device__ static int bytes(int warps) { return slots * slot(warps) + chunks * (int)sizeof(Chunk<P>); }
};

// A chunk that holds infinities or NaN, token by token: within the products a token meets every other one, if only as 0
// times it, which these values pass. S: the warp's accumulators, in memory.
template <class T, class P, class R, int KP, int MT>
__device__ __noinline__ void odd_chunk(const Forward &f, float *S, const typename P::E *Q, const typename P::E *K,
                                       const typename P::E *V, int vp, int64_t n, int h, int64_t at, int v0, int lane) {
    const goib2d_delta_desc &d = f.d;
    const int g = lane >> 2, t = lane & 3, tokens = (int)(d.n_steps - at < kChunk ? d.n_steps - at : kChunk);
    for (int i = 0; i < tokens; ++i) {
        const Gate gate = Gates<T>(d, n, h).at(at + i).get();
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
            const float r = to_float(V[i * vp + v - v0]) - sk, u = gate.b * r;
            for (int j = 0; j < KP / 8; ++j)
                for (int e = 0; e < 2; ++e) s[4 * j + e] += to_float(K[i * (KP + 8) + 8 * j + 2 * t + e]) * u;
            if (t == 0 && v < d.value_dim) {
                row<T>(d.out, d.out_stride, n, at + i, h)[v] = from_float<T>(d.scale * (sq + kq * u));
                if (f.r)
                    ((R *)f.r)[((n * d.heads + h) * d.n_steps + at + i) * d.value_dim + v] = from_float<R>(r);
            }
        }
    }
}

// R: the type of what is kept
template <class T, class P, class R, int KP, int MT, int AHEAD>
__global__ void __maxnreg__(AHEAD == 1 ? 232 : 168)  // 168: 12 warps an SM, two blocks ahead
    goib2d_delta_forward_kernel(const __grid_constant__ Forward f) {
    using L = Layout<P, KP, MT, AHEAD != 0>;
    using E = typename P::E;
    constexpr int KT = KP / 16;
    constexpr bool half = sizeof(E) == 2;
    extern __shared__ __align__(16) char sm[];
    const goib2d_delta_desc &d = f.d;
    const int K = d.key_dim, V = d.value_dim, w = threadIdx.x / 32, lane = threadIdx.x % 32, t = lane & 3;
    const int warps = blockDim.x / 32 - (AHEAD ? 2 : 0), threads = blockDim.x;
    const int64_t nh = blockIdx.x, n = nh / d.heads;
    const int steps = (int)d.n_steps, count = (steps + kChunk - 1) / kChunk;
    const int h = (int)(nh - n * d.heads), hk = h / (d.heads / d.key_heads);
    const int slot = L::slot(warps), vp = L::v_pitch(warps), block0 = blockIdx.y * warps * 16 * MT;
    Chunk<P> *chunks = (Chunk<P> *)(sm + L::slots * slot);
    const T *const q = row<T>(d.q, d.q_stride, n, 0, hk), *const k = row<T>(d.k, d.k_stride, n, 0, hk);
    const T *const v = row<T>(d.v, d.v_stride, n, 0, h) + block0;
    const int qs = (int)d.q_stride[1], ks = (int)d.k_stride[1], vs = (int)d.v_stride[1];
    const Gates<T> gates(d, n, h);

    if (AHEAD && w >= warps) {
        // every second chunk; two slots of rows and one chunk's matrices are this warp's
        const int me = w - warps;
        auto load = [&](int i) {
            const int at = i * kChunk, left = steps - at;
            if (left > 0) {
                E *Q = (E *)(sm + (i & 3) * slot), *Kb = Q + kChunk * L::pitch, *Vb = Kb + kChunk * L::pitch;
                chunk_rows(Q, L::pitch, q + (int64_t)at * qs, qs, left, K, KP, f.grain_q, lane);
                chunk_rows(Kb, L::pitch, k + (int64_t)at * ks, ks, left, K, KP, f.grain_k, lane);
                chunk_rows(Vb, vp, v + (int64_t)at * vs, vs, left, V - block0, warps * 16 * MT, f.grain_v, lane);
            }
            cp_commit();
        };
        load(me);
        RawGate<T> next = gates.at(me * kChunk + (lane & 15));
        for (int i = me; i < count; i += 2) {
            if (i >= 2) bar_wait(3 + me, 32 + 32 * warps);  // chunk i - 2 is solved: its slot and its matrices are free
            load(i + 2);
            const RawGate<T> gate = next;
            next = gates.at((i + 2) * kChunk + (lane & 15));
            cp_wait<1>();
            __syncwarp();
            const E *Q = (const E *)(sm + (i & 3) * slot);
            prepare<P, KP, false>(chunks[me], Q, Q + kChunk * L::pitch, L::pitch, gate.get(), d.scale, lane);
            __threadfence_block();
            bar_arrive(1 + me, 32 + 32 * warps);
        }
        return;
    }

    const int v0 = w * 16 * MT, tile0 = block0 / 16 + w * MT;  // columns within the block; the first tile of V
    float S[MT][KP / 8][4];  // S^T: rows v, columns k
    load_state<MT, KP>(S, d.state_in ? d.state_in + nh * K * V : nullptr, K, V, block0 + v0, lane);
    T *const out = row<T>(d.out, d.out_stride, n, 0, h) + block0;
    R *const r = f.r ? (R *)f.r + nh * steps * V + block0 : nullptr;
    const int os = (int)d.out_stride[1];
    auto solve = [&](int at, const E *Qs, const E *Ks, E *Vs, const Chunk<P> &c) {
            if (f.kept && at % f.keep == 0) {
                const int64_t x = (nh * ((steps + f.keep - 1) / f.keep) + at / f.keep) * f.tiles_v + tile0;
#pragma unroll
                for (int m = 0; m < MT; ++m)
                    if (tile0 + m < f.tiles_v) keep_state<KT>((R *)f.kept + (x + m) * 16 * KP, S[m], lane);
            }
            const uint32_t tokens = steps - at < kChunk ? (1u << (steps - at)) - 1 : 0xffffu;
            float Y[MT][2][4] = {}, O[MT][2][4] = {};
#pragma unroll
            for (int j = 0; j < KT; ++j) {
                const typename P::B1 kb = P::n_rows(Ks, L::pitch, 0, 16 * j, lane), qb = P::n_rows(Qs, L::pitch, 0, 16 * j, lane);
#pragma unroll
                for (int m = 0; m < MT; ++m) {
                    const typename P::A2 a = P::exact(S[m][2 * j], S[m][2 * j + 1]);
                    P::mul(Y[m][0], Y[m][1], a, kb);
                    P::mul(O[m][0], O[m][1], P::first(a), qb);  // Half: S is rounded once, as o is: 1.9e-3 off, 1.7e-3 is o's own rounding
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
                odd_chunk<T, P, R, KP, MT>(f, s, Qs, Ks, Vs + v0, vp, n, h, at, block0 + v0, lane);
#pragma unroll
                for (int i = 0; i < MT * (KP / 8) * 4; ++i) S[i / (KP / 2)][i / 4 % (KP / 8)][i % 4] = s[i];
                return;
            }
            if (r) {
                R *to = r + (int64_t)at * V;
                if (sizeof(R) == 2)
                    store_rows<MT>((bf16 *)to, V, tokens, v0, V - block0, f.wide_r, (bf16 *)Vs, vp, Y, lane);
                else
#pragma unroll
                    for (int m = 0; m < MT; ++m) store_direct<R>(to, V, tokens, v0 + 16 * m, V - block0, Y[m], lane);
            }
            typename P::A2 u[MT];
            {
                const typename P::B2 p = c.p.n_rows(lane);
#pragma unroll
                for (int m = 0; m < MT; ++m) {
                    P::mul(O[m][0], O[m][1], P::exact(Y[m][0], Y[m][1]), p);
#pragma unroll
                    for (int j = 0; j < 2; ++j)
#pragma unroll
                        for (int e = 0; e < 4; ++e) Y[m][j][e] *= c.bd[j * 8 + 2 * t + (e & 1)];
                    u[m] = P::exact(Y[m][0], Y[m][1]);
                }
            }
            T *to = out + (int64_t)at * os;
            if (half)
                store_rows<MT>((bf16 *)to, os, tokens, v0, V - block0, f.wide_o, (bf16 *)Vs, vp, O, lane);
            else
#pragma unroll
                for (int m = 0; m < MT; ++m) store_direct<T>(to, os, tokens, v0 + 16 * m, V - block0, O[m], lane);
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
    };
    if constexpr (AHEAD) {
#pragma unroll 1
        for (int i = 0; i < count; ++i) {
            E *Q = (E *)(sm + (i & 3) * slot);
            bar_wait(1 + (i & 1), 32 + 32 * warps);
            solve(i * kChunk, Q, Q + kChunk * L::pitch, Q + 2 * kChunk * L::pitch, chunks[i & 1]);
            if (i + 2 < count) bar_arrive(3 + (i & 1), 32 + 32 * warps);
        }
    } else {
        constexpr int TILE = kTile<P>, N = TILE / kChunk;
        const int tiles = (steps + TILE - 1) / TILE;
        auto load = [&](int tile) {
            E *Q = (E *)(sm + (tile & 1) * slot), *Kb = Q + TILE * L::pitch, *Vb = Kb + TILE * L::pitch;
            const int at = tile * TILE, left = steps - at < TILE ? steps - at : TILE;
            load_rows(Q, L::pitch, q + (int64_t)at * qs, qs, left, TILE, K, KP, f.grain_q, threadIdx.x, threads);
            load_rows(Kb, L::pitch, k + (int64_t)at * ks, ks, left, TILE, K, KP, f.grain_k, threadIdx.x, threads);
            load_rows(Vb, vp, v + (int64_t)at * vs, vs, left, TILE, V - block0, warps * 16 * MT, f.grain_v, threadIdx.x, threads);
            cp_commit();
        };
        RawGate<T> gate[N];
        // the tiles' chunks are prepared by the warps in turn; `first`: the warp of the tile's first one
        auto turn_of = [&](int first, int s) { 
            const int x = first + s;  // at most three over
            return x < warps ? x : x - warps < warps ? x - warps : x - 2 * warps < warps ? x - 2 * warps : 0;
        };
        auto gates_of = [&](int tile, int first) {
#pragma unroll
            for (int s = 0; s < N; ++s)
                if (turn_of(first, s) == w) gate[s] = gates.at(tile * TILE + s * kChunk + (lane & 15));
        };
        if (tiles) load(0), gates_of(0, 0);
        int turn = 0;
#pragma unroll 1
        for (int tile = 0; tile < tiles; ++tile) {
            E *Q = (E *)(sm + (tile & 1) * slot), *Kb = Q + TILE * L::pitch, *Vb = Kb + TILE * L::pitch;
            cp_wait<0>();
            __syncthreads();
            if (tile + 1 < tiles) load(tile + 1);
#pragma unroll
            for (int s = 0; s < N; ++s)
                if (turn_of(turn, s) == w)
                    prepare<P, KP, false>(chunks[s], Q + s * kChunk * L::pitch, Kb + s * kChunk * L::pitch, L::pitch, gate[s].get(),
                                          d.scale, lane);
            turn = turn_of(turn, N);
            if (tile + 1 < tiles) gates_of(tile + 1, turn);
            __syncthreads();
#pragma unroll 1
            for (int s = 0; s < N && tile * TILE + s * kChunk < steps; ++s)
                solve(tile * TILE + s * kChunk, Q + s * kChunk * L::pitch, Kb + s * kChunk * L::pitch, Vb + s * kChunk * vp,
                      chunks[s]);
        }
    }
    store_state<MT, KP>(d.state_out + nh * K * V, S, K, V, block0 + v0, lane);
}

template <class T, class P, class R, int KP, int MT, int AHEAD>
cudaError_t forward_of(const Forward &f, const Split &b, cudaStream_t s) {
    const size_t smem = Layout<P, KP, MT, AHEAD != 0>::bytes(b.warps);
    cudaError_t e = allow_smem(goib2d_delta_forward_kernel<T, P, R, KP, MT, AHEAD>, smem);
    if (e != cudaSuccess) return e;
    goib2d_delta_forward_kernel<T, P, R, KP, MT, AHEAD>
        <<<dim3((unsigned)(f.d.n_worlds * f.d.heads), b.blocks), 32 * (b.warps + (AHEAD ? 2 : 0)), smem, s>>>(f);
    return cudaGetLastError();
}

template <class T, class P, class R, int KP>
cudaError_t forward_wide(const Forward &f, cudaStream_t s) {
    const Split b(f.d);
    if (b.ahead == 1) return forward_of<T, P, R, KP, 1, 1>(f, b, s);
    if constexpr (KP < 128) {
        if (b.ahead == 0) return b.MT == 2 ? forward_of<T, P, R, KP, 2, 0>(f, b, s) : forward_of<T, P, R, KP, 1, 0>(f, b, s);
    }
    return forward_of<T, P, R, KP, 1, 2>(f, b, s);
}

template <class T, class P, class R>
cudaError_t forward_typed(const goib2d_delta_desc &d, void *saved, cudaStream_t s) {
    Forward f{d};
    const Saved at = delta_saved(d);
    f.r = saved, f.kept = saved ? (char *)saved + at.r : nullptr, f.keep = at.keep, f.tiles_v = at.tiles_v;
    const int V = d.value_dim, z = sizeof(T);
    f.grain_q = rows_grain(d.q, d.q_stride, d.n_worlds, d.n_steps, d.key_heads, d.key_dim, z);
    f.grain_k = rows_grain(d.k, d.k_stride, d.n_worlds, d.n_steps, d.key_heads, d.key_dim, z);
    f.grain_v = rows_grain(d.v, d.v_stride, d.n_worlds, d.n_steps, d.heads, V, z);
    f.wide_o = rows_grain(d.out, d.out_stride, d.n_worlds, d.n_steps, d.heads, V, z) == 16;
    f.wide_r = V % 8 == 0;
    switch (padded_keys(d.key_dim)) {
        case 32: return forward_wide<T, P, R, 32>(f, s);
        case 64: return forward_wide<T, P, R, 64>(f, s);
        default: return forward_wide<T, P, R, 128>(f, s);
    }
}

}  // namespace

int64_t delta_saved_bytes(const goib2d_delta_desc &d) { return delta_saved(d).bytes; }

// What is kept for gradients in full products is float32. The forward products do not change with it, so that o and the
// last state are the same bits whether gradients are wanted or not.
cudaError_t launch_delta_forward(const goib2d_delta_desc &d, void *saved, cudaStream_t s) {
    if (d.dtype == GOIB2D_FLOAT32) return forward_typed<float, Full, float>(d, saved, s);
    return saved && delta_full(d) ? forward_typed<bf16, Half, float>(d, saved, s) : forward_typed<bf16, Half, bf16>(d, saved, s);
}

}  // namespace gb
