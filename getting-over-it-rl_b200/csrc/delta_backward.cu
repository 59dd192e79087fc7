// Gradients of the gated delta rule (goib2d_delta_backward), in two kernels around the states that the forward pass kept,
// and a third that redoes what came out with infinities or NaN.
//
// The first goes backwards through the rollout as the forward kernel goes forwards: a warp holds dS^T for its columns
// of V in the accumulators of its products. With X the gradient that reaches u from outside the chunk's own recurrence,
//     X = P^T dO + d (K dS1),  du = (I + diag(b) W)^-T X,  dv = b du,  db = du . r,
//     dS0 = a_16 dS1 + Q^T (scale a dO) - K^T (a dv);
// it writes dv and db, and dS at the ends of the spans of `keep` tokens.
//
// The second takes every span by itself, as there is nothing left to carry: with the span's first state S0 and last
// gradient dS1, and D over the span's tokens,
//     A_ij = scale D_ij b_j dO_i.r_j (j <= i),  M_ij = -D_ij b_j dv_i.r_j (j < i),
//     dq = scale a (dO S0^T) + A K,   dk = -a (dv S0^T) + M K + d b (r dS1^T) + A^T Q + M^T K.
// A decay's gradient is the sum of all that passes from before its token to its token or after: pairs j < l <= i of
// A_ij q_i.k_j + M_ij k_i.k_j, what i >= l reads of S0, what j < l leaves in the last state, and a_end <S0, dS1>. Summing
// these pairs keeps the relative precision where decays are strong; the difference q.dq - k.dk cancels there.
//
// What only bfloat16 results depend on is rounded to bfloat16 (Half): r, S0, dS1, dv, A and M as operands here, of one
// product each, and held so between the kernels. dq, dk, dg and db are 2.3e-3 to 3.0e-3 off by it where the rounding of the
// results alone gives 1.7e-3. A and M unrounded on the row side: dq 2.9e-3 -> 2.3e-3, and 5 % more time.
//
// 4096 worlds x 64 steps x 4 heads of 64 x 64, bfloat16: 0.42 ms, bound as the forward pass, and 0.61 ms, 38 % of the issue
// slots at 12 warps an SM (74 KB of rows and 168 registers allow three blocks): loads, barriers and instruction latency.
// 32 channels of dq and dk a warp instead of 64 (16 warps an SM) makes A and M twice: 0.25 ms slower.
#include "delta_chunk.cuh"

namespace gb {
namespace {

struct Backward {
    goib2d_delta_desc d;
    goib2d_delta_grads gr;
    const void *r, *kept_s;  // what the forward pass saved (Saved)
    void *kept_ds;           // dS after each span, in the same layout
    void *dv;                // dv as the second kernel reads it: gr.dv, or float32 in the workspace
    int64_t dv_stride[3];
    float *db;               // db by warps' columns: [n][h][parts][t]
    int32_t *odd;            // [n][key head][span]: whether a result is not finite
    int32_t keep, tiles_v, parts;
    int grain_q, grain_k, grain_do, grain_dv, grain_r;  // rows_grain
    bool wide_dv;            // rows of dv are 16-byte pieces
    bool wide_dqk;           // pairs of channels of dq and dk are aligned
};

// ---- dS through the rollout, dv and db

template <class P, int KP, int MT, bool AHEAD>
struct Layout {
    using E = typename P::E;
    static constexpr int pitch = KP + 8, chunks = AHEAD ? 2 : kTile<P> / kChunk;
    static constexpr int rows = AHEAD ? kChunk : kTile<P>;  // of a slot
    static constexpr int keys = AHEAD ? 4 : 2, values = AHEAD ? 4 : 1;  // slots of q and k, of dO and r
    __host__ __device__ static int v_pitch(int warps) { return warps * 16 * MT + (sizeof(E) == 2 ? 8 : 4); }
    __host__ __device__ static int bytes(int warps) {
        return 2 * rows * (keys * pitch + values * v_pitch(warps)) * (int)sizeof(E) + chunks * (int)sizeof(Chunk<P>);
    }
};

template <class T, class P, int KP, int MT, int AHEAD>
__global__ void __maxnreg__(AHEAD == 1 ? 232 : 168)  // 168: 12 warps an SM, two blocks ahead
    goib2d_delta_back_state_kernel(const __grid_constant__ Backward f) {
    using L = Layout<P, KP, MT, AHEAD != 0>;
    using E = typename P::E;
    constexpr int KT = KP / 16;
    constexpr bool half = sizeof(E) == 2;
    extern __shared__ __align__(16) char sm[];
    const goib2d_delta_desc &d = f.d;
    const int K = d.key_dim, V = d.value_dim, w = threadIdx.x / 32, lane = threadIdx.x % 32, g = lane >> 2, t = lane & 3;
    const int warps = blockDim.x / 32 - (AHEAD ? 2 : 0), threads = blockDim.x;
    const int64_t nh = blockIdx.x, n = nh / d.heads;
    const int steps = (int)d.n_steps, count = (steps + kChunk - 1) / kChunk;
    const int h = (int)(nh - n * d.heads), hk = h / (d.heads / d.key_heads);
    const int vp = L::v_pitch(warps), cols = warps * 16 * MT, block0 = blockIdx.y * cols;
    const int key_slot = 2 * L::rows * L::pitch, value_slot = 2 * L::rows * vp;
    E *const keys = (E *)sm, *const values = keys + L::keys * key_slot;
    Chunk<P> *chunks = (Chunk<P> *)(values + L::values * value_slot);
    const T *const q = row<T>(d.q, d.q_stride, n, 0, hk), *const k = row<T>(d.k, d.k_stride, n, 0, hk);
    const T *const o = f.gr.dout ? row<T>(f.gr.dout, f.gr.dout_stride, n, 0, h) + block0 : nullptr;
    const E *const r = (const E *)f.r + nh * steps * V + block0;
    const int qs = (int)d.q_stride[1], ks = (int)d.k_stride[1], os = (int)f.gr.dout_stride[1];
    const Gates<T> gates(d, n, h);

    if (AHEAD && w >= warps) {
        // every second chunk, from the last down (i-th: chunk count - 1 - i); two slots and one chunk's matrices
        const int me = w - warps;
        auto load = [&](int i) {
            const int at = (count - 1 - i) * kChunk, left = steps - at;
            if (at >= 0) {
                E *Q = keys + (i & 3) * key_slot, *Ob = values + (i & 3) * value_slot;
                chunk_rows(Q, L::pitch, q + (int64_t)at * qs, qs, left, K, KP, f.grain_q, lane);
                chunk_rows(Q + kChunk * L::pitch, L::pitch, k + (int64_t)at * ks, ks, left, K, KP, f.grain_k, lane);
                chunk_rows(Ob, vp, o + (int64_t)at * os, os, o ? left : 0, V - block0, cols, f.grain_do, lane);
                chunk_rows(Ob + kChunk * vp, vp, r + (int64_t)at * V, V, left, V - block0, cols, f.grain_r, lane);
            }
            cp_commit();
        };
        auto gate_of = [&](int i) { return gates.at((int64_t)(count - 1 - i) * kChunk + (lane & 15)); };
        load(me);
        RawGate<T> next = gate_of(me);
        for (int i = me; i < count; i += 2) {
            if (i >= 2) bar_wait(3 + me, 32 + 32 * warps);  // i - 2 is done: its slot and its matrices are free
            load(i + 2);
            const RawGate<T> gate = next;
            next = gate_of(i + 2);
            cp_wait<1>();
            __syncwarp();
            const E *Q = keys + (i & 3) * key_slot;
            prepare<P, KP, true>(chunks[me], Q, Q + kChunk * L::pitch, L::pitch, gate.get(), d.scale, lane);
            __threadfence_block();
            bar_arrive(1 + me, 32 + 32 * warps);
        }
        return;
    }

    const int v0 = w * 16 * MT, tile0 = block0 / 16 + w * MT;
    float S[MT][KP / 8][4];  // dS^T: rows v, columns k
    load_state<MT, KP>(S, f.gr.dstate_out ? f.gr.dstate_out + nh * K * V : nullptr, K, V, block0 + v0, lane);
    T *const dv = row<T>(f.gr.dv, f.gr.dv_stride, n, 0, h) + block0;
    E *const also = !half && f.dv != f.gr.dv ? row<E>(f.dv, f.dv_stride, n, 0, h) + block0 : nullptr;
    float *const db = tile0 < f.tiles_v ? f.db + (nh * f.parts + tile0 / MT) * steps : nullptr;
    const int dvs = (int)f.gr.dv_stride[1];
    auto solve = [&](int at, const E *Qs, const E *Ks, const E *Os, E *Rs, const Chunk<P> &c) {
            if ((at + kChunk) % f.keep == 0 || at + kChunk >= steps) {
                const int64_t x = (nh * ((steps + f.keep - 1) / f.keep) + at / f.keep) * f.tiles_v + tile0;
#pragma unroll
                for (int m = 0; m < MT; ++m)
                    if (tile0 + m < f.tiles_v) keep_state<KT>((E *)f.kept_ds + (x + m) * 16 * KP, S[m], lane);
            }
            const uint32_t tokens = steps - at < kChunk ? (1u << (steps - at)) - 1 : 0xffffu;
            float X[MT][2][4] = {};
#pragma unroll
            for (int j = 0; j < KT; ++j) {
                const typename P::B1 kb = P::n_rows(Ks, L::pitch, 0, 16 * j, lane);
#pragma unroll
                for (int m = 0; m < MT; ++m) P::mul(X[m][0], X[m][1], P::exact(S[m][2 * j], S[m][2 * j + 1]), kb);
            }
            typename P::A2 o[MT], y[MT];
            float sum[4] = {};
            {
                const typename P::B2 z = c.z.n_rows(lane), p = c.p.k_rows(lane);
#pragma unroll
                for (int m = 0; m < MT; ++m) {
#pragma unroll
                    for (int j = 0; j < 2; ++j)
#pragma unroll
                        for (int e = 0; e < 4; ++e) X[m][j][e] *= c.d[j * 8 + 2 * t + (e & 1)];
                    P::mul(X[m][0], X[m][1], P::a_cols(Os, vp, 0, v0 + 16 * m, lane), p);
                    const typename P::A2 x = P::exact(X[m][0], X[m][1]);
                    float r[2][4];
                    P::values_t(r, Rs, vp, 0, v0 + 16 * m, lane);
#pragma unroll
                    for (int j = 0; j < 2; ++j)
#pragma unroll
                        for (int e = 0; e < 4; ++e) X[m][j][e] = 0.0f;
                    P::mul(X[m][0], X[m][1], x, z);  // du
#pragma unroll
                    for (int j = 0; j < 2; ++j)
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            sum[2 * j + (e & 1)] += X[m][j][e] * r[j][e];
                            X[m][j][e] *= c.b[j * 8 + 2 * t + (e & 1)];  // dv
                        }
                }
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                for (int i = 4; i < 32; i *= 2) sum[e] += __shfl_xor_sync(~0u, sum[e], i);
                const int token = (e >> 1) * 8 + 2 * t + (e & 1);
                if (g == 0 && db && at + token < steps) db[at + token] = sum[e];
            }
            T *to = dv + (int64_t)at * dvs;
            if (half) {
                store_rows<MT>((bf16 *)to, dvs, tokens, v0, V - block0, f.wide_dv, (bf16 *)Rs, vp, X, lane);
            } else {
#pragma unroll
                for (int m = 0; m < MT; ++m) store_direct<T>(to, dvs, tokens, v0 + 16 * m, V - block0, X[m], lane);
                if (also)
#pragma unroll
                    for (int m = 0; m < MT; ++m)
                        store_direct<E>(also + (int64_t)at * f.dv_stride[1], (int)f.dv_stride[1], tokens, v0 + 16 * m, V - block0,
                                        X[m], lane);
            }
#pragma unroll
            for (int m = 0; m < MT; ++m) {
                float x[2][4];
                P::values_t(x, Os, vp, 0, v0 + 16 * m, lane);
#pragma unroll
                for (int j = 0; j < 2; ++j)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        x[j][e] *= c.sa[j * 8 + 2 * t + (e & 1)];
                        X[m][j][e] *= -c.a[j * 8 + 2 * t + (e & 1)];
                    }
                o[m] = P::exact(x[0], x[1]);
                y[m] = P::exact(X[m][0], X[m][1]);
            }
            const float a_end = c.a_end;
#pragma unroll
            for (int j = 0; j < KT; ++j) {
                const typename P::B1 qb = P::k_rows(Qs, L::pitch, 0, 16 * j, lane);
#pragma unroll
                for (int m = 0; m < MT; ++m) {
                    float(&c0)[4] = S[m][2 * j], (&c1)[4] = S[m][2 * j + 1];
#pragma unroll
                    for (int e = 0; e < 4; ++e) c0[e] *= a_end, c1[e] *= a_end;
                    P::mul(c0, c1, o[m], qb);
                }
                const typename P::B1 kb = P::k_rows(Ks, L::pitch, 0, 16 * j, lane);
#pragma unroll
                for (int m = 0; m < MT; ++m) P::mul(S[m][2 * j], S[m][2 * j + 1], y[m], kb);
            }
    };
    if constexpr (AHEAD) {
#pragma unroll 1
        for (int i = 0; i < count; ++i) {
            const E *Q = keys + (i & 3) * key_slot;
            E *Ob = values + (i & 3) * value_slot;
            bar_wait(1 + (i & 1), 32 + 32 * warps);
            solve((count - 1 - i) * kChunk, Q, Q + kChunk * L::pitch, Ob, Ob + kChunk * vp, chunks[i & 1]);
            if (i + 2 < count) bar_arrive(3 + (i & 1), 32 + 32 * warps);
        }
    } else {
        // q and k twice, the next tile's coming while this one is solved; dO and r once, coming while the chunks are prepared
        constexpr int TILE = kTile<P>, N = TILE / kChunk;
        const int tiles = (steps + TILE - 1) / TILE;
        E *const Ob = values, *const Rb = values + TILE * vp;
        auto load_keys = [&](int tile) {
            E *Q = keys + (tile & 1) * key_slot;
            const int at = tile * TILE, left = steps - at < TILE ? steps - at : TILE;
            load_rows(Q, L::pitch, q + (int64_t)at * qs, qs, left, TILE, K, KP, f.grain_q, threadIdx.x, threads);
            load_rows(Q + TILE * L::pitch, L::pitch, k + (int64_t)at * ks, ks, left, TILE, K, KP, f.grain_k, threadIdx.x, threads);
            cp_commit();
        };
        auto load_values = [&](int tile) {
            const int at = tile * TILE, left = steps - at < TILE ? steps - at : TILE;
            load_rows(Ob, vp, o + (int64_t)at * os, os, o ? left : 0, TILE, V - block0, cols, f.grain_do, threadIdx.x, threads);
            load_rows(Rb, vp, r + (int64_t)at * V, V, left, TILE, V - block0, cols, f.grain_r, threadIdx.x, threads);
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
        if (tiles) load_keys(tiles - 1), gates_of(tiles - 1, 0);
        int turn = 0;
#pragma unroll 1
        for (int tile = tiles - 1; tile >= 0; --tile) {
            const E *Q = keys + (tile & 1) * key_slot, *Kb = Q + TILE * L::pitch;
            cp_wait<0>();
            __syncthreads();
            load_values(tile);
            if (tile > 0) load_keys(tile - 1);
#pragma unroll
            for (int s = 0; s < N; ++s)
                if (turn_of(turn, s) == w)
                    prepare<P, KP, true>(chunks[s], Q + s * kChunk * L::pitch, Kb + s * kChunk * L::pitch, L::pitch, gate[s].get(),
                                         d.scale, lane);
            turn = turn_of(turn, N);
            if (tile > 0) gates_of(tile - 1, turn), cp_wait<1>();
            else cp_wait<0>();
            __syncthreads();
#pragma unroll 1
            for (int s = N - 1; s >= 0; --s)
                if (tile * TILE + s * kChunk < steps)
                    solve(tile * TILE + s * kChunk, Q + s * kChunk * L::pitch, Kb + s * kChunk * L::pitch, Ob + s * kChunk * vp,
                          Rb + s * kChunk * vp, chunks[s]);
        }
    }
    if (f.gr.dstate_in) store_state<MT, KP>(f.gr.dstate_in + nh * K * V, S, K, V, block0 + v0, lane);
}

// ---- dq, dk and dg, span by span
//
// A span is cut into blocks of 16 tokens, one a warp. Between two blocks D_ij = a_i m d_j, a_i the decay from i's
// block's start, d_j that to j's block's end, m that of the blocks between: products instead of exponentials, all of
// them at most what they make. A warp takes its tokens first as i, over the blocks before them, then as j, over those
// behind: A and M go through shared memory where they fit (Half), and are made again from the other side otherwise.

template <class P, int KP, int C>
struct Span {
    using E = typename P::E;
    static constexpr int RB = C / 16;                   // blocks
    static constexpr int KH = KP < 64 ? KP : 64;        // channels of dq and dk a warp holds
    static constexpr int warps = RB * (KP / KH);
    static constexpr int pitch = KP + 8;
    static constexpr bool store = sizeof(E) == 2;
    struct Tokens {
        float a[C], d[C], b[C], hi[C], lo[C];           // within the block; hi + lo: the running sum of g / ln 2
        float through[RB];                              // a block's whole decay
        int since[C];                                   // tokens of the block up to this one that start afresh
        float row[KP / KH][C], col[KP / KH][C];         // what a token reads of S0, leaves in the last state
        float own[C], rows[C], cols[RB][C], end[warps]; // the pairs of a decay, see below
    };
    E *Q, *K, *O, *V, *R, *S, *A, *M;                   // S: S0^T, then dS1^T (rows v, columns k); A, M: 16 x 24 a block
    Tokens *x;
    __host__ __device__ static int v_pitch(int tiles_v) { return tiles_v * 16 + 8; }
    __host__ __device__ static int bytes(int tiles_v) {
        return (int)sizeof(E) * (2 * C * pitch + 3 * C * v_pitch(tiles_v) + tiles_v * 16 * pitch +
                                 (store ? RB * (RB + 1) * 16 * 24 : 0)) + (int)sizeof(Tokens);
    }
    __device__ Span(char *sm, int tiles_v) {
        const int vp = v_pitch(tiles_v);
        Q = (E *)sm, K = Q + C * pitch, O = K + C * pitch, V = O + C * vp, R = V + C * vp, S = R + C * vp;
        A = S + tiles_v * 16 * pitch, M = A + (store ? RB * (RB + 1) / 2 * 16 * 24 : 0);
        x = (Tokens *)(M + (store ? RB * (RB + 1) / 2 * 16 * 24 : 0));
    }
    static __device__ __forceinline__ int block(int ib, int jb) { return (ib * (ib + 1) / 2 + jb) * 16 * 24; }
};

__device__ __forceinline__ void store_pair(bf16 *p, float x, float y) { *(uint32_t *)p = pack(x, y); }
__device__ __forceinline__ void store_pair(float *p, float x, float y) { *(float2 *)p = make_float2(x, y); }
__device__ __forceinline__ void put_block(bf16 *p, const Half::A1 &a, int lane) {  // rows and columns as accumulators
    bf16 *q = p + (lane >> 2) * 24 + 2 * (lane & 3);
    *(uint32_t *)q = a.x[0], *(uint32_t *)(q + 8 * 24) = a.x[1];
    *(uint32_t *)(q + 8) = a.x[2], *(uint32_t *)(q + 8 * 24 + 8) = a.x[3];
}

template <class T, class P, int KP, int C>
__global__ void __launch_bounds__(Span<P, KP, C>::warps * 32, sizeof(typename P::E) == 4 ? 1 : KP == 128 ? 1 : KP == 64 ? 3 : 4)
    goib2d_delta_back_span_kernel(const __grid_constant__ Backward f) {
    using L = Span<P, KP, C>;
    using E = typename P::E;
    constexpr int RB = L::RB, KH = L::KH, threads = L::warps * 32, PL = C / 32;
    constexpr int N = 16 / sizeof(E), B = 4;
    extern __shared__ __align__(16) char sm[];
    const goib2d_delta_desc &d = f.d;
    const int K = d.key_dim, V = d.value_dim, tv = f.tiles_v, vp = L::v_pitch(tv), cols = tv * 16;
    const int tid = threadIdx.x, w = tid / 32, lane = tid % 32, g = lane >> 2, t = lane & 3;
    const int rb = w % RB, part = w / RB, k0 = part * KH;  // the warp's block of tokens, and its channels
    const int i0 = rb * 16 + g;                            // the thread's rows: i0, i0 + 8
    const int64_t steps = d.n_steps, spans = (steps + C - 1) / C;
    const int64_t item = blockIdx.x / spans, span = blockIdx.x - item * spans, at = span * C, n = item / d.key_heads;
    const int hk = (int)(item - n * d.key_heads), group = d.heads / d.key_heads;
    const int left = (int)(steps - at < C ? steps - at : C);
    const L s(sm, tv);
    auto &x = *s.x;

    load_rows(s.Q, L::pitch, row<T>(d.q, d.q_stride, n, at, hk), (int)d.q_stride[1], left, C, K, KP, f.grain_q, tid, threads);
    load_rows(s.K, L::pitch, row<T>(d.k, d.k_stride, n, at, hk), (int)d.k_stride[1], left, C, K, KP, f.grain_k, tid, threads);
    float dq[KH / 8][4] = {}, dk[KH / 8][4] = {};
#pragma unroll 1
    for (int j = 0; j < group; ++j) {
        const int h = hk * group + j;
        const int64_t nh = n * d.heads + h, kept = (nh * spans + span) * cols * KP;
        const Gates<T> gates(d, n, h);
        const RawGate<T> raw = gates.at(at + rb * 16 + (lane & 15)), first = gates.at(at);
        __syncthreads();
        const bool o = f.gr.dout != nullptr;
        load_rows(s.O, vp, o ? row<T>(f.gr.dout, f.gr.dout_stride, n, at, h) : nullptr, (int)f.gr.dout_stride[1], o ? left : 0, C, V,
                  cols, f.grain_do, tid, threads);
        load_rows(s.V, vp, row<E>((const void *)f.dv, f.dv_stride, n, at, h), (int)f.dv_stride[1], left, C, V, cols, f.grain_dv, tid,
                  threads);
        load_rows(s.R, vp, (const E *)f.r + (nh * steps + at) * V, V, left, C, V, cols, f.grain_r, tid, threads);
        // S0 may hold anything where the span's first token starts afresh: it is not used then
        const E *kept_s = (const E *)f.kept_s + kept, *kept_ds = (const E *)f.kept_ds + kept;
        load_rows(s.S, L::pitch, kept_s, KP, cols, cols, KP, KP, 16, tid, threads);
        cp_commit();
        const bool anew = first.get().fresh;
        float end = 0.0f;
        for (int i = tid * N; i < cols * KP; i += threads * N * B) {  // B pairs of loads in flight
            uint4 u[B], v[B];
#pragma unroll
            for (int e = 0; e < B; ++e) {
                const bool in = i + e * threads * N < cols * KP;
                u[e] = in ? *(const uint4 *)(kept_s + i + e * threads * N) : make_uint4(0, 0, 0, 0);
                v[e] = in ? *(const uint4 *)(kept_ds + i + e * threads * N) : make_uint4(0, 0, 0, 0);
            }
#pragma unroll
            for (int e = 0; e < B; ++e) end += dot16<E>(u[e], v[e]);
        }
        for (int i = 16; i > 0; i >>= 1) end += __shfl_xor_sync(~0u, end, i);
        if (lane == 0) x.end[w] = anew ? 0.0f : end;
        if (part == 0) {
            const int i = lane & 15;
            const Gate gate = raw.get();
            const double G = running_sum(gate, lane), last = __shfl_sync(~0u, G, 15);
            const uint32_t fresh = __ballot_sync(~0u, gate.fresh) & 0xffffu;
            const int since = __popc(fresh & ((2u << i) - 1)), all = __popc(fresh);
            if (lane < 16) {
                const int l = rb * 16 + i;
                x.a[l] = since ? 0.0f : exp2_fast((float)G), x.d[l] = since == all ? exp2_fast((float)(last - G)) : 0.0f;
                x.b[l] = gate.b, x.hi[l] = (float)G, x.lo[l] = (float)(G - (double)(float)G), x.since[l] = since;
                if (i == 0) x.through[rb] = all ? 0.0f : exp2_fast((float)last);
                if (l < left) {
                    float db = 0.0f;
                    for (int e = 0; e < f.parts; ++e) db += f.db[(nh * f.parts + e) * steps + at + l];
                    *row<T>(f.gr.dbeta, f.gr.dbeta_stride, n, at + l, h) = from_float<T>(db);
                    dq[0][0] = fmaf(0.0f, db, dq[0][0]);  // nothing, or NaN: looked for below
                }
            }
        }
        cp_wait<0>();
        __syncthreads();

        const float a_i[2] = {x.a[i0], x.a[i0 + 8]}, b_i[2] = {x.b[i0], x.b[i0 + 8]}, d_i[2] = {x.d[i0], x.d[i0 + 8]};
        float to = 1.0f, from = 1.0f;  // the decay of the blocks before, and behind
        for (int i = 0; i < rb; ++i) to *= x.through[i];
        for (int i = rb + 1; i < RB; ++i) from *= x.through[i];
        // what the tokens read of S0
        float sum[2] = {};
        if (!anew) {
#pragma unroll
            for (int which = 0; which < 2; ++which) {
                float acc[KH / 8][4] = {};
                const E *A = which ? s.V : s.O, *with = which ? s.K : s.Q;
#pragma unroll 1
                for (int v = 0; v < tv; ++v) {
                    const typename P::A1 fa = P::a_rows(A, vp, rb * 16, v * 16, lane);
#pragma unroll
                    for (int c = 0; c < KH / 16; ++c)
                        P::mul(acc[2 * c], acc[2 * c + 1], fa, P::k_rows(s.S, L::pitch, v * 16, k0 + c * 16, lane));
                }
#pragma unroll
                for (int r = 0; r < 2; ++r) {
                    const float scaled = (which ? -1.0f : d.scale) * a_i[r] * to;
                    const E *p = with + (i0 + 8 * r) * L::pitch + k0 + 2 * t;
#pragma unroll
                    for (int c = 0; c < KH / 8; ++c) {
                        const float y0 = scaled * acc[c][2 * r], y1 = scaled * acc[c][2 * r + 1];
                        const float2 z = pair_at(p + 8 * c);
                        sum[r] += z.x * y0 + z.y * y1;
                        if (which) dk[c][2 * r] += y0, dk[c][2 * r + 1] += y1;
                        else dq[c][2 * r] += y0, dq[c][2 * r + 1] += y1;
                    }
                }
            }
        }
        // the tokens as i: A and M over the tokens up to them. For dg, the pairs A_ij q_i.k_j + M_ij k_i.k_j: those of one
        // block by the tokens l between (own[l]), the others by rows (rows[i]) and by columns (cols[block of i][j])
        float rows[2] = {}, m = 1.0f;
#pragma unroll 1
        for (int jb = rb; jb >= 0; --jb) {
            float A[2][4] = {}, M[2][4] = {}, qk[2][4] = {}, kk[2][4] = {};
#pragma unroll 2
            for (int v = 0; v < tv; ++v) {
                const typename P::B1 fr = P::n_rows(s.R, vp, jb * 16, v * 16, lane);
                P::mul(A[0], A[1], P::a_rows(s.O, vp, rb * 16, v * 16, lane), fr);
                P::mul(M[0], M[1], P::a_rows(s.V, vp, rb * 16, v * 16, lane), fr);
            }
            if (part == 0)
#pragma unroll
                for (int c = 0; c < KP / 16; ++c) {
                    const typename P::B1 fj = P::n_rows(s.K, L::pitch, jb * 16, c * 16, lane);
                    P::mul(qk[0], qk[1], P::a_rows(s.Q, L::pitch, rb * 16, c * 16, lane), fj);
                    P::mul(kk[0], kk[1], P::a_rows(s.K, L::pitch, rb * 16, c * 16, lane), fj);
                }
            if (jb == rb) {
#pragma unroll
                for (int r = 0; r < 2; ++r) {
                    const float hi = x.hi[i0 + 8 * r], lo = x.lo[i0 + 8 * r];
                    const int since = x.since[i0 + 8 * r];
                    float upto = 0.0f;  // the sum over the columns before
#pragma unroll
                    for (int nt = 0; nt < 2; ++nt) {
                        float pair[2];
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            const int col = nt * 8 + 2 * t + e, jj = rb * 16 + col;
                            const bool seen = col <= g + 8 * r && x.since[jj] == since, past = seen && col < g + 8 * r;
                            const float D = seen ? exp2_fast((hi - x.hi[jj]) + (lo - x.lo[jj])) * x.b[jj] : 0.0f;
                            float &y = A[nt][2 * r + e], &z = M[nt][2 * r + e];
                            y = seen ? d.scale * D * y : 0.0f;
                            z = past ? -D * z : 0.0f;
                            pair[e] = past ? y * qk[nt][2 * r + e] + z * kk[nt][2 * r + e] : 0.0f;
                        }
                        float incl = pair[0] + pair[1], y = __shfl_up_sync(~0u, incl, 1, 4);
                        if (t >= 1) incl += y;
                        y = __shfl_up_sync(~0u, incl, 2, 4);
                        if (t >= 2) incl += y;
                        const float excl = __shfl_up_sync(~0u, incl, 1, 4), before = upto + (t ? excl : 0.0f);
                        // tokens l = these columns, up to the row: pairs over the columns before l
                        qk[nt][2 * r] = nt * 8 + 2 * t <= g + 8 * r ? before : 0.0f;
                        qk[nt][2 * r + 1] = nt * 8 + 2 * t < g + 8 * r ? before + pair[0] : 0.0f;
                        upto += __shfl_sync(~0u, incl, 3, 4);
                    }
                }
#pragma unroll
                for (int nt = 0; nt < 2; ++nt)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        float y = qk[nt][e] + qk[nt][2 + e];
                        for (int i = 4; i < 32; i *= 2) y += __shfl_xor_sync(~0u, y, i);
                        if (part == 0 && g == 0) x.own[rb * 16 + nt * 8 + 2 * t + e] = y;
                    }
            } else {
                const float f0 = a_i[0] * m, f1 = a_i[1] * m;
#pragma unroll
                for (int nt = 0; nt < 2; ++nt)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const int jj = jb * 16 + nt * 8 + 2 * t + e;
                        const float fc = x.d[jj] * x.b[jj], fs = fc * d.scale;
                        float &y0 = A[nt][e], &y1 = A[nt][2 + e], &z0 = M[nt][e], &z1 = M[nt][2 + e];
                        y0 *= f0 * fs, y1 *= f1 * fs, z0 *= -f0 * fc, z1 *= -f1 * fc;
                        const float p0 = y0 * qk[nt][e] + z0 * kk[nt][e], p1 = y1 * qk[nt][2 + e] + z1 * kk[nt][2 + e];
                        rows[0] += p0, rows[1] += p1;
                        float y = p0 + p1;
                        for (int i = 4; i < 32; i *= 2) y += __shfl_xor_sync(~0u, y, i);
                        if (part == 0 && g == 0) x.cols[rb][jj] = y;
                    }
                m *= x.through[jb];
            }
            const typename P::A1 fa = P::rounded(A[0], A[1]), fm = P::rounded(M[0], M[1]);
            if constexpr (L::store)
                if (part == 0) put_block(s.A + L::block(rb, jb), fa, lane), put_block(s.M + L::block(rb, jb), fm, lane);
#pragma unroll
            for (int c = 0; c < KH / 16; ++c) {
                const typename P::B1 fk = P::k_rows(s.K, L::pitch, jb * 16, k0 + c * 16, lane);
                P::mul(dq[2 * c], dq[2 * c + 1], fa, fk);
                P::mul(dk[2 * c], dk[2 * c + 1], fm, fk);
            }
        }
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            for (int i = 1; i < 4; i *= 2) sum[r] += __shfl_xor_sync(~0u, sum[r], i), rows[r] += __shfl_xor_sync(~0u, rows[r], i);
            if (t == 0) x.row[part][i0 + 8 * r] = sum[r];
            if (t == 0 && part == 0) x.rows[i0 + 8 * r] = rows[r];
        }
        __syncthreads();
        load_rows(s.S, L::pitch, kept_ds, KP, cols, cols, KP, KP, 16, tid, threads);
        cp_commit();
        // the tokens as j: A and M over the tokens from them on
        m = 1.0f;
#pragma unroll 1
        for (int ib = rb; ib < RB; ++ib) {
            typename P::A1 fa, fm;
            if constexpr (L::store) {
                fa = P::a_cols(s.A + L::block(ib, rb), 24, 0, 0, lane), fm = P::a_cols(s.M + L::block(ib, rb), 24, 0, 0, lane);
            } else {
                float A[2][4] = {}, M[2][4] = {};
#pragma unroll 2
                for (int v = 0; v < tv; ++v) {
                    const typename P::A1 fr = P::a_rows(s.R, vp, rb * 16, v * 16, lane);
                    P::mul(A[0], A[1], fr, P::n_rows(s.O, vp, ib * 16, v * 16, lane));
                    P::mul(M[0], M[1], fr, P::n_rows(s.V, vp, ib * 16, v * 16, lane));
                }
                if (ib == rb) {
#pragma unroll
                    for (int nt = 0; nt < 2; ++nt)
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const int r = e >> 1, jj = i0 + 8 * r, i = ib * 16 + nt * 8 + 2 * t + (e & 1);
                            const bool seen = jj <= i && x.since[i] == x.since[jj];
                            const float D = seen ? exp2_fast((x.hi[i] - x.hi[jj]) + (x.lo[i] - x.lo[jj])) * b_i[r] : 0.0f;
                            A[nt][e] = seen ? d.scale * D * A[nt][e] : 0.0f;
                            M[nt][e] = seen && jj < i ? -D * M[nt][e] : 0.0f;
                        }
                } else {
#pragma unroll
                    for (int nt = 0; nt < 2; ++nt)
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const float D = x.a[ib * 16 + nt * 8 + 2 * t + (e & 1)] * m * (d_i[e >> 1] * b_i[e >> 1]);
                            A[nt][e] *= d.scale * D, M[nt][e] *= -D;
                        }
                    m *= x.through[ib];
                }
                fa = P::rounded(A[0], A[1]), fm = P::rounded(M[0], M[1]);
            }
#pragma unroll
            for (int c = 0; c < KH / 16; ++c) {
                P::mul(dk[2 * c], dk[2 * c + 1], fa, P::k_rows(s.Q, L::pitch, ib * 16, k0 + c * 16, lane));
                P::mul(dk[2 * c], dk[2 * c + 1], fm, P::k_rows(s.K, L::pitch, ib * 16, k0 + c * 16, lane));
            }
        }
        cp_wait<0>();
        __syncthreads();
        // what they leave in the last state
        {
            float acc[KH / 8][4] = {};
#pragma unroll 1
            for (int v = 0; v < tv; ++v) {
                const typename P::A1 fa = P::a_rows(s.R, vp, rb * 16, v * 16, lane);
#pragma unroll
                for (int c = 0; c < KH / 16; ++c)
                    P::mul(acc[2 * c], acc[2 * c + 1], fa, P::k_rows(s.S, L::pitch, v * 16, k0 + c * 16, lane));
            }
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                const float scaled = d_i[r] * from * b_i[r];
                const E *p = s.K + (i0 + 8 * r) * L::pitch + k0 + 2 * t;
                float y = 0.0f;
#pragma unroll
                for (int c = 0; c < KH / 8; ++c) {
                    const float y0 = scaled * acc[c][2 * r], y1 = scaled * acc[c][2 * r + 1];
                    const float2 z = pair_at(p + 8 * c);
                    y += z.x * y0 + z.y * y1;
                    dk[c][2 * r] += y0, dk[c][2 * r + 1] += y1;
                }
                y += __shfl_xor_sync(~0u, y, 1);
                y += __shfl_xor_sync(~0u, y, 2);
                if (t == 0) x.col[part][i0 + 8 * r] = y;
            }
        }
        __syncthreads();
        if (w == 0) {  // dg, PL neighbouring tokens a lane
            float reads[PL], leaves[PL], own[PL], behind[PL];
            float read_sum = 0.0f, leave_sum = 0.0f, own_sum = 0.0f, behind_sum = 0.0f, middle[RB] = {};
            const int lb = lane * PL / 16;
#pragma unroll
            for (int e = 0; e < PL; ++e) {
                const int l = lane * PL + e;
                reads[e] = x.row[0][l], leaves[e] = x.col[0][l], own[e] = x.rows[l], behind[e] = 0.0f;
                for (int i = 1; i < KP / KH; ++i) reads[e] += x.row[i][l], leaves[e] += x.col[i][l];
#pragma unroll
                for (int i = 1; i < RB; ++i) {
                    const float y = i > lb ? x.cols[i][l] : 0.0f;
                    behind[e] += y;
#pragma unroll
                    for (int b = 1; b < i; ++b) middle[b] += lb < b ? y : 0.0f;  // pairs that pass over the whole block b
                }
                read_sum += reads[e], leave_sum += leaves[e], own_sum += own[e], behind_sum += behind[e];
            }
            float read_all = read_sum, leave_all = leave_sum, own_all = own_sum, behind_all = behind_sum;
            constexpr int LB = 16 / PL;  // lanes of a block
#pragma unroll
            for (int i = 1; i < 32; i *= 2) {
                float y = __shfl_down_sync(~0u, read_all, i);
                if (lane + i < 32) read_all += y;
                y = __shfl_up_sync(~0u, leave_all, i);
                if (lane >= i) leave_all += y;
                if (i < LB) {
                    y = __shfl_down_sync(~0u, own_all, i, LB);
                    if (lane % LB + i < LB) own_all += y;
                    y = __shfl_up_sync(~0u, behind_all, i, LB);
                    if (lane % LB >= i) behind_all += y;
                }
#pragma unroll
                for (int b = 1; b < RB - 1; ++b) middle[b] += __shfl_xor_sync(~0u, middle[b], i);
            }
            float through = 0.0f, y;
            for (int i = 0; i < L::warps; ++i) through += x.end[i];
            for (int i = 0; i < RB; ++i) through *= x.through[i];
            // of the lanes behind (reads; own pairs' rows in the block), and of the lanes before (leaves; columns in the block)
            y = __shfl_down_sync(~0u, read_all, 1), read_sum = lane < 31 ? y : 0.0f;
            y = __shfl_up_sync(~0u, leave_all, 1), leave_sum = lane ? y : 0.0f;
            y = __shfl_down_sync(~0u, own_all, 1, LB), own_sum = lane % LB < LB - 1 ? y : 0.0f;
            y = __shfl_up_sync(~0u, behind_all, 1, LB), behind_sum = lane % LB ? y : 0.0f;
#pragma unroll
            for (int b = 1; b < RB - 1; ++b)
                if (b == lb) through += middle[b];
            float mine[PL];
#pragma unroll
            for (int e = 0; e < PL; ++e) {
                mine[e] = through + leave_sum + behind_sum + x.own[lane * PL + e];
                leave_sum += leaves[e], behind_sum += behind[e];
            }
#pragma unroll
            for (int e = PL - 1; e >= 0; --e) {
                const int l = lane * PL + e;
                read_sum += reads[e], own_sum += own[e];
                const bool fresh = x.since[l] != (l % 16 ? x.since[l - 1] : 0);
                const float dg = fresh ? 0.0f : mine[e] + read_sum + own_sum;
                dq[0][0] = fmaf(0.0f, dg, dq[0][0]);
                if (l < left) *row<T>(f.gr.dg, f.gr.dg_stride, n, at + l, h) = from_float<T>(dg);
            }
        }
    }
    float odd[4] = {};
#pragma unroll
    for (int c = 0; c < KH / 8; ++c)
#pragma unroll
        for (int e = 0; e < 4; ++e) odd[e] = fmaf(0.0f, dq[c][e], fmaf(0.0f, dk[c][e], odd[e]));
#pragma unroll
    for (int r = 0; r < 2; ++r) {
        if (i0 + 8 * r >= left) continue;
        T *q = row<T>(f.gr.dq, f.gr.dq_stride, n, at + i0 + 8 * r, hk) + k0 + 2 * t;
        T *k = row<T>(f.gr.dk, f.gr.dk_stride, n, at + i0 + 8 * r, hk) + k0 + 2 * t;
#pragma unroll
        for (int c = 0; c < KH / 8; ++c) {
            const int left_k = K - (k0 + c * 8 + 2 * t);
            if (left_k >= 2 && f.wide_dqk) {
                store_pair(q + 8 * c, dq[c][2 * r], dq[c][2 * r + 1]), store_pair(k + 8 * c, dk[c][2 * r], dk[c][2 * r + 1]);
            } else {
                if (left_k >= 1) q[8 * c] = from_float<T>(dq[c][2 * r]), k[8 * c] = from_float<T>(dk[c][2 * r]);
                if (left_k >= 2) q[8 * c + 1] = from_float<T>(dq[c][2 * r + 1]), k[8 * c + 1] = from_float<T>(dk[c][2 * r + 1]);
            }
        }
    }
    const bool any = __syncthreads_or((odd[0] + odd[1]) + (odd[2] + odd[3]) != 0.0f);
    if (tid == 0) f.odd[blockIdx.x] = any;
}

// ---- what is not finite, token by token
//
// Within the products above a token meets every other one, if only as 0 times it, which infinities and NaN pass: from a
// world that blew up they would reach the gradients of its episodes before and after. Whatever is not finite in the
// inputs shows in dq, dk, dg or db of its span, or of one before. This kernel takes the (world, key head)s of such spans, a
// block each, and replaces all their gradients by those of the definition, where they end at the tokens that start
// afresh. A thread holds 16 channels of a column of S and of dS; S at a token is made again from the last one put down in
// shared memory (every 8 tokens, or as many as fit). Latency: 1.1 ms for 64 tokens of 64 x 64 (4.1 without what is put
// down); 0.13 s where a head of each of 4096 worlds is odd. Otherwise it reads the flags: 5 to 9 us.
constexpr int kOddThreads = 1024, kOddColumns = 128, kOddParts = kOddThreads / kOddColumns, kOddRows = 128 / kOddParts;

template <class T, class E>
__global__ void __launch_bounds__(kOddThreads) goib2d_delta_back_odd_kernel(const __grid_constant__ Backward f, int KP, int stride) {
    extern __shared__ __align__(16) float sums[];  // dq, dk of the span's tokens; S before every stride-th one
    __shared__ float du_of[kOddParts][kOddColumns], dqk_of[2][kOddColumns / 32][128], dgb_of[kOddThreads / 32][2];
    __shared__ int found[kOddThreads / 32];
    const goib2d_delta_desc &d = f.d;
    const goib2d_delta_grads &gr = f.gr;
    const int K = d.key_dim, V = d.value_dim, group = d.heads / d.key_heads, tid = threadIdx.x, w = tid / 32, lane = tid % 32;
    const int v = tid % kOddColumns, part = tid / kOddColumns, count = part < K ? (K - part + kOddParts - 1) / kOddParts : 0;
    const bool live = v < V;
    float *const down = sums + 2 * f.keep * K;
    const int64_t steps = d.n_steps, spans = (steps + f.keep - 1) / f.keep, items = d.n_worlds * d.key_heads;

    auto redo = [&](int64_t item) {
        const int64_t n = item / d.key_heads;
        const int hk = (int)(item - n * d.key_heads);
        for (int64_t span = spans - 1; span >= 0; --span) {
            const int64_t at = span * f.keep;
            const int tokens = (int)(steps - at < f.keep ? steps - at : f.keep);
            for (int i = tid; i < 2 * tokens * K; i += kOddThreads) sums[i] = 0.0f;
            for (int j = 0; j < group; ++j) {
                const int h = hk * group + j;
                const int64_t nh = n * d.heads + h, states = nh * spans * f.tiles_v * 16 * KP;
                const E *const first = (const E *)f.kept_s + states + (span * f.tiles_v * 16 + v) * KP;
                const E *const r = (const E *)f.r + (nh * steps + at) * V + v;
                // dS between spans, in float32: over the head's kept dS, which are used up, and larger where there are two
                float *const carry = (float *)((E *)f.kept_ds + states) + (int64_t)part * V + v;
                const float *const last = gr.dstate_out ? gr.dstate_out + nh * K * V + (int64_t)part * V + v : nullptr;
                const Gates<T> gates(d, n, h);
                float S[kOddRows], dS[kOddRows], k[kOddRows];
                auto load_key = [&](int64_t l) {
                    const T *p = row<T>(d.k, d.k_stride, n, l, hk) + part;
#pragma unroll
                    for (int e = 0; e < kOddRows; ++e) k[e] = e < count ? to_float(p[e * kOddParts]) : 0.0f;
                };
#pragma unroll
                for (int e = 0; e < kOddRows; ++e) {
                    dS[e] = 0.0f;
                    if (live && e < count) {
                        if (span + 1 < spans) dS[e] = carry[e * kOddParts * V];
                        else if (last) dS[e] = last[e * kOddParts * V];
                    }
                }
                // S from before token `from` to token i, decayed but not written to; what is passed at whole strides is
                // put down. Each thread reads only what it put down itself.
                Gate gate;
                auto replay = [&](int from, int i, bool put) {
                    for (int l = from;; ++l) {
                        if (put && l && l % stride == 0)
#pragma unroll
                            for (int e = 0; e < kOddRows; ++e)
                                if (live && e < count) down[((int64_t)(l / stride - 1) * K + part + e * kOddParts) * V + v] = S[e];
                        gate = gates.at(at + l).get();
                        load_key(at + l);
                        const float a = expf(gate.g);
#pragma unroll
                        for (int e = 0; e < kOddRows; ++e) S[e] = gate.fresh ? 0.0f : a * S[e];
                        if (l == i) break;
                        const float u = live ? gate.b * to_float(r[(int64_t)l * V]) : 0.0f;
#pragma unroll
                        for (int e = 0; e < kOddRows; ++e) S[e] += k[e] * u;
                    }
                };
                for (int i = tokens - 1; i >= 0; --i) {
                    const bool all = i == tokens - 1;
                    const int slot = all ? 0 : i / stride;
#pragma unroll
                    for (int e = 0; e < kOddRows; ++e) {
                        S[e] = 0.0f;
                        if (live && e < count)
                            S[e] = slot ? down[((int64_t)(slot - 1) * K + part + e * kOddParts) * V + v] : to_float(first[part + e * kOddParts]);
                    }
                    replay(slot * stride, i, all);
                    const float rest = live ? to_float(r[(int64_t)i * V]) : 0.0f, u = live ? gate.b * rest : 0.0f;
                    const float dout = live && gr.dout ? to_float(row<T>(gr.dout, gr.dout_stride, n, at + i, h)[v]) : 0.0f;
                    const T *const q = row<T>(d.q, d.q_stride, n, at + i, hk) + part;
                    float du = 0.0f;
#pragma unroll
                    for (int e = 0; e < kOddRows; ++e) {
                        if (live && e < count) dS[e] += d.scale * to_float(q[e * kOddParts]) * dout;
                        du += dS[e] * k[e];
                    }
                    du_of[part][v] = du;
                    __syncthreads();
                    du = 0.0f;
                    for (int e = 0; e < kOddParts; ++e) du += du_of[e][v];
                    const float dv = live ? gate.b * du : 0.0f, a = expf(gate.g);
                    float dg = 0.0f, db = live && part == 0 ? du * rest : 0.0f;
#pragma unroll
                    for (int e = 0; e < kOddRows; ++e) {
                        float x = (S[e] + k[e] * u) * dout, y = dS[e] * u - S[e] * dv;
                        for (int o = 16; o > 0; o /= 2) x += __shfl_xor_sync(~0u, x, o), y += __shfl_xor_sync(~0u, y, o);
                        if (lane == 0) dqk_of[0][w % 4][part + e * kOddParts] = x, dqk_of[1][w % 4][part + e * kOddParts] = y;
                        dS[e] -= k[e] * dv;  // of S before the write
                        dg += S[e] * dS[e];
                        dS[e] = gate.fresh ? 0.0f : a * dS[e];
                    }
                    for (int o = 16; o > 0; o /= 2) dg += __shfl_xor_sync(~0u, dg, o), db += __shfl_xor_sync(~0u, db, o);
                    if (lane == 0) dgb_of[w][0] = dg, dgb_of[w][1] = db;
                    if (live && part == 0) row<T>(gr.dv, gr.dv_stride, n, at + i, h)[v] = from_float<T>(dv);
                    __syncthreads();
                    if (tid < 2 * K) {
                        const int of_k = tid >= K, c = tid - of_k * K;
                        float x = 0.0f;
                        for (int e = 0; e < kOddColumns / 32; ++e) x += dqk_of[of_k][e][c];
                        sums[(of_k * tokens + i) * K + c] += of_k ? x : d.scale * x;
                    }
                    if (tid == kOddThreads - 1) {
                        dg = db = 0.0f;
                        for (int e = 0; e < kOddThreads / 32; ++e) dg += dgb_of[e][0], db += dgb_of[e][1];
                        *row<T>(gr.dg, gr.dg_stride, n, at + i, h) = from_float<T>(gate.fresh ? 0.0f : dg);
                        *row<T>(gr.dbeta, gr.dbeta_stride, n, at + i, h) = from_float<T>(db);
                    }
                }
                float *const to = span ? carry : gr.dstate_in ? gr.dstate_in + nh * K * V + (int64_t)part * V + v : nullptr;
                if (to)
#pragma unroll
                    for (int e = 0; e < kOddRows; ++e)
                        if (live && e < count) to[e * kOddParts * V] = dS[e];
            }
            __syncthreads();
            for (int i = tid; i < tokens * K; i += kOddThreads) {
                const int l = i / K, c = i - l * K;
                row<T>(gr.dq, gr.dq_stride, n, at + l, hk)[c] = from_float<T>(sums[i]);
                row<T>(gr.dk, gr.dk_stride, n, at + l, hk)[c] = from_float<T>(sums[tokens * K + i]);
            }
            __syncthreads();
        }
    };
    for (int64_t i = blockIdx.x; i < items; i += (int64_t)gridDim.x * (kOddThreads / 32)) {
        const int64_t mine = i + (int64_t)w * gridDim.x;  // a warp looks at one
        int odd = 0;
        if (mine < items)
            for (int64_t s = lane; s < spans; s += 32) odd |= f.odd[mine * spans + s];
        odd = __any_sync(~0u, odd);
        if (lane == 0) found[w] = odd;
        if (!__syncthreads_or(odd)) continue;
        for (int e = 0; e < kOddThreads / 32; ++e)
            if (found[e]) redo(i + (int64_t)e * gridDim.x);
        __syncthreads();
    }
}

template <class T, class E>
cudaError_t back_odd(const Backward &f, cudaStream_t s) {
    const int64_t items = f.d.n_worlds * f.d.key_heads;
    if (!items || !f.d.n_steps) return cudaSuccess;
    int stride = 8;
    auto bytes = [&] { return 4ll * f.d.key_dim * (2 * f.keep + (f.keep - 1) / stride * f.d.value_dim); };
    while (bytes() > 200 << 10) stride *= 2;
    cudaError_t e = allow_smem(goib2d_delta_back_odd_kernel<T, E>, bytes());
    if (e != cudaSuccess) return e;
    goib2d_delta_back_odd_kernel<T, E>
        <<<(unsigned)(items < 148 ? items : 148), kOddThreads, bytes(), s>>>(f, padded_keys(f.d.key_dim), stride);
    return cudaGetLastError();
}

template <class T, class P, int KP, int MT, int AHEAD>
cudaError_t back_state(const Backward &f, const Split &b, cudaStream_t s) {
    const size_t smem = Layout<P, KP, MT, AHEAD != 0>::bytes(b.warps);
    cudaError_t e = allow_smem(goib2d_delta_back_state_kernel<T, P, KP, MT, AHEAD>, smem);
    if (e != cudaSuccess) return e;
    goib2d_delta_back_state_kernel<T, P, KP, MT, AHEAD>
        <<<dim3((unsigned)(f.d.n_worlds * f.d.heads), b.blocks), 32 * (b.warps + (AHEAD ? 2 : 0)), smem, s>>>(f);
    return cudaGetLastError();
}

template <class T, class P, int KP, int C>
cudaError_t back_span(const Backward &f, cudaStream_t s) {
    using L = Span<P, KP, C>;
    const int64_t blocks = f.d.n_worlds * f.d.key_heads * ((f.d.n_steps + C - 1) / C);
    if (!blocks) return cudaSuccess;
    cudaError_t e = allow_smem(goib2d_delta_back_span_kernel<T, P, KP, C>, L::bytes(f.tiles_v));
    if (e != cudaSuccess) return e;
    goib2d_delta_back_span_kernel<T, P, KP, C><<<(unsigned)blocks, L::warps * 32, L::bytes(f.tiles_v), s>>>(f);
    return cudaGetLastError();
}

template <class T, class P, int KP>
cudaError_t back_wide(Backward &f, cudaStream_t s) {
    const Split b(f.d);
    f.parts = (f.tiles_v + b.MT - 1) / b.MT;
    if (b.ahead == 1) return back_state<T, P, KP, 1, 1>(f, b, s);
    if constexpr (KP < 128) {
        if (b.ahead == 0) return b.MT == 2 ? back_state<T, P, KP, 2, 0>(f, b, s) : back_state<T, P, KP, 1, 0>(f, b, s);
    }
    return back_state<T, P, KP, 1, 2>(f, b, s);
}

template <class T, class P, int KP>
cudaError_t backward_of(Backward &f, cudaStream_t s) {
    const cudaError_t e = back_wide<T, P, KP>(f, s);
    if (e != cudaSuccess) return e;
    if constexpr (sizeof(typename P::E) == 2 || KP <= 64)
        if (f.keep == 64) return back_span<T, P, KP, 64>(f, s);
    if constexpr (sizeof(typename P::E) == 4) return back_span<T, P, KP, 32>(f, s);
    return cudaErrorUnknown;
}

int64_t odd_bytes(const goib2d_delta_desc &d, int keep) {
    return (d.n_worlds * d.key_heads * ((d.n_steps + keep - 1) / keep) * 4 + 15) / 16 * 16;
}
int64_t db_bytes(const goib2d_delta_desc &d) {  // [n][h][16-column tiles of V][t], in whole 16 bytes
    return (d.n_worlds * d.heads * ((d.value_dim + 15) / 16) * d.n_steps * 4 + 15) / 16 * 16;
}

template <class T, class P>
cudaError_t backward_typed(const goib2d_delta_desc &d, const goib2d_delta_grads &gr, const void *saved, void *workspace,
                           cudaStream_t s) {
    Backward f{d, gr};
    const Saved at = delta_saved(d);
    f.r = saved, f.kept_s = (const char *)saved + at.r, f.kept_ds = workspace, f.keep = at.keep, f.tiles_v = at.tiles_v;
    const int V = d.value_dim, z = sizeof(T);
    f.dv = gr.dv;
    for (int i = 0; i < 3; ++i) f.dv_stride[i] = gr.dv_stride[i];
    f.db = (float *)((char *)workspace + at.states);
    f.odd = (int32_t *)((char *)f.db + db_bytes(d));
    if (sizeof(T) != sizeof(typename P::E)) {
        f.dv = (char *)f.odd + odd_bytes(d, at.keep);
        f.dv_stride[0] = d.n_steps * d.heads * V, f.dv_stride[1] = (int64_t)d.heads * V, f.dv_stride[2] = V;
    }
    f.grain_q = rows_grain(d.q, d.q_stride, d.n_worlds, d.n_steps, d.key_heads, d.key_dim, z);
    f.grain_k = rows_grain(d.k, d.k_stride, d.n_worlds, d.n_steps, d.key_heads, d.key_dim, z);
    f.grain_do = rows_grain(gr.dout, gr.dout_stride, d.n_worlds, d.n_steps, d.heads, V, z);
    f.grain_dv = rows_grain(f.dv, f.dv_stride, d.n_worlds, d.n_steps, d.heads, V, sizeof(typename P::E));
    f.wide_dv = f.grain_dv == 16;
    f.grain_r = dense_grain(V, sizeof(typename P::E));
    f.wide_dqk = (uintptr_t)gr.dq % (2 * z) == 0 && (uintptr_t)gr.dk % (2 * z) == 0;
    for (int i = 0; i < 3; ++i) f.wide_dqk = f.wide_dqk && gr.dq_stride[i] % 2 == 0 && gr.dk_stride[i] % 2 == 0;
    cudaError_t e;
    switch (padded_keys(d.key_dim)) {
        case 32: e = backward_of<T, P, 32>(f, s); break;
        case 64: e = backward_of<T, P, 64>(f, s); break;
        default: e = backward_of<T, P, 128>(f, s);
    }
    return e == cudaSuccess ? back_odd<T, typename P::E>(f, s) : e;
}

}  // namespace

int64_t delta_workspace_bytes(const goib2d_delta_desc &d) {
    const Saved s = delta_saved(d);
    return s.states + db_bytes(d) + odd_bytes(d, s.keep) + (d.dtype == GOIB2D_BFLOAT16 && s.size == 4 ? s.r : 0);
}

cudaError_t launch_delta_backward(const goib2d_delta_desc &d, const goib2d_delta_grads &gr, const void *saved,
                                  void *workspace, cudaStream_t s) {
    if (d.dtype == GOIB2D_FLOAT32) return backward_typed<float, Full>(d, gr, saved, workspace, s);
    return delta_full(d) ? backward_typed<bf16, Full>(d, gr, saved, workspace, s)
                         : backward_typed<bf16, Half>(d, gr, saved, workspace, s);
}

}  // namespace gb
