// Gradients of the gated delta rule (goib2d_delta_backward), in two kernels around the states that the forward pass kept.
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
    int32_t keep, tiles_v;
    bool wide_q, wide_k, wide_do, wide_dv, wide_r;
};

// ---- dS through the rollout, dv and db

template <class P, int KP, int MT>
struct Layout {
    static constexpr int pitch = KP + 8, E = sizeof(typename P::E);
    __host__ __device__ static int v_pitch(int warps) { return warps * 16 * MT + (E == 2 ? 8 : 4); }
    __host__ __device__ static int stage(int warps) { return kTile * (2 * pitch + 2 * v_pitch(warps)) * E; }
    __host__ __device__ static int bytes(int warps) {
        return 2 * stage(warps) + kTile / kChunk * (int)sizeof(Chunk<P>) + warps * kTile * 4;
    }
};

template <class T, class P, int KP, int MT>
__global__ void __launch_bounds__(MT == 2 ? 128 : 256) goib2d_delta_back_state_kernel(const __grid_constant__ Backward f) {
    using L = Layout<P, KP, MT>;
    using E = typename P::E;
    constexpr int KT = KP / 16;
    constexpr bool half = sizeof(E) == 2;
    extern __shared__ __align__(16) char sm[];
    const goib2d_delta_desc &d = f.d;
    const int K = d.key_dim, V = d.value_dim, threads = blockDim.x, warps = threads / 32;
    const int tid = threadIdx.x, w = tid / 32, lane = tid % 32, g = lane >> 2, t = lane & 3;
    const int64_t nh = blockIdx.x, n = nh / d.heads, steps = d.n_steps;
    const int h = (int)(nh - n * d.heads), hk = h / (d.heads / d.key_heads);
    const int stage = L::stage(warps), vp = L::v_pitch(warps), v0 = w * 16 * MT, cols = warps * 16 * MT;
    Chunk<P> *chunks = (Chunk<P> *)(sm + 2 * stage);
    float *db = (float *)(chunks + kTile / kChunk);  // [warp][token of the tile]

    float S[MT][KP / 8][4];  // dS^T: rows v, columns k
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int j = 0; j < KP / 8; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int v = v0 + 16 * m + g + (e >> 1) * 8, k = j * 8 + 2 * t + (e & 1);
                S[m][j][e] = f.gr.dstate_out && v < V && k < K ? f.gr.dstate_out[(nh * K + k) * V + v] : 0.0f;
            }
    const int64_t tiles = (steps + kTile - 1) / kTile;
    const T *q0 = row<T>(d.q, d.q_stride, n, 0, hk), *k0 = row<T>(d.k, d.k_stride, n, 0, hk);
    const T *o0 = f.gr.dout ? row<T>(f.gr.dout, f.gr.dout_stride, n, 0, h) : nullptr;
    const E *r0 = (const E *)f.r + nh * steps * V;
    auto load = [&](int64_t tile) {
        E *Q = (E *)(sm + (tile & 1) * stage), *Kb = Q + kTile * L::pitch, *Ob = Kb + kTile * L::pitch, *Rb = Ob + kTile * vp;
        const int64_t at = tile * kTile;
        const int left = (int)(steps - at < kTile ? steps - at : kTile);
        load_rows(Q, L::pitch, q0 + at * d.q_stride[1], d.q_stride[1], left, kTile, K, KP, f.wide_q, tid, threads);
        load_rows(Kb, L::pitch, k0 + at * d.k_stride[1], d.k_stride[1], left, kTile, K, KP, f.wide_k, tid, threads);
        load_rows(Ob, vp, o0 + at * f.gr.dout_stride[1], f.gr.dout_stride[1], o0 ? left : 0, kTile, V, cols, f.wide_do, tid,
                  threads);
        load_rows(Rb, vp, r0 + at * V, V, left, kTile, V, cols, f.wide_r, tid, threads);
        cp_commit();
    };
    Gate gate[kTile / kChunk];
    auto gates = [&](int64_t tile) {
#pragma unroll
        for (int s = 0; s < kTile / kChunk; ++s)
            if (s % warps == w) gate[s] = load_gate<T>(d, n, tile * kTile + s * kChunk + (lane & 15), h);
    };
    // db of the tile before, from the warps' parts
    auto finish = [&](int64_t tile) {
        const int64_t at = tile * kTile + tid;
        if (tid < kTile && at < steps) {
            float x = 0.0f;
            for (int i = 0; i < warps; ++i) x += db[i * kTile + tid];
            *row<T>(f.gr.dbeta, f.gr.dbeta_stride, n, at, h) = from_float<T>(x);
        }
    };
    if (tiles) load(tiles - 1), gates(tiles - 1);
    for (int64_t tile = tiles - 1; tile >= 0; --tile) {
        const E *Q = (const E *)(sm + (tile & 1) * stage), *Kb = Q + kTile * L::pitch, *Ob = Kb + kTile * L::pitch;
        E *Rb = (E *)(Ob + kTile * vp);
        cp_wait<0>();
        __syncthreads();
        if (tile + 1 < tiles) finish(tile + 1);
        if (tile > 0) load(tile - 1);
#pragma unroll
        for (int s = 0; s < kTile / kChunk; ++s)
            if (s % warps == w)
                prepare<P, KP, true>(chunks[s], Q + s * kChunk * L::pitch, Kb + s * kChunk * L::pitch, L::pitch, gate[s],
                                     d.scale, lane);
        if (tile > 0) gates(tile - 1);
        __syncthreads();
        if ((tile + 1) * kTile % f.keep == 0 || tile == tiles - 1) {
            const int64_t at = nh * ((steps + f.keep - 1) / f.keep) + tile * kTile / f.keep;
#pragma unroll
            for (int m = 0; m < MT; ++m)
                if (w * MT + m < f.tiles_v) keep_state<E, KT>(f.kept_ds, (at * f.tiles_v + w * MT + m) * KT, S[m], lane);
        }
#pragma unroll 1
        for (int s = kTile / kChunk - 1; s >= 0; --s) {
            const int64_t at = tile * kTile + s * kChunk;
            if (at >= steps) continue;
            const Chunk<P> &c = chunks[s];
            const E *Qs = Q + s * kChunk * L::pitch, *Ks = Kb + s * kChunk * L::pitch, *Os = Ob + s * kChunk * vp;
            E *Rs = Rb + s * kChunk * vp;
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
                const typename P::B2 z = c.z.k_rows(lane), p = c.p.k_rows(lane);
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
                if (g == 0) db[w * kTile + s * kChunk + (e >> 1) * 8 + 2 * t + (e & 1)] = sum[e];
            }
            T *to = row<T>(f.gr.dv, f.gr.dv_stride, n, at, h);
            if (half) {
                store_rows<MT>((bf16 *)to, f.gr.dv_stride[1], tokens, v0, V, f.wide_dv, (bf16 *)Rs, vp, X, lane);
            } else {
#pragma unroll
                for (int m = 0; m < MT; ++m) store_direct<T>(to, f.gr.dv_stride[1], tokens, v0 + 16 * m, V, X[m], lane);
                if (f.dv != f.gr.dv) {
                    E *also = row<E>(f.dv, f.dv_stride, n, at, h);
#pragma unroll
                    for (int m = 0; m < MT; ++m) store_direct<E>(also, f.dv_stride[1], tokens, v0 + 16 * m, V, X[m], lane);
                }
            }
#pragma unroll
            for (int m = 0; m < MT; ++m) {
                float x[2][4];
                P::values_t(x, Os, vp, 0, v0 + 16 * m, lane);
#pragma unroll
                for (int j = 0; j < 2; ++j)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const float a = c.a[j * 8 + 2 * t + (e & 1)];
                        x[j][e] *= d.scale * a;
                        X[m][j][e] *= -a;
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
        }
    }
    __syncthreads();
    if (tiles) finish(0);
    if (f.gr.dstate_in)
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
            for (int j = 0; j < KP / 8; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int v = v0 + 16 * m + g + (e >> 1) * 8, k = j * 8 + 2 * t + (e & 1);
                    if (v < V && k < K) f.gr.dstate_in[(nh * K + k) * V + v] = S[m][j][e];
                }
}

// ---- dq, dk and dg, span by span

template <class P, int KP, int C>
struct Span {
    static constexpr int RB = C / 16;                   // row blocks: warps that share the tokens
    static constexpr int KH = KP < 64 ? KP : 64;        // channels of dq and dk a warp holds
    static constexpr int warps = RB * (KP / KH);
    static constexpr int pitch = KP + 8;
    struct Tokens {
        float a[C], d[C], b[C], hi[C], lo[C];           // hi + lo: the running sum of g
        int since[C];
        float row[KP / KH][C], col[KP / KH][C], pairs[RB][C], end[warps];
        float a_end;
    };
    __host__ __device__ static int v_pitch(int tiles_v) { return tiles_v * 16 + 8; }
    __host__ __device__ static int bytes(int tiles_v) {
        return (int)sizeof(typename P::E) * (2 * C * pitch + 3 * C * v_pitch(tiles_v) + tiles_v * 16 * pitch) +
               (int)sizeof(Tokens);
    }
};

template <class T, class P, int KP, int C>
__global__ void __launch_bounds__(Span<P, KP, C>::warps * 32) goib2d_delta_back_span_kernel(const __grid_constant__ Backward f) {
    using L = Span<P, KP, C>;
    using E = typename P::E;
    constexpr int RB = L::RB, KH = L::KH, threads = L::warps * 32;
    extern __shared__ __align__(16) char sm[];
    const goib2d_delta_desc &d = f.d;
    const int K = d.key_dim, V = d.value_dim, tv = f.tiles_v, vp = L::v_pitch(tv), cols = tv * 16;
    const int tid = threadIdx.x, w = tid / 32, lane = tid % 32, g = lane >> 2, t = lane & 3;
    const int rb = w % RB, part = w / RB, k0 = part * KH;  // 16 tokens, and KH channels of keys
    const int64_t steps = d.n_steps, spans = (steps + C - 1) / C;
    const int64_t item = blockIdx.x / spans, span = blockIdx.x - item * spans, at = span * C, n = item / d.key_heads;
    const int hk = (int)(item - n * d.key_heads), group = d.heads / d.key_heads;
    const int left = (int)(steps - at < C ? steps - at : C);

    E *Q = (E *)sm, *Kb = Q + C * L::pitch, *Ob = Kb + C * L::pitch, *Vb = Ob + C * vp, *Rb = Vb + C * vp;
    E *St = Rb + C * vp;                                // S0^T, then dS1^T: rows v, columns k
    auto &x = *(typename L::Tokens *)(St + cols * L::pitch);

    load_rows(Q, L::pitch, row<T>(d.q, d.q_stride, n, at, hk), d.q_stride[1], left, C, K, KP, f.wide_q, tid, threads);
    load_rows(Kb, L::pitch, row<T>(d.k, d.k_stride, n, at, hk), d.k_stride[1], left, C, K, KP, f.wide_k, tid, threads);
    float dq[KH / 8][4] = {}, dk[KH / 8][4] = {};
    for (int j = 0; j < group; ++j) {
        const int h = hk * group + j;
        const int64_t nh = n * d.heads + h;
        __syncthreads();
        const bool o = f.gr.dout != nullptr;
        load_rows(Ob, vp, o ? row<T>(f.gr.dout, f.gr.dout_stride, n, at, h) : nullptr, f.gr.dout_stride[1], o ? left : 0, C, V,
                  cols, f.wide_do, tid, threads);
        load_rows(Vb, vp, row<E>((const void *)f.dv, f.dv_stride, n, at, h), f.dv_stride[1], left, C, V, cols, f.wide_dv, tid,
                  threads);
        load_rows(Rb, vp, (const E *)f.r + (nh * steps + at) * V, V, left, C, V, cols, f.wide_r, tid, threads);
        cp_commit();
        const int64_t kept = (nh * spans + span) * tv * (KP / 16) * 32;
        float end = 0.0f;
        for (int i = tid; i < tv * (KP / 16) * 32; i += threads) {
            float s[8], ds[8];
            kept_values<E>(s, f.kept_s, kept + i);
            kept_values<E>(ds, f.kept_ds, kept + i);
            put_state<E>(St, L::pitch, i / 32 / (KP / 16), i / 32 % (KP / 16), s, i % 32);
#pragma unroll
            for (int e = 0; e < 8; ++e) end += s[e] * ds[e];
        }
        for (int i = 16; i > 0; i >>= 1) end += __shfl_xor_sync(~0u, end, i);
        if (lane == 0) x.end[w] = end;
        if (w == 0) {
            // the tokens' gates: C / 32 neighbouring tokens a lane
            constexpr int PL = C / 32;
            Gate gt[PL];
            double G = 0.0;
            uint32_t fresh[PL];
#pragma unroll
            for (int e = 0; e < PL; ++e) {
                gt[e] = load_gate<T>(d, n, at + lane * PL + e, h);
                G += gt[e].fresh ? 0.0 : (double)gt[e].g;
                fresh[e] = __ballot_sync(~0u, gt[e].fresh);
            }
            const double mine = G;
#pragma unroll
            for (int i = 1; i < 32; i *= 2) {
                const double y = __shfl_up_sync(~0u, G, i);
                if (lane >= i) G += y;
            }
            const double last = __shfl_sync(~0u, G, 31);
            int all = 0, before = 0;
#pragma unroll
            for (int e = 0; e < PL; ++e) all += __popc(fresh[e]), before += __popc(fresh[e] & ((1u << lane) - 1));
            G -= mine;
#pragma unroll
            for (int e = 0; e < PL; ++e) {
                const int i = lane * PL + e;
                G = (e == 0 && lane == 0 ? 0.0 : G) + (gt[e].fresh ? 0.0 : (double)gt[e].g);
                before += gt[e].fresh;
                const float hi = (float)G;
                x.hi[i] = hi, x.lo[i] = (float)(G - (double)hi), x.b[i] = gt[e].b, x.since[i] = before;
                x.a[i] = before ? 0.0f : expf(hi);
                x.d[i] = before == all ? expf((float)(last - G)) : 0.0f;
            }
            if (lane == 0) x.a_end = all ? 0.0f : expf((float)last);
        }
        cp_wait<0>();
        __syncthreads();

        const int i0 = rb * 16 + g;  // the thread's rows: i0, i0 + 8
        // what the tokens read of S0
        float row_sum[2] = {};
#pragma unroll 1
        for (int which = 0; which < 2; ++which) {
            float acc[KH / 8][4] = {};
            const E *A = which ? Vb : Ob, *with = which ? Kb : Q;
#pragma unroll 1
            for (int v = 0; v < tv; ++v) {
                const typename P::A1 fa = P::a_rows(A, vp, rb * 16, v * 16, lane);
#pragma unroll
                for (int c = 0; c < KH / 16; ++c)
                    P::mul(acc[2 * c], acc[2 * c + 1], fa, P::k_rows(St, L::pitch, v * 16, k0 + c * 16, lane));
            }
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                const float a = x.a[i0 + 8 * r], scaled = which ? -a : d.scale * a;
                const E *p = with + (i0 + 8 * r) * L::pitch + k0 + 2 * t;
                float sum = 0.0f;
#pragma unroll
                for (int c = 0; c < KH / 8; ++c) {
                    float(&y)[4] = acc[c];
                    y[2 * r] = a == 0.0f ? 0.0f : scaled * y[2 * r];
                    y[2 * r + 1] = a == 0.0f ? 0.0f : scaled * y[2 * r + 1];
                    sum += to_float(p[8 * c]) * y[2 * r] + to_float(p[8 * c + 1]) * y[2 * r + 1];
                }
                row_sum[r] += sum;
            }
            if (which == 0) {
#pragma unroll
                for (int c = 0; c < KH / 8; ++c)
#pragma unroll
                    for (int e = 0; e < 4; ++e) dq[c][e] += acc[c][e];
            } else {
#pragma unroll
                for (int c = 0; c < KH / 8; ++c)
#pragma unroll
                    for (int e = 0; e < 4; ++e) dk[c][e] += acc[c][e];
            }
        }
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            row_sum[r] += __shfl_xor_sync(~0u, row_sum[r], 1);
            row_sum[r] += __shfl_xor_sync(~0u, row_sum[r], 2);
            if (t == 0) x.row[part][i0 + 8 * r] = row_sum[r];
        }
        const float hi_i[2] = {x.hi[i0], x.hi[i0 + 8]}, lo_i[2] = {x.lo[i0], x.lo[i0 + 8]};
        const int since_i[2] = {x.since[i0], x.since[i0 + 8]};
        // the warp's tokens as i, those before them as j
        float before[2] = {};  // sum over the columns so far
#pragma unroll 1
        for (int jb = 0; jb <= rb; ++jb) {
            float A[2][4] = {}, M[2][4] = {}, qk[2][4] = {}, kk[2][4] = {};
#pragma unroll 1
            for (int v = 0; v < tv; ++v) {
                const typename P::B1 fr = P::n_rows(Rb, vp, jb * 16, v * 16, lane);
                P::mul(A[0], A[1], P::a_rows(Ob, vp, rb * 16, v * 16, lane), fr);
                P::mul(M[0], M[1], P::a_rows(Vb, vp, rb * 16, v * 16, lane), fr);
            }
#pragma unroll
            for (int c = 0; c < KP / 16; ++c) {
                const typename P::B1 fj = P::n_rows(Kb, L::pitch, jb * 16, c * 16, lane);
                P::mul(qk[0], qk[1], P::a_rows(Q, L::pitch, rb * 16, c * 16, lane), fj);
                P::mul(kk[0], kk[1], P::a_rows(Kb, L::pitch, rb * 16, c * 16, lane), fj);
            }
            float pair[2][4];
#pragma unroll
            for (int nt = 0; nt < 2; ++nt)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int jj = jb * 16 + nt * 8 + 2 * t + (e & 1), r = e >> 1, i = i0 + 8 * r;
                    const bool seen = jj <= i && x.since[jj] == since_i[r];
                    const float D = seen ? expf((hi_i[r] - x.hi[jj]) + (lo_i[r] - x.lo[jj])) * x.b[jj] : 0.0f;
                    A[nt][e] = seen ? d.scale * D * A[nt][e] : 0.0f;
                    M[nt][e] = seen && jj < i ? -D * M[nt][e] : 0.0f;
                    pair[nt][e] = seen && jj < i ? A[nt][e] * qk[nt][e] + M[nt][e] * kk[nt][e] : 0.0f;
                }
            // pairs[l] = sum over rows i >= l of the sums over columns j < l
            float upto[2][2][2];  // [row][tile][column]
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                float base = before[r];
#pragma unroll
                for (int nt = 0; nt < 2; ++nt) {
                    const float p0 = pair[nt][2 * r], p1 = pair[nt][2 * r + 1];
                    float incl = p0 + p1;
                    float y = __shfl_up_sync(~0u, incl, 1, 4);
                    if (t >= 1) incl += y;
                    y = __shfl_up_sync(~0u, incl, 2, 4);
                    if (t >= 2) incl += y;
                    float excl = __shfl_up_sync(~0u, incl, 1, 4);
                    excl = t ? excl : 0.0f;
                    upto[r][nt][0] = base + excl, upto[r][nt][1] = base + excl + p0;
                    base += __shfl_sync(~0u, incl, 3, 4);
                }
                before[r] = base;
            }
#pragma unroll
            for (int nt = 0; nt < 2; ++nt)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const int l = jb * 16 + nt * 8 + 2 * t + e;
                    float y = (l <= i0 ? upto[0][nt][e] : 0.0f) + (l <= i0 + 8 ? upto[1][nt][e] : 0.0f);
                    for (int o = 4; o < 32; o *= 2) y += __shfl_xor_sync(~0u, y, o);
                    if (part == 0 && g == 0) x.pairs[rb][l] = y;
                }
            const typename P::A1 fa = P::rounded(A[0], A[1]), fm = P::rounded(M[0], M[1]);
#pragma unroll
            for (int c = 0; c < KH / 16; ++c) {
                const typename P::B1 fk = P::k_rows(Kb, L::pitch, jb * 16, k0 + c * 16, lane);
                P::mul(dq[2 * c], dq[2 * c + 1], fa, fk);
                P::mul(dk[2 * c], dk[2 * c + 1], fm, fk);
            }
        }
        // the warp's tokens as j, those after them as i
        const float b_j[2] = {x.b[i0], x.b[i0 + 8]};
#pragma unroll 1
        for (int ib = rb; ib < RB; ++ib) {
            float A[2][4] = {}, M[2][4] = {};
#pragma unroll 1
            for (int v = 0; v < tv; ++v) {
                const typename P::A1 fr = P::a_rows(Rb, vp, rb * 16, v * 16, lane);
                P::mul(A[0], A[1], fr, P::n_rows(Ob, vp, ib * 16, v * 16, lane));
                P::mul(M[0], M[1], fr, P::n_rows(Vb, vp, ib * 16, v * 16, lane));
            }
#pragma unroll
            for (int nt = 0; nt < 2; ++nt)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int i = ib * 16 + nt * 8 + 2 * t + (e & 1), r = e >> 1, jj = i0 + 8 * r;
                    const bool seen = jj <= i && x.since[i] == since_i[r];
                    const float D = seen ? expf((x.hi[i] - hi_i[r]) + (x.lo[i] - lo_i[r])) * b_j[r] : 0.0f;
                    A[nt][e] = seen ? d.scale * D * A[nt][e] : 0.0f;
                    M[nt][e] = seen && jj < i ? -D * M[nt][e] : 0.0f;
                }
            const typename P::A1 fa = P::rounded(A[0], A[1]), fm = P::rounded(M[0], M[1]);
#pragma unroll
            for (int c = 0; c < KH / 16; ++c) {
                P::mul(dk[2 * c], dk[2 * c + 1], fa, P::k_rows(Q, L::pitch, ib * 16, k0 + c * 16, lane));
                P::mul(dk[2 * c], dk[2 * c + 1], fm, P::k_rows(Kb, L::pitch, ib * 16, k0 + c * 16, lane));
            }
        }
        // what the tokens leave in the last state
        __syncthreads();
        for (int i = tid; i < tv * (KP / 16) * 32; i += threads) {
            float ds[8];
            kept_values<E>(ds, f.kept_ds, kept + i);
            put_state<E>(St, L::pitch, i / 32 / (KP / 16), i / 32 % (KP / 16), ds, i % 32);
        }
        __syncthreads();
        {
            float acc[KH / 8][4] = {};
#pragma unroll 1
            for (int v = 0; v < tv; ++v) {
                const typename P::A1 fa = P::a_rows(Rb, vp, rb * 16, v * 16, lane);
#pragma unroll
                for (int c = 0; c < KH / 16; ++c)
                    P::mul(acc[2 * c], acc[2 * c + 1], fa, P::k_rows(St, L::pitch, v * 16, k0 + c * 16, lane));
            }
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                const float dd = x.d[i0 + 8 * r], scaled = dd * b_j[r];
                const E *p = Kb + (i0 + 8 * r) * L::pitch + k0 + 2 * t;
                float sum = 0.0f;
#pragma unroll
                for (int c = 0; c < KH / 8; ++c) {
                    const float y0 = dd == 0.0f ? 0.0f : scaled * acc[c][2 * r], y1 = dd == 0.0f ? 0.0f : scaled * acc[c][2 * r + 1];
                    sum += to_float(p[8 * c]) * y0 + to_float(p[8 * c + 1]) * y1;
                    dk[c][2 * r] += y0, dk[c][2 * r + 1] += y1;
                }
                sum += __shfl_xor_sync(~0u, sum, 1);
                sum += __shfl_xor_sync(~0u, sum, 2);
                if (t == 0) x.col[part][i0 + 8 * r] = sum;
            }
        }
        __syncthreads();
        if (w == 0) {
            constexpr int PL = C / 32;
            float rows[PL], before_l[PL], row_all = 0.0f, col_all = 0.0f;
#pragma unroll
            for (int e = 0; e < PL; ++e) {
                const int l = lane * PL + e;
                before_l[e] = col_all;
                float rs = 0.0f, cs = 0.0f;
                for (int i = 0; i < KP / KH; ++i) rs += x.row[i][l], cs += x.col[i][l];
                rows[e] = rs, row_all += rs, col_all += cs;
            }
            float after = row_all, ahead = col_all;  // of this lane on; up to this lane
#pragma unroll
            for (int i = 1; i < 32; i *= 2) {
                const float y = __shfl_down_sync(~0u, after, i), z = __shfl_up_sync(~0u, ahead, i);
                if (lane + i < 32) after += y;
                if (lane >= i) ahead += z;
            }
            after = __shfl_down_sync(~0u, after, 1);  // of the lanes behind
            if (lane == 31) after = 0.0f;
            ahead = __shfl_up_sync(~0u, ahead, 1);
            if (lane == 0) ahead = 0.0f;
            float through = 0.0f;
            for (int i = 0; i < L::warps; ++i) through += x.end[i];
            through = x.a_end == 0.0f ? 0.0f : x.a_end * through;
            float suffix = after;
#pragma unroll
            for (int e = PL - 1; e >= 0; --e) {
                const int l = lane * PL + e;
                suffix += rows[e];
                float y = through + suffix + (ahead + before_l[e]);
                for (int i = l / 16; i < RB; ++i) y += x.pairs[i][l];
                const bool is_fresh = x.since[l] != (l ? x.since[l - 1] : 0);
                if (l < left) *row<T>(f.gr.dg, f.gr.dg_stride, n, at + l, h) = from_float<T>(is_fresh ? 0.0f : y);
            }
        }
    }
#pragma unroll
    for (int c = 0; c < KH / 8; ++c)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int i = rb * 16 + g + (e >> 1) * 8, k = k0 + c * 8 + 2 * t + (e & 1);
            if (i >= left || k >= K) continue;
            row<T>(f.gr.dq, f.gr.dq_stride, n, at + i, hk)[k] = from_float<T>(dq[c][e]);
            row<T>(f.gr.dk, f.gr.dk_stride, n, at + i, hk)[k] = from_float<T>(dk[c][e]);
        }
}

template <class T, class P, int KP, int MT>
cudaError_t back_state(const Backward &f, cudaStream_t s) {
    const int warps = (f.d.value_dim + 16 * MT - 1) / (16 * MT);
    const size_t smem = Layout<P, KP, MT>::bytes(warps);
    cudaError_t e = allow_smem(goib2d_delta_back_state_kernel<T, P, KP, MT>, smem);
    if (e != cudaSuccess) return e;
    goib2d_delta_back_state_kernel<T, P, KP, MT><<<(unsigned)(f.d.n_worlds * f.d.heads), 32 * warps, smem, s>>>(f);
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
cudaError_t backward_of(const Backward &f, cudaStream_t s) {
    const cudaError_t e = f.d.value_dim <= 16 ? back_state<T, P, KP, 1>(f, s) : back_state<T, P, KP, 2>(f, s);
    if (e != cudaSuccess) return e;
    if constexpr (sizeof(typename P::E) == 2 || KP <= 64)
        if (f.keep == 64) return back_span<T, P, KP, 64>(f, s);
    if constexpr (sizeof(typename P::E) == 4) return back_span<T, P, KP, 32>(f, s);
    return cudaErrorUnknown;
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
    if (sizeof(T) != sizeof(typename P::E)) {
        f.dv = (char *)workspace + at.states;
        f.dv_stride[0] = d.n_steps * d.heads * V, f.dv_stride[1] = (int64_t)d.heads * V, f.dv_stride[2] = V;
    }
    f.wide_q = rows_aligned(d.q, d.q_stride, d.n_worlds, d.n_steps, d.key_heads, d.key_dim, z);
    f.wide_k = rows_aligned(d.k, d.k_stride, d.n_worlds, d.n_steps, d.key_heads, d.key_dim, z);
    f.wide_do = rows_aligned(gr.dout, gr.dout_stride, d.n_worlds, d.n_steps, d.heads, V, z);
    f.wide_dv = rows_aligned(f.dv, f.dv_stride, d.n_worlds, d.n_steps, d.heads, V, sizeof(typename P::E));
    f.wide_r = V % 8 == 0;
    switch (padded_keys(d.key_dim)) {
        case 16: return backward_of<T, P, 16>(f, s);
        case 32: return backward_of<T, P, 32>(f, s);
        case 64: return backward_of<T, P, 64>(f, s);
        default: return backward_of<T, P, 128>(f, s);
    }
}

}  // namespace

int64_t delta_workspace_bytes(const goib2d_delta_desc &d) {
    const Saved s = delta_saved(d);
    return s.states + (d.dtype == GOIB2D_BFLOAT16 && s.size == 4 ? s.r : 0);
}

cudaError_t launch_delta_backward(const goib2d_delta_desc &d, const goib2d_delta_grads &gr, const void *saved,
                                  void *workspace, cudaStream_t s) {
    if (d.dtype == GOIB2D_FLOAT32) return backward_typed<float, Full>(d, gr, saved, workspace, s);
    return delta_full(d) ? backward_typed<bf16, Full>(d, gr, saved, workspace, s)
                         : backward_typed<bf16, Half>(d, gr, saved, workspace, s);
}

}  // namespace gb
