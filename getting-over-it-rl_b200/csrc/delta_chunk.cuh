// Chunks of 16 tokens of the gated delta rule as small matrix products (delta_forward.cu, delta_backward.cu).
//
// With G the running sum of g in the chunk, a_i = exp(G_i) and D_ij = exp(G_i - G_j) (both 0 across a token that
// starts afresh), W_ij = D_ij k_i.k_j for j < i and P_ij = scale D_ij q_i.k_j for j <= i, the tokens of the chunk obey
//     (I + W diag(b)) r = V - a (K S0),   u = b r,   O = scale a (Q S0) + P u,   S1 = a_16 S0 + K^T (d u),
// d_j = exp(G_16 - G_j). Chunks of 16 because that is one tile of the matrix instructions in both directions: the
// work inside a chunk grows with its length, that on the state does not shrink below it, and the triangular system is
// solved in registers. The inverse Z of its matrix is formed by forward substitution in float32: a product of
// powers of W would cancel catastrophically where the keys of neighbouring tokens are alike.
//
// The products' precision (mma.cuh): Half for bfloat16 inputs, Full for float32 ones. Gradients of a few tokens in
// bfloat16 take Full too (delta_full).
#pragma once
#include "delta.cuh"
#include "mma.cuh"

namespace gb {

constexpr int kChunk = 16;

// The passes over rollouts come in two shapes. With blocks for every SM, all warps of a block load a tile of chunks,
// prepare one each and solve them in turn: nothing waits idle, as others have the SM meanwhile. Where all blocks run at
// once a chunk's latency is the rollout's: then two warps more run ahead of the others and prepare every second chunk
// each (AHEAD), and the columns are spread over more warps. Split (delta.cuh) chooses, with both measured.
template <class P>
constexpr int kTile = sizeof(typename P::E) == 2 ? 32 : 16;  // tokens of a tile, so that six blocks of 64 channels fit

// One warp that prepares and the ones that solve, by the hardware's named barriers: `threads` counts both.
__device__ __forceinline__ void bar_wait(int id, int threads) { asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(threads) : "memory"); }
__device__ __forceinline__ void bar_arrive(int id, int threads) { asm volatile("bar.arrive %0, %1;" ::"r"(id), "r"(threads) : "memory"); }
// 2^x within 2^-22 of it, one instruction in place of expf's dozen for every pair of tokens: of the size of the products'
// own errors. 0 below 2^-126: a decay that small leaves nothing of a state in float32, but does not count as a fresh start.
__device__ __forceinline__ float exp2_fast(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// A 16 x 16 matrix that a chunk's products use: two bfloat16 each, or float32.
template <class P>
struct Square;
template <>
struct Square<Half> {
    bf16 hi[kChunk][24], lo[kChunk][24];
    __device__ __forceinline__ void put(int r, int c, float x, float y) {  // (r, c) and (r, c + 1), c even
        uint32_t h, l;
        split(x, y, h, l);
        *(uint32_t *)&hi[r][c] = h, *(uint32_t *)&lo[r][c] = l;
    }
    __device__ __forceinline__ void put(int r, int c, const float (&x)[8]) {  // (r, c) to (r, c + 7), c 0 or 8
        uint4 h, l;
        split(x[0], x[1], h.x, l.x), split(x[2], x[3], h.y, l.y), split(x[4], x[5], h.z, l.z), split(x[6], x[7], h.w, l.w);
        *(uint4 *)&hi[r][c] = h, *(uint4 *)&lo[r][c] = l;
    }
    __device__ __forceinline__ Half::B2 n_rows(int lane) const {
        Half::B2 b;
        ldsm(b.hi, at_b(&hi[0][0], 24, 0, 0, lane)), ldsm(b.lo, at_b(&lo[0][0], 24, 0, 0, lane));
        return b;
    }
    __device__ __forceinline__ Half::B2 k_rows(int lane) const {
        Half::B2 b;
        ldsm_t(b.hi, at_a(&hi[0][0], 24, 0, 0, lane)), ldsm_t(b.lo, at_a(&lo[0][0], 24, 0, 0, lane));
        return b;
    }
};
template <>
struct Square<Full> {
    float x[kChunk][24];
    __device__ __forceinline__ void put(int r, int c, float u, float v) { *(float2 *)&x[r][c] = make_float2(u, v); }
    __device__ __forceinline__ void put(int r, int c, const float (&y)[8]) {
        *(float4 *)&x[r][c] = make_float4(y[0], y[1], y[2], y[3]);
        *(float4 *)&x[r][c + 4] = make_float4(y[4], y[5], y[6], y[7]);
    }
    __device__ __forceinline__ Full::B1 n_rows(int lane) const { return Full::n_rows(&x[0][0], 24, 0, 0, lane); }
    __device__ __forceinline__ Full::B1 k_rows(int lane) const { return Full::k_rows(&x[0][0], 24, 0, 0, lane); }
};

// What one chunk needs besides its rows: Z (or T) transposed, P, and the tokens' factors.
template <class P>
struct alignas(16) Chunk {
    union {
        Square<P> z;
        float wt[kChunk][20];   // before Z is there: the strictly lower matrix, transposed
    };
    Square<P> p;
    float4 gate[kChunk];        // hi, lo (hi + lo: G / ln 2), b, and the tokens up to this one that start afresh
    float a[kChunk], sa[kChunk], d[kChunk], b[kChunk], bd[kChunk];  // sa = scale a, bd = b d
    float a_end;
    int odd;                    // whether a write strength is not finite
};

// A token's gates, held by lanes i and i + 16 of the warp that prepares the chunk.
struct Gate {
    float g, b;
    bool fresh;
};

// The same as loaded: nothing is done with the values until they are asked for, so that a load for the next chunk is
// not waited for.
template <class T>
struct RawGate {
    T g, b;
    uint8_t reset;
    bool live;
    __device__ __forceinline__ Gate get() const {
        if (!live) return {0.0f, 0.0f, false};
        const float x = to_float(g);
        return {x, to_float(b), reset || expf(x) == 0.0f};
    }
};

// The gates of one (world, head).
template <class T>
struct Gates {
    const T *g, *b;
    const uint8_t *reset;
    int gs, bs, rs, steps;
    __device__ __forceinline__ Gates(const goib2d_delta_desc &d, int64_t n, int h)
        : g(row<T>(d.g, d.g_stride, n, 0, h)), b(row<T>(d.beta, d.beta_stride, n, 0, h)),
          reset(d.reset ? d.reset + n * d.reset_stride[0] : nullptr), gs((int)d.g_stride[1]), bs((int)d.beta_stride[1]),
          rs((int)d.reset_stride[1]), steps((int)d.n_steps) {}
    __device__ __forceinline__ RawGate<T> at(int64_t t) const {
        RawGate<T> r;
        r.live = t >= 0 && t < steps;
        r.reset = 0, r.g = r.b = T(0.0f);
        if (r.live) {
            r.g = g[t * gs], r.b = b[t * bs];
            if (reset) r.reset = reset[t * rs];
        }
        return r;
    }
};

// The running sums of 16 tokens' g / ln 2, in float64: differences of sums over a chunk of strong decays keep
// float32's precision. Lanes i and i + 16 hold token i.
__device__ __forceinline__ double running_sum(const Gate &gate, int lane) {
    double G = gate.fresh ? 0.0 : (double)gate.g * 1.4426950408889634;
#pragma unroll
    for (int o = 1; o < 16; o *= 2) {
        const double y = __shfl_up_sync(~0u, G, o, 16);
        if ((lane & 15) >= o) G += y;
    }
    return G;
}

// A warp prepares one chunk from its 16 rows of Q and K. Forwards Z = (I + W diag(b))^-1 and P diag(b); BACK: T =
// (I + diag(b) W)^-1 and P.
template <class P, int KP, bool BACK>
__device__ __forceinline__ void prepare(Chunk<P> &c, const typename P::E *Q, const typename P::E *K, int pitch, Gate gate,
                                        float scale, int lane) {
    const int i = lane & 15, g = lane >> 2, t = lane & 3;
    const double G = running_sum(gate, lane), end = __shfl_sync(~0u, G, 15);
    const uint32_t fresh = __ballot_sync(~0u, gate.fresh) & 0xffffu;
    const int since = __popc(fresh & ((2u << i) - 1)), all = __popc(fresh);
    const int odd = __any_sync(~0u, 0.0f * gate.b != 0.0f);
    if (lane < 16) {
        const float hi = (float)G, a = since ? 0.0f : exp2_fast(hi), d = since == all ? exp2_fast((float)(end - G)) : 0.0f;
        c.a[i] = a, c.sa[i] = scale * a, c.d[i] = d, c.b[i] = gate.b, c.bd[i] = gate.b * d;
        c.gate[i] = make_float4(hi, (float)(G - (double)hi), gate.b, (float)since);
        if (lane == 0) c.a_end = all ? 0.0f : exp2_fast((float)end), c.odd = odd;
    }
    float kk[2][4] = {}, qk[2][4] = {};
#pragma unroll
    for (int x = 0; x < KP; x += 16) {
        const auto kb = P::n_rows(K, pitch, 0, x, lane);
        P::mul(kk[0], kk[1], P::a_rows(K, pitch, 0, x, lane), kb);
        P::mul(qk[0], qk[1], P::a_rows(Q, pitch, 0, x, lane), kb);
    }
    __syncwarp();
    const float4 rows[2] = {c.gate[g], c.gate[g + 8]};
#pragma unroll
    for (int n = 0; n < 2; ++n) {
        const float4 cols[2] = {c.gate[n * 8 + 2 * t], c.gate[n * 8 + 2 * t + 1]};
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            const int row = g + 8 * r;
            float p[2];
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const int col = n * 8 + 2 * t + e;
                const bool seen = col <= row && cols[e].w == rows[r].w;
                const float D = exp2_fast((rows[r].x - cols[e].x) + (rows[r].y - cols[e].y));
                const float w = D * kk[n][2 * r + e] * (BACK ? rows[r].z : cols[e].z);
                c.wt[col][row] = seen && col < row ? w : 0.0f;
                const float x = scale * D * qk[n][2 * r + e];
                p[e] = seen ? (BACK ? x : x * cols[e].z) : 0.0f;
            }
            c.p.put(row, n * 8 + 2 * t, p[0], p[1]);
        }
    }
    __syncwarp();
    // column i of the inverse, right-looking
    float z[kChunk];
#pragma unroll
    for (int r = 0; r < kChunk; ++r) z[r] = r == i ? 1.0f : 0.0f;
#pragma unroll
    for (int j = 0; j < kChunk - 1; ++j) {
        const float zj = j < i ? 0.0f : z[j];  // 0 above the diagonal, whatever W holds there
#pragma unroll
        for (int q4 = (j + 1) / 4 * 4; q4 < kChunk; q4 += 4) {
            const float4 w = *(const float4 *)&c.wt[j][q4];
            if (q4 > j) z[q4] -= w.x * zj;
            if (q4 + 1 > j) z[q4 + 1] -= w.y * zj;
            if (q4 + 2 > j) z[q4 + 2] -= w.z * zj;
            z[q4 + 3] -= w.w * zj;
        }
    }
    if (fresh)  // 0 times what is not finite before such a token
#pragma unroll
        for (int r = 0; r < kChunk; ++r)
            if (r < i || __popc(fresh & ((2u << r) - 1)) != since) z[r] = 0.0f;
    __syncwarp();
    float half[8];  // of the column, a half-warp each
#pragma unroll
    for (int r = 0; r < 8; ++r) half[r] = lane < 16 ? z[r] : z[8 + r];
    c.z.put(i, lane / 16 * 8, half);
}

// Rows of a strided tensor into shared memory, zeros past `rows` and `cols`: by asynchronous copies of `grain` bytes
// (rows_grain) where the types are the same, eight neighbouring threads to a row.
template <int BYTES, class E>
__device__ __forceinline__ void copy_rows(E *to, int pitch, const E *from, int64_t step, int r0, int dr, int rows, int count,
                                          int cols, int padded, int tid) {
    constexpr int N = BYTES / sizeof(E);
    for (int c = tid % 8 * N; c < padded; c += 8 * N) {
        const E *p = from + c;
        E *q = to + c;
        const int live = c < cols ? rows : 0;
        for (int r = r0; r < count; r += dr, p += step, q += dr * pitch) {
            if (r < live) {
                cp_async<BYTES>(q, p);
            } else {
#pragma unroll
                for (int e = 0; e < BYTES / 4; ++e) ((uint32_t *)q)[e] = 0;
            }
        }
    }
}
template <class E, class T>
__device__ __noinline__ void load_rows_odd(E *to, int pitch, const T *from, int stride, int rows, int count, int cols,
                                          int padded, int grain, int tid, int threads) {
    const int r0 = tid / 8, dr = threads / 8;
    const int64_t step = (int64_t)dr * stride;
    from += (int64_t)r0 * stride, to += r0 * pitch;
    if constexpr (sizeof(T) == sizeof(E)) {
        if (grain == 8) return copy_rows<8>(to, pitch, from, step, r0, dr, rows, count, cols, padded, tid);
        if (sizeof(T) == 4 || grain == 4) return copy_rows<4>(to, pitch, from, step, r0, dr, rows, count, cols, padded, tid);
    }
    constexpr int U = 4;  // rows whose loads are in flight together
    for (int c = tid % 8 * 2; c < padded; c += 16) {
        const T *p = from + c;
        E *q = to + c;
        for (int r = r0; r < count; r += U * dr, p += U * step, q += U * dr * pitch) {
            T u[U], v[U];
#pragma unroll
            for (int e = 0; e < U; ++e) {
                u[e] = r + e * dr < rows && c < cols ? p[e * step] : T(0.0f);
                v[e] = r + e * dr < rows && c + 1 < cols ? p[e * step + 1] : T(0.0f);
            }
#pragma unroll
            for (int e = 0; e < U; ++e) {
                if (r + e * dr >= count) break;
                if constexpr (sizeof(E) == 2) *(uint32_t *)(q + e * dr * pitch) = pack(to_float(u[e]), to_float(v[e]));
                else *(float2 *)(q + e * dr * pitch) = make_float2(to_float(u[e]), to_float(v[e]));
            }
        }
    }
}
template <class E, class T>
__device__ __forceinline__ void load_rows(E *to, int pitch, const T *from, int stride, int rows, int count, int cols,
                                          int padded, int grain, int tid, int threads) {
    if constexpr (sizeof(T) == sizeof(E)) {
        if (grain == 16) {
            const int r0 = tid / 8, dr = threads / 8;
            return copy_rows<16>(to + r0 * pitch, pitch, from + (int64_t)r0 * stride, (int64_t)dr * stride, r0, dr, rows, count,
                                 cols, padded, tid);
        }
    }
    load_rows_odd(to, pitch, from, stride, rows, count, cols, padded, grain, tid, threads);
}
// The same for 16 rows by one warp.
template <class E, class T>
__device__ __forceinline__ void chunk_rows(E *to, int pitch, const T *from, int stride, int rows, int cols, int padded,
                                           int grain, int lane) {
    if constexpr (sizeof(T) == sizeof(E)) {
        if (grain == 16) {
            constexpr int N = 16 / sizeof(E);
            for (int c = lane % 8 * N; c < padded; c += 8 * N) {
                const T *p = from + (int64_t)(lane / 8) * stride + c;
                E *q = to + lane / 8 * pitch + c;
                const int left = c < cols ? rows - lane / 8 : 0;
#pragma unroll
                for (int r = 0; r < kChunk; r += 4, p += (int64_t)4 * stride, q += 4 * pitch) {
                    if (r < left) cp_async<16>(q, p);
                    else *(uint4 *)q = make_uint4(0, 0, 0, 0);
                }
            }
            return;
        }
    }
    load_rows_odd(to, pitch, from, stride, rows, kChunk, cols, padded, grain, lane, 32);
}

// A warp's MT * 16 columns of a state [K][V] as accumulators of S^T (rows v, columns k), and back.
template <int MT, int KP>
__device__ __forceinline__ void load_state(float (&S)[MT][KP / 8][4], const float *from, int K, int V, int v0, int lane) {
    const int k0 = (lane & 3) * 2, v1 = v0 + (lane >> 2);
    if (from && K == KP && v0 + 16 * MT <= V) {
        const float *p = from + k0 * V + v1, *q = p + V;
#pragma unroll
        for (int j = 0; j < KP / 8; ++j, p += 8 * V, q += 8 * V)
#pragma unroll
            for (int m = 0; m < MT; ++m) {
                S[m][j][0] = p[16 * m], S[m][j][1] = q[16 * m];
                S[m][j][2] = p[16 * m + 8], S[m][j][3] = q[16 * m + 8];
            }
        return;
    }
#pragma unroll
    for (int j = 0; j < KP / 8; ++j)
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int k = 8 * j + k0 + (e & 1), v = v1 + 16 * m + (e >> 1) * 8;
                S[m][j][e] = from && k < K && v < V ? from[k * V + v] : 0.0f;
            }
}
template <int MT, int KP>
__device__ __forceinline__ void store_state(float *to, const float (&S)[MT][KP / 8][4], int K, int V, int v0, int lane) {
    const int k0 = (lane & 3) * 2, v1 = v0 + (lane >> 2);
    if (K == KP && v0 + 16 * MT <= V) {
        float *p = to + k0 * V + v1, *q = p + V;
#pragma unroll
        for (int j = 0; j < KP / 8; ++j, p += 8 * V, q += 8 * V)
#pragma unroll
            for (int m = 0; m < MT; ++m) {
                p[16 * m] = S[m][j][0], q[16 * m] = S[m][j][1];
                p[16 * m + 8] = S[m][j][2], q[16 * m + 8] = S[m][j][3];
            }
        return;
    }
#pragma unroll
    for (int j = 0; j < KP / 8; ++j)
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int k = 8 * j + k0 + (e & 1), v = v1 + 16 * m + (e >> 1) * 8;
                if (k < K && v < V) to[k * V + v] = S[m][j][e];
            }
}

// 16 x 16 values (rows v, columns tokens) of one accumulator pair, to the rows of a strided tensor; tokens: a bit each
template <class T>
__device__ __forceinline__ void store_direct(T *to, int stride, uint32_t tokens, int v0, int V, const float (&c)[2][4],
                                             int lane) {
    const int g = lane >> 2, t = lane & 3;
#pragma unroll
    for (int n = 0; n < 2; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int token = n * 8 + 2 * t + (e & 1), v = v0 + g + (e >> 1) * 8;
            if (tokens >> token & 1 && v < V) to[(int64_t)token * stride + v] = from_float<T>(c[n][e]);
        }
}

// The same for MT tiles by way of the warp's own columns of a [token][v] buffer, for rows of 16-byte pieces.
template <int MT>
__device__ __forceinline__ void store_rows(bf16 *to, int stride, uint32_t tokens, int v0, int V, bool wide, bf16 *buf,
                                           int pitch, const float (&c)[MT][2][4], int lane) {
    __syncwarp();
#pragma unroll
    for (int m = 0; m < MT; ++m)
        stsm_t((void *)at_b(buf, pitch, 0, v0 + 16 * m, lane), Half::rounded(c[m][0], c[m][1]).x);
    __syncwarp();
#pragma unroll
    for (int m = 0; m < MT; ++m) {
        const int x = lane + 32 * m, token = x / (2 * MT), v = v0 + x % (2 * MT) * 8;
        if (!(tokens >> token & 1) || v >= V) continue;
        const bf16 *p = buf + token * pitch + v;
        bf16 *q = to + (int64_t)token * stride + v;
        if (wide) *(uint4 *)q = *(const uint4 *)p;
        else
            for (int e = 0; e < 8 && v + e < V; ++e) q[e] = p[e];
    }
    __syncwarp();
}

// 16 rows of S^T to what is kept for the backward pass (Saved): rows v of KT * 16 channels.
template <int KT>
__device__ __forceinline__ void keep_state(bf16 *to, const float (&S)[2 * KT][4], int lane) {
    uint32_t *p = (uint32_t *)to + (lane >> 2) * KT * 8 + (lane & 3);
#pragma unroll
    for (int j = 0; j < 2 * KT; ++j) p[4 * j] = pack(S[j][0], S[j][1]), p[KT * 64 + 4 * j] = pack(S[j][2], S[j][3]);
}
template <int KT>
__device__ __forceinline__ void keep_state(float *to, const float (&S)[2 * KT][4], int lane) {
    float2 *p = (float2 *)to + (lane >> 2) * KT * 8 + (lane & 3);
#pragma unroll
    for (int j = 0; j < 2 * KT; ++j)
        p[4 * j] = make_float2(S[j][0], S[j][1]), p[KT * 64 + 4 * j] = make_float2(S[j][2], S[j][3]);
}

// Two neighbouring values.
__device__ __forceinline__ float2 pair_at(const bf16 *p) {
    const uint32_t x = *(const uint32_t *)p;
    return make_float2(low(x), high(x));
}
__device__ __forceinline__ float2 pair_at(const float *p) { return *(const float2 *)p; }

// The sum of the products of 16 bytes of values.
template <class E>
__device__ __forceinline__ float dot16(const uint4 &x, const uint4 &y) {
    const uint32_t u[4] = {x.x, x.y, x.z, x.w}, v[4] = {y.x, y.y, y.z, y.w};
    float s = 0.0f;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        if constexpr (sizeof(E) == 2) s += low(u[e]) * low(v[e]) + high(u[e]) * high(v[e]);
        else s += __uint_as_float(u[e]) * __uint_as_float(v[e]);
    }
    return s;
}

}  // namespace gb
