// Causal attention under a visibility rule: a sliding window, a few first positions that stay visible (sinks), a learned bias by distance
// bucket.  Forward, backward with the bias table's gradient, and the form for one new position per sequence over a cache.  The reference
// has the causal form alone (frontend/tensor_other.hpp:53-93).
//
// This file holds the entry points, the fp32 FMA kernels, which take any strides and heads of up to 128 columns, and the kernel for single
// positions.
#include <algorithm>
#include <type_traits>
#include <utility>

#include "attention_fma.cuh"
#include "attention_tc.cuh"
#include "attention_window.cuh"

namespace gcb {

// ---- fp32 FMA kernels ----------------------------------------------------------------------------------------------------------
// A CTA owns 16 R queries (forward, dQ) or keys (dK, dV) of a head, R 2 or 4, and walks over tiles of 64 of the other side, skipping those that the
// rule hides as a whole.  The bias of a tile is looked up once per distance and read from shared memory
// (from the buckets themselves: a table by distance first would be a launch).
__host__ __device__ constexpr int aw_diag(int R) { return 16 * R + AS_T - 1; }

// ROWS rows of D columns from row r0 into [row][Dp + 4], zero beyond T and D.  VEC: rows start on 16 bytes and D is a multiple of four.
template <int ROWS, bool VEC>
__device__ __forceinline__ void aw_load(float* sm, const float* p, int64_t ld, int r0, int T, int D, int Dp) {
    if (VEC) { as_load<ROWS>(sm, p, ld, r0, T, D); return; }
    for (int i = threadIdx.x; i < ROWS * Dp; i += 256) {
        const int r = i / Dp, c = i - r * Dp;
        sm[r * (Dp + 4) + c] = r0 + r < T && c < D ? p[(r0 + r) * ld + c] : 0.0f;
    }
}
template <bool VEC>
__device__ __forceinline__ float4 aw_ld4(const float* p, int c, int D) {
    if (VEC) return c < D ? ld4(p + c) : make_float4(0.f, 0.f, 0.f, 0.f);
    return make_float4(c < D ? p[c] : 0.0f, c + 1 < D ? p[c + 1] : 0.0f, c + 2 < D ? p[c + 2] : 0.0f, c + 3 < D ? p[c + 3] : 0.0f);
}
template <bool VEC>
__device__ __forceinline__ void aw_st4(float* p, int c, int D, float4 x) {
    if (VEC) { if (c < D) st4(p + c, x); return; }
    if (c < D) p[c] = x.x;
    if (c + 1 < D) p[c + 1] = x.y;
    if (c + 2 < D) p[c + 2] = x.z;
    if (c + 3 < D) p[c + 3] = x.w;
}
// c[i][j] = a[ty + 16 i] . b[tx + 16 j], even and odd columns apart until the end
template <int R, int C>
__device__ __forceinline__ void aw_abt(float (&c)[R][C], const float* a, const float* b, int D, int ty, int tx) {
    const int P = D + 4;
    unsigned long long sum[R][C] = {};
#pragma unroll 4
    for (int d = 0; d < D; d += 4) {
        F4 x[R], y[C];
#pragma unroll
        for (int i = 0; i < R; ++i) x[i].f = ld4(a + (ty + 16 * i) * P + d);
#pragma unroll
        for (int j = 0; j < C; ++j) y[j].f = ld4(b + (tx + 16 * j) * P + d);
#pragma unroll
        for (int i = 0; i < R; ++i)
#pragma unroll
            for (int j = 0; j < C; ++j) sum[i][j] = fma2(x[i].d[1], y[j].d[1], fma2(x[i].d[0], y[j].d[0], sum[i][j]));
    }
#pragma unroll
    for (int i = 0; i < R; ++i)
#pragma unroll
        for (int j = 0; j < C; ++j) {
            float even, odd;
            asm("mov.b64 {%0, %1}, %2;" : "=f"(even), "=f"(odd) : "l"(sum[i][j]));
            c[i][j] = even + odd;
        }
}
// A head's row of the bias table and the buckets' first distances, kept by the CTA behind its other tables; ready after the next barrier.
template <int R>
__device__ __forceinline__ float* aw_lut(float* tab, const WindowAttn& p, int64_t h) {
    float* lut = tab + 2 * (aw_diag(R) + 1);
    const int t = threadIdx.x;
    if (t < p.rule.buckets) { lut[t] = p.rule.bias[h * p.rule.buckets + t]; lut[AW_MAX_BUCKETS + t] = __int_as_float(p.rule.starts[t]); }
    return lut;
}
// bias of a tile's distances, the first of which is d0
template <int R>
__device__ __forceinline__ void aw_tab(float* sm, const WindowAttn& p, const float* lut, int d0) {
    if (p.rule.bias == nullptr || threadIdx.x >= aw_diag(R)) return;
    const int d = max(0, d0 + (int)threadIdx.x);
    int n = 0;
#pragma unroll
    for (int step = AW_MAX_BUCKETS / 2; step > 0; step >>= 1)
        if (n + step < p.rule.buckets && __float_as_int(lut[AW_MAX_BUCKETS + n + step]) <= d) n += step;
    sm[threadIdx.x] = lut[n];
}
// the tile of keys after k0 that the queries from q0 on look at
__device__ __forceinline__ int aw_first_tile(const WindowRule& r, int q0) { return r.S > 0 ? 0 : r.window_first(q0) / AS_T * AS_T; }
__device__ __forceinline__ int aw_next_tile(const WindowRule& r, int q0, int k0) {
    const int k1 = k0 + AS_T, lo = r.window_first(q0) / AS_T * AS_T;
    return k1 >= r.S && k1 < lo ? lo : k1;
}
static size_t aw_floats(int R, int own, int other, int blocks, int64_t Dp) { return (size_t)(own * 16 * R + other * AS_T) * (Dp + 4) + (size_t)blocks * AS_T * (16 * R + 4) + 2 * (aw_diag(R) + 1) + 2 * AW_MAX_BUCKETS; }

template <int R, int NC, bool VEC>
__global__ void __launch_bounds__(256, 2) window_attention_fwd_kernel(const __grid_constant__ WindowAttn p) {
    constexpr int OWN = 16 * R;
    extern __shared__ __align__(16) float aw_sm[];
    pdl_trigger();
    pdl_wait();
    const int D = p.D, Dp = (D + 3) / 4 * 4, tx = threadIdx.x & 15, ty = threadIdx.x >> 4, head = blockIdx.x / p.tiles, q0 = (blockIdx.x - head * p.tiles) * OWN, last = min(q0 + OWN, p.T);
    const int64_t b = head / p.H, h = head - b * p.H;
    float *sq = aw_sm, *sk = sq + OWN * (Dp + 4), *sv = sk + AS_T * (Dp + 4), *sp = sv + AS_T * (Dp + 4), *tab = sp + AS_T * (OWN + 4);
    const float* lut = aw_lut<R>(tab, p, h);
    const float *k = p.k + b * p.k_so + h * p.k_si, *v = p.v + b * p.v_so + h * p.v_si;
    aw_load<OWN, VEC>(sq, p.q + b * p.q_so + h * p.q_si, p.q_ld, q0, p.T, D, Dp);
    float acc[R][4 * NC] = {}, m[R], sum[R] = {};
#pragma unroll
    for (int i = 0; i < R; ++i) m[i] = -INFINITY;
    for (int k0 = aw_first_tile(p.rule, q0); k0 < last; k0 = aw_next_tile(p.rule, q0, k0)) {
        __syncthreads();
        aw_load<AS_T, VEC>(sk, k, p.k_ld, k0, p.T, D, Dp);
        aw_load<AS_T, VEC>(sv, v, p.v_ld, k0, p.T, D, Dp);
        aw_tab<R>(tab, p, lut, q0 - k0 - (AS_T - 1));
        as_landed();
        float s[R][4];
        aw_abt(s, sq, sk, Dp, ty, tx);
#pragma unroll
        for (int i = 0; i < R; ++i) {
            const int row = q0 + ty + 16 * i;
            float mx = m[i];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float z = p.rule.bias ? fmaf(s[i][j], p.scale, tab[ty + 16 * i - (tx + 16 * j) + AS_T - 1]) : s[i][j] * p.scale;
                s[i][j] = p.rule.sees(row, k0 + tx + 16 * j) ? z : -INFINITY;
                mx = fmaxf(mx, s[i][j]);
            }
            mx = as_row(mx, true);
            const float rel = mx == -INFINITY ? 0.0f : mx, f = __expf(m[i] - rel);  // nothing seen yet: every term below is exp(-inf)
            m[i] = mx;
            float part = 0.0f;
#pragma unroll
            for (int j = 0; j < 4; ++j) { const float e = __expf(s[i][j] - rel); part += e; sp[(ty + 16 * i) * (AS_T + 4) + tx + 16 * j] = e; }
            sum[i] = sum[i] * f + as_row(part, false);
#pragma unroll
            for (int e = 0; e < 4 * NC; ++e) acc[i][e] *= f;
        }
        __syncthreads();
        as_ab<NC>(acc, sp, sv, Dp, ty, tx);
    }
    float* out = p.out + b * p.o_so + h * p.o_si;
#pragma unroll
    for (int i = 0; i < R; ++i) {
        const int row = q0 + ty + 16 * i;
        if (row >= p.T) continue;
        const bool empty = m[i] == -INFINITY;
        const float inv = empty ? 0.0f : 1.0f / sum[i];
#pragma unroll
        for (int n = 0; n < NC; ++n)
            aw_st4<VEC>(out + row * p.o_ld, 64 * n + 4 * tx, D, make_float4(acc[i][4 * n] * inv, acc[i][4 * n + 1] * inv, acc[i][4 * n + 2] * inv, acc[i][4 * n + 3] * inv));
        if (tx == 0) { p.row_max[head * p.Tp + row] = empty ? INFINITY : m[i]; p.row_inv[head * p.Tp + row] = inv; }
    }
}

// dO . O and the statistics of this thread's rows ty + 16 i of a query tile (dO in shared memory, O requested before it has landed)
template <int R, int NC, bool VEC>
struct AwRows {
    float delta[R], m[R], inv[R];
    float4 y[R][NC];
    __device__ __forceinline__ void request(const WindowAttn& p, int head, const float* o, int r0, int ty, int tx) {
#pragma unroll
        for (int i = 0; i < R; ++i) {
            const int row = r0 + ty + 16 * i;
            const bool live = row < p.T;
            m[i] = live ? p.row_max[head * p.Tp + row] : INFINITY;
            inv[i] = live ? p.row_inv[head * p.Tp + row] : 0.0f;
#pragma unroll
            for (int n = 0; n < NC; ++n) y[i][n] = live ? aw_ld4<VEC>(o + row * p.o_ld, 64 * n + 4 * tx, p.D) : make_float4(0.f, 0.f, 0.f, 0.f);
        }
    }
    __device__ __forceinline__ void finish(const float* sg, int Dp, int ty, int tx) {
#pragma unroll
        for (int i = 0; i < R; ++i) {
            float d = 0.0f;
#pragma unroll
            for (int n = 0; n < NC; ++n)
                if (64 * n + 4 * tx < Dp) {
                    const float4 x = ld4(sg + (ty + 16 * i) * (Dp + 4) + 64 * n + 4 * tx);
                    d = fmaf(x.x, y[i][n].x, fmaf(x.y, y[i][n].y, fmaf(x.z, y[i][n].z, fmaf(x.w, y[i][n].w, d))));
                }
            delta[i] = as_row(d, false);
        }
    }
};

// dQ of 16 R queries; with a bias table also its gradient over them: thread n < buckets keeps bucket n, dbias_part is [head][tile][buckets].
// Sums of a bucket go along the tile's diagonals, in a fixed order.
template <int R, int NC, bool VEC>
__device__ __forceinline__ void aw_dq(const WindowAttn& p, float* aw_sm, int item) {
    constexpr int OWN = 16 * R;
    const int D = p.D, Dp = (D + 3) / 4 * 4, tx = threadIdx.x & 15, ty = threadIdx.x >> 4, head = item / p.tiles, tile = item - head * p.tiles, q0 = tile * OWN;
    const int64_t b = head / p.H, h = head - b * p.H;
    float *s0 = aw_sm, *s1 = s0 + OWN * (Dp + 4), *s2 = s1 + OWN * (Dp + 4), *s3 = s2 + AS_T * (Dp + 4), *ss = s3 + AS_T * (Dp + 4), *tab = ss + AS_T * (OWN + 4), *diag = tab + aw_diag(R) + 1;
    const float* lut = aw_lut<R>(tab, p, h);
    const float *k = p.k + b * p.k_so + h * p.k_si, *v = p.v + b * p.v_so + h * p.v_si;
    float dq[R][4 * NC] = {}, db = 0.0f;
    AwRows<R, NC, VEC> rows;
    aw_load<OWN, VEC>(s0, p.q + b * p.q_so + h * p.q_si, p.q_ld, q0, p.T, D, Dp);
    aw_load<OWN, VEC>(s1, p.g + b * p.g_so + h * p.g_si, p.g_ld, q0, p.T, D, Dp);
    rows.request(p, head, p.o + b * p.o_so + h * p.o_si, q0, ty, tx);
    bool first = true;
    for (int k0 = aw_first_tile(p.rule, q0); k0 < min(q0 + OWN, p.T); k0 = aw_next_tile(p.rule, q0, k0)) {
        const int d0 = q0 - k0 - (AS_T - 1);
        __syncthreads();
        aw_load<AS_T, VEC>(s2, k, p.k_ld, k0, p.T, D, Dp);
        aw_load<AS_T, VEC>(s3, v, p.v_ld, k0, p.T, D, Dp);
        aw_tab<R>(tab, p, lut, d0);
        as_landed();
        if (first) {
            rows.finish(s1, Dp, ty, tx);
#pragma unroll
            for (int i = 0; i < R; ++i)
                if (tx == 0 && q0 + ty + 16 * i < p.T) p.delta[head * p.Tp + q0 + ty + 16 * i] = rows.delta[i];
        }
        first = false;
        float s[R][4], dp[R][4];
        aw_abt(s, s0, s2, Dp, ty, tx);
        aw_abt(dp, s1, s3, Dp, ty, tx);
#pragma unroll
        for (int i = 0; i < R; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int r = ty + 16 * i, c = tx + 16 * j;
                const float z = p.rule.bias ? fmaf(s[i][j], p.scale, tab[r - c + AS_T - 1]) : s[i][j] * p.scale;
                const float pr = p.rule.sees(q0 + r, k0 + c) ? __expf(z - rows.m[i]) * rows.inv[i] : 0.0f;
                ss[r * (AS_T + 4) + c] = pr * (dp[i][j] - rows.delta[i]);
            }
        __syncthreads();
        as_ab<NC>(dq, ss, s2, Dp, ty, tx);
        if (p.dbias_part) {
            const int t = threadIdx.x;
            if (t < aw_diag(R)) {
                float a = 0.0f;
                for (int r = max(0, t - (AS_T - 1)); r <= min(OWN - 1, t); ++r) a += ss[r * (AS_T + 4) + r - t + AS_T - 1];
                diag[t] = a;
            }
            __syncthreads();
            if (t < p.rule.buckets) {
                const int end = t + 1 < p.rule.buckets ? p.rule.starts[t + 1] - d0 : aw_diag(R);
                float a = 0.0f;
                for (int i = max(0, p.rule.starts[t] - d0); i < min(end, aw_diag(R)); ++i) a += diag[i];
                db += a;
            }
        }
    }
#pragma unroll
    for (int i = 0; i < R; ++i) {
        const int r = q0 + ty + 16 * i;
        if (r >= p.T) continue;
#pragma unroll
        for (int n = 0; n < NC; ++n)
            aw_st4<VEC>(p.dq + b * p.d_so + h * p.d_si + r * p.d_ld, 64 * n + 4 * tx, D,
                        make_float4(p.scale * dq[i][4 * n], p.scale * dq[i][4 * n + 1], p.scale * dq[i][4 * n + 2], p.scale * dq[i][4 * n + 3]));
    }
    if (p.dbias_part && threadIdx.x < p.rule.buckets) p.dbias_part[(int64_t)item * p.rule.buckets + threadIdx.x] = db;
}

// dK and dV of 16 R keys from the queries that see them through the window, and with far_inside from those beyond that still see the first keys.
template <int R, int NC, bool VEC>
__device__ __forceinline__ void aw_dkv(const WindowAttn& p, float* aw_sm, int item) {
    constexpr int OWN = 16 * R;
    const int D = p.D, Dp = (D + 3) / 4 * 4, tx = threadIdx.x & 15, ty = threadIdx.x >> 4, head = item / p.tiles, t0 = (item - head * p.tiles) * OWN;
    const int64_t b = head / p.H, h = head - b * p.H;
    float *s0 = aw_sm, *s1 = s0 + OWN * (Dp + 4), *s2 = s1 + OWN * (Dp + 4), *s3 = s2 + AS_T * (Dp + 4), *sp = s3 + AS_T * (Dp + 4), *ss = sp + AS_T * (OWN + 4), *tab = ss + AS_T * (OWN + 4);
    const float* lut = aw_lut<R>(tab, p, h);
    const float *q = p.q + b * p.q_so + h * p.q_si, *g = p.g + b * p.g_so + h * p.g_si, *o = p.o + b * p.o_so + h * p.o_si;
    float dk[R][4 * NC] = {}, dv[R][4 * NC] = {};
    aw_load<OWN, VEC>(s0, p.k + b * p.k_so + h * p.k_si, p.k_ld, t0, p.T, D, Dp);
    aw_load<OWN, VEC>(s1, p.v + b * p.v_so + h * p.v_si, p.v_ld, t0, p.T, D, Dp);
    const int W = p.rule.W, keys_end = min(t0 + OWN, p.T), always = p.far_inside ? p.rule.S : 0;
    const int r_end = t0 >= always && W > 0 && W < p.T - keys_end ? keys_end - 1 + W : p.T;
    for (int r0 = t0 / AS_T * AS_T; r0 < r_end; r0 += AS_T) {
        __syncthreads();
        AwRows<4, NC, VEC> rows;
        aw_load<AS_T, VEC>(s2, q, p.q_ld, r0, p.T, D, Dp);
        aw_load<AS_T, VEC>(s3, g, p.g_ld, r0, p.T, D, Dp);
        aw_tab<R>(tab, p, lut, r0 - t0 - (OWN - 1));
        rows.request(p, head, o, r0, ty, tx);
        as_landed();
        rows.finish(s3, Dp, ty, tx);
        float s[4][R], dp[4][R];
        aw_abt(s, s2, s0, Dp, ty, tx);
        aw_abt(dp, s3, s1, Dp, ty, tx);
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int j = 0; j < R; ++j) {
                const int r = ty + 16 * i, c = tx + 16 * j, d = r0 + r - (t0 + c);
                const float z = p.rule.bias ? fmaf(s[i][j], p.scale, tab[r - c + OWN - 1]) : s[i][j] * p.scale;
                const bool seen = d >= 0 && (W == 0 || d < W || t0 + c < always);
                const float pr = seen ? __expf(z - rows.m[i]) * rows.inv[i] : 0.0f;
                sp[r * (OWN + 4) + c] = pr;
                ss[r * (OWN + 4) + c] = pr * (dp[i][j] - rows.delta[i]);
            }
        __syncthreads();
        as_atb<NC>(dv, sp, s3, Dp, ty, tx);
        as_atb<NC>(dk, ss, s2, Dp, ty, tx);
    }
#pragma unroll
    for (int i = 0; i < R; ++i)
#pragma unroll
        for (int n = 0; n < NC; ++n) {
            const int c = 64 * n + 4 * tx, r = t0 + R * ty + i;
            const float4 a = make_float4(p.scale * dk[i][4 * n], p.scale * dk[i][4 * n + 1], p.scale * dk[i][4 * n + 2], p.scale * dk[i][4 * n + 3]);
            const float4 e = make_float4(dv[i][4 * n], dv[i][4 * n + 1], dv[i][4 * n + 2], dv[i][4 * n + 3]);
            if (r < p.T) {
                const int64_t at = b * p.d_so + h * p.d_si + r * p.d_ld;
                aw_st4<VEC>(p.dk + at, c, D, a);
                aw_st4<VEC>(p.dv + at, c, D, e);
            }
        }
}
// One launch for both sides: they share nothing that one would have to wait for, since each takes dO . O for itself.  The CTAs of dK and dV come first:
// theirs is the longer work.
template <int R, int NC, bool VEC>
__global__ void __launch_bounds__(256) window_attention_bwd_kernel(const __grid_constant__ WindowAttn p, int items) {
    extern __shared__ __align__(16) float aw_sm[];
    pdl_trigger();
    pdl_wait();
    if (blockIdx.x < items) aw_dkv<R, NC, VEC>(p, aw_sm, blockIdx.x);
    else aw_dq<R, NC, VEC>(p, aw_sm, blockIdx.x - items);
}
// What the queries beyond the window, which see the first S keys alone, add to those keys' gradients.  Tiles of keys would spend most of their work on
// keys that are not seen: here four keys lie in registers, a column quadruple a lane, and a warp passes over the rows of q and dO, 32 / LPR at a time.
// A CTA takes far_rows queries of a head and four of the keys, and leaves its sums in far_part, [head][chunk][S][dk, dv][Dp].
// Bound by memory (q and dO once for every four keys) and, about as much, by the eight sums over a row's lanes.
// 256 heads of 768 queries beyond a window: 54 us with four keys, 228 as tiles of 32 keys.  Its time grows with the number of keys: a backward pass of 16 x 16 x 1024 x 64, window 256, takes
// 490 us without first keys, 569 with four, 687 with sixteen and 1148 with 64; of 1 x 16 x 8192 x 64, window 1024, 559, 616, 685 and 948.
constexpr int AW_KEYS = 4;
template <int LPR>
__device__ __forceinline__ void sum_eight(float (&v)[8], int lane) {  // every lane gets all eight sums over its LPR lanes: halves change hands until each lane has one
    const bool b0 = lane & (LPR / 2), b1 = lane & (LPR / 4), b2 = lane & (LPR / 8);
    float w[4], x[2], y;
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = (b0 ? v[4 + i] : v[i]) + __shfl_xor_sync(0xffffffffu, b0 ? v[i] : v[4 + i], LPR / 2);
#pragma unroll
    for (int i = 0; i < 2; ++i) x[i] = (b1 ? w[2 + i] : w[i]) + __shfl_xor_sync(0xffffffffu, b1 ? w[i] : w[2 + i], LPR / 4);
    y = (b2 ? x[1] : x[0]) + __shfl_xor_sync(0xffffffffu, b2 ? x[0] : x[1], LPR / 8);
#pragma unroll
    for (int s = LPR / 16; s > 0; s >>= 1) y += __shfl_xor_sync(0xffffffffu, y, s);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = __shfl_sync(0xffffffffu, y, (lane & ~(LPR - 1)) | ((i & 4) ? LPR / 2 : 0) | ((i & 2) ? LPR / 4 : 0) | ((i & 1) ? LPR / 8 : 0));
}
template <int LPR, bool VEC>
__global__ void __launch_bounds__(256, 2) window_attention_far_kernel(const __grid_constant__ WindowAttn p) {
    constexpr int RPW = 32 / LPR, U = 2, DP = 4 * LPR, STEP = 8 * RPW;
    __shared__ __align__(16) float sums[8][2 * AW_KEYS][DP];
    pdl_trigger();
    pdl_wait();
    const int groups = (p.rule.S + AW_KEYS - 1) / AW_KEYS, per_head = groups * p.far_chunks, head = blockIdx.x / per_head, item = blockIdx.x - head * per_head, j0 = item / p.far_chunks * AW_KEYS, chunk = item % p.far_chunks;
    const int64_t b = head / p.H, h = head - b * p.H;
    const int D = p.D, W = p.rule.W, warp = threadIdx.x >> 5, lane = threadIdx.x & 31, col = 4 * (lane % LPR), r_end = min(p.T, W + (chunk + 1) * p.far_rows);
    const float *qb = p.q + b * p.q_so + h * p.q_si, *gb = p.g + b * p.g_so + h * p.g_si, *tab = p.tab ? p.tab + h * p.tab_len : nullptr;
    float4 k[AW_KEYS], v[AW_KEYS], dk[AW_KEYS] = {}, dv[AW_KEYS] = {};
    const float4 zero = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int x = 0; x < AW_KEYS; ++x) {
        const bool there = j0 + x < min(p.rule.S, p.T);
        k[x] = there ? aw_ld4<VEC>(p.k + b * p.k_so + h * p.k_si + (j0 + x) * p.k_ld, col, D) : zero;
        v[x] = there ? aw_ld4<VEC>(p.v + b * p.v_so + h * p.v_si + (j0 + x) * p.v_ld, col, D) : zero;
    }
    for (int r0 = W + chunk * p.far_rows + warp * RPW; r0 < r_end; r0 += U * STEP) {
        float4 q[U], g[U];
        float m[U], inv[U], delta[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int r = r0 + u * STEP + lane / LPR;
            const bool live = r < r_end;
            q[u] = live ? aw_ld4<VEC>(qb + r * p.q_ld, col, D) : zero;
            g[u] = live ? aw_ld4<VEC>(gb + r * p.g_ld, col, D) : zero;
            m[u] = live ? p.row_max[head * p.Tp + r] : INFINITY;
            inv[u] = live ? p.row_inv[head * p.Tp + r] : 0.0f;
            delta[u] = live ? p.delta[head * p.Tp + r] : 0.0f;
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int r = r0 + u * STEP + lane / LPR;
            float s[2 * AW_KEYS];
#pragma unroll
            for (int x = 0; x < AW_KEYS; ++x) {
                s[x] = fmaf(q[u].x, k[x].x, fmaf(q[u].y, k[x].y, fmaf(q[u].z, k[x].z, q[u].w * k[x].w)));
                s[AW_KEYS + x] = fmaf(g[u].x, v[x].x, fmaf(g[u].y, v[x].y, fmaf(g[u].z, v[x].z, g[u].w * v[x].w)));
            }
            sum_eight<LPR>(s, lane);
#pragma unroll
            for (int x = 0; x < AW_KEYS; ++x) {
                const int d = r - j0 - x;
                const float z = tab ? fmaf(s[x], p.scale, tab[clamp_distance(d, p.tab_len)]) : s[x] * p.scale;
                const float pr = d >= W && j0 + x < p.rule.S ? __expf(z - m[u]) * inv[u] : 0.0f, ds = pr * (s[AW_KEYS + x] - delta[u]);
                dk[x].x = fmaf(ds, q[u].x, dk[x].x); dk[x].y = fmaf(ds, q[u].y, dk[x].y); dk[x].z = fmaf(ds, q[u].z, dk[x].z); dk[x].w = fmaf(ds, q[u].w, dk[x].w);
                dv[x].x = fmaf(pr, g[u].x, dv[x].x); dv[x].y = fmaf(pr, g[u].y, dv[x].y); dv[x].z = fmaf(pr, g[u].z, dv[x].z); dv[x].w = fmaf(pr, g[u].w, dv[x].w);
            }
        }
    }
#pragma unroll
    for (int x = 0; x < AW_KEYS; ++x) {
        float e[8] = {p.scale * dk[x].x, p.scale * dk[x].y, p.scale * dk[x].z, p.scale * dk[x].w, dv[x].x, dv[x].y, dv[x].z, dv[x].w};
#pragma unroll
        for (int s = LPR; s < 32; s <<= 1)
#pragma unroll
            for (int i = 0; i < 8; ++i) e[i] += __shfl_xor_sync(0xffffffffu, e[i], s);
        if (lane < LPR) {
            st4(&sums[warp][2 * x][col], make_float4(e[0], e[1], e[2], e[3]));
            st4(&sums[warp][2 * x + 1][col], make_float4(e[4], e[5], e[6], e[7]));
        }
    }
    __syncthreads();
    const int Dp = (D + 3) / 4 * 4;
    for (int i = threadIdx.x; i < 2 * AW_KEYS * DP; i += 256) {
        const int x = i / DP, c = i - x * DP, key = j0 + x / 2;
        if (c >= Dp || key >= p.rule.S) continue;
        float a = 0.0f;
#pragma unroll
        for (int w = 0; w < 8; ++w) a += sums[w][x][c];
        p.far_part[((((int64_t)head * p.far_chunks + chunk) * p.rule.S + key) * 2 + (x & 1)) * Dp + c] = a;
    }
}
// Adds the chunks of far_part, in their order, to dK and dV of the first keys.  A block per (head, key), a thread per column.
__global__ void __launch_bounds__(128) window_attention_far_sum_kernel(const __grid_constant__ WindowAttn p, int keys) {
    pdl_trigger();
    pdl_wait();
    const int head = blockIdx.x / keys, key = blockIdx.x - head * keys, c = threadIdx.x, Dp = (p.D + 3) / 4 * 4;
    if (c >= p.D) return;
    const int64_t b = head / p.H, h = head - b * p.H, stride = (int64_t)p.rule.S * 2 * Dp;
    const float* part = p.far_part + (int64_t)head * p.far_chunks * stride + key * 2 * Dp + c;
    float dk = 0.0f, dv = 0.0f;
#pragma unroll 8
    for (int i = 0; i < p.far_chunks; ++i) { dk += part[i * stride]; dv += part[i * stride + Dp]; }
    const int64_t at = b * p.d_so + h * p.d_si + key * p.d_ld + c;
    p.dk[at] += dk;
    p.dv[at] += dv;
}
// dbias[h, n] (+)= the sum of dbias_part over sequences and tiles, a warp each, in a fixed order
__global__ void __launch_bounds__(256) window_attention_dbias_kernel(float* __restrict__ dbias, const float* __restrict__ part, int H, int B, int tiles, int buckets, int accumulate) {
    pdl_trigger();
    pdl_wait();
    const int w = blockIdx.x * 8 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
    if (w >= H * buckets) return;
    const int h = w / buckets, n = w - h * buckets;
    double a = 0.0;  // terms of both signs over the whole batch
    for (int64_t i = lane; i < (int64_t)B * tiles; i += 32) { const int64_t b = i / tiles; a += part[((b * H + h) * tiles + i - b * tiles) * buckets + n]; }
#pragma unroll
    for (int s = 16; s > 0; s >>= 1) a += __shfl_xor_sync(0xffffffffu, a, s);
    if (lane == 0) dbias[w] = (accumulate ? dbias[w] : 0.0f) + (float)a;
}

// ---- one new position per sequence ----------------------------------------------------------------------------------------------
// A cluster of up to eight CTAs takes one head of one sequence and cuts the keys it sees (the first S, then the window) into as many
// stretches; each of a CTA's eight warps reads four groups of rows at a time, a lane four columns, with a running maximum per lane group.
// The stretches are joined through distributed shared memory, in their order, by the first CTA.
// Bound by memory: 8 D bytes a key and head.
constexpr int ST_WARPS = 8, ST_MAX_SPLIT = 8;
struct StepAttn {
    const float *q, *k, *v;
    float* out;
    const int64_t* lengths;
    int* status;
    int64_t o_so, o_si, q_so, q_si, k_ld, k_so, k_si, v_ld, v_so, v_si, cache_len;
    int D, H;
    float scale;
    WindowRule rule;
};
__device__ __forceinline__ uint32_t cluster_rank() { uint32_t r; asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(r)); return r; }
__device__ __forceinline__ uint32_t cluster_size() { uint32_t r; asm("mov.u32 %0, %%cluster_nctarank;" : "=r"(r)); return r; }
__device__ __forceinline__ void cluster_sync() { asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory"); }
__device__ __forceinline__ float peer_float(const float* p, uint32_t rank) {
    uint32_t a = (uint32_t)__cvta_generic_to_shared(p), m;
    float f;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(m) : "r"(a), "r"(rank));
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(f) : "r"(m) : "memory");
    return f;
}

template <int LPR, bool VEC>  // lanes a row: 8, 16 or 32 of four columns each
__global__ void __launch_bounds__(32 * ST_WARPS) window_attention_step_kernel(const __grid_constant__ StepAttn p) {
    constexpr int RPW = 32 / LPR, U = 4, GROUPS = ST_WARPS * RPW, STEP = GROUPS * U, DP = 4 * LPR;
    __shared__ __align__(16) float g_o[GROUPS][DP + 4];
    __shared__ float g_m[GROUPS], g_sum[GROUPS], c_o[DP], c_m, c_sum;
    pdl_trigger();
    pdl_wait();
    const int rank = (int)cluster_rank(), split = (int)cluster_size(), item = blockIdx.x / split, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int64_t b = item / p.H, h = item - b * p.H;
    const int D = p.D, col = 4 * (lane % LPR), group = warp * RPW + lane / LPR;
    int64_t len = p.lengths[b];
    if (len < 0 || len > p.cache_len) {  // reported, not read
        if (threadIdx.x == 0 && rank == 0 && h == 0) { atomicExch(&p.status[0], 2); atomicExch(&p.status[1], (int)b); }
        len = 0;
    }
    const int last = (int)len - 1, lo = p.rule.window_first(last), s0 = min(p.rule.S, lo), count = len > 0 ? s0 + (int)len - lo : 0;
    const int per = (count + split - 1) / split, v0 = min(count, rank * per), v1 = min(count, v0 + per);
    const float *kb = p.k + b * p.k_so + h * p.k_si, *vb = p.v + b * p.v_so + h * p.v_si;
    float4 q = aw_ld4<VEC>(p.q + b * p.q_so + h * p.q_si, col, D), o = make_float4(0.f, 0.f, 0.f, 0.f);
    q.x *= p.scale; q.y *= p.scale; q.z *= p.scale; q.w *= p.scale;
    float m = -INFINITY, sum = 0.0f;
    auto key_of = [&](int x) { return x < s0 ? x : lo + (x - s0); };
    float4 kk[U], vv[U], kn[U], vn[U];  // rows in hand, and the next ones
    auto rows = [&](int x, float4 (&kr)[U], float4 (&vr)[U]) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int y = x + u * GROUPS;
            const bool live = y < v1;
            const int64_t key = live ? key_of(y) : 0;
            kr[u] = live ? aw_ld4<VEC>(kb + key * p.k_ld, col, D) : make_float4(0.f, 0.f, 0.f, 0.f);
            vr[u] = live ? aw_ld4<VEC>(vb + key * p.v_ld, col, D) : make_float4(0.f, 0.f, 0.f, 0.f);
        }
    };
    rows(v0 + group, kk, vv);
    int bucket = p.rule.buckets - 1;
    float bias = p.rule.bias != nullptr ? p.rule.bias[h * p.rule.buckets + bucket] : 0.0f;
    for (int x0 = v0; x0 < v1; x0 += STEP) {  // the same trips for every lane
        const int x = x0 + group;
        rows(x + STEP, kn, vn);
        float z[U];
#pragma unroll
        for (int u = 0; u < U; ++u) z[u] = fmaf(q.x, kk[u].x, fmaf(q.y, kk[u].y, fmaf(q.z, kk[u].z, q.w * kk[u].w)));
#pragma unroll
        for (int s = LPR / 2; s > 0; s >>= 1)
#pragma unroll
            for (int u = 0; u < U; ++u) z[u] += __shfl_xor_sync(0xffffffffu, z[u], s);
        float mx = m;
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int y = x + u * GROUPS;
            if (p.rule.bias != nullptr && y < v1) {  // distances only go down along the walk, and so do buckets
                const int d = last - key_of(y);
                if (p.rule.starts[bucket] > d) {
                    do --bucket; while (p.rule.starts[bucket] > d);
                    bias = p.rule.bias[h * p.rule.buckets + bucket];
                }
                if (bias == -INFINITY) { z[u] = -INFINITY; vv[u] = make_float4(0.f, 0.f, 0.f, 0.f); }  // hidden: may hold anything
                else z[u] += bias;
            }
            if (y >= v1) z[u] = -INFINITY;
            mx = fmaxf(mx, z[u]);
        }
        const float rel = mx == -INFINITY ? 0.0f : mx, f = __expf(m - rel);
        m = mx;
        sum *= f;
        o.x *= f; o.y *= f; o.z *= f; o.w *= f;
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const float e = __expf(z[u] - rel);
            sum += e;
            o.x = fmaf(e, vv[u].x, o.x); o.y = fmaf(e, vv[u].y, o.y); o.z = fmaf(e, vv[u].z, o.z); o.w = fmaf(e, vv[u].w, o.w);
            kk[u] = kn[u]; vv[u] = vn[u];
        }
    }
    if (lane % LPR == 0) { g_m[group] = m; g_sum[group] = sum; }
    st4(&g_o[group][col], o);
    __syncthreads();
    const int t = threadIdx.x;
    if (t < DP) {  // this CTA's stretch: its groups in their order
        float mx = -INFINITY;
#pragma unroll
        for (int i = 0; i < GROUPS; ++i) mx = fmaxf(mx, g_m[i]);
        const float rel = mx == -INFINITY ? 0.0f : mx;
        float a = 0.0f, total = 0.0f;
#pragma unroll
        for (int i = 0; i < GROUPS; ++i) {
            const float f = __expf(g_m[i] - rel);
            a = fmaf(f, g_o[i][t], a);
            total = fmaf(f, g_sum[i], total);
        }
        c_o[t] = a;
        if (t == 0) { c_m = mx; c_sum = total; }
    }
    cluster_sync();
    if (rank == 0 && t < D) {
        float mx = -INFINITY;
        for (int i = 0; i < split; ++i) mx = fmaxf(mx, peer_float(&c_m, i));
        const float rel = mx == -INFINITY ? 0.0f : mx;
        float a = 0.0f, total = 0.0f;
        for (int i = 0; i < split; ++i) {
            const float f = __expf(peer_float(&c_m, i) - rel);
            a = fmaf(f, peer_float(c_o + t, i), a);
            total = fmaf(f, peer_float(&c_sum, i), total);
        }
        p.out[b * p.o_so + h * p.o_si + t] = total == 0.0f ? 0.0f : a / total;  // nothing seen; scores that are not numbers leave no maximum either, but a sum that is none
    }
    cluster_sync();  // nobody leaves while its shared memory is read
}

// Long caches: one CTA an SM, all of which share the tiles of all heads and sequences evenly, whatever their lengths.  A tile is 16 KB of keys and as
// much of values, brought by TMA into a ring of six, so that 192 KB an SM are on their way; eight warps read it as above.  A head whose tiles
// lie in several CTAs leaves partial results, which a second kernel joins in their order.
// Bound by memory: 8 x 16 heads of 16384 keys x 64 (1.07 GB) 196 us after a flush of L2, 64 x 16 of 1028 (539 MB) 114, so that the second half of a long call passes
// at 6.5 TB/s; the cluster kernel above took 137 for the latter.
constexpr int SM_STAGES = 6, SM_TILE = 16384, SM_MAX_SEQ = 1024, SM_THREADS = 32 * ST_WARPS + 32;
struct StreamAttn {
    StepAttn a;
    float* part;  // [CTA][head that began before it, head that goes on after it][D + 2]: o, maximum, sum
    int* head;    // [CTA]: the head that its first tile continues, or -1
    int n_seq;
};
struct StreamKeys {  // the keys of one sequence in tiles of R: the first s0 ones, then lo .. len - 1
    int len, s0, lo, first_tiles, tiles;
    __device__ __forceinline__ StreamKeys(const StepAttn& p, int b, int R) {
        const int64_t n = p.lengths[b];
        len = n < 0 || n > p.cache_len ? 0 : (int)n;
        lo = p.rule.window_first(len - 1);
        s0 = min(p.rule.S, lo);
        first_tiles = (s0 + R - 1) / R;
        tiles = len > 0 ? first_tiles + (len - lo + R - 1) / R : 0;
    }
    __device__ __forceinline__ int row(int t, int R) const { return t < first_tiles ? t * R : lo + (t - first_tiles) * R; }
    __device__ __forceinline__ int rows(int t, int R) const { return min(R, (t < first_tiles ? s0 : len) - row(t, R)); }
};
__device__ __forceinline__ void consumers_sync() { asm volatile("bar.sync 1, 256;" ::: "memory"); }

// Whether a bias of -inf hides a bucket of this head: the same for a whole warp.
__device__ __forceinline__ bool hides_some(const WindowRule& r, int64_t h, int lane) {
    bool x = false;
    if (r.bias != nullptr)
        for (int n = lane; n < r.buckets; n += 32) x = x || r.bias[h * r.buckets + n] == -INFINITY;
    return __any_sync(0xffffffffu, x);
}
__device__ __forceinline__ bool hides(const WindowRule& r, int64_t h, int distance) { return r.bias[h * r.buckets + r.bucket(distance)] == -INFINITY; }

template <int LPR>
__global__ void __launch_bounds__(SM_THREADS, 1) window_attention_stream_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, const __grid_constant__ StreamAttn g) {
    constexpr int RPW = 32 / LPR, U = 4, GROUPS = ST_WARPS * RPW, R = GROUPS * U, DP = 4 * LPR;
    static_assert(R * DP * 4 == SM_TILE, "a tile is 16 KB");
    extern __shared__ uint8_t smem_raw[];
    const uint32_t base = (smem_u32(smem_raw) + 127u) & ~127u;
    uint8_t* gen = smem_raw + (base - smem_u32(smem_raw));
    __shared__ __align__(8) uint64_t bars[2 * SM_STAGES];
    __shared__ __align__(16) float g_o[GROUPS][DP + 4];
    __shared__ float g_m[GROUPS], g_sum[GROUPS];
    __shared__ int pre[SM_MAX_SEQ + 1];  // tiles of the sequences before, of one head
    const StepAttn& p = g.a;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, D = p.D, H = p.H;
    auto full = [&](int s) { return smem_u32(bars + s); };
    auto empty = [&](int s) { return smem_u32(bars + SM_STAGES + s); };
    if (threadIdx.x == 0) {
        for (int s = 0; s < SM_STAGES; ++s) { mbar_init(full(s), 1); mbar_init(empty(s), ST_WARPS); }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    pdl_trigger();
    pdl_wait();
    for (int b = threadIdx.x; b < g.n_seq; b += SM_THREADS) {
        pre[b + 1] = StreamKeys(p, b, R).tiles;
        if (blockIdx.x == 0 && (p.lengths[b] < 0 || p.lengths[b] > p.cache_len)) { atomicExch(&p.status[0], 2); atomicExch(&p.status[1], b); }
    }
    __syncthreads();
    if (warp == 0) {
        int run = 0;
        for (int b0 = 0; b0 < g.n_seq; b0 += 32) {
            int x = b0 + lane < g.n_seq ? pre[b0 + lane + 1] : 0;
#pragma unroll
            for (int s = 1; s < 32; s <<= 1) { const int y = __shfl_up_sync(0xffffffffu, x, s); if (lane >= s) x += y; }
            if (b0 + lane < g.n_seq) pre[b0 + lane + 1] = run + x;
            run += __shfl_sync(0xffffffffu, x, 31);
        }
        if (lane == 0) pre[0] = 0;
    }
    __syncthreads();
    const int64_t total = (int64_t)pre[g.n_seq] * H, begin = total * blockIdx.x / gridDim.x, end = total * (blockIdx.x + 1) / gridDim.x;
    for (int b = blockIdx.x; b < g.n_seq; b += gridDim.x)  // sequences without a key
        if (pre[b] == pre[b + 1])
            for (int i = threadIdx.x; i < H * D; i += SM_THREADS) p.out[b * p.o_so + i / D * p.o_si + i % D] = 0.0f;
    // where the first tile lies: sequence, head, tile
    int b = 0;
    for (int step = SM_MAX_SEQ / 2; step > 0; step >>= 1)
        if (b + step < g.n_seq && (int64_t)pre[b + step] * H <= begin) b += step;
    StreamKeys keys(p, b, R);
    int h = 0, t = 0;
    if (begin < total) {
        const int64_t at = begin - (int64_t)pre[b] * H;
        h = (int)(at / keys.tiles);
        t = (int)(at - (int64_t)h * keys.tiles);
    }
    auto next_unit = [&]() {
        t = 0;
        if (++h < H) return;
        h = 0;
        do { ++b; } while (b < g.n_seq && pre[b] == pre[b + 1]);
        if (b < g.n_seq) keys = StreamKeys(p, b, R);
    };
    if (threadIdx.x == 0) g.head[blockIdx.x] = begin < total && t > 0 ? b * H + h : -1;
    if (begin == end && begin < total && t > 0 && threadIdx.x < D + 2) {  // fewer tiles than CTAs, and none for this one in the middle of a head: an empty part
        g.part[(int64_t)blockIdx.x * 2 * (D + 2) + threadIdx.x] = threadIdx.x == D ? -INFINITY : 0.0f;
    }

    if (warp == ST_WARPS) {
        if (lane == 0) {
            bool ok = true;
            for (int64_t i = begin; i < end && ok; ++i) {
                const uint32_t n = (uint32_t)(i - begin), s = n % SM_STAGES;
                ok = mbar_wait(empty(s), ((n / SM_STAGES) & 1u) ^ 1u, p.status, 71);
                if (!ok) break;
                mbar_expect_tx(full(s), 2 * R * D * 4);
                tma_load_4d(base + s * 2 * SM_TILE, &map_k, full(s), 0, keys.row(t, R), h, b);
                tma_load_4d(base + s * 2 * SM_TILE + SM_TILE, &map_v, full(s), 0, keys.row(t, R), h, b);
                if (++t == keys.tiles) next_unit();
            }
        }
        return;
    }
    const int col = 4 * (lane % LPR), group = warp * RPW + lane / LPR;
    const float4 zero = make_float4(0.f, 0.f, 0.f, 0.f);
    bool good = true;
    for (int64_t i = begin; i < end;) {
        const bool continues = t > 0;  // only the first one of this CTA
        const int last = keys.len - 1;
        float4 q = col < D ? ld4(p.q + b * p.q_so + h * p.q_si + col) : zero, o = zero;
        q.x *= p.scale; q.y *= p.scale; q.z *= p.scale; q.w *= p.scale;
        float m = -INFINITY, sum = 0.0f;
        int bucket = p.rule.buckets - 1;
        float bias = p.rule.bias != nullptr ? p.rule.bias[(int64_t)h * p.rule.buckets + bucket] : 0.0f;
        auto walk = [&](auto hidden) {
            for (; t < keys.tiles && i < end; ++t, ++i) {
                const uint32_t n = (uint32_t)(i - begin), s = n % SM_STAGES;
                const int rows = keys.rows(t, R), r0 = keys.row(t, R);
                good = good && __all_sync(0xffffffffu, mbar_wait(full(s), (n / SM_STAGES) & 1u, p.status, 72));
                const float* kt = reinterpret_cast<const float*>(gen + s * 2 * SM_TILE);
                const float* vt = kt + SM_TILE / 4;
                float z[U];
                float4 vv[U];
#pragma unroll
                for (int u = 0; u < U; ++u) {  // rows that are not there, or hidden, hold anything and are not looked at
                    const int y = u * GROUPS + group;
                    const bool live = y < rows && col < D && !(decltype(hidden)::value && hides(p.rule, h, last - (r0 + y)));
                    const float4 kk = live ? ld4(kt + y * D + col) : zero;
                    vv[u] = live ? ld4(vt + y * D + col) : zero;
                    z[u] = fmaf(q.x, kk.x, fmaf(q.y, kk.y, fmaf(q.z, kk.z, q.w * kk.w)));
                }
                __syncwarp();
                if (lane == 0) mbar_arrive(empty(s));  // everything of this warp's is in registers
#pragma unroll
                for (int x = LPR / 2; x > 0; x >>= 1)
#pragma unroll
                    for (int u = 0; u < U; ++u) z[u] += __shfl_xor_sync(0xffffffffu, z[u], x);
                float mx = m;
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    const int y = u * GROUPS + group;
                    if (p.rule.bias != nullptr && y < rows) {  // distances only go down along the walk, and so do buckets
                        const int d = last - (r0 + y);
                        if (p.rule.starts[bucket] > d) {
                            do --bucket; while (p.rule.starts[bucket] > d);
                            bias = p.rule.bias[(int64_t)h * p.rule.buckets + bucket];
                        }
                        z[u] += bias;
                    }
                    if (y >= rows) z[u] = -INFINITY;
                    mx = fmaxf(mx, z[u]);
                }
                const float rel = mx == -INFINITY ? 0.0f : mx, f = __expf(m - rel);
                m = mx;
                sum *= f;
                o.x *= f; o.y *= f; o.z *= f; o.w *= f;
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    const float e = __expf(z[u] - rel);
                    sum += e;
                    o.x = fmaf(e, vv[u].x, o.x); o.y = fmaf(e, vv[u].y, o.y); o.z = fmaf(e, vv[u].z, o.z); o.w = fmaf(e, vv[u].w, o.w);
                }
            }
        };
        if (hides_some(p.rule, h, lane)) walk(std::true_type());  // a loop of its own: a test of every row cost all biased calls 4 to 10 %
        else walk(std::false_type());
        // this CTA's tiles of the head: its groups in their order
        consumers_sync();  // the head before has been written
        if (lane % LPR == 0) { g_m[group] = m; g_sum[group] = sum; }
        st4(&g_o[group][col], o);
        consumers_sync();
        const int c = threadIdx.x;
        if (c < D) {
            float mx = -INFINITY;
#pragma unroll
            for (int x = 0; x < GROUPS; ++x) mx = fmaxf(mx, g_m[x]);
            const float rel = mx == -INFINITY ? 0.0f : mx;
            float a = 0.0f, all = 0.0f;
#pragma unroll
            for (int x = 0; x < GROUPS; ++x) {
                const float f = __expf(g_m[x] - rel);
                a = fmaf(f, g_o[x][c], a);
                all = fmaf(f, g_sum[x], all);
            }
            const bool whole = !continues && t == keys.tiles;
            if (whole) {
                p.out[b * p.o_so + h * p.o_si + c] = all == 0.0f ? 0.0f : a / all;
            } else {
                float* part = g.part + ((int64_t)blockIdx.x * 2 + (continues ? 0 : 1)) * (D + 2);
                part[c] = a;
                if (c == 0) { part[D] = mx; part[D + 1] = all; }
            }
        }
        if (t == keys.tiles) next_unit();
    }
}
// Joins the parts of the heads that lie in several CTAs: the block of the second of them does it.
__global__ void __launch_bounds__(128) window_attention_join_kernel(const __grid_constant__ StreamAttn g) {
    pdl_trigger();
    pdl_wait();
    const int i = blockIdx.x + 1, ctas = gridDim.x + 1, unit = g.head[i], c = threadIdx.x, D = g.a.D;
    if (unit < 0 || g.head[i - 1] == unit || c >= D) return;
    auto part = [&](int cta, int which) { return g.part + ((int64_t)cta * 2 + which) * (D + 2); };
    int end = i;
    while (end < ctas && g.head[end] == unit) ++end;
    float mx = part(i - 1, 1)[D];
    for (int x = i; x < end; ++x) mx = fmaxf(mx, part(x, 0)[D]);
    const float rel = mx == -INFINITY ? 0.0f : mx;
    float f = __expf(part(i - 1, 1)[D] - rel), a = f * part(i - 1, 1)[c], all = f * part(i - 1, 1)[D + 1];
    for (int x = i; x < end; ++x) {
        f = __expf(part(x, 0)[D] - rel);
        a = fmaf(f, part(x, 0)[c], a);
        all = fmaf(f, part(x, 0)[D + 1], all);
    }
    g.a.out[unit / g.a.H * g.a.o_so + unit % g.a.H * g.a.o_si + c] = all == 0.0f ? 0.0f : a / all;
}

// ---- host side ----------------------------------------------------------------------------------------------------------------
static bool vec_rows(const float* p, int64_t ld, int64_t so, int64_t si) { return aligned16(p) && ld % 4 == 0 && so % 4 == 0 && si % 4 == 0; }
// Rows that are written lie apart: by ascending stride, each one reaches past the stretch that the smaller ones cover, as in a dense tensor or a slice of one.
static bool own_rows(int64_t B, int64_t H, int64_t T, int64_t D, int64_t ld, int64_t so, int64_t si) {
    std::pair<int64_t, int64_t> d[3] = {{ld, T}, {si, H}, {so, B}};
    std::sort(d, d + 3);
    double stretch = (double)D;
    for (const auto& [stride, n] : d) {
        if (n <= 1) continue;
        if ((double)stride < stretch) return false;
        stretch += (double)(n - 1) * (double)stride;
    }
    return true;
}
// Floats of keys in sight from which the streaming kernel and its join are taken instead of the one launch of clusters (either, us, after a flush of L2:
// 1 x 16 heads of 2048 x 64 16.4 clusters, 19.5 streamed; 8 x 16 of 512 20.5, 21.5; 4 x 16 of 2048 30.8, 29.7; 1 x 16 of 8192 36.9, 29.7; 32 x 16 of 512 47.1, 42.0).
constexpr int64_t ST_STREAM = int64_t(1) << 22;
constexpr int64_t AW_MAX_T = int64_t(1) << 24, AW_MAX_D = 128, AW_MAX_H = 65535;

template <class K, class... A>
static int fma_launch(gcb_ctx* ctx, K kernel, bool* done, int64_t ctas, size_t floats, const char* name, const WindowAttn& p, A... more) {
    GCB_REQUIRE(ctas < (int64_t(1) << 31), "window attention: more tiles than a grid holds");
    if (!done[ctx->device]) { GCB_CHECK_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 232448 - 1024)); done[ctx->device] = true; }
    GCB_CHECK_CUDA(launch_next(ctx->stream, dim3((unsigned)ctas), 256, sizeof(float) * floats, kernel, p, more...));
    return after_launch(ctx, name);
}
template <int R, int NC, bool VEC>
static int fma_fwd(gcb_ctx* ctx, int64_t heads, const WindowAttn& p) {
    static bool done[kMaxDevices] = {};
    return fma_launch(ctx, window_attention_fwd_kernel<R, NC, VEC>, done, heads * p.tiles, aw_floats(R, 1, 2, 1, (p.D + 3) / 4 * 4), "window_attention_fwd", p);
}
template <int R, int NC, bool VEC>
static int fma_bwd(gcb_ctx* ctx, int64_t heads, const WindowAttn& p) {
    static bool done[kMaxDevices] = {};
    return fma_launch(ctx, window_attention_bwd_kernel<R, NC, VEC>, done, 2 * heads * p.tiles, aw_floats(R, 2, 2, 2, (p.D + 3) / 4 * 4), "window_attention_bwd", p, (int)(heads * p.tiles));
}
// R, with 16 R rows of a CTA's own: 64 rows take 8 reads of shared memory for 32 double FMAs where 32 rows take 6 for 16; 32 rows where 64 would leave three fifths
// of the SMs idle.  Either, us, forward and backward: 16 x 16 x 1024 x 128 with a window of 256 1508 and 5898 with 32, 1339 and 4006 with 64; 4 x 8 x 256 x 128
// 51 and 134, 42 and 114; 4 x 4 x 256 x 128 47 and 84, 42 and 73; 1 x 4 x 256 x 128 31 and 55, 41 and 73; 64 x 12 x 32 x 64 25 and 86, 33 and 116.  Twice the
// threads for 64 rows, which leaves the reads as they are, was slower than twice the rows a thread (6028 and 5537 in the first of these, at an earlier step).
static int fma_rows(int64_t heads, int64_t T) { return T > 32 && 5 * heads * ((T + 63) / 64) >= 2 * kSMs ? 4 : 2; }
template <int R>
static int fma_run(gcb_ctx* ctx, int64_t heads, const WindowAttn& p, bool vec) {
    if (p.dq) return p.D <= 64 ? (vec ? fma_bwd<R, 1, true>(ctx, heads, p) : fma_bwd<R, 1, false>(ctx, heads, p)) : (vec ? fma_bwd<R, 2, true>(ctx, heads, p) : fma_bwd<R, 2, false>(ctx, heads, p));
    return p.D <= 64 ? (vec ? fma_fwd<R, 1, true>(ctx, heads, p) : fma_fwd<R, 1, false>(ctx, heads, p)) : (vec ? fma_fwd<R, 2, true>(ctx, heads, p) : fma_fwd<R, 2, false>(ctx, heads, p));
}
// What queries beyond the window add to the first keys' gradients; after dK and dV have been written, and delta.
static int far_gradients(gcb_ctx* ctx, int64_t heads, WindowAttn& p, bool vec, Scratch& mem) {
    const int Dp = (p.D + 3) / 4 * 4, groups = (p.rule.S + AW_KEYS - 1) / AW_KEYS, keys = std::min(p.rule.S, p.T);
    // 256 queries a CTA, and where that leaves SMs idle 64
    p.far_rows = heads * groups * ((p.T - p.rule.W + 255) / 256) >= 2 * kSMs ? 256 : 64;
    p.far_chunks = (p.T - p.rule.W + p.far_rows - 1) / p.far_rows;
    const int64_t ctas = heads * groups * p.far_chunks;
    GCB_REQUIRE(ctas < (int64_t(1) << 31) && heads * keys < (int64_t(1) << 31), "window attention: more tiles than a grid holds");
    const int rc = mem.get(sizeof(float) * (size_t)(heads * p.far_chunks * p.rule.S * 2 * Dp));
    if (rc) return rc;
    p.far_part = mem.as<float>();
    auto run = [&](auto kernel) { return launch_next(ctx->stream, dim3((unsigned)ctas), 256, 0, kernel, p); };
    if (p.D <= 32) GCB_CHECK_CUDA(vec ? run(window_attention_far_kernel<8, true>) : run(window_attention_far_kernel<8, false>));
    else if (p.D <= 64) GCB_CHECK_CUDA(vec ? run(window_attention_far_kernel<16, true>) : run(window_attention_far_kernel<16, false>));
    else GCB_CHECK_CUDA(vec ? run(window_attention_far_kernel<32, true>) : run(window_attention_far_kernel<32, false>));
    const int launched = after_launch(ctx, "window_attention_far");
    if (launched) return launched;
    GCB_CHECK_CUDA(launch_next(ctx->stream, dim3((unsigned)(heads * keys)), 128, 0, window_attention_far_sum_kernel, p, keys));
    return after_launch(ctx, "window_attention_far_sum");
}
// The bias by distance of every head, up to the first distance of the last bucket, which holds for all beyond.
__global__ void __launch_bounds__(256) window_attention_table_kernel(float* __restrict__ tab, int len, const __grid_constant__ WindowRule r) {
    pdl_trigger();
    pdl_wait();
    const int d = blockIdx.x * 256 + threadIdx.x, h = blockIdx.y;
    if (d < len) tab[(int64_t)h * len + d] = r.bias[(int64_t)h * r.buckets + r.bucket(d)];
}
static int make_table(gcb_ctx* ctx, WindowAttn& p, Scratch& mem) {
    if (p.rule.bias == nullptr) return GCB_OK;
    p.tab_len = std::min(p.T, p.rule.starts[p.rule.buckets - 1] + 1);
    const int rc = mem.get(sizeof(float) * (size_t)p.H * p.tab_len);
    if (rc) return rc;
    p.tab = mem.as<float>();
    GCB_CHECK_CUDA(launch_next(ctx->stream, dim3((unsigned)((p.tab_len + 255) / 256), (unsigned)p.H), 256, 0, window_attention_table_kernel, mem.as<float>(), p.tab_len, p.rule));
    return after_launch(ctx, "window_attention_table");
}

template <int LPR>
static int stream_launch(gcb_ctx* ctx, const StreamAttn& g, const float* k, const float* v, int ctas) {
    const StepAttn& p = g.a;
    const int rows = SM_TILE / (16 * LPR);
    CUtensorMap mk, mv;
    auto rows_of = [&](CUtensorMap& map, const float* x, int64_t ld, int64_t so, int64_t si) {
        return encode_rows(tma_encode(ctx), &map, x, p.D, p.cache_len, ld, si, so, p.H, g.n_seq, p.D, rows, CU_TENSOR_MAP_SWIZZLE_NONE);
    };
    GCB_REQUIRE(rows_of(mk, k, p.k_ld, p.k_so, p.k_si) && rows_of(mv, v, p.v_ld, p.v_so, p.v_si), "window attention: strides beyond what TMA can address");
    constexpr size_t smem = 2 * SM_STAGES * SM_TILE + 128;
    static bool done[kMaxDevices] = {};
    if (!done[ctx->device]) { GCB_CHECK_CUDA(cudaFuncSetAttribute(window_attention_stream_kernel<LPR>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem)); done[ctx->device] = true; }
    GCB_CHECK_CUDA(launch_chained(ctx->stream, dim3((unsigned)ctas), SM_THREADS, smem, window_attention_stream_kernel<LPR>, mk, mv, g));
    const int rc = after_launch(ctx, "window_attention_stream");
    if (rc) return rc;
    GCB_CHECK_CUDA(launch_chained(ctx->stream, dim3((unsigned)ctas - 1), 128, 0, window_attention_join_kernel, g));
    return after_launch(ctx, "window_attention_join");
}

}  // namespace gcb

using namespace gcb;

extern "C" {

int gcb_relative_bucket_starts(int64_t buckets, int64_t reach, int64_t* starts) {
    GCB_REQUIRE(buckets >= 1 && buckets <= AW_MAX_BUCKETS && reach >= 1 && reach < (int64_t(1) << 30) && starts, "gcb_relative_bucket_starts: 1 to %d buckets and a positive distance are needed", AW_MAX_BUCKETS);
    // Bucket e + k of e + m starts at the least n with n^m e^k >= reach^k e^m: whole numbers of up to 64 factors of 30 bits, so that no
    // border hangs on the rounding of a logarithm.
    const int64_t e = std::max<int64_t>(1, buckets / 2), m = buckets - e, far = std::max(reach, e);
    struct Big {
        uint32_t w[128];
        int n;
    };
    auto times = [](Big& x, uint64_t f, int64_t times) {
        for (; times > 0; --times) {
            uint64_t carry = 0;
            for (int i = 0; i < x.n; ++i) { carry += x.w[i] * f; x.w[i] = (uint32_t)carry; carry >>= 32; }
            if (carry) x.w[x.n++] = (uint32_t)carry;
        }
    };
    auto less = [](const Big& a, const Big& b) {
        if (a.n != b.n) return a.n < b.n;
        for (int i = a.n - 1; i >= 0; --i) if (a.w[i] != b.w[i]) return a.w[i] < b.w[i];
        return false;
    };
    for (int64_t n = 0; n < e; ++n) starts[n] = n;
    for (int64_t k = 0; k < m; ++k) {
        Big right = {{1}, 1};
        times(right, (uint64_t)far, k);
        times(right, (uint64_t)e, m);
        int64_t lo = 0, hi = far;  // lo is too small, hi is not
        while (hi - lo > 1) {
            const int64_t mid = lo + (hi - lo) / 2;
            Big left = {{1}, 1};
            times(left, (uint64_t)mid, m);
            times(left, (uint64_t)e, k);
            (less(left, right) ? lo : hi) = mid;
        }
        starts[e + k] = hi;
    }
    return GCB_OK;
}

int gcb_window_attention_fwd_f32(gcb_ctx* ctx, int64_t B, int64_t H, int64_t T, int64_t D, float* out, int64_t o_ld, int64_t o_so, int64_t o_si, float* stats, const float* q, int64_t q_ld, int64_t q_so, int64_t q_si,
                                 const float* k, int64_t k_ld, int64_t k_so, int64_t k_si, const float* v, int64_t v_ld, int64_t v_so, int64_t v_si, float scale, int64_t window, int64_t sinks, const float* bias,
                                 int64_t buckets, const int64_t* bucket_starts) {
    GCB_REQUIRE(ctx && B >= 0 && H >= 0 && T >= 0 && D >= 0, "gcb_window_attention_fwd_f32: bad arguments");
    WindowAttn p = {};
    int rc = make_rule(p.rule, "gcb_window_attention_fwd_f32", window, sinks, bias, buckets, bucket_starts);
    if (rc) return rc;
    if (B == 0 || H == 0 || T == 0 || D == 0) return GCB_OK;
    if (D > AW_MAX_D || T > AW_MAX_T || H > AW_MAX_H) { set_error("gcb_window_attention_fwd_f32: at most %lld heads of %lld columns and sequences of %lld positions", (long long)AW_MAX_H, (long long)AW_MAX_D, (long long)AW_MAX_T); return GCB_UNSUPPORTED; }
    GCB_REQUIRE(out && stats && q && k && v && own_rows(B, H, T, D, o_ld, o_so, o_si), "gcb_window_attention_fwd_f32: NULL pointer, or output rows that overlap");
    cudaSetDevice(ctx->device);
    p.q = q; p.q_ld = q_ld; p.q_so = q_so; p.q_si = q_si;
    p.k = k; p.k_ld = k_ld; p.k_so = k_so; p.k_si = k_si;
    p.v = v; p.v_ld = v_ld; p.v_so = v_so; p.v_si = v_si;
    p.out = out; p.o_ld = o_ld; p.o_so = o_so; p.o_si = o_si;
    p.Tp = gcb_attention_stats_floats(1, 1, T) / 2; p.T = (int)T; p.D = (int)D; p.H = (int)H; p.scale = scale;
    p.row_max = stats; p.row_inv = stats + B * H * p.Tp;
    const int R = fma_rows(B * H, T);
    p.tiles = (int)((T + 16 * R - 1) / (16 * R));
    const bool vec = D % 4 == 0 && vec_rows(q, q_ld, q_so, q_si) && vec_rows(k, k_ld, k_so, k_si) && vec_rows(v, v_ld, v_so, v_si) && vec_rows(out, o_ld, o_so, o_si);
    Scratch tab(ctx);
    const bool tc = window_tc_takes(ctx, B, p);
    if (tc && (rc = make_table(ctx, p, tab))) return rc;
    if (tc) rc = window_tc_fwd(ctx, B, p);
    else rc = R == 4 ? fma_run<4>(ctx, B * H, p, vec) : fma_run<2>(ctx, B * H, p, vec);
    if (rc) return rc;
    note_write(ctx, out, span_bytes(B, H, T, D, o_ld, o_so, o_si));
    return GCB_OK;
}

int gcb_window_attention_bwd_f32(gcb_ctx* ctx, int64_t B, int64_t H, int64_t T, int64_t D, float* dq, float* dk, float* dv, int64_t d_ld, int64_t d_so, int64_t d_si, float* dbias, int accumulate_dbias,
                                 const float* dout, int64_t g_ld, int64_t g_so, int64_t g_si, const float* out, int64_t o_ld, int64_t o_so, int64_t o_si, const float* stats, const float* q, int64_t q_ld, int64_t q_so,
                                 int64_t q_si, const float* k, int64_t k_ld, int64_t k_so, int64_t k_si, const float* v, int64_t v_ld, int64_t v_so, int64_t v_si, float scale, int64_t window, int64_t sinks,
                                 const float* bias, int64_t buckets, const int64_t* bucket_starts) {
    GCB_REQUIRE(ctx && B >= 0 && H >= 0 && T >= 0 && D >= 0, "gcb_window_attention_bwd_f32: bad arguments");
    WindowAttn p = {};
    int rc = make_rule(p.rule, "gcb_window_attention_bwd_f32", window, sinks, bias, buckets, bucket_starts);
    if (rc) return rc;
    GCB_REQUIRE(bias || !dbias, "gcb_window_attention_bwd_f32: a gradient of the bias without a bias");
    if (B == 0 || H == 0 || T == 0 || D == 0) return dbias && !accumulate_dbias && H > 0 ? gcb_fill_f32(ctx, dbias, 0.0f, H * buckets) : GCB_OK;
    if (D > AW_MAX_D || T > AW_MAX_T || H > AW_MAX_H) { set_error("gcb_window_attention_bwd_f32: at most %lld heads of %lld columns and sequences of %lld positions", (long long)AW_MAX_H, (long long)AW_MAX_D, (long long)AW_MAX_T); return GCB_UNSUPPORTED; }
    GCB_REQUIRE(dq && dk && dv && dout && out && stats && q && k && v && own_rows(B, H, T, D, d_ld, d_so, d_si), "gcb_window_attention_bwd_f32: NULL pointer, or gradient rows that overlap");
    cudaSetDevice(ctx->device);
    p.q = q; p.q_ld = q_ld; p.q_so = q_so; p.q_si = q_si;
    p.k = k; p.k_ld = k_ld; p.k_so = k_so; p.k_si = k_si;
    p.v = v; p.v_ld = v_ld; p.v_so = v_so; p.v_si = v_si;
    p.g = dout; p.g_ld = g_ld; p.g_so = g_so; p.g_si = g_si;
    p.o = out; p.o_ld = o_ld; p.o_so = o_so; p.o_si = o_si;
    p.dq = dq; p.dk = dk; p.dv = dv; p.d_ld = d_ld; p.d_so = d_so; p.d_si = d_si;
    p.Tp = gcb_attention_stats_floats(1, 1, T) / 2; p.T = (int)T; p.D = (int)D; p.H = (int)H; p.scale = scale;
    p.row_max = const_cast<float*>(stats); p.row_inv = p.row_max + B * H * p.Tp;
    const int R = fma_rows(B * H, T);
    p.tiles = (int)((T + 16 * R - 1) / (16 * R));
    const int64_t heads = B * H;
    const bool vec = D % 4 == 0 && vec_rows(q, q_ld, q_so, q_si) && vec_rows(k, k_ld, k_so, k_si) && vec_rows(v, v_ld, v_so, v_si) && vec_rows(dout, g_ld, g_so, g_si) && vec_rows(out, o_ld, o_so, o_si) &&
                     vec_rows(dq, d_ld, d_so, d_si) && vec_rows(dk, d_ld, d_so, d_si) && vec_rows(dv, d_ld, d_so, d_si);
    const bool tc = window_tc_takes(ctx, B, p);
    const int tiles = tc ? (int)((T + AW_TC_TILE - 1) / AW_TC_TILE) : p.tiles;
    Scratch part(ctx), far(ctx), tab(ctx), delta(ctx);
    // Few queries beyond the window: the tiles of the first keys go on to the last query, which saves two launches (4 x 4 x 64 13 us, 18 with them;
    // 5 x 6 x 331, window 100, 135 and 136; 8 x 8 x 200, window 30, 122 and 117; 2 x 4 x 512, window 64, 91 and 54).
    p.far_inside = !tc && T - p.rule.W <= 128;
    const bool beyond = p.rule.S > 0 && p.rule.W < T && !p.far_inside;  // some query looks past its window
    if (((tc || beyond) && (rc = make_table(ctx, p, tab))) || (rc = delta.get(sizeof(float) * (size_t)(heads * p.Tp)))) return rc;
    p.delta = delta.as<float>();
    if (dbias) {
        if ((rc = part.get(sizeof(float) * (size_t)(heads * tiles * buckets)))) return rc;
        p.dbias_part = part.as<float>();
    }
    if (tc) rc = window_tc_bwd(ctx, B, p);
    else rc = R == 4 ? fma_run<4>(ctx, heads, p, vec) : fma_run<2>(ctx, heads, p, vec);
    if (rc) return rc;
    if (beyond && (rc = far_gradients(ctx, heads, p, vec, far))) return rc;
    for (float* d : {dq, dk, dv}) note_write(ctx, d, span_bytes(B, H, T, D, d_ld, d_so, d_si));
    if (dbias) {
        GCB_CHECK_CUDA(launch_next(ctx->stream, dim3((unsigned)((H * buckets + 7) / 8)), 256, 0, window_attention_dbias_kernel, dbias, part.as<float>(), (int)H, (int)B, tiles, (int)buckets, accumulate_dbias));
        note_write(ctx, dbias, sizeof(float) * (size_t)(H * buckets));
        return after_launch(ctx, "window_attention_dbias");
    }
    return GCB_OK;
}

int gcb_window_attention_step_f32(gcb_ctx* ctx, int64_t n_seq, int64_t H, int64_t D, float* out, int64_t o_so, int64_t o_si, const float* q, int64_t q_so, int64_t q_si, const float* k, int64_t k_ld, int64_t k_so,
                                  int64_t k_si, const float* v, int64_t v_ld, int64_t v_so, int64_t v_si, int64_t cache_len, const int64_t* lengths, float scale, int64_t window, int64_t sinks, const float* bias,
                                  int64_t buckets, const int64_t* bucket_starts) {
    GCB_REQUIRE(ctx && n_seq >= 0 && H >= 0 && D >= 0 && cache_len >= 0, "gcb_window_attention_step_f32: bad arguments");
    StepAttn p = {};
    int rc = make_rule(p.rule, "gcb_window_attention_step_f32", window, sinks, bias, buckets, bucket_starts);
    if (rc) return rc;
    if (n_seq == 0 || H == 0 || D == 0) return GCB_OK;
    if (D > AW_MAX_D || cache_len >= (int64_t(1) << 30)) { set_error("gcb_window_attention_step_f32: heads of up to %lld columns and caches of less than 2^30 positions", (long long)AW_MAX_D); return GCB_UNSUPPORTED; }
    GCB_REQUIRE(out && q && (cache_len == 0 || (k && v)) && lengths && own_rows(n_seq, H, 1, D, 0, o_so, o_si), "gcb_window_attention_step_f32: NULL pointer, or output rows that overlap");
    cudaSetDevice(ctx->device);
    p.q = q; p.q_so = q_so; p.q_si = q_si;
    p.k = k; p.k_ld = k_ld; p.k_so = k_so; p.k_si = k_si;
    p.v = v; p.v_ld = v_ld; p.v_so = v_so; p.v_si = v_si;
    p.out = out; p.o_so = o_so; p.o_si = o_si;
    p.lengths = lengths; p.status = ctx->d_status; p.cache_len = cache_len; p.D = (int)D; p.H = (int)H; p.scale = scale;
    const bool vec = D % 4 == 0 && vec_rows(q, 0, q_so, q_si) && vec_rows(k, k_ld, k_so, k_si) && vec_rows(v, v_ld, v_so, v_si);
    const int64_t seen = p.rule.W ? std::min<int64_t>(cache_len, (int64_t)p.rule.W + p.rule.S) : cache_len;
    if (vec && n_seq <= SM_MAX_SEQ && n_seq * H < (int64_t(1) << 31) && n_seq * cache_len < (int64_t(1) << 34) && n_seq * H * seen * D >= ST_STREAM && rows_ok(k, k_ld, k_so, k_si, n_seq, H) && rows_ok(v, v_ld, v_so, v_si, n_seq, H) && tma_encode(ctx) != nullptr) {
        StreamAttn g = {p, nullptr, nullptr, (int)n_seq};
        Scratch mem(ctx);
        if ((rc = mem.get(sizeof(float) * (size_t)kSMs * (2 * (D + 2) + 1)))) return rc;
        g.part = mem.as<float>();
        g.head = reinterpret_cast<int*>(g.part + kSMs * 2 * (D + 2));
        rc = D <= 32 ? stream_launch<8>(ctx, g, k, v, kSMs) : D <= 64 ? stream_launch<16>(ctx, g, k, v, kSMs) : stream_launch<32>(ctx, g, k, v, kSMs);
        if (!rc) note_write(ctx, out, span_bytes(n_seq, H, 1, D, 0, o_so, o_si));
        return rc;
    }
    // As many stretches as fill the SMs about twice over, none shorter than 64 keys.
    int64_t split = 1;
    while (split < ST_MAX_SPLIT && n_seq * H * split < 2 * kSMs && seen / (2 * split) >= 64) split *= 2;
    GCB_REQUIRE(n_seq * H * split < (int64_t(1) << 31), "gcb_window_attention_step_f32: more heads than a grid holds");
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(n_seq * H * split));
    cfg.blockDim = dim3(32 * ST_WARPS);
    cfg.stream = ctx->stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = (unsigned)split; attr[0].val.clusterDim.y = 1; attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = n_seq * H * split <= kSMs ? 2 : 1;
    auto run = [&](auto kernel) { return cudaLaunchKernelEx(&cfg, kernel, p); };
    if (D <= 32) GCB_CHECK_CUDA(vec ? run(window_attention_step_kernel<8, true>) : run(window_attention_step_kernel<8, false>));
    else if (D <= 64) GCB_CHECK_CUDA(vec ? run(window_attention_step_kernel<16, true>) : run(window_attention_step_kernel<16, false>));
    else GCB_CHECK_CUDA(vec ? run(window_attention_step_kernel<32, true>) : run(window_attention_step_kernel<32, false>));
    note_write(ctx, out, span_bytes(n_seq, H, 1, D, 0, o_so, o_si));
    return after_launch(ctx, "window_attention_step");
}

}  // extern "C"
