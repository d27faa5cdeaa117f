// Tiles of fp32 FMA attention: 16 R rows of a CTA's own (R 2, or 4) against 64 of the other side, 256 threads as 16 x 16, rows of D + 4 floats
// (D a multiple of four) in shared memory.
#pragma once
#include "common.cuh"

namespace gcb {

constexpr int AS_OWN = 32, AS_T = 64;

// ROWS rows of D columns from row r0 into [row][D + 4], asynchronously; rows beyond T are zero
template <int ROWS>
__device__ __forceinline__ void as_load(float* sm, const float* p, int64_t ld, int r0, int T, int D) {
    const int d4 = D >> 2, down = 256 / d4, across = 256 - down * d4;
    int r = threadIdx.x / d4, q = threadIdx.x - r * d4;
    while (r < ROWS) {
        const int c = 4 * q;
        const bool live = r0 + r < T;
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"((uint32_t)__cvta_generic_to_shared(sm + r * (D + 4) + c)), "l"(live ? p + (r0 + r) * ld + c : p), "r"(live ? 16 : 0) : "memory");
        r += down;
        q += across;
        if (q >= d4) { q -= d4; ++r; }
    }
}
__device__ __forceinline__ void as_landed() {
    asm volatile("cp.async.wait_all;" ::: "memory");
    __syncthreads();
}
// c[i][j] = a[ty + 16 i] . b[tx + 16 j]
template <int R, int C>
__device__ __forceinline__ void as_abt(float (&c)[R][C], const float* a, const float* b, int D, int ty, int tx) {
#pragma unroll
    for (int i = 0; i < R; ++i)
#pragma unroll
        for (int j = 0; j < C; ++j) c[i][j] = 0.0f;
    const int P = D + 4;
#pragma unroll 4
    for (int d = 0; d < D; d += 4) {
        float4 x[R], y[C];
#pragma unroll
        for (int i = 0; i < R; ++i) x[i] = ld4(a + (ty + 16 * i) * P + d);
#pragma unroll
        for (int j = 0; j < C; ++j) y[j] = ld4(b + (tx + 16 * j) * P + d);
#pragma unroll
        for (int i = 0; i < R; ++i)
#pragma unroll
            for (int j = 0; j < C; ++j) c[i][j] = fmaf(x[i].x, y[j].x, fmaf(x[i].y, y[j].y, fmaf(x[i].z, y[j].z, fmaf(x[i].w, y[j].w, c[i][j]))));
    }
}
// two fused multiply-adds in one instruction
union F4 { float4 f; unsigned long long d[2]; };
__device__ __forceinline__ unsigned long long twice(float x) {
    unsigned long long r;
    asm("mov.b64 %0, {%1, %1};" : "=l"(r) : "f"(x));
    return r;
}
__device__ __forceinline__ unsigned long long fma2(unsigned long long a, unsigned long long b, unsigned long long c) {
    asm("fma.rn.f32x2 %0, %1, %2, %0;" : "+l"(c) : "l"(a), "l"(b));
    return c;
}
__device__ __forceinline__ void fma2_to(float& x, float& y, unsigned long long a, unsigned long long b) {  // (x, y) += a b
    unsigned long long c;
    asm("mov.b64 %0, {%1, %2};" : "=l"(c) : "f"(x), "f"(y));
    c = fma2(a, b, c);
    asm("mov.b64 {%0, %1}, %2;" : "=f"(x), "=f"(y) : "l"(c));
}
// acc[i][4 n + e] += sum_k p[ty + 16 i][k] b[k][64 n + 4 tx + e], k < 64
template <int NC, int R>
__device__ __forceinline__ void as_ab(float (&acc)[R][4 * NC], const float* p, const float* b, int D, int ty, int tx) {
    const int P = D + 4;
#pragma unroll 4
    for (int k = 0; k < AS_T; k += 4) {
        float a[R][4];
#pragma unroll
        for (int i = 0; i < R; ++i) { const float4 x = ld4(p + (ty + 16 * i) * (AS_T + 4) + k); a[i][0] = x.x; a[i][1] = x.y; a[i][2] = x.z; a[i][3] = x.w; }
#pragma unroll
        for (int n = 0; n < NC; ++n) {
            const int c = min(64 * n + 4 * tx, D - 4);  // what lies beyond D is not used, and a branch would keep the loads of several rows apart
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                F4 y;
                y.f = ld4(b + (k + q) * P + c);
#pragma unroll
                for (int i = 0; i < R; ++i) {
                    const unsigned long long w = twice(a[i][q]);
                    fma2_to(acc[i][4 * n], acc[i][4 * n + 1], w, y.d[0]);
                    fma2_to(acc[i][4 * n + 2], acc[i][4 * n + 3], w, y.d[1]);
                }
            }
        }
    }
}
// acc[i][4 n + e] += sum_r p[r][R ty + i] b[r][64 n + 4 tx + e], r < 64
template <int NC, int R>
__device__ __forceinline__ void as_atb(float (&acc)[R][4 * NC], const float* p, const float* b, int D, int ty, int tx) {
    static_assert(R == 2 || R == 4, "a thread's rows are one load");
    const int P = D + 4;
#pragma unroll 8
    for (int r = 0; r < AS_T; ++r) {
        float a[R];
        const float* row = p + r * (16 * R + 4) + R * ty;
        if (R == 2) { const float2 x = *reinterpret_cast<const float2*>(row); a[0] = x.x; a[1] = x.y; }
        else { const float4 x = ld4(row); a[0] = x.x; a[1] = x.y; a[R - 2] = x.z; a[R - 1] = x.w; }
#pragma unroll
        for (int n = 0; n < NC; ++n) {
            const int c = min(64 * n + 4 * tx, D - 4);  // what lies beyond D is not used, and a branch would keep the loads of several rows apart
            F4 y;
            y.f = ld4(b + r * P + c);
#pragma unroll
            for (int i = 0; i < R; ++i) {
                const unsigned long long w = twice(a[i]);
                fma2_to(acc[i][4 * n], acc[i][4 * n + 1], w, y.d[0]);
                fma2_to(acc[i][4 * n + 2], acc[i][4 * n + 3], w, y.d[1]);
            }
        }
    }
}
__device__ __forceinline__ float as_row(float v, bool is_max) {  // over the 16 threads of a row
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) { const float w = __shfl_xor_sync(0xffffffffu, v, o); v = is_max ? fmaxf(v, w) : v + w; }
    return v;
}

}  // namespace gcb
