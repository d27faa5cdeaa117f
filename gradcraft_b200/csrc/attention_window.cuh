// What the kernels of attention under a visibility rule share: the rule, the operands, the bias by distance.
//   key j is seen by query i   <=>   j <= i and (W == 0 or i - j < W or j < S)
//   score(i, j) = scale q_i . k_j + bias[h, n],  n = the last bucket whose first distance is at most i - j
#pragma once
#include "common.cuh"

namespace gcb {

constexpr int AW_MAX_BUCKETS = 64, AW_MAX_SINKS = 64;

struct WindowRule {
    int W, S, buckets;
    const float* bias;            // [H][buckets], or NULL
    int starts[AW_MAX_BUCKETS];   // first distance of every bucket, ascending from 0
    __host__ __device__ bool sees(int i, int j) const { return j <= i && (W == 0 || i - j < W || j < S); }
    // first key a query sees through the window
    __host__ __device__ int window_first(int i) const { return W > 0 && i >= W ? i - W + 1 : 0; }
    __device__ __forceinline__ int bucket(int d) const {
        int n = 0;
#pragma unroll
        for (int step = AW_MAX_BUCKETS / 2; step > 0; step >>= 1)
            if (n + step < buckets && starts[n + step] <= d) n += step;
        return n;
    }
};

__device__ __forceinline__ int clamp_distance(int d, int len) { return max(0, min(d, len - 1)); }

// Checks and copies the rule of an entry point.
inline int make_rule(WindowRule& r, const char* who, int64_t window, int64_t sinks, const float* bias, int64_t buckets, const int64_t* starts) {
    GCB_REQUIRE(window >= 0, "%s: the window must be a number of positions, or 0 for all of them", who);
    GCB_REQUIRE(sinks >= 0 && sinks <= AW_MAX_SINKS, "%s: at most %d first positions stay visible", who, AW_MAX_SINKS);
    constexpr int64_t most = 1 << 30;
    r.W = (int)(window < most ? window : 0);  // no distance is that large
    r.S = r.W ? (int)sinks : 0;
    r.bias = bias;
    r.buckets = 0;
    if (bias == nullptr) return GCB_OK;
    GCB_REQUIRE(buckets >= 1 && buckets <= AW_MAX_BUCKETS && starts && starts[0] == 0, "%s: a bias takes 1 to %d buckets, the first of which starts at distance 0", who, AW_MAX_BUCKETS);
    r.buckets = (int)buckets;
    for (int64_t n = 0; n < buckets; ++n) {
        GCB_REQUIRE(n == 0 || starts[n] >= starts[n - 1], "%s: bucket %lld starts before the one in front of it", who, (long long)n);
        r.starts[n] = (int)(starts[n] < most ? starts[n] : most);
    }
    return GCB_OK;
}

struct WindowAttn {
    const float *q, *k, *v, *g, *o;
    float *out, *dq, *dk, *dv, *row_max, *row_inv;  // statistics: per query the maximum score and 1 / sum (infinity and 0 where nothing is seen: P is then 0 whatever a score is), Tp a head
    float *dbias_part, *far_part;                   // backward: partial sums, see the kernels that fill them
    float* delta;                                   // backward: dO . O per query, Tp a head, written with dQ
    const float* tab;                               // [H][tab_len]: bias by distance, the last one for all distances beyond; NULL: no bias
    int64_t q_ld, q_so, q_si, k_ld, k_so, k_si, v_ld, v_so, v_si, g_ld, g_so, g_si, o_ld, o_so, o_si, d_ld, d_so, d_si, Tp;
    int T, D, H, tiles, tab_len, far_chunks, far_rows, far_inside;
    float scale;
    WindowRule rule;
};

// The kernels of attention_window_tc.cu.
bool window_tc_takes(gcb_ctx* ctx, int64_t B, const WindowAttn& a);
int window_tc_fwd(gcb_ctx* ctx, int64_t B, const WindowAttn& a);
int window_tc_bwd(gcb_ctx* ctx, int64_t B, const WindowAttn& a);
constexpr int AW_TC_TILE = 128;  // queries of a tile there

}  // namespace gcb
