// Dropout whose mask follows from a seed and a counter and is never stored: the backward pass, or a repeat of the forward, draws it again.
//
// Numbers come from Philox4x32-10 (Salmon, Moraes, Dror, Shaw: Parallel random numbers: as easy as 1, 2, 3; SC 2011): a block of four
// words from a 128-bit counter and a 64-bit key.  Element i takes word i % 4 of the counter offset + i / 4 under the key `seed`, and is dropped when
// that word is below p 2^32; what is kept is divided by 1 - p.  So the mask hangs on nothing but (seed, offset, i): not on the grid, the
// alignment or the width of the accesses.
// Bound by memory: 8 bytes an element, 12 with a residual (or a gradient that is added to).  Ten rounds are 20 wide multiplications for
// four elements, about half of what the integer units could do meanwhile.  32768 x 1024 elements, forward with a residual and backward (671 MB): 110 us,
// 6.1 TB/s.
#include "common.cuh"

namespace gcb {

__device__ __forceinline__ uint4 philox(uint64_t counter, uint64_t key) {
    uint32_t c0 = (uint32_t)counter, c1 = (uint32_t)(counter >> 32), c2 = 0, c3 = 0, k0 = (uint32_t)key, k1 = (uint32_t)(key >> 32);
#pragma unroll
    for (int r = 0; r < 10; ++r) {
        const uint64_t a = (uint64_t)c0 * 0xD2511F53u, b = (uint64_t)c2 * 0xCD9E8D57u;
        c0 = (uint32_t)(b >> 32) ^ c1 ^ k0;
        c1 = (uint32_t)b;
        c2 = (uint32_t)(a >> 32) ^ c3 ^ k1;
        c3 = (uint32_t)a;
        k0 += 0x9E3779B9u;
        k1 += 0xBB67AE85u;
    }
    return make_uint4(c0, c1, c2, c3);
}

struct DropoutArgs {
    float* out;
    const float *x, *add;  // add: what the result is added to, or NULL
    int64_t n;
    uint64_t seed, offset;
    uint32_t below;  // words below this are dropped
    bool all;        // p == 1
    float scale;
};

// A thread takes U blocks of four elements, all loads first.  out may be x or add.
template <int U, bool VEC>
__global__ void __launch_bounds__(256) dropout_kernel(const DropoutArgs p) {
    pdl_trigger();
    pdl_wait();
    const int64_t b0 = (int64_t)blockIdx.x * (256 * U) + threadIdx.x;
    float x[U][4], r[U][4];
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const int64_t i = (b0 + 256 * u) * 4;
        if (VEC && i + 4 <= p.n) {
            const float4 a = ld4_stream(p.x + i), b = p.add ? ld4_stream(p.add + i) : make_float4(0.f, 0.f, 0.f, 0.f);
            x[u][0] = a.x; x[u][1] = a.y; x[u][2] = a.z; x[u][3] = a.w;
            r[u][0] = b.x; r[u][1] = b.y; r[u][2] = b.z; r[u][3] = b.w;
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                x[u][e] = i + e < p.n ? p.x[i + e] : 0.0f;
                r[u][e] = p.add && i + e < p.n ? p.add[i + e] : 0.0f;
            }
        }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const int64_t block = b0 + 256 * u, i = block * 4;
        if (i >= p.n) break;
        const uint4 w4 = philox(p.offset + (uint64_t)block, p.seed);
        const uint32_t w[4] = {w4.x, w4.y, w4.z, w4.w};
        float y[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) y[e] = w[e] < p.below || p.all ? r[u][e] : fmaf(x[u][e], p.scale, r[u][e]);  // a dropped value is not looked at: it may be anything
        if (VEC && i + 4 <= p.n) {
            st4_stream(p.out + i, make_float4(y[0], y[1], y[2], y[3]));
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) if (i + e < p.n) p.out[i + e] = y[e];
        }
    }
}

static int dropout(gcb_ctx* ctx, const char* who, float* out, const float* x, const float* add, int64_t n, float p, int64_t seed, int64_t offset) {
    GCB_REQUIRE(ctx && n >= 0 && n < (int64_t(1) << 40), "%s: bad arguments", who);
    GCB_REQUIRE(p >= 0.0f && p <= 1.0f, "%s: the probability must lie between 0 and 1", who);
    if (n == 0) return GCB_OK;
    GCB_REQUIRE(out && x, "%s: NULL pointer", who);
    cudaSetDevice(ctx->device);
    DropoutArgs a = {};
    a.out = out; a.x = x; a.add = add; a.n = n;
    a.seed = (uint64_t)seed; a.offset = (uint64_t)offset;
    a.all = p == 1.0f;
    a.below = a.all ? 0u : (uint32_t)((double)p * 4294967296.0);
    a.scale = a.all ? 0.0f : (float)(1.0 / (1.0 - (double)p));
    const bool vec = aligned16(out) && aligned16(x) && aligned16(add);
    const int64_t blocks = (n + 3) / 4;
    auto run = [&](auto kernel, int u) { return launch_next(ctx->stream, dim3((unsigned)((blocks + 256 * u - 1) / (256 * u))), 256, 0, kernel, a); };
    if (blocks <= (int64_t)kSMs * 1024) GCB_CHECK_CUDA(vec ? run(dropout_kernel<1, true>, 1) : run(dropout_kernel<1, false>, 1));
    else GCB_CHECK_CUDA(vec ? run(dropout_kernel<4, true>, 4) : run(dropout_kernel<4, false>, 4));
    note_write(ctx, out, sizeof(float) * (size_t)n);
    return after_launch(ctx, "dropout");
}

}  // namespace gcb

using namespace gcb;

extern "C" {

int gcb_dropout_fwd_f32(gcb_ctx* ctx, float* out, const float* x, const float* residual, int64_t n, float p, int64_t seed, int64_t offset) { return dropout(ctx, "gcb_dropout_fwd_f32", out, x, residual, n, p, seed, offset); }
int gcb_dropout_bwd_f32(gcb_ctx* ctx, float* dx, const float* dy, int64_t n, float p, int64_t seed, int64_t offset, int accumulate) {
    return dropout(ctx, "gcb_dropout_bwd_f32", dx, dy, accumulate ? dx : nullptr, n, p, seed, offset);
}

}  // extern "C"
