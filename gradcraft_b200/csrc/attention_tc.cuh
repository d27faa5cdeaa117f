// What the tensor-core attention kernels share: items and their order, tiles in shared and tensor memory, the products of a 128-row side with 64-row
// blocks of the other in split-fp32 arithmetic, and the tensor maps of their operands.
#pragma once
#include <algorithm>

#include "gemm.cuh"
#include "tcgen05.cuh"

namespace gcb {

constexpr int AT_ROWS = 128, AT_KEYS = 64;  // rows of tensor memory; the other side's block
constexpr int AT_FWD_THREADS = 768, AT_BWD_THREADS = 896;  // six / seven groups of four warps

struct AttnItem {
    int b, h, unit;
    bool skip;
};
// Items run from the heaviest unit of a group of heads to its lightest, dealt out in snake order (left to right, right to left), so
// that CTAs end together and a group's k and v stay in the L2 cache.  `ascending`: unit 0 is the heaviest (backward).
template <class Params>
__device__ __forceinline__ AttnItem attn_item(const Params& p, int64_t w, bool ascending) {
    AttnItem it;
    const int64_t G = gridDim.x, round = w / G, c = w - round * G, x = round * G + ((round & 1) ? G - 1 - c : c);
    it.skip = x >= p.items;
    const int64_t per_group = (int64_t)p.group * p.units;
    const int g = (int)(x / per_group), r = (int)(x - g * per_group), gh = min(p.group, p.heads - g * p.group);
    const int cls = gh > 0 ? r / gh : 0, head = g * p.group + (gh > 0 ? r - cls * gh : 0);
    it.unit = ascending ? cls : p.units - 1 - cls;
    it.b = head / p.H;
    it.h = head - it.b * p.H;
    return it;
}

template <int DP>
struct AttnSmem {
    static constexpr int TWIN = AT_ROWS * DP * 4;          // BF16 companions of a 128-row operand
    static constexpr int RAW = AT_KEYS * DP * 4;           // a landed 64-row block; its companions take as much again
    static constexpr int BLOCK = 2 * RAW;
    static constexpr int BLOCKS_OFF = 2 * TWIN;            // four blocks: forward k0 k1 v0 v1, backward q, dO (K-major), dO, q (MN-major)
    static constexpr int STAGE_OFF = BLOCKS_OFF + 4 * BLOCK;  // backward: 4 KB a warp on the way out; forward: words two threads of a row exchange
    static constexpr int BAR_OFF = STAGE_OFF + 8 * 4096;
    static constexpr int STATS_OFF = BAR_OFF + 256;        // backward: row maximum, 1 / sum and dO . O of a block's queries, two blocks
    static constexpr int TOTAL = STATS_OFF + 2 * 3 * AT_KEYS * 4 + 1024;
    static_assert(TOTAL <= 232448, "shared memory");
};

// D[128 x 64] = A[128 x DP] B[64 x DP]^T.  A: t in tensor memory, companions in shared memory; B: K-major block and companions (addresses in 16-byte units).
template <int DP>
__device__ __forceinline__ void issue_scores(uint32_t d, uint32_t a_t, uint32_t a_twin, uint32_t b_raw) {
    constexpr uint32_t idesc = (1u << 4) | (2u << 7) | (2u << 10) | ((uint32_t)(AT_KEYS >> 3) << 17) | ((uint32_t)(AT_ROWS >> 4) << 24);
    constexpr uint32_t idesc_bf = (1u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(AT_KEYS >> 3) << 17) | ((uint32_t)(AT_ROWS >> 4) << 24);
    constexpr uint32_t twin = AT_KEYS * DP * 4 / 16;
    asm volatile("" : "+r"(a_t), "+r"(a_twin), "+r"(b_raw));  // descriptors are made here, one addition each: kept across the loop they are spilled
#pragma unroll
    for (int kb = 0; kb < DP / 16; ++kb) {
        const uint32_t b = b_raw + kb * 256, a = a_twin + kb * 512;
        umma_tf32_ts(d, a_t + 16 * kb, tile_desc<16, 512, 4>(b), idesc, kb > 0 ? 1u : 0u);
        umma_tf32_ts(d, a_t + 16 * kb + 8, tile_desc<16, 512, 4>(b + 2), idesc, 1u);
        umma_bf16(d, tile_desc<128, 256, 0>(a + 256), tile_desc<128, 256, 0>(b + twin), idesc_bf, 1u);
        umma_bf16(d, tile_desc<128, 256, 0>(a), tile_desc<128, 256, 0>(b + twin + 128), idesc_bf, 1u);
    }
}
// D[128 x DP] (+)= A[128 x 64] B[64 x DP].  A: its three parts in tensor memory, the companions of 16 columns STEP apart; B: MN-major block and K-major companions.
template <int DP, int STEP = 8>
__device__ __forceinline__ void issue_values(uint32_t d, uint32_t a_t, uint32_t a_big, uint32_t a_sml, uint32_t b_raw, bool accumulate) {
    constexpr uint32_t idesc = (1u << 4) | (2u << 7) | (2u << 10) | (1u << 16) | ((uint32_t)(DP >> 3) << 17) | ((uint32_t)(AT_ROWS >> 4) << 24);
    constexpr uint32_t idesc_bf = (1u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(DP >> 3) << 17) | ((uint32_t)(AT_ROWS >> 4) << 24);
    constexpr uint32_t twin = AT_KEYS * DP * 4 / 16;
    asm volatile("" : "+r"(a_t), "+r"(a_big), "+r"(a_sml), "+r"(b_raw));
#pragma unroll
    for (int kb = 0; kb < AT_KEYS / 16; ++kb) {
        const uint32_t b = b_raw + kb * 128, tw = b_raw + twin + kb * DP * 4;
        umma_tf32_ts(d, a_t + 16 * kb, tile_desc<8192, 512, 1>(b), idesc, (kb > 0 || accumulate) ? 1u : 0u);
        umma_tf32_ts(d, a_t + 16 * kb + 8, tile_desc<8192, 512, 1>(b + 64), idesc, 1u);
        umma_bf16_ts(d, a_sml + STEP * kb, tile_desc<128, 256, 0>(tw), idesc_bf, 1u);
        umma_bf16_ts(d, a_big + STEP * kb, tile_desc<128, 256, 0>(tw + DP * 2), idesc_bf, 1u);
    }
}
// Copies of a 64-row block starting at row r0: 16-wide slabs of 64-byte rows (K-major), or 32-wide chunks (MN-major).
template <int DP>
__device__ __forceinline__ void load_k_major(uint32_t dst, const CUtensorMap* map, uint32_t bar, int r0, int h, int b) {
    mbar_expect_tx(bar, AttnSmem<DP>::RAW);
#pragma unroll
    for (int kb = 0; kb < DP / 16; ++kb) tma_load_4d(dst + kb * 4096, map, bar, 16 * kb, r0, h, b);
}
template <int DP>
__device__ __forceinline__ void load_mn_major(uint32_t dst, const CUtensorMap* map, uint32_t bar, int r0, int h, int b) {
    mbar_expect_tx(bar, AttnSmem<DP>::RAW);
#pragma unroll
    for (int c = 0; c < DP / 32; ++c) tma_load_4d(dst + c * 8192, map, bar, 32 * c, r0, h, b);
}
template <int DP>
__device__ __forceinline__ void split_k_major(uint8_t* raw, int t) {  // a thread: one half row (8 columns) of every slab, as in split_hybrid; all loads first
    const int q = t >> 3, h = q & 1, row = (q >> 1) * 8 + (t & 7), sw = (row >> 1) & 3;
    float4 x[DP / 8];
#pragma unroll
    for (int kb = 0; kb < DP / 16; ++kb)
#pragma unroll
        for (int e = 0; e < 2; ++e) x[2 * kb + e] = *reinterpret_cast<const float4*>(raw + kb * 4096 + row * 64 + (((2 * h + e) ^ sw) << 4));
    uint8_t* big = raw + AttnSmem<DP>::RAW + (row >> 3) * 256 + h * 128 + (row & 7) * 16;
#pragma unroll
    for (int kb = 0; kb < DP / 16; ++kb) {
        const float4 a = x[2 * kb], b = x[2 * kb + 1];
        *reinterpret_cast<uint4*>(big + kb * 4096) = make_uint4(pack_bf16(a.x, a.y), pack_bf16(a.z, a.w), pack_bf16(b.x, b.y), pack_bf16(b.z, b.w));
        *reinterpret_cast<uint4*>(big + kb * 4096 + 2048) = make_uint4(pack_bf16(a.x - trunc_tf32(a.x), a.y - trunc_tf32(a.y)), pack_bf16(a.z - trunc_tf32(a.z), a.w - trunc_tf32(a.w)),
                                                                       pack_bf16(b.x - trunc_tf32(b.x), b.y - trunc_tf32(b.y)), pack_bf16(b.z - trunc_tf32(b.z), b.w - trunc_tf32(b.w)));
    }
}
template <int DP>
__device__ __forceinline__ void split_mn_major(const uint8_t* raw, uint8_t* twin, int t) {  // a thread: one column, 16 rows at a time
    const int n = t % DP, j = n & 31;
#pragma unroll
    for (int kb = t / DP; kb < AT_KEYS / 16; kb += 128 / DP) {
        const uint8_t* box = raw + (n >> 5) * 8192 + kb * 2048;
        float x[16];
#pragma unroll
        for (int k = 0; k < 16; ++k) x[k] = *reinterpret_cast<const float*>(box + k * 128 + ((((j >> 3) ^ (k & 3)) << 5) | ((j & 7) << 2)));
        uint8_t* big = twin + kb * DP * 64 + (n >> 3) * 256 + (n & 7) * 16;
#pragma unroll
        for (int kc = 0; kc < 2; ++kc) {
            const float* y = x + 8 * kc;
            *reinterpret_cast<uint4*>(big + kc * 128) = make_uint4(pack_bf16(y[0], y[1]), pack_bf16(y[2], y[3]), pack_bf16(y[4], y[5]), pack_bf16(y[6], y[7]));
            float s[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) s[e] = y[e] - trunc_tf32(y[e]);
            *reinterpret_cast<uint4*>(big + DP * 32 + kc * 128) = make_uint4(pack_bf16(s[0], s[1]), pack_bf16(s[2], s[3]), pack_bf16(s[4], s[5]), pack_bf16(s[6], s[7]));
        }
    }
}
// KBS 16-column slabs of this thread's row of a 128-row A operand: from global memory, then t to tensor memory and the companions to shared memory.
template <int KBS>
__device__ __forceinline__ void load_row(float (&x)[16 * KBS], const float* src, bool live, int cols) {
#pragma unroll
    for (int e = 0; e < 4 * KBS; ++e) {
        const float4 f = live && 4 * e < cols ? ld4(src + 4 * e) : make_float4(0.f, 0.f, 0.f, 0.f);
        x[4 * e] = f.x; x[4 * e + 1] = f.y; x[4 * e + 2] = f.z; x[4 * e + 3] = f.w;
    }
}
template <int KBS>
__device__ __forceinline__ void place_row(const float (&row_x)[16 * KBS], uint32_t t_addr, uint8_t* twin, int row) {
#pragma unroll
    for (int kb = 0; kb < KBS; ++kb) {
        const float* x = row_x + 16 * kb;
        uint32_t t[16];
        float s[16];
#pragma unroll
        for (int k = 0; k < 16; ++k) { t[k] = __float_as_uint(x[k]) & 0xffffe000u; s[k] = x[k] - __uint_as_float(t[k]); }
        tmem_st16(t_addr + 16 * kb, t);
        uint8_t* big = twin + kb * 8192 + (row >> 3) * 256 + (row & 7) * 16;
#pragma unroll
        for (int kc = 0; kc < 2; ++kc) {
            const float *y = x + 8 * kc, *z = s + 8 * kc;
            *reinterpret_cast<uint4*>(big + kc * 128) = make_uint4(pack_bf16(y[0], y[1]), pack_bf16(y[2], y[3]), pack_bf16(y[4], y[5]), pack_bf16(y[6], y[7]));
            *reinterpret_cast<uint4*>(big + 4096 + kc * 128) = make_uint4(pack_bf16(z[0], z[1]), pack_bf16(z[2], z[3]), pack_bf16(z[4], z[5]), pack_bf16(z[6], z[7]));
        }
    }
}
__device__ __forceinline__ void place_parts16(const float* x, uint32_t t_addr, uint32_t big, uint32_t sml) {  // 16 columns of an A operand in tensor memory
    uint32_t t[16], b[8], s[8];
#pragma unroll
    for (int k = 0; k < 16; ++k) t[k] = __float_as_uint(x[k]) & 0xffffe000u;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        b[i] = pack_bf16(x[2 * i], x[2 * i + 1]);
        s[i] = pack_bf16(x[2 * i] - __uint_as_float(t[2 * i]), x[2 * i + 1] - __uint_as_float(t[2 * i + 1]));
    }
    tmem_st16(t_addr, t);
    tmem_st8(big, b);
    tmem_st8(sml, s);
}
__device__ __forceinline__ void place_parts(const float (&x)[32], uint32_t t_addr, uint32_t big, uint32_t sml) {
    place_parts16(x, t_addr, big, sml);
    place_parts16(x + 16, t_addr + 16, big + 8, sml + 8);
}
__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ void tmem_stores_done() {
    asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
}
__device__ __forceinline__ void after_sync() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ bool warp_wait(uint32_t bar, uint32_t parity, int* status, int where) { return __all_sync(0xffffffffu, mbar_wait(bar, parity, status, where)) != 0; }

template <int R>
__device__ __forceinline__ void regs_give() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(R)); }
template <int R>
__device__ __forceinline__ void regs_take() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(R)); }
__device__ __forceinline__ void pair_sync(int id) { asm volatile("bar.sync %0, 256;" ::"r"(id) : "memory"); }
__device__ __forceinline__ bool pair_any(int id, bool x) {  // barrier of the 256 threads of a query tile, with the or of their x
    uint32_t r;
    asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %1, 0;\n\tbarrier.cta.red.or.pred q, %2, 256, p;\n\tselp.b32 %0, 1, 0, q;\n\t}" : "=r"(r) : "r"((uint32_t)x), "r"(id) : "memory");
    return r != 0;
}
__device__ __forceinline__ float max32(const float (&v)[32]) {
    float m[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) m[e] = v[e];
#pragma unroll
    for (int e = 4; e < 32; ++e) m[e & 3] = fmaxf(m[e & 3], v[e]);
    return fmaxf(fmaxf(m[0], m[1]), fmaxf(m[2], m[3]));
}

// Tensor memory, shared by both kernels: all 512 columns, taken by warp 1, given back at the end.
__device__ __forceinline__ uint32_t tmem_take(uint32_t slot, volatile uint32_t* slot_gen, int warp) {
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(slot), "r"(512u) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    after_sync();
    return *slot_gen;
}
__device__ __forceinline__ void tmem_give(uint32_t tmem, int warp) {
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    if (warp == 1) {
        after_sync();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
    }
}

// ---- host side ----------------------------------------------------------------------------------------------------------------
// (column, row, head, sequence) view of one operand in boxes of `cols` x 64.
static bool encode_rows(TmaEncodeFn enc, CUtensorMap* map, const float* ptr, int64_t cols, int64_t T, int64_t ld, int64_t si, int64_t so, int64_t H, int64_t B, int box_cols, int box_rows, CUtensorMapSwizzle swizzle) {
    const cuuint64_t row_bytes = (cuuint64_t)ld * 4;
    cuuint64_t dims[4] = {(cuuint64_t)cols, (cuuint64_t)T, (cuuint64_t)H, (cuuint64_t)B};
    cuuint64_t strides[3] = {row_bytes, H > 1 ? (cuuint64_t)si * 4 : row_bytes * (cuuint64_t)T, B > 1 ? (cuuint64_t)so * 4 : row_bytes * (cuuint64_t)T};
    cuuint32_t box[4] = {(cuuint32_t)box_cols, (cuuint32_t)box_rows, 1u, 1u}, estr[4] = {1, 1, 1, 1};
    return enc(map, CU_TENSOR_MAP_DATA_TYPE_FLOAT32, 4, const_cast<float*>(ptr), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle, CU_TENSOR_MAP_L2_PROMOTION_L2_128B,
               CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}
static bool rows_ok(const float* p, int64_t ld, int64_t so, int64_t si, int64_t B, int64_t H) {
    constexpr int64_t reach = int64_t(1) << 38;  // a tensor map's strides stay below 2^40 bytes
    return p && aligned16(p) && ld > 0 && ld < reach && ld % 4 == 0 && (H == 1 || (si > 0 && si < reach && si % 4 == 0)) && (B == 1 || (so > 0 && so < reach && so % 4 == 0));
}
static size_t span_bytes(int64_t B, int64_t H, int64_t T, int64_t D, int64_t ld, int64_t so, int64_t si) { return sizeof(float) * (size_t)((B - 1) * so + (H - 1) * si + (T - 1) * ld + D); }
static int64_t padded(int64_t T) { return (T + AT_ROWS - 1) / AT_ROWS * AT_ROWS; }

// Items and grid of `tiles_per_unit` 128-row tiles a CTA.
template <class Params>
static void plan(Params& p, int64_t B, int64_t H, int64_t T, int tiles_per_unit) {
    p.H = (int)H; p.heads = (int)(B * H); p.Tp = padded(T);
    p.tiles_per_unit = tiles_per_unit;
    p.units = (int)((p.Tp / AT_ROWS + tiles_per_unit - 1) / tiles_per_unit);
    p.items = (int64_t)p.units * p.heads;
    const int64_t grid = std::min<int64_t>(p.items, kSMs);
    p.loop_end = (p.items + grid - 1) / grid * grid;
    p.group = (int)std::max<int64_t>(1, std::min<int64_t>(p.heads, 2 * grid / p.units));
}

}  // namespace gcb
