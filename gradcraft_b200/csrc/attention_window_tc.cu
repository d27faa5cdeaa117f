// Attention under a visibility rule (attention_window.cuh) on tcgen05 / TMEM, in the split-fp32 arithmetic of the GEMMs, for heads of up to 64
// columns: the forward, dK and dV of 128 keys, dQ and the bias gradient of 128 queries, one kernel each.  Nothing T x T goes through
// memory, and blocks that the rule hides as a whole are not visited, so that a sequence costs T (window + sinks).
// Reference counterpart: the causal form alone (frontend/tensor_other.hpp:53-93).
//
// Tiles, roles and the order of products are those of attention.cu, with these differences:
//   - a unit's key blocks are the blocks of the first S keys and those of its window; the two query tiles of a forward CTA share the union;
//   - scores are masked only in blocks that a border of the rule passes through, a test per warp;
//   - a bias is read from a table by distance, 191 entries a block through shared memory, beyond its last distance from a register;
//   - a query may see nothing of a block that its tile visits: a maximum of -inf stands for "nothing yet" until the first key;
//   - dQ is a kernel of its own that forms P and dS again (three products a block), because dS of a long sequence is too much memory: five
//     products and T^2 floats there, seven products here.
// The gradients of the first S keys from queries beyond the window are left to the FMA kernel of attention_window.cu: 128-key tiles would
// spend T / 64 blocks on a handful of keys.
// 1 x 16 heads of 8192 x 64, window 1024, four first positions: forward 252 us, dQ 261, dK and dV 346 (with a bias of 32 buckets 288, 342, 386); 16 x 16 heads of
// 1024, window 256: 212, 252, 266; each after a flush of the L2 cache.  The tensor cores are at work for 31, 42 and 44 % of a call at 4096 positions, and 45, 52 and 48 % of the issue
// slots go to what turns scores into probabilities and rows into companions; what is left is the way of a block from role to role, a barrier each time.
// Every wait is bounded, as in the GEMM kernels.
#include "attention_tc.cuh"
#include "attention_window.cuh"

namespace gcb {

constexpr int WT_FLUSH = 4;                     // backward: blocks whose products are added up in tensor memory before the sum moves on
constexpr int WT_DIAG = AT_ROWS + AT_KEYS - 1;  // distances in a block of scores
constexpr int WT_TAB = 192;                     // their place in shared memory, in floats
constexpr float kLog2e = 1.4426950408889634f;

struct WindowTc {
    int64_t q_ld, q_so, q_si, k_ld, k_so, k_si, v_ld, v_so, v_si, g_ld, g_so, g_si, o_ld, o_so, o_si, d_ld, d_so, d_si;
    const float *q, *k, *v, *g, *o;
    float *out, *dq, *dk, *dv, *row_max, *row_inv, *delta, *dbias_part;
    float* moved;      // 64 KB a CTA, for what leaves tensor memory before an item's end
    const float* tab;  // [H][tab_len]: bias by distance, the last one for all distances beyond; NULL: no bias
    int tab_len;
    int64_t Tp;
    float scale;
    int T, D, H, heads, units, group, tiles_per_unit;
    int64_t items, loop_end;
    int* status;
    WindowRule rule;
};

// The key blocks that a 128-query tile from row r0 looks at: 0 .. sinks - 1, then first .. last.  None where r0 lies beyond the sequence.
struct TileKeys {
    int sinks, first, last;
    __device__ __forceinline__ TileKeys(const WindowTc& p, int r0) {
        const bool there = r0 < p.T;
        first = p.rule.window_first(r0) / AT_KEYS;
        last = there ? (min(p.T, r0 + AT_ROWS) - 1) / AT_KEYS : -1;
        sinks = there ? min((p.rule.S + AT_KEYS - 1) / AT_KEYS, first) : 0;
    }
    __device__ __forceinline__ int count() const { return last < 0 ? 0 : sinks + last - first + 1; }
    __device__ __forceinline__ int block(int j) const { return j < sinks ? j : first + j - sinks; }
    __device__ __forceinline__ bool has(int b) const { return b < sinks || (b >= first && b <= last); }
    __device__ __forceinline__ int begin() const { return sinks > 0 ? 0 : first; }
};
__device__ __forceinline__ bool all_any(bool x) {  // barrier of the 512 threads of the query warps, with the or of their x
    uint32_t r;
    asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %1, 0;\n\tbarrier.cta.red.or.pred q, 1, 512, p;\n\tselp.b32 %0, 1, 0, q;\n\t}" : "=r"(r) : "r"((uint32_t)x) : "memory");
    return r != 0;
}
// Keeps score e of a row (query i against key j0 + e) or hides it; `room` = i - j0.
__device__ __forceinline__ bool keeps(int e, int room, int window_from, int sinks_to) { return e <= room && (e >= window_from || e < sinks_to); }

// Blocks of the 64-row side: raw tiles from TMA, 32 columns of 64 rows a copy (rows of 128 bytes, 128-byte swizzle: K-major; in 32-byte units:
// MN-major), and BF16 companions, bf16(x) then bf16(x - t), as 8 x 8 core matrices in rows of DP / 8.  A core matrix holds 8 rows of 8 columns either
// way, so one set of companions serves a product over the columns (K-major: scores, dP) and one over the rows (MN-major: values).
template <int DP>
struct WinTile {
    static constexpr int RAW = AT_KEYS * DP * 4, TWIN = RAW, SMALL = RAW / 2, ROWS8 = DP * 16;
};
template <int DP>
__device__ __forceinline__ void win_load(uint32_t dst, const CUtensorMap* map, uint32_t bar, int r0, int h, int b) {
    mbar_expect_tx(bar, WinTile<DP>::RAW);
#pragma unroll
    for (int c = 0; c < DP / 32; ++c) tma_load_4d(dst + c * 8192, map, bar, 32 * c, r0, h, b);
}
// Companions of a raw tile by THREADS threads, a core-matrix row (8 columns) at a time, all loads first.
template <int DP, int THREADS, bool MN>
__device__ __forceinline__ void win_split(const uint8_t* raw, uint8_t* twin, int t) {
    constexpr int U = 8 * DP / THREADS;
    float4 x[U][2];
#pragma unroll
    for (int v = 0; v < U; ++v) {
        const int u = t + THREADS * v, r = u & 7, j = (u >> 3) % (DP / 8), row = u / DP * 8 + r;
        const uint8_t* at = raw + (j >> 2) * 8192 + row * 128;
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const int half = MN ? e ^ (r >> 2) : e;  // rows four apart have their unit in the same place: they take its halves in turn
            x[v][e] = *reinterpret_cast<const float4*>(at + (MN ? ((((j & 3) ^ (r & 3)) << 5) | (half << 4)) : (((2 * (j & 3) + e) ^ r) << 4)));
        }
    }
#pragma unroll
    for (int v = 0; v < U; ++v) {
        const int u = t + THREADS * v, r = u & 7, j = (u >> 3) % (DP / 8);
        const bool swap = MN && (r >> 2);
        const float4 a = swap ? x[v][1] : x[v][0], b = swap ? x[v][0] : x[v][1];
        uint8_t* at = twin + u / DP * WinTile<DP>::ROWS8 + j * 128 + r * 16;
        *reinterpret_cast<uint4*>(at) = make_uint4(pack_bf16(a.x, a.y), pack_bf16(a.z, a.w), pack_bf16(b.x, b.y), pack_bf16(b.z, b.w));
        *reinterpret_cast<uint4*>(at + WinTile<DP>::SMALL) = make_uint4(pack_bf16(a.x - trunc_tf32(a.x), a.y - trunc_tf32(a.y)), pack_bf16(a.z - trunc_tf32(a.z), a.w - trunc_tf32(a.w)),
                                                                        pack_bf16(b.x - trunc_tf32(b.x), b.y - trunc_tf32(b.y)), pack_bf16(b.z - trunc_tf32(b.z), b.w - trunc_tf32(b.w)));
    }
}
// Every addition of the tensor core cuts off up to 2^-23 of the sum that it adds to, always towards zero.  Both products therefore begin with those of the remainders, while
// the sum is still 2^-10 of what it will be.
// D[128 x 64] = A[128 x DP] B[64 x DP]^T.  A: t in tensor memory, companions in shared memory (place_row); B: K-major raw tile and companions (addresses in 16-byte units).
template <int DP>
__device__ __forceinline__ void win_scores(uint32_t d, uint32_t a_t, uint32_t a_twin, uint32_t b_raw, uint32_t b_twin) {
    constexpr uint32_t idesc = (1u << 4) | (2u << 7) | (2u << 10) | ((uint32_t)(AT_KEYS >> 3) << 17) | ((uint32_t)(AT_ROWS >> 4) << 24);
    constexpr uint32_t idesc_bf = (1u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(AT_KEYS >> 3) << 17) | ((uint32_t)(AT_ROWS >> 4) << 24);
    constexpr uint32_t small = WinTile<DP>::SMALL / 16;
    asm volatile("" : "+r"(a_t), "+r"(a_twin), "+r"(b_raw), "+r"(b_twin));  // descriptors are made here, one addition each: kept across the loop they are spilled
#pragma unroll
    for (int kb = 0; kb < DP / 16; ++kb) {
        const uint32_t tw = b_twin + kb * 16, a = a_twin + kb * 512;
        umma_bf16(d, tile_desc<128, 256, 0>(a + 256), tile_desc<128, WinTile<DP>::ROWS8, 0>(tw), idesc_bf, kb > 0 ? 1u : 0u);
        umma_bf16(d, tile_desc<128, 256, 0>(a), tile_desc<128, WinTile<DP>::ROWS8, 0>(tw + small), idesc_bf, 1u);
    }
#pragma unroll
    for (int kb = 0; kb < DP / 16; ++kb) {
        const uint32_t b = b_raw + (kb >> 1) * 512 + (kb & 1) * 4;
        umma_tf32_ts(d, a_t + 16 * kb, tile_desc<16, 1024, 2>(b), idesc, 1u);
        umma_tf32_ts(d, a_t + 16 * kb + 8, tile_desc<16, 1024, 2>(b + 2), idesc, 1u);
    }
}
// D[128 x DP] (+)= A[128 x 64] B[64 x DP].  A: its three parts in tensor memory, the companions of 16 columns STEP apart; B: MN-major raw tile and companions.
template <int DP, int STEP>
__device__ __forceinline__ void win_values(uint32_t d, uint32_t a_t, uint32_t a_big, uint32_t a_sml, uint32_t b_raw, uint32_t b_twin, bool accumulate) {
    constexpr uint32_t idesc = (1u << 4) | (2u << 7) | (2u << 10) | (1u << 16) | ((uint32_t)(DP >> 3) << 17) | ((uint32_t)(AT_ROWS >> 4) << 24);
    constexpr uint32_t idesc_bf = (1u << 4) | (1u << 7) | (1u << 10) | (1u << 16) | ((uint32_t)(DP >> 3) << 17) | ((uint32_t)(AT_ROWS >> 4) << 24);
    constexpr uint32_t small = WinTile<DP>::SMALL / 16;
    asm volatile("" : "+r"(a_t), "+r"(a_big), "+r"(a_sml), "+r"(b_raw), "+r"(b_twin));
#pragma unroll
    for (int kb = 0; kb < AT_KEYS / 16; ++kb) {
        const uint32_t tw = b_twin + kb * 2 * (WinTile<DP>::ROWS8 / 16);
        umma_bf16_ts(d, a_sml + STEP * kb, tile_desc<WinTile<DP>::ROWS8, 128, 0>(tw), idesc_bf, (kb > 0 || accumulate) ? 1u : 0u);
        umma_bf16_ts(d, a_big + STEP * kb, tile_desc<WinTile<DP>::ROWS8, 128, 0>(tw + small), idesc_bf, 1u);
    }
#pragma unroll
    for (int kb = 0; kb < AT_KEYS / 16; ++kb) {
        const uint32_t b = b_raw + kb * 128;
        umma_tf32_ts(d, a_t + 16 * kb, tile_desc<8192, 512, 1>(b), idesc, 1u);
        umma_tf32_ts(d, a_t + 16 * kb + 8, tile_desc<8192, 512, 1>(b + 64), idesc, 1u);
    }
}
// The 128 rows a CTA owns of an operand or of a result pass through shared memory, as TMA moves them: [32 columns][128 rows][128 bytes], 128-byte swizzle.
// (Threads that load and store the row they own, 16 bytes of 32 different lines an instruction, took 20 000 cycles an item where this takes 4000.)
// A loaded tile lies where its companions go: threads read their rows, wait for one another, and write the companions over it.
template <int DP>
__device__ __forceinline__ void own_load(uint32_t dst, const CUtensorMap* map, uint32_t bar, int r0, int h, int b) {
    mbar_expect_tx(bar, AT_ROWS * DP * 4);
#pragma unroll
    for (int c = 0; c < DP / 32; ++c)
#pragma unroll
        for (int x = 0; x < 2; ++x) tma_load_4d(dst + c * 16384 + x * 8192, map, bar, 32 * c, r0 + 64 * x, h, b);
}
template <int DP>
__device__ __forceinline__ void own_store(const CUtensorMap* map, uint32_t src, const WindowTc& p, int r0, int h, int b) {
#pragma unroll
    for (int c = 0; c < DP / 32; ++c)
#pragma unroll
        for (int x = 0; x < 2; ++x)
            if (32 * c < p.D && r0 + 64 * x < p.T) tma_store_4d(map, src + c * 16384 + x * 8192, 32 * c, r0 + 64 * x, h, b);
}
__device__ __forceinline__ float4* own_at(uint8_t* tile, int row, int col) { return reinterpret_cast<float4*>(tile + (col >> 5) * 16384 + row * 128 + ((((col & 31) >> 2) ^ (row & 7)) << 4)); }
template <int N>
__device__ __forceinline__ void own_read(float (&x)[N], uint8_t* tile, int row, int col) {
#pragma unroll
    for (int e = 0; e < N; e += 4) {
        const float4 f = *own_at(tile, row, col + e);
        x[e] = f.x; x[e + 1] = f.y; x[e + 2] = f.z; x[e + 3] = f.w;
    }
}
// Moves 16 columns of a sum from tensor memory to a CTA's place in `moved`, [which][column / 4][row][4]: moved = (there ? moved : 0) + sum.
// A sum over hundreds of instructions comes out too small (8192 keys in one sum: 6e-5 of the result); one of WT_FLUSH blocks, 64 instructions, by at most 8e-6 where all terms have
// one sign, and these are added here with rounding.  Every eight blocks instead: 2.5 % off the backward pass; every two: 5 % more.
__device__ __forceinline__ void move_sum(uint32_t taddr, float* moved, bool there) {
    uint32_t x[16];
    tmem_ld16(taddr, x);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        float* at = moved + e * 4 * AT_ROWS;
        const float4 o = there ? ld4(at) : make_float4(0.f, 0.f, 0.f, 0.f);
        st4(at, make_float4(o.x + __uint_as_float(x[4 * e]), o.y + __uint_as_float(x[4 * e + 1]), o.z + __uint_as_float(x[4 * e + 2]), o.w + __uint_as_float(x[4 * e + 3])));
    }
}
// 16 columns of a result on their way out: f times a sum in tensor memory and what has moved.
__device__ __forceinline__ void place_result(uint8_t* tile, int row, int col, uint32_t taddr, const float* moved, bool there, float f) {
    uint32_t x[16];
    tmem_ld16(taddr, x);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const float4 o = there ? ld4(moved + e * 4 * AT_ROWS) : make_float4(0.f, 0.f, 0.f, 0.f);
        *own_at(tile, row, col + 4 * e) = make_float4((o.x + __uint_as_float(x[4 * e])) * f, (o.y + __uint_as_float(x[4 * e + 1])) * f, (o.z + __uint_as_float(x[4 * e + 2])) * f, (o.w + __uint_as_float(x[4 * e + 3])) * f);
    }
}
__device__ __forceinline__ void tmem_read(uint32_t taddr, float (&x)[32]) { tmem_ld32(taddr, x); }
__device__ __forceinline__ void tmem_read(uint32_t taddr, float (&x)[16]) {
    uint32_t u[16];
    tmem_ld16(taddr, u);
#pragma unroll
    for (int e = 0; e < 16; ++e) x[e] = __uint_as_float(u[e]);
}
__device__ __forceinline__ float* moved_at(const WindowTc& p, int which, int col, int row) { return p.moved + ((int64_t)blockIdx.x * 2 + which) * 64 * AT_ROWS + (col * AT_ROWS + row * 4); }

__device__ __forceinline__ bool ready_wait(uint32_t bar, uint32_t parity, int* status, int where) { return __all_sync(0xffffffffu, mbar_test(bar, parity) || mbar_wait(bar, parity, status, where)) != 0; }
// The issuing thread's waits are mostly over before they begin, and it is the one that everybody waits for: a plain test first (dQ 264 -> 247 us, dK and dV 363 -> 345).
__device__ __forceinline__ bool issuer_wait(uint32_t bar, uint32_t parity, int* status, int where) { return mbar_test(bar, parity) || mbar_wait(bar, parity, status, where); }

// ---- forward ------------------------------------------------------------------------------------------------------------------
// Tensor memory of query tile q, from column 256 q: scores / t of P [0, 64), bf16(P) [64, 96), bf16(P - t) [96, 128), a block's share of O [128, 192), t of q [192, 256).
// O itself is added up by the threads, with rounding: dO . O has to agree with the dP of the backward pass, or gradients that are small differences of the two are wrong
// (2048 positions, window 1024, values whose common part is ten times as large as the rest: bias gradient off by 1e-2 of its largest with sums of eight blocks in tensor memory, 2e-4
// so, 3e-5 by the FMA kernels; dQ 1e-3, 2e-4, 8e-5).  A thread's sums lie in shared memory as far as there is room, 12 of 32 columns, and the others in L2, requested before the wait
// for the block: 214 us at 16 x 16 x 1024, window 256 (all of them in L2: 225; 20 in registers, 12 in shared memory: 262; sums of eight blocks in tensor memory: 206).
template <int DP, bool BIAS>
__global__ void __launch_bounds__(AT_FWD_THREADS, 1) window_attention_tc_fwd_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, const __grid_constant__ CUtensorMap map_q,
                                                                                    const __grid_constant__ CUtensorMap map_o, const __grid_constant__ WindowTc p) {
    using S = AttnSmem<DP>;
    extern __shared__ uint8_t smem_raw[];
    const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
    uint8_t* gen = smem_raw + (base - smem_u32(smem_raw));
    const uint32_t bars = base + S::BAR_OFF;
    auto full = [&](int b) { return bars + 8u * b; };        // blocks k0 k1 v0 v1: landed
    auto conv = [&](int b) { return bars + 8u * (4 + b); };  // companions written
    auto empty = [&](int b) { return bars + 8u * (8 + b); }; // products have read it
    auto s_full = [&](int q) { return bars + 8u * (12 + q); };
    auto p_ready = [&](int q) { return bars + 8u * (14 + q); };
    auto o_full = [&](int q) { return bars + 8u * (16 + q); };
    auto q_ready = [&](int q) { return bars + 8u * (18 + q); };
    auto own_full = [&](int q) { return bars + 8u * (20 + q); };
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        for (int b = 0; b < 4; ++b) { mbar_init(full(b), 1); mbar_init(conv(b), 4); mbar_init(empty(b), 1); }
        for (int q = 0; q < 2; ++q) { mbar_init(s_full(q), 1); mbar_init(p_ready(q), 8); mbar_init(o_full(q), 1); mbar_init(q_ready(q), 8); mbar_init(own_full(q), 1); }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    const uint32_t tmem = tmem_take(bars + 8u * 24, reinterpret_cast<volatile uint32_t*>(gen + S::BAR_OFF + 8 * 24), warp);
    pdl_trigger();
    pdl_wait();
    auto tile_row = [&](const AttnItem& it, int q) { return q < p.tiles_per_unit ? (it.unit * p.tiles_per_unit + q) * AT_ROWS : p.T; };
    // both tiles' blocks: those of tile 0 up to the end of tile 1's (the second tile's window begins before the first one's ends)
    struct Union {
        TileKeys a, b;
        int blocks;
        __device__ __forceinline__ Union(const TileKeys& x, const TileKeys& y) : a(x), b(y), blocks(x.sinks + max(x.last, y.last) - x.first + 1) {}
        __device__ __forceinline__ int block(int n) const { return a.block(n); }
    };
    auto slot = [&](int kind, uint32_t n) { return (int)(2 * kind + (n & 1u)); };  // kind 0: k, 1: v; n: running block number

    if (warp < 4) regs_give<40>();
    if (warp == 0) {
        if (lane == 0) {
            uint32_t n = 0;
            bool ok = true;
            for (int64_t w = blockIdx.x; w < p.loop_end && ok; w += gridDim.x) {
                const AttnItem it = attn_item(p, w, false);
                if (it.skip) continue;
                const Union u(TileKeys(p, tile_row(it, 0)), TileKeys(p, tile_row(it, 1)));
                for (int j = 0; j < u.blocks && ok; ++j, ++n) {
                    const uint32_t ph = ((n >> 1) & 1u) ^ 1u;
                    const int kb = slot(0, n), vb = slot(1, n), r0 = u.block(j) * AT_KEYS;
                    ok = mbar_wait(empty(kb), ph, p.status, 41);
                    if (!ok) break;
                    win_load<DP>(base + S::BLOCKS_OFF + kb * S::BLOCK, &map_k, full(kb), r0, it.h, it.b);
                    ok = mbar_wait(empty(vb), ph, p.status, 41);
                    if (!ok) break;
                    win_load<DP>(base + S::BLOCKS_OFF + vb * S::BLOCK, &map_v, full(vb), r0, it.h, it.b);
                }
            }
        }
    } else if (warp == 1) {
        if (elect_one()) {
            const uint32_t base16 = base >> 4;
            uint32_t n = 0, q_phase[2] = {0, 0}, p_phase[2] = {0, 0};
            bool ok = true;
            for (int64_t w = blockIdx.x; w < p.loop_end && ok; w += gridDim.x) {
                const AttnItem it = attn_item(p, w, false);
                if (it.skip) continue;
                const Union u(TileKeys(p, tile_row(it, 0)), TileKeys(p, tile_row(it, 1)));
                const int blocks = u.blocks;
                auto scores = [&](int q, int j) {
                    const uint32_t raw = base16 + S::BLOCKS_OFF / 16 + slot(0, n + j) * (S::BLOCK / 16);
                    win_scores<DP>(tmem + 256 * q, tmem + 256 * q + 192, base16 + q * (S::TWIN / 16), raw, raw + S::RAW / 16);
                    umma_commit(s_full(q));
                };
                auto k_landed = [&](int j) {
                    const bool r = issuer_wait(conv(slot(0, n + j)), ((n + j) >> 1) & 1u, p.status, 42);
                    after_sync();
                    return r;
                };
#pragma unroll
                for (int q = 0; q < 2; ++q)
                    if (ok && (q ? u.b : u.a).last >= 0) { ok = issuer_wait(q_ready(q), q_phase[q] & 1u, p.status, 43); ++q_phase[q]; }
                if (ok) ok = k_landed(0);
                if (!ok) break;
#pragma unroll
                for (int q = 0; q < 2; ++q)
                    if ((q ? u.b : u.a).has(u.block(0))) scores(q, 0);
                umma_commit(empty(slot(0, n)));
                for (int j = 0; j < blocks && ok; ++j) {
                    const int vb = slot(1, n + j), now = u.block(j), next = u.block(j + 1);
                    const uint32_t v_raw = base16 + S::BLOCKS_OFF / 16 + vb * (S::BLOCK / 16);
                    ok = issuer_wait(conv(vb), ((n + j) >> 1) & 1u, p.status, 44);
                    bool k_here = false;
#pragma unroll
                    for (int q = 0; q < 2; ++q) {
                        const TileKeys& t = q ? u.b : u.a;
                        if (ok && t.has(now)) {
                            ok = issuer_wait(p_ready(q), p_phase[q] & 1u, p.status, 45);
                            ++p_phase[q];
                            if (ok) {
                                after_sync();
                                const uint32_t t0 = tmem + 256 * q;
                                win_values<DP, 8>(t0 + 128, t0, t0 + 64, t0 + 96, v_raw, v_raw + S::RAW / 16, false);
                                if (now == t.last) umma_commit(o_full(q));
                            }
                        }
                        if (ok && j + 1 < blocks && t.has(next)) {
                            if (!k_here) { ok = k_landed(j + 1); k_here = true; }
                            if (ok) scores(q, j + 1);
                        }
                    }
                    if (!ok) break;
                    umma_commit(empty(vb));
                    if (j + 1 < blocks) umma_commit(empty(slot(0, n + j + 1)));
                }
                n += blocks;
            }
        }
    } else if (warp >= 4 && warp < 8) {
        regs_give<56>();
        const int t = threadIdx.x - 128;
        uint32_t n = 0;
        bool ok = true;
        for (int64_t w = blockIdx.x; w < p.loop_end && ok; w += gridDim.x) {
            const AttnItem it = attn_item(p, w, false);
            if (it.skip) continue;
            const Union u(TileKeys(p, tile_row(it, 0)), TileKeys(p, tile_row(it, 1)));
            for (int j = 0; j < u.blocks && ok; ++j, ++n) {
#pragma unroll
                for (int kind = 0; kind < 2; ++kind) {
                    const int b = slot(kind, n);
                    ok = ready_wait(full(b), (n >> 1) & 1u, p.status, 46);
                    if (!ok) break;
                    uint8_t* raw = gen + S::BLOCKS_OFF + b * S::BLOCK;
                    if (kind == 0) win_split<DP, 128, false>(raw, raw + S::RAW, t);
                    else win_split<DP, 128, true>(raw, raw + S::RAW, t);
                    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                    __syncwarp();
                    if (lane == 0) mbar_arrive(conv(b));
                }
            }
        }
    } else if (warp >= 8) {
        regs_take<96>();
        // two threads a query: each has 32 of a block's 64 keys, and half of the columns of q and O
        const int q = (warp - 8) >> 3, half = ((warp - 8) >> 2) & 1, row = 32 * (warp & 3) + lane, bar = 1 + q, at_tile = (threadIdx.x - 256) & 255;
        const uint32_t t0 = tmem + 256 * q + ((uint32_t)(32 * (warp & 3)) << 16);
        float* xch = reinterpret_cast<float*>(gen + S::STAGE_OFF) + q * 256;  // [half][row]
        float* tabs = reinterpret_cast<float*>(gen + S::STAGE_OFF + 2048) + q * 2 * WT_TAB;
        constexpr int OC = DP / 2, NEAR = 12;  // columns of a thread, and how many of their sums lie in shared memory
        float4* near_by = reinterpret_cast<float4*>(gen + S::STAGE_OFF + 2048 + 4 * WT_TAB * 4) + (threadIdx.x - 256);
        static_assert(2048 + 4 * WT_TAB * 4 + NEAR * 4 * 512 <= 8 * 4096, "shared memory");
        const float c = BIAS ? kLog2e : p.scale * kLog2e;  // scores, or scores before the scale, to log2 units
        uint32_t s_phase = 0, o_phase = 0, items = 0;
        bool ok = true;
        uint8_t* own = gen + q * S::TWIN;
        // this tile's rows of the item at w or the next one that has any
        auto fetch = [&](int64_t w) {
            for (; w < p.loop_end; w += gridDim.x) {
                const AttnItem it = attn_item(p, w, false);
                if (it.skip || tile_row(it, q) >= p.T) continue;
                own_load<DP>(base + q * S::TWIN, &map_q, own_full(q), tile_row(it, q), it.h, it.b);
                break;
            }
        };
        if (at_tile == 0) fetch(blockIdx.x);
        for (int64_t w = blockIdx.x; w < p.loop_end && ok; w += gridDim.x) {
            const AttnItem it = attn_item(p, w, false);
            if (it.skip) continue;
            const int r0 = tile_row(it, q);
            const TileKeys keys(p, r0);
            const int blocks = keys.count();
            if (!blocks) continue;
            const int r = r0 + row;
            const bool live = r < p.T;
            bool good = ready_wait(own_full(q), items & 1u, p.status, 49);  // every thread keeps step with the barriers below, whatever a wait says
            ++items;
            {
                float x[OC];
                own_read(x, own, row, half * OC);
                pair_sync(bar);
                place_row<DP / 32>(x, t0 + 192 + half * OC, gen + q * S::TWIN + half * (OC / 16) * 8192, row);
            }
            tmem_stores_done();
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            if (lane == 0) mbar_arrive(q_ready(q));
            // the bias of a block's 191 distances: requested a block ahead, in shared memory before the barrier of the block in front
            const float* tab = BIAS ? p.tab + (int64_t)it.h * p.tab_len : nullptr;
            const float beyond = BIAS ? __ldg(tab + p.tab_len - 1) : 0.0f;
            auto distance = [&](int b) { return r0 - (b + 1) * AT_KEYS + 1; };  // the smallest one of a block
            auto request = [&](int b) { return at_tile < WT_DIAG ? __ldg(tab + clamp_distance(distance(b) + at_tile, p.tab_len)) : 0.0f; };
            if (BIAS) {
                if (at_tile < WT_DIAG) tabs[at_tile] = request(keys.begin());
                pair_sync(bar);
            }
            float* moved = moved_at(p, q, half * OC, row);
            float m = -INFINITY, sum = 0.0f, m_out = -INFINITY;  // m: the maximum the probabilities are relative to; m_out: the one the sums are
            auto sums = [&](int e) { return e < NEAR / 4 ? near_by[512 * e] : __ldcg(reinterpret_cast<const float4*>(moved + e * 4 * AT_ROWS)); };
            for (int j = 0; j < blocks; ++j) {
                const int b = keys.block(j);
                float ahead = 0.0f;
                if (BIAS && j + 1 < blocks) ahead = request(keys.block(j + 1));
                float4 was[OC / 4];
#pragma unroll
                for (int e = NEAR / 4; e < OC / 4; ++e) was[e] = j > 1 ? sums(e) : make_float4(0.f, 0.f, 0.f, 0.f);
                good = good && ready_wait(s_full(q), s_phase & 1u, p.status, 47);
                ++s_phase;
                after_sync();
                if (j > 0) {  // the products of the block before came before these scores
                    const float f = m_out == m ? 1.0f : ex2((m_out - m) * c);
                    float x[OC];
                    tmem_read(t0 + 128 + half * OC, x);
#pragma unroll
                    for (int e = 0; e < OC / 4; ++e) {
                        if (e < NEAR / 4) was[e] = j > 1 ? sums(e) : make_float4(0.f, 0.f, 0.f, 0.f);
                        const float4 now = make_float4(fmaf(was[e].x, f, x[4 * e]), fmaf(was[e].y, f, x[4 * e + 1]), fmaf(was[e].z, f, x[4 * e + 2]), fmaf(was[e].w, f, x[4 * e + 3]));
                        if (e < NEAR / 4) near_by[512 * e] = now;
                        else __stcg(reinterpret_cast<float4*>(moved + e * 4 * AT_ROWS), now);
                    }
                    m_out = m;
                }
                float v[32];
                tmem_ld32(t0 + 32 * half, v);
                const int j0 = b * AT_KEYS + 32 * half, room = r - j0;
                if (BIAS) {
                    if (distance(b) >= p.tab_len - 1) {
#pragma unroll
                        for (int e = 0; e < 32; ++e) v[e] = fmaf(v[e], p.scale, beyond);
                    } else {
                        const float* mine = tabs + (j & 1) * WT_TAB + row - 32 * half + AT_KEYS - 1;
#pragma unroll
                        for (int e = 0; e < 32; ++e) v[e] = fmaf(v[e], p.scale, mine[-e]);
                    }
                    if (j + 1 < blocks && at_tile < WT_DIAG) tabs[((j + 1) & 1) * WT_TAB + at_tile] = ahead;
                }
                // a border passes through where the warp's first query does not see its last key or its last query not the first one
                if (room - lane < 31 || (p.rule.W > 0 && room - lane + 31 >= p.rule.W && j0 + 31 >= p.rule.S)) {
                    const int from = p.rule.W > 0 ? room - p.rule.W + 1 : 0, to = p.rule.S - j0;
#pragma unroll
                    for (int e = 0; e < 32; ++e) v[e] = keeps(e, room, from, to) ? v[e] : -INFINITY;
                }
                float mx = max32(v);
                if (pair_any(bar, j == 0 || (mx - m) * c > 8.0f)) {  // almost only in the first block
                    xch[half * 128 + row] = mx;
                    pair_sync(bar);
                    mx = fmaxf(mx, xch[(half ^ 1) * 128 + row]);
                    if (j == 0) {
                        m = mx;
                    } else {
                        sum *= mx > m ? ex2((m - mx) * c) : 1.0f;
                        m = fmaxf(m, mx);
                    }
                    pair_sync(bar);  // both have read before either writes again
                }
                const float rel = m == -INFINITY ? 0.0f : m, m2 = rel * c;  // nothing seen yet: every score is -inf
                float acc[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int e = 0; e < 32; ++e) {
                    v[e] = BIAS ? ex2((v[e] - rel) * c) : ex2(fmaf(v[e], c, -m2));  // a bias may be the type's lowest value, which log2 units cannot hold
                    acc[e & 3] += v[e];
                }
                sum += (acc[0] + acc[1]) + (acc[2] + acc[3]);
                place_parts(v, t0 + 32 * half, t0 + 64 + 16 * half, t0 + 96 + 16 * half);
                tmem_stores_done();
                __syncwarp();
                if (lane == 0) mbar_arrive(p_ready(q));
            }
            good = good && ready_wait(o_full(q), o_phase & 1u, p.status, 48);
            ++o_phase;
            after_sync();
            xch[half * 128 + row] = sum;
            ok = !pair_any(bar, !good);  // all of a tile's threads leave together
            const bool empty_row = m == -INFINITY;
            const float inv = empty_row ? 0.0f : 1.0f / (sum + xch[(half ^ 1) * 128 + row]);
            pair_sync(bar);
            if (!ok) break;
            const float inv_sums = inv * (m_out == m ? 1.0f : ex2((m_out - m) * c));
            float x[OC];
            tmem_read(t0 + 128 + half * OC, x);
#pragma unroll
            for (int e = 0; e < OC / 4; ++e) {
                const float4 o = blocks > 1 ? sums(e) : make_float4(0.f, 0.f, 0.f, 0.f);
                *own_at(own, row, half * OC + 4 * e) = make_float4(fmaf(o.x, inv_sums, x[4 * e] * inv), fmaf(o.y, inv_sums, x[4 * e + 1] * inv), fmaf(o.z, inv_sums, x[4 * e + 2] * inv), fmaf(o.w, inv_sums, x[4 * e + 3] * inv));
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            pair_sync(bar);
            if (at_tile == 0) {
                own_store<DP>(&map_o, base + q * S::TWIN, p, r0, it.h, it.b);
                tma_store_commit();
                tma_store_wait_read<0>();
                fetch(w + gridDim.x);
            }
            if (half == 0 && live) {
                const int64_t at = ((int64_t)it.b * p.H + it.h) * p.Tp + r;
                p.row_max[at] = empty_row ? INFINITY : BIAS ? m : m * p.scale;
                p.row_inv[at] = inv;
            }
        }
        if (at_tile == 0) tma_store_wait_all();
    }
    tmem_give(tmem, warp);
}

// ---- dK and dV ----------------------------------------------------------------------------------------------------------------
// A thread owns a key and sixteen of a block's queries, everything transposed: S^T = k q^T, dP^T = v dO^T, dV += P^T dO, dK += dS^T q, for the
// queries from the diagonal to the window's end.  Products are ordered so that the tensor core has dV(i), S(i+1) to do while dS(i) is made
// and dK(i), dP(i+1) while P(i+1) is.
//   warps 0, 2   TMA producers: K-major tiles, MN-major tiles       warp 1  MMA issuer
//   warps 4..11  companions, the statistics of a block's queries and its bias        warps 12..27  four threads a key
// A tile of q arrives K-major and once more MN-major; so does dO.  Its companions serve both products and stay until the second has read them.
// Tensor memory: S^T / t of P^T [0, 64), dP^T / t of dS^T [64, 128), P^T companions [128, 192), dS^T companions [192, 256), dV [256, 320), dK [320, 384),
// t of k [384, 448), t of v [448, 512).
template <int DP, bool BIAS>
struct DkvSmem {
    using T = WinTile<DP>;
    static constexpr int OWN = AT_ROWS * DP * 4;  // companions of a 128-row operand
    static constexpr int O_RAWS = BIAS ? 1 : 2;   // with a bias its table takes the place of the second one
    static constexpr int Q_RAW = 2 * OWN, O_RAW = Q_RAW + 2 * T::RAW, Q_MN = O_RAW + O_RAWS * T::RAW, O_MN = Q_MN + T::RAW, Q_TWIN = O_MN + 2 * T::RAW, O_TWIN = Q_TWIN + 2 * T::TWIN;
    static constexpr int STATS = O_TWIN + T::TWIN;  // row maximum, dO . O and (with a bias) 1 / sum of a block's queries, two blocks; then the bias of its distances, two blocks
    static constexpr int STATS_BLOCK = (BIAS ? 3 : 2) * AT_KEYS * 4, TABS = STATS + 2 * STATS_BLOCK, BAR = TABS + (BIAS ? 2 * WT_TAB * 4 : 0), TOTAL = BAR + 256 + 1024;
    static_assert(TOTAL <= 232448, "shared memory");
};
template <int DP, bool BIAS>
__global__ void __launch_bounds__(AT_BWD_THREADS, 1) window_attention_tc_dkv_kernel(const __grid_constant__ CUtensorMap map_qk, const __grid_constant__ CUtensorMap map_qn, const __grid_constant__ CUtensorMap map_ok,
                                                                                const __grid_constant__ CUtensorMap map_on, const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
                                                                                const __grid_constant__ CUtensorMap map_dk, const __grid_constant__ CUtensorMap map_dv, const __grid_constant__ WindowTc p) {
    using S = DkvSmem<DP, BIAS>;
    using T = WinTile<DP>;
    extern __shared__ uint8_t smem_raw[];
    const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
    uint8_t* gen = smem_raw + (base - smem_u32(smem_raw));
    const uint32_t bars = base + S::BAR;
    auto bar = [&](int i) { return bars + 8u * i; };
    // n: running number of a block; parities of what has two places and of what has one
    auto two = [](uint32_t n) { return (n >> 1) & 1u; };
    auto one = [](uint32_t n) { return n & 1u; };
    auto o_place = [](uint32_t n) { return S::O_RAWS == 2 ? n & 1u : 0u; };
    auto q_full = [&](uint32_t n) { return bar(0 + (n & 1u)); };
    auto o_full = [&](uint32_t n) { return bar(2 + o_place(n)); };
    auto on_full = [&](uint32_t n) { return bar(4 + (n & 1u)); };
    auto q_conv = [&](uint32_t n) { return bar(6 + (n & 1u)); };
    // One barrier a product, in two turns: it tells the threads that the result is there, and the producers and the companion warps that what it read may go.
    auto s_done = [&](uint32_t n) { return bar(8 + (n & 1u)); };
    auto dp_done = [&](uint32_t n) { return bar(10 + (n & 1u)); };
    auto dv_done = [&](uint32_t n) { return bar(12 + (n & 1u)); };
    auto dk_done = [&](uint32_t n) { return bar(14 + (n & 1u)); };
    const uint32_t qn_full = bar(16), o_conv = bar(17), p_ready = bar(18), ds_ready = bar(19), kv_ready = bar(20), own_full = bar(21);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        for (int i = 0; i < 22; ++i) mbar_init(bar(i), i == 6 || i == 7 || i == 17 ? 8 : i >= 18 && i <= 20 ? 16 : i == 21 ? 2 : 1);  // own_full: two tiles
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    const uint32_t tmem = tmem_take(bars + 8u * 28, reinterpret_cast<volatile uint32_t*>(gen + S::BAR + 8 * 28), warp);
    pdl_trigger();
    pdl_wait();
    auto steps = [&](const AttnItem& it) {  // blocks of queries from the tile's first key to the last query that sees its last one
        const int k0 = it.unit * AT_ROWS, k1 = min(p.T, k0 + AT_ROWS), end = p.rule.W > 0 && p.rule.W < p.T - k1 ? k1 - 1 + p.rule.W : p.T;
        return (end - k0 + AT_KEYS - 1) / AT_KEYS;
    };

    if (warp < 4) regs_give<64>();
    if (warp == 0 || warp == 2) {  // K-major tiles by warp 0, up to two blocks ahead, MN-major ones by warp 2
        if (lane == 0) {
            uint32_t n0 = 0;
            bool ok = true;
            for (int64_t w = blockIdx.x; w < p.loop_end && ok; w += gridDim.x) {
                const AttnItem it = attn_item(p, w, true);
                if (it.skip) continue;
                const int n = steps(it);
                // `back` blocks ago the place was last filled, and `done` is the product that read it
                auto load = [&](auto done, uint32_t back, int dst, const CUtensorMap* map, uint32_t landed, int i) {
                    const uint32_t at = n0 + i;
                    if (at >= back && !mbar_wait(done(at - back), two(at - back), p.status, 51)) return false;
                    win_load<DP>(base + dst, map, landed, it.unit * AT_ROWS + i * AT_KEYS, it.h, it.b);
                    return true;
                };
                for (int i = 0; i < n && ok; ++i) {
                    const uint32_t at = n0 + i, place = (at & 1u) * T::RAW;
                    if (warp == 0) ok = load(s_done, 2, S::Q_RAW + place, &map_qk, q_full(at), i) && load(dp_done, S::O_RAWS, S::O_RAW + o_place(at) * T::RAW, &map_ok, o_full(at), i);
                    else ok = load(dv_done, 2, S::O_MN + place, &map_on, on_full(at), i) && load(dk_done, 1, S::Q_MN, &map_qn, qn_full, i);
                }
                n0 += n;
            }
        }
    } else if (warp == 1) {
        if (elect_one()) {
            const uint32_t base16 = base >> 4;
            uint32_t n0 = 0, items = 0;
            bool ok = true;
            for (int64_t w = blockIdx.x; w < p.loop_end && ok; w += gridDim.x, ++items) {
                const AttnItem it = attn_item(p, w, true);
                if (it.skip) break;  // only the last round has items left out
                const int n = steps(it);
                auto landed = [&](uint32_t b, uint32_t parity) {
                    const bool r = issuer_wait(b, parity, p.status, 52);
                    after_sync();
                    return r;
                };
                auto scores = [&](uint32_t at) {
                    if (!landed(q_conv(at), two(at))) return false;
                    win_scores<DP>(tmem, tmem + 384, base16, base16 + (S::Q_RAW + (at & 1u) * T::RAW) / 16, base16 + (S::Q_TWIN + (at & 1u) * T::TWIN) / 16);
                    umma_commit(s_done(at));
                    return true;
                };
                auto dprobs = [&](uint32_t at) {
                    if (!landed(o_conv, one(at))) return false;
                    win_scores<DP>(tmem + 64, tmem + 448, base16 + S::OWN / 16, base16 + (S::O_RAW + o_place(at) * T::RAW) / 16, base16 + S::O_TWIN / 16);
                    umma_commit(dp_done(at));
                    return true;
                };
                ok = issuer_wait(kv_ready, items & 1u, p.status, 53) && scores(n0) && dprobs(n0);
                for (int i = 0; i < n && ok; ++i) {
                    const uint32_t at = n0 + i;
                    const bool more = i + 1 < n;
                    ok = issuer_wait(on_full(at), two(at), p.status, 54) && landed(p_ready, one(at));
                    if (!ok) break;
                    win_values<DP, 8>(tmem + 256, tmem, tmem + 128, tmem + 160, base16 + (S::O_MN + (at & 1u) * T::RAW) / 16, base16 + S::O_TWIN / 16, i % WT_FLUSH != 0);
                    umma_commit(dv_done(at));
                    ok = (!more || scores(at + 1)) && issuer_wait(qn_full, one(at), p.status, 55) && landed(ds_ready, one(at));
                    if (!ok) break;
                    win_values<DP, 8>(tmem + 320, tmem + 64, tmem + 192, tmem + 224, base16 + S::Q_MN / 16, base16 + (S::Q_TWIN + (at & 1u) * T::TWIN) / 16, i % WT_FLUSH != 0);
                    umma_commit(dk_done(at));
                    ok = !more || dprobs(at + 1);
                }
                if (!ok) break;
                n0 += n;
            }
        }
    } else if (warp >= 4 && warp < 12) {
        regs_give<56>();
        const int t = threadIdx.x - 128;
        uint32_t n0 = 0;
        bool ok = true;
        for (int64_t w = blockIdx.x; w < p.loop_end && ok; w += gridDim.x) {
            const AttnItem it = attn_item(p, w, true);
            if (it.skip) continue;
            const int n = steps(it), q_at = it.unit * AT_ROWS + t;
            const int64_t at_head = ((int64_t)it.b * p.H + it.h) * p.Tp;
            const float* tab = BIAS ? p.tab + (int64_t)it.h * p.tab_len : nullptr;
            float nm = 0.f, ni = 0.f, nd = 0.f, nb = 0.f;  // the next block's, loaded a block ahead
            auto request = [&](int i) {
                const int q = q_at + i * AT_KEYS, d0 = i * AT_KEYS - (AT_ROWS - 1);
                const bool live = t < AT_KEYS && q < p.T;  // queries beyond the sequence have no statistics: P is then zero
                nm = live ? __ldg(p.row_max + at_head + q) : INFINITY;
                ni = live ? __ldg(p.row_inv + at_head + q) : 0.0f;
                nd = live ? __ldg(p.delta + at_head + q) : 0.0f;
                if (BIAS) nb = __ldg(tab + clamp_distance(d0 + t, p.tab_len));
            };
            request(0);
            for (int i = 0; i < n && ok; ++i) {
                const uint32_t at = n0 + i, place = (at & 1u) * T::RAW;
                // dK of the block before last has read the companions that these replace; its statistics were used before that
                ok = ready_wait(q_full(at), two(at), p.status, 56) && (at < 2u || ready_wait(dk_done(at - 2u), two(at - 2u), p.status, 56));
                if (!ok) break;
                if (t < AT_KEYS) {
                    float* slot = reinterpret_cast<float*>(gen + S::STATS + (at & 1u) * S::STATS_BLOCK) + t;
                    slot[0] = BIAS ? nm : nm * kLog2e - log2f(ni);
                    slot[AT_KEYS] = nd;
                    if (BIAS) slot[2 * AT_KEYS] = ni;
                }
                if (BIAS && t < WT_TAB) reinterpret_cast<float*>(gen + S::TABS)[(at & 1u) * WT_TAB + t] = nb;
                if (i + 1 < n) request(i + 1);
                win_split<DP, 256, false>(gen + S::Q_RAW + place, gen + S::Q_TWIN + (at & 1u) * T::TWIN, t);
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                __syncwarp();
                if (lane == 0) mbar_arrive(q_conv(at));
                ok = ready_wait(o_full(at), S::O_RAWS == 2 ? two(at) : one(at), p.status, 56) && (at < 1u || ready_wait(dv_done(at - 1u), two(at - 1u), p.status, 56));
                if (!ok) break;
                win_split<DP, 256, false>(gen + S::O_RAW + o_place(at) * T::RAW, gen + S::O_TWIN, t);
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                __syncwarp();
                if (lane == 0) mbar_arrive(o_conv);
            }
            n0 += n;
        }
    } else if (warp >= 12) {
        regs_take<80>();
        const int part = (warp - 12) >> 2, row = 32 * (warp & 3) + lane;  // this warp: 32 keys x 16 of the block's 64 queries
        constexpr int OC = DP / 2;                                       // and half of the columns of k and dK (parts 0, 1) or v and dV (2, 3)
        const int half = part & 1;
        const uint32_t lanes = tmem + ((uint32_t)(32 * (warp & 3)) << 16);
        const float c = p.scale * kLog2e;
        uint32_t n = 0, items = 0;
        bool good = true;
        uint8_t* own = gen + (part >> 1) * S::OWN;
        auto fetch = [&](int64_t w) {  // the rows of the item at w
            if (w >= p.loop_end) return;
            const AttnItem it = attn_item(p, w, true);
            if (it.skip) return;
            own_load<DP>(base, &map_k, own_full, it.unit * AT_ROWS, it.h, it.b);
            own_load<DP>(base + S::OWN, &map_v, own_full, it.unit * AT_ROWS, it.h, it.b);
        };
        if (threadIdx.x == 384) fetch(blockIdx.x);
        for (int64_t w = blockIdx.x; w < p.loop_end; w += gridDim.x, ++items) {
            const AttnItem it = attn_item(p, w, true);
            if (it.skip) break;
            good = good && ready_wait(own_full, items & 1u, p.status, 50);  // every thread keeps step with the barriers of the items, whatever a wait says
            {
                float x[OC];
                own_read(x, own, row, half * OC);
                all_any(false);
                place_row<DP / 32>(x, lanes + (part < 2 ? 384 : 448) + half * OC, own + half * (OC / 16) * 8192, row);
            }
            tmem_stores_done();
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            if (lane == 0) mbar_arrive(kv_ready);
            const int cnt = steps(it);
            float* moved = moved_at(p, part >> 1, half * OC, row);
            auto move = [&](bool there) {
#pragma unroll
                for (int g = 0; g < OC / 16; ++g) move_sum(lanes + (part < 2 ? 320 : 256) + half * OC + 16 * g, moved + 16 * g * AT_ROWS, there);
            };
#pragma unroll 1
            for (int i = 0; i < cnt; ++i, ++n) {
                const float4* mp = reinterpret_cast<const float4*>(gen + S::STATS + (n & 1u) * S::STATS_BLOCK) + 4 * part;
                const float4 *dp = mp + AT_KEYS / 4, *ip = dp + AT_KEYS / 4;
                good = good && ready_wait(s_done(n), two(n), p.status, 57);
                after_sync();
                if (part >= 2 && i > 0 && i % WT_FLUSH == 0) move(i > WT_FLUSH);  // dV of the blocks before came before these scores
                uint32_t u[16];
                float pr[16];
                tmem_ld16(lanes + 16 * part, u);
                const int first = row - i * AT_KEYS - 16 * part;  // queries from here on look at this key, as many as the window is long
                const float* bias = reinterpret_cast<const float*>(gen + S::TABS) + (n & 1u) * WT_TAB + (AT_ROWS - 1) + 16 * part - row;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float4 m = mp[e];
                    const float mm[4] = {m.x, m.y, m.z, m.w};
                    if (BIAS) {
                        const float4 iv = ip[e];
                        const float ii[4] = {iv.x, iv.y, iv.z, iv.w};
#pragma unroll
                        for (int x = 0; x < 4; ++x) pr[4 * e + x] = ex2((fmaf(__uint_as_float(u[4 * e + x]), p.scale, bias[4 * e + x]) - mm[x]) * kLog2e) * ii[x];
                    } else {
#pragma unroll
                        for (int x = 0; x < 4; ++x) pr[4 * e + x] = ex2(fmaf(__uint_as_float(u[4 * e + x]), c, -mm[x]));
                    }
                }
                if (i < 2 || (p.rule.W > 0 && (i + 1) * AT_KEYS > p.rule.W)) {  // the diagonal block, and those the window ends in
                    const int end = p.rule.W > 0 ? min(16, first + p.rule.W) : 16;
#pragma unroll
                    for (int e = 0; e < 16; ++e) pr[e] = e >= first && e < end ? pr[e] : 0.0f;
                }
                place_parts16(pr, lanes + 16 * part, lanes + 128 + 8 * part, lanes + 160 + 8 * part);
                tmem_stores_done();
                __syncwarp();
                if (lane == 0) mbar_arrive(p_ready);
                good = good && ready_wait(dp_done(n), two(n), p.status, 58);
                after_sync();
                tmem_ld16(lanes + 64 + 16 * part, u);
#pragma unroll
                for (int e = 0; e < 4; ++e) {  // a masked P is zero whatever dP holds; the scale comes last
                    const float4 d = dp[e];
                    const float dd[4] = {d.x, d.y, d.z, d.w};
#pragma unroll
                    for (int x = 0; x < 4; ++x) pr[4 * e + x] *= __uint_as_float(u[4 * e + x]) - dd[x];
                }
                place_parts16(pr, lanes + 64 + 16 * part, lanes + 192 + 8 * part, lanes + 224 + 8 * part);
                if (part < 2 && i > 0 && i % WT_FLUSH == 0) move(i > WT_FLUSH);  // dK of the blocks before came before this dP
                tmem_stores_done();
                __syncwarp();
                if (lane == 0) mbar_arrive(ds_ready);
            }
            good = good && ready_wait(dk_done(n - 1u), two(n - 1u), p.status, 59);  // the last product of all
            after_sync();
            const float f = part < 2 ? p.scale : 1.0f;
#pragma unroll
            for (int g = 0; g < OC / 16; ++g) place_result(own, row, half * OC + 16 * g, lanes + (part < 2 ? 320 : 256) + half * OC + 16 * g, moved + 16 * g * AT_ROWS, cnt > WT_FLUSH, f);
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            if (all_any(!good)) break;  // all of them leave together
            if (threadIdx.x == 384) {
                own_store<DP>(&map_dk, base, p, it.unit * AT_ROWS, it.h, it.b);
                own_store<DP>(&map_dv, base + S::OWN, p, it.unit * AT_ROWS, it.h, it.b);
                tma_store_commit();
                tma_store_wait_read<0>();
                fetch(w + gridDim.x);
            }
        }
        if (threadIdx.x == 384) tma_store_wait_all();
    }
    tmem_give(tmem, warp);
}

// ---- dQ and the bias gradient ---------------------------------------------------------------------------------------------------
// A CTA takes 128 queries and walks over their keys: S = q k^T and dP = dO v^T of one block while dQ += dS k of the block before passes.  Four
// threads a query, sixteen of a block's keys each.  dO . O is formed here, from the rows that are loaded anyway, and kept for dK.
// Roles as above.
// Scores and dP alternate between two places, x = 0 and 1; dS takes the place of both, a thread's columns where it has read them.
// Tensor memory: S / companions of dS [128 x, + 64) (of 16 keys: 8 columns bf16(dS), 8 bf16(dS - t)), dP / t of dS [128 x + 64, + 64), dQ [256, 320), t of q [320, 384), t of dO [384, 448).
// Bias gradient: a warp adds up the dS of its 32 x 16 block along the diagonals, 47 of them, in sixteen shuffles; lane n keeps buckets n and n + 32, as
// differences of running sums over the diagonals.  A block that lies in one bucket as a whole is added up row by row in registers instead.
template <int DP, bool BIAS>
struct DqSmem {
    using T = WinTile<DP>;
    static constexpr int OWN = AT_ROWS * DP * 4;
    static constexpr uint32_t MNS = BIAS ? 1 : 2;  // with a bias its table takes the place of the second MN-major tile (a third place for companions is worth more: 264 us against 383)
    static constexpr int K_RAW = 2 * OWN, V_RAW = K_RAW + 2 * T::RAW, K_MN = V_RAW + 2 * T::RAW, K_TWIN = K_MN + (int)MNS * T::RAW, V_TWIN = K_TWIN + 3 * T::TWIN;
    static constexpr int XCH = V_TWIN + T::TWIN, TABS = XCH + AT_ROWS * 4, BAR = TABS + (BIAS ? 3 * WT_TAB * 4 : 0);  // dO . O of every row; bias of a block's distances, three blocks
    static constexpr int TOTAL = BAR + 256 + 1024;
    static_assert(TOTAL <= 232448 && AW_MAX_BUCKETS == 64, "shared memory");
};
template <int DP, bool BIAS>
__global__ void __launch_bounds__(AT_BWD_THREADS, 1) window_attention_tc_dq_kernel(const __grid_constant__ CUtensorMap map_kk, const __grid_constant__ CUtensorMap map_vk, const __grid_constant__ CUtensorMap map_kn, const __grid_constant__ CUtensorMap map_q,
                                                                               const __grid_constant__ CUtensorMap map_do, const __grid_constant__ CUtensorMap map_dq,
                                                                               const __grid_constant__ WindowTc p) {
    using S = DqSmem<DP, BIAS>;
    using T = WinTile<DP>;
    extern __shared__ uint8_t smem_raw[];
    const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
    uint8_t* gen = smem_raw + (base - smem_u32(smem_raw));
    const uint32_t bars = base + S::BAR;
    auto bar = [&](int i) { return bars + 8u * i; };
    auto two = [](uint32_t n) { return (n >> 1) & 1u; };
    auto one = [](uint32_t n) { return n & 1u; };
    auto k_full = [&](uint32_t n) { return bar(0 + (n & 1u)); };
    auto v_full = [&](uint32_t n) { return bar(2 + (n & 1u)); };
    auto kn_place = [](uint32_t n) { return S::MNS == 2 ? n & 1u : 0u; };
    auto kn_full = [&](uint32_t n) { return bar(4 + kn_place(n)); };
    auto k_conv = [&](uint32_t n) { return bar(6 + n % 3u); };
    // one barrier a product, in two turns, as above
    auto s_done = [&](uint32_t n) { return bar(9 + (n & 1u)); };
    auto dp_done = [&](uint32_t n) { return bar(11 + (n & 1u)); };
    auto dq_done = [&](uint32_t n) { return bar(13 + (n & 1u)); };
    auto ds_ready = [&](uint32_t n) { return bar(15 + (n & 1u)); };
    const uint32_t v_conv = bar(17), q_ready = bar(18), own_full = bar(19);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        for (int i = 0; i < 20; ++i) mbar_init(bar(i), (i >= 6 && i <= 8) || i == 17 ? 8 : i == 15 || i == 16 || i == 18 ? 16 : i == 19 ? 2 : 1);  // own_full: two tiles
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    const uint32_t tmem = tmem_take(bars + 8u * 30, reinterpret_cast<volatile uint32_t*>(gen + S::BAR + 8 * 30), warp);
    pdl_trigger();
    pdl_wait();

    if (warp < 4) regs_give<64>();
    if (warp == 0 || warp == 2) {  // K-major tiles by warp 0, up to two blocks ahead, MN-major ones by warp 2
        if (lane == 0) {
            uint32_t n0 = 0;
            bool ok = true;
            for (int64_t w = blockIdx.x; w < p.loop_end && ok; w += gridDim.x) {
                const AttnItem it = attn_item(p, w, false);
                if (it.skip) continue;
                const TileKeys keys(p, it.unit * AT_ROWS);
                const int n = keys.count();
                // `back` blocks ago the place was last filled, and `done` is the product that read it
                auto load = [&](auto done, uint32_t back, int dst, const CUtensorMap* map, uint32_t landed, int i) {
                    const uint32_t at = n0 + i;
                    if (at >= back && !mbar_wait(done(at - back), two(at - back), p.status, 61)) return false;
                    win_load<DP>(base + dst, map, landed, keys.block(i) * AT_KEYS, it.h, it.b);
                    return true;
                };
                for (int i = 0; i < n && ok; ++i) {
                    const uint32_t at = n0 + i, place = (at & 1u) * T::RAW;
                    if (warp == 0) ok = load(s_done, 2, S::K_RAW + place, &map_kk, k_full(at), i) && load(dp_done, 2, S::V_RAW + place, &map_vk, v_full(at), i);
                    else ok = load(dq_done, S::MNS, S::K_MN + kn_place(at) * T::RAW, &map_kn, kn_full(at), i);
                }
                n0 += n;
            }
        }
    } else if (warp == 1) {
        if (elect_one()) {
            const uint32_t base16 = base >> 4;
            uint32_t n0 = 0, items = 0;
            bool ok = true;
            for (int64_t w = blockIdx.x; w < p.loop_end && ok; w += gridDim.x, ++items) {
                const AttnItem it = attn_item(p, w, false);
                if (it.skip) break;  // only the last round has items left out
                const int n = TileKeys(p, it.unit * AT_ROWS).count();
                auto products = [&](uint32_t at) {  // S and dP
                    const uint32_t place = tmem + 128 * (at & 1u), raw = (at & 1u) * (T::RAW / 16);
                    if (!issuer_wait(k_conv(at), (at / 3u) & 1u, p.status, 62) || !issuer_wait(v_conv, one(at), p.status, 62)) return false;
                    after_sync();
                    win_scores<DP>(place, tmem + 320, base16, base16 + S::K_RAW / 16 + raw, base16 + (S::K_TWIN + at % 3u * T::TWIN) / 16);
                    umma_commit(s_done(at));
                    win_scores<DP>(place + 64, tmem + 384, base16 + S::OWN / 16, base16 + S::V_RAW / 16 + raw, base16 + S::V_TWIN / 16);
                    umma_commit(dp_done(at));
                    return true;
                };
                ok = issuer_wait(q_ready, items & 1u, p.status, 63);
                if (!ok) break;
                ok = products(n0);
                for (int i = 0; i < n && ok; ++i) {
                    const uint32_t at = n0 + i, place = tmem + 128 * (at & 1u);
                    ok = (i + 1 == n || products(at + 1)) && issuer_wait(kn_full(at), S::MNS == 2 ? two(at) : one(at), p.status, 64) && issuer_wait(ds_ready(at), two(at), p.status, 64);
                    if (!ok) break;
                    after_sync();
                    win_values<DP, 16>(tmem + 256, place + 64, place, place + 8, base16 + (S::K_MN + kn_place(at) * T::RAW) / 16, base16 + (S::K_TWIN + at % 3u * T::TWIN) / 16, i % WT_FLUSH != 0);
                    umma_commit(dq_done(at));
                }
                if (!ok) break;
                n0 += n;
            }
        }
    } else if (warp >= 4 && warp < 12) {
        regs_give<56>();
        const int t = threadIdx.x - 128;
        uint32_t n0 = 0;
        bool ok = true;
        for (int64_t w = blockIdx.x; w < p.loop_end && ok; w += gridDim.x) {
            const AttnItem it = attn_item(p, w, false);
            if (it.skip) continue;
            const TileKeys keys(p, it.unit * AT_ROWS);
            const int n = keys.count();
            const float* tab = BIAS ? p.tab + (int64_t)it.h * p.tab_len : nullptr;
            float nb = 0.f;  // the next block's, loaded a block ahead
            auto request = [&](int i) { nb = __ldg(tab + clamp_distance(it.unit * AT_ROWS - (keys.block(i) + 1) * AT_KEYS + 1 + t, p.tab_len)); };
            if (BIAS) request(0);
            for (int i = 0; i < n && ok; ++i) {
                const uint32_t at = n0 + i, place = (at & 1u) * T::RAW;
                // dQ has read the companions that these replace; that block's bias was used before
                ok = ready_wait(k_full(at), two(at), p.status, 65) && (at < 3u || ready_wait(dq_done(at - 3u), two(at - 3u), p.status, 65));
                if (!ok) break;
                if (BIAS) {
                    if (t < WT_TAB) reinterpret_cast<float*>(gen + S::TABS)[at % 3u * WT_TAB + t] = nb;
                    if (i + 1 < n) request(i + 1);
                }
                win_split<DP, 256, false>(gen + S::K_RAW + place, gen + S::K_TWIN + at % 3u * T::TWIN, t);
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                __syncwarp();
                if (lane == 0) mbar_arrive(k_conv(at));
                ok = ready_wait(v_full(at), two(at), p.status, 65) && (at < 1u || ready_wait(dp_done(at - 1u), two(at - 1u), p.status, 65));
                if (!ok) break;
                win_split<DP, 256, false>(gen + S::V_RAW + place, gen + S::V_TWIN, t);
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                __syncwarp();
                if (lane == 0) mbar_arrive(v_conv);
            }
            n0 += n;
        }
    } else if (warp >= 12) {
        regs_take<80>();
        const int part = (warp - 12) >> 2, row = 32 * (warp & 3) + lane;  // this warp: 32 queries x 16 of the block's 64 keys
        constexpr int OC = DP / 2;                                       // and half of the columns of q (parts 0, 1) or dO (2, 3)
        const int half = part & 1;
        const uint32_t lanes = tmem + ((uint32_t)(32 * (warp & 3)) << 16);
        float* sums = reinterpret_cast<float*>(gen + S::OWN);  // [warp][bucket], at an item's end, when dO's companions have been read
        float* xch = reinterpret_cast<float*>(gen + S::XCH);  // dO . O of every row
        const float c = p.scale * kLog2e;
        const bool wants_dbias = BIAS && p.dbias_part != nullptr;
        uint32_t n = 0, items = 0;
        bool good = true;
        uint8_t* own = gen + (part >> 1) * S::OWN;
        auto fetch = [&](int64_t w) {  // the rows of the item at w
            if (w >= p.loop_end) return;
            const AttnItem it = attn_item(p, w, false);
            if (it.skip) return;
            own_load<DP>(base, &map_q, own_full, it.unit * AT_ROWS, it.h, it.b);
            own_load<DP>(base + S::OWN, &map_do, own_full, it.unit * AT_ROWS, it.h, it.b);
        };
        if (threadIdx.x == 384) fetch(blockIdx.x);
        for (int64_t w = blockIdx.x; w < p.loop_end; w += gridDim.x, ++items) {
            const AttnItem it = attn_item(p, w, false);
            if (it.skip) break;
            const int r0 = it.unit * AT_ROWS, r = r0 + row;
            const bool live = r < p.T;
            const int64_t at = ((int64_t)it.b * p.H + it.h) * p.Tp + r;
            // dO . O: a warp's eight rows, DP / 4 lanes each, while the tiles arrive
            constexpr int LANES = DP / 4, STEP = 32 / LANES;
            float a[8 / STEP];
#pragma unroll
            for (int x = 0; x < 8 / STEP; ++x) {
                const int rr = r0 + 8 * (warp - 12) + x * STEP + lane / LANES, col = 4 * (lane % LANES);
                const bool in = rr < p.T && col < p.D;
                const float4 u = in ? ld4(p.g + it.b * p.g_so + it.h * p.g_si + rr * p.g_ld + col) : make_float4(0.f, 0.f, 0.f, 0.f);
                const float4 y = in ? ld4(p.o + it.b * p.o_so + it.h * p.o_si + rr * p.o_ld + col) : make_float4(0.f, 0.f, 0.f, 0.f);
                a[x] = fmaf(u.x, y.x, fmaf(u.y, y.y, fmaf(u.z, y.z, u.w * y.w)));
            }
#pragma unroll
            for (int s = LANES / 2; s > 0; s >>= 1)
#pragma unroll
                for (int x = 0; x < 8 / STEP; ++x) a[x] += __shfl_xor_sync(0xffffffffu, a[x], s);
            if (lane % LANES == 0)
#pragma unroll
                for (int x = 0; x < 8 / STEP; ++x) xch[8 * (warp - 12) + x * STEP + lane / LANES] = a[x];
            good = good && ready_wait(own_full, items & 1u, p.status, 60);  // every thread keeps step with the barriers of the items, whatever a wait says
            {
                float x[OC];
                own_read(x, own, row, half * OC);
                all_any(false);
                place_row<DP / 32>(x, lanes + (part < 2 ? 320 : 384) + half * OC, own + half * (OC / 16) * 8192, row);
            }
            tmem_stores_done();
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            if (lane == 0) mbar_arrive(q_ready);
            const float delta = xch[row];
            if (part == 0 && live) p.delta[at] = delta;
            const float inv = live ? p.row_inv[at] : 0.0f, m = !live ? INFINITY : BIAS ? p.row_max[at] : p.row_max[at] * kLog2e - log2f(inv);
            const float* tab = BIAS ? p.tab + (int64_t)it.h * p.tab_len : nullptr;
            const float beyond = BIAS ? __ldg(tab + p.tab_len - 1) : 0.0f;
            const TileKeys keys(p, r0);
            const int cnt = keys.count();
            float* moved = moved_at(p, 0, 16 * part, row);
            // bias gradient: this lane's buckets, and what belongs to bucket `run_of` as a whole; buckets only go down along the walk
            float sum0 = 0.0f, sum1 = 0.0f, run = 0.0f;
            int run_of = p.rule.buckets - 1, near_of = run_of, far_of = run_of;
            auto settle = [&]() {
                const float a = warp_sum(run);
                if (lane == (run_of & 31)) { if (run_of < 32) sum0 += a; else sum1 += a; }
                run = 0.0f;
            };
#pragma unroll 1
            for (int i = 0; i < cnt; ++i, ++n) {
                const uint32_t place = lanes + 128 * (n & 1u);
                const int b = keys.block(i), j0 = b * AT_KEYS + 16 * part, room = r - j0;
                good = good && ready_wait(s_done(n), two(n), p.status, 66);
                after_sync();
                uint32_t u[16];
                float pr[16];
                tmem_ld16(place + 16 * part, u);
                if (BIAS) {
                    if (r0 - (b + 1) * AT_KEYS + 1 >= p.tab_len - 1) {
#pragma unroll
                        for (int e = 0; e < 16; ++e) pr[e] = ex2((fmaf(__uint_as_float(u[e]), p.scale, beyond) - m) * kLog2e) * inv;
                    } else {
                        const float* mine = reinterpret_cast<const float*>(gen + S::TABS) + n % 3u * WT_TAB + row - 16 * part + AT_KEYS - 1;
#pragma unroll
                        for (int e = 0; e < 16; ++e) pr[e] = ex2((fmaf(__uint_as_float(u[e]), p.scale, mine[-e]) - m) * kLog2e) * inv;
                    }
                } else {
#pragma unroll
                    for (int e = 0; e < 16; ++e) pr[e] = ex2(fmaf(__uint_as_float(u[e]), c, -m));
                }
                if (room - lane < 15 || (p.rule.W > 0 && room - lane + 31 >= p.rule.W && j0 + 15 >= p.rule.S)) {
                    const int from = p.rule.W > 0 ? room - p.rule.W + 1 : 0, to = p.rule.S - j0;
#pragma unroll
                    for (int e = 0; e < 16; ++e) pr[e] = keeps(e, room, from, to) ? pr[e] : 0.0f;
                }
                good = good && ready_wait(dp_done(n), two(n), p.status, 67);
                after_sync();
                tmem_ld16(place + 64 + 16 * part, u);
#pragma unroll
                for (int e = 0; e < 16; ++e) pr[e] *= __uint_as_float(u[e]) - delta;  // a masked P is zero whatever dP holds
                place_parts16(pr, place + 64 + 16 * part, place + 16 * part, place + 16 * part + 8);
                if (i > 0 && i % WT_FLUSH == 0) {
                    good = good && ready_wait(dq_done(n - 1u), two(n - 1u), p.status, 68);
                    after_sync();
                    if (16 * part < DP) move_sum(lanes + 256 + 16 * part, moved, i > WT_FLUSH);
                }
                tmem_stores_done();
                __syncwarp();
                if (lane == 0) mbar_arrive(ds_ready(n));
                const int d1 = room - lane + 31, d0 = room - lane - 15;  // largest and smallest distance of the warp's 32 x 16 block
                if (wants_dbias && d1 >= 0) {
                    while (p.rule.starts[far_of] > d1) --far_of;
                    while (p.rule.starts[near_of] > max(d0, 0)) --near_of;
                    if (near_of == far_of) {
                        if (run_of != near_of) { settle(); run_of = near_of; }
                        float a[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                        for (int e = 0; e < 16; ++e) a[e & 3] += pr[e];
                        run += (a[0] + a[1]) + (a[2] + a[3]);
                    } else {
                        float a = 0.0f, a2 = 0.0f;  // diagonals `lane` and `lane` + 32: distances d0 + lane, d0 + lane + 32
#pragma unroll
                        for (int e = 0; e < 16; ++e) {  // key e meets diagonal t at query t - 15 + e, and diagonal t + 32 at the same lane's number modulo 32
                            const float x = __shfl_sync(0xffffffffu, pr[e], (lane + 17 + e) & 31);
                            if (lane - 15 + e >= 0) a += x;
                            else a2 += x;
                        }
                        // sums of the first x diagonals, in order; a bucket is a difference of two of them
#pragma unroll
                        for (int x = 1; x < 32; x <<= 1) {
                            const float y = __shfl_up_sync(0xffffffffu, a, x), y2 = __shfl_up_sync(0xffffffffu, a2, x);
                            if (lane >= x) { a += y; a2 += y2; }
                        }
                        a2 += __shfl_sync(0xffffffffu, a, 31);
                        auto first = [&](int x) {  // x from 0 to 47
                            const float y = __shfl_sync(0xffffffffu, a, (x - 1) & 31), y2 = __shfl_sync(0xffffffffu, a2, (x - 1) & 31);
                            return x == 0 ? 0.0f : x <= 32 ? y : y2;
                        };
                        auto edge = [&](int bucket) { return bucket < p.rule.buckets ? max(0, min(47, p.rule.starts[bucket] - d0)) : 47; };
                        sum0 += first(edge(lane + 1)) - first(edge(lane));
                        if (p.rule.buckets > 32) sum1 += first(edge(lane + 33)) - first(edge(lane + 32));
                    }
                }
            }
            good = good && ready_wait(dq_done(n - 1u), two(n - 1u), p.status, 68);  // the last product of all
            after_sync();
            if (wants_dbias) {
                settle();
                sums[(warp - 12) * 64 + lane] = sum0;
                sums[(warp - 12) * 64 + 32 + lane] = sum1;
            }
            if (16 * part < DP) place_result(gen, row, 16 * part, lanes + 256 + 16 * part, moved, cnt > WT_FLUSH, p.scale);
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            if (all_any(!good)) break;  // all of them leave together
            if (wants_dbias && warp == 12) {  // before the next item's dO takes their place
                float t[2] = {0.f, 0.f};
#pragma unroll
                for (int x = 0; x < 16; ++x) { t[0] += sums[x * 64 + lane]; t[1] += sums[x * 64 + 32 + lane]; }
                float* part_out = p.dbias_part + (((int64_t)it.b * p.H + it.h) * p.units + it.unit) * p.rule.buckets;
#pragma unroll
                for (int x = 0; x < 2; ++x)
                    if (lane + 32 * x < p.rule.buckets) part_out[lane + 32 * x] = t[x];
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                __syncwarp();
            }
            if (threadIdx.x == 384) {
                own_store<DP>(&map_dq, base, p, r0, it.h, it.b);
                tma_store_commit();
                tma_store_wait_read<0>();
                fetch(w + gridDim.x);
            }
        }
        if (threadIdx.x == 384) tma_store_wait_all();
    }
    tmem_give(tmem, warp);
}

// ---- host side ----------------------------------------------------------------------------------------------------------------
static WindowTc operands(gcb_ctx* ctx, int64_t B, const WindowAttn& a, int tiles_per_unit) {
    WindowTc p = {};
    p.q = a.q; p.q_ld = a.q_ld; p.q_so = a.q_so; p.q_si = a.q_si;
    p.k = a.k; p.k_ld = a.k_ld; p.k_so = a.k_so; p.k_si = a.k_si;
    p.v = a.v; p.v_ld = a.v_ld; p.v_so = a.v_so; p.v_si = a.v_si;
    p.g = a.g; p.g_ld = a.g_ld; p.g_so = a.g_so; p.g_si = a.g_si;
    p.o = a.o; p.o_ld = a.o_ld; p.o_so = a.o_so; p.o_si = a.o_si;
    p.dq = a.dq; p.dk = a.dk; p.dv = a.dv; p.d_ld = a.d_ld; p.d_so = a.d_so; p.d_si = a.d_si;
    p.out = a.out; p.row_max = a.row_max; p.row_inv = a.row_inv; p.dbias_part = a.dbias_part;
    p.delta = a.delta; p.tab = a.tab; p.tab_len = a.tab_len; p.scale = a.scale; p.T = a.T; p.D = a.D; p.rule = a.rule; p.status = ctx->d_status;
    plan(p, B, a.H, a.T, tiles_per_unit);
    // Heads are taken all together, the heaviest tiles of every one first, so that the lightest are left for the end; not where every tile goes back to the first keys
    // and k and v of all heads are more than the L2 cache holds, 126 MB: groups of heads then stay in it (kernels as they are here and in groups, us: 16 x 16 x 1024 x 64,
    // window 256, forward 212 and 220, dQ 252 and 274, dK and dV 266 and 350; 8 x 12 x 512, no window, 45, 56, 68 and 45, 60, 83; 16 x 16 x 1024, no window, 254, 305,
    // 373 and 248, 303, 372).
    if (a.rule.W > 0 || 2 * sizeof(float) * p.heads * (int64_t)a.T * a.D <= (int64_t(126) << 20)) p.group = p.heads;
    return p;
}
template <class K, class... Maps>
static int tc_launch(gcb_ctx* ctx, K kernel, bool* done, unsigned threads, size_t smem, const WindowTc& p, const Maps&... maps) {
    if (!done[ctx->device]) { GCB_CHECK_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem)); done[ctx->device] = true; }
    GCB_CHECK_CUDA(launch_chained(ctx->stream, dim3((unsigned)std::min<int64_t>(p.items, kSMs)), threads, smem, kernel, maps..., p));
    return GCB_OK;
}
template <int DP, bool BIAS>
static int run_fwd(gcb_ctx* ctx, const WindowTc& p, const CUtensorMap& k, const CUtensorMap& v, const CUtensorMap& q, const CUtensorMap& o) {
    static bool done[kMaxDevices] = {};
    return tc_launch(ctx, window_attention_tc_fwd_kernel<DP, BIAS>, done, AT_FWD_THREADS, AttnSmem<DP>::TOTAL, p, k, v, q, o);
}
struct BwdMaps {
    CUtensorMap kk, vk, kn, qk, qn, ok, on, dq, dk, dv;
};
template <int DP, bool BIAS>
static int run_bwd(gcb_ctx* ctx, const WindowTc& p, const BwdMaps& m) {
    static bool done_q[kMaxDevices] = {}, done_kv[kMaxDevices] = {};
    int rc = tc_launch(ctx, window_attention_tc_dq_kernel<DP, BIAS>, done_q, AT_BWD_THREADS, DqSmem<DP, BIAS>::TOTAL, p, m.kk, m.vk, m.kn, m.qk, m.ok, m.dq);
    if (!rc) rc = after_launch(ctx, "window_attention_tc_dq");
    if (!rc) rc = tc_launch(ctx, window_attention_tc_dkv_kernel<DP, BIAS>, done_kv, AT_BWD_THREADS, DkvSmem<DP, BIAS>::TOTAL, p, m.qk, m.qn, m.ok, m.on, m.kk, m.vk, m.dk, m.dv);
    return rc ? rc : after_launch(ctx, "window_attention_tc_dkv");
}
// Room for the sums that leave tensor memory before an item's end, where an item may have more than `blocks` blocks.
static int make_moved(WindowTc& p, Scratch& mem, int blocks) {
    if (p.T <= blocks * AT_KEYS) return GCB_OK;
    const int rc = mem.get((size_t)std::min<int64_t>(p.items, kSMs) * 2 * 64 * AT_ROWS * sizeof(float));
    p.moved = mem.as<float>();
    return rc;
}

// Short sequences that the FMA kernels do sooner: up to 32 positions, up to 64 where every SM has a tile of 32 at most, up to 128 where a quarter of them has
// (forward and backward, us, there and here: 64 x 12 x 32 x 64 25 and 86, 41 and 94; 4 x 4 x 64 x 32, window 16 and 2 sinks, 5.2 and 8.0, 7.1 and 22.7; 1 x 4 x 64 x 64
// 5.9 and 9.5, 7.7 and 18.4; 16 x 4 x 64 x 64 9.9 and 13.3, 8.2 and 20.8; 32 x 4 x 64 x 64 11.7 and 23.3, 8.8 and 21.8; 64 x 12 x 64 x 64 34 and 125, 41 and 106;
// 1 x 4 x 128 x 64 10.3 and 16.8, 10.7 and 22.5; 4 x 4 x 128 x 64 12.5 and 17.1, 10.9 and 23.8; 4 x 12 x 128 x 64 18.4 and 31.1, 10.9 and 24.0).
static bool short_enough(int64_t heads, int T) {
    const int64_t tiles = heads * ((T + 31) / 32);
    return T <= 32 || (T <= 64 && tiles <= kSMs) || (T <= 128 && 4 * tiles <= kSMs);
}
// Heads of up to 64 columns (tensor memory holds two query tiles of that width), the split arithmetic of mode 2, rows that TMA can address: strides that grow, so that one k and v for
// all heads or sequences (a stride of 0), or rows backwards, go to the FMA kernels.
bool window_tc_takes(gcb_ctx* ctx, int64_t B, const WindowAttn& a) {
    if (ctx->gemm_engine == 1 || ctx->gemm_split_mode != 2 || a.D > 64 || a.D % 4 != 0 || !(a.scale > 0.0f) || a.scale > 1e30f) return false;
    if (ctx->gemm_engine == 0 && short_enough(B * a.H, a.T)) return false;
    if (!rows_ok(a.q, a.q_ld, a.q_so, a.q_si, B, a.H) || !rows_ok(a.k, a.k_ld, a.k_so, a.k_si, B, a.H) || !rows_ok(a.v, a.v_ld, a.v_so, a.v_si, B, a.H)) return false;
    if (a.out && !rows_ok(a.out, a.o_ld, a.o_so, a.o_si, B, a.H)) return false;
    if (a.g && (!rows_ok(a.g, a.g_ld, a.g_so, a.g_si, B, a.H) || !rows_ok(a.o, a.o_ld, a.o_so, a.o_si, B, a.H) || !rows_ok(a.dq, a.d_ld, a.d_so, a.d_si, B, a.H) || !rows_ok(a.dk, a.d_ld, a.d_so, a.d_si, B, a.H) ||
                !rows_ok(a.dv, a.d_ld, a.d_so, a.d_si, B, a.H)))
        return false;
    return B * a.H * ((a.T + 127) / 128) < (int64_t(1) << 30) && tma_encode(ctx) != nullptr;
}

int window_tc_fwd(gcb_ctx* ctx, int64_t B, const WindowAttn& a) {
    TmaEncodeFn enc = tma_encode(ctx);
    // two query tiles share their key blocks; one tile a CTA where pairs would leave SMs idle (in pairs and one by one, us: 16 x 16 x 1024, window 256, 205 and 273;
    // 1 x 12 x 4099, window 512, 89 and 99; 2 x 12 x 1024 48 and 46; 1 x 4 x 512 27 and 25; 3 x 12 x 700 36 and 36)
    WindowTc p = operands(ctx, B, a, B * a.H * ((a.T + 255) / 256) < kSMs ? 1 : 2);
    Scratch moved(ctx);
    int rc = make_moved(p, moved, 1);
    if (rc) return rc;
    CUtensorMap k, v, q, o;
    GCB_REQUIRE(encode_rows(enc, &k, a.k, a.D, a.T, a.k_ld, a.k_si, a.k_so, a.H, B, 32, AT_KEYS, CU_TENSOR_MAP_SWIZZLE_128B) &&
                    encode_rows(enc, &q, a.q, a.D, a.T, a.q_ld, a.q_si, a.q_so, a.H, B, 32, AT_KEYS, CU_TENSOR_MAP_SWIZZLE_128B) &&
                    encode_rows(enc, &o, a.out, a.D, a.T, a.o_ld, a.o_si, a.o_so, a.H, B, 32, AT_KEYS, CU_TENSOR_MAP_SWIZZLE_128B) &&
                    encode_rows(enc, &v, a.v, a.D, a.T, a.v_ld, a.v_si, a.v_so, a.H, B, 32, AT_KEYS, CU_TENSOR_MAP_SWIZZLE_128B_ATOM_32B),
                "window attention: strides beyond what TMA can address");
    rc = p.tab ? (a.D <= 32 ? run_fwd<32, true>(ctx, p, k, v, q, o) : run_fwd<64, true>(ctx, p, k, v, q, o)) : (a.D <= 32 ? run_fwd<32, false>(ctx, p, k, v, q, o) : run_fwd<64, false>(ctx, p, k, v, q, o));
    return rc ? rc : after_launch(ctx, "window_attention_tc_fwd");
}

// a.dbias_part: [head][tile of 128 queries][bucket], or NULL.
int window_tc_bwd(gcb_ctx* ctx, int64_t B, const WindowAttn& a) {
    TmaEncodeFn enc = tma_encode(ctx);
    WindowTc p = operands(ctx, B, a, 1);
    Scratch moved(ctx);
    const int rc = make_moved(p, moved, WT_FLUSH);
    if (rc) return rc;
    BwdMaps m;
    auto rows = [&](CUtensorMap& map, const float* x, int64_t ld, int64_t so, int64_t si, bool k_major) {
        return encode_rows(enc, &map, x, a.D, a.T, ld, si, so, a.H, B, 32, AT_KEYS, k_major ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_128B_ATOM_32B);
    };
    GCB_REQUIRE(rows(m.kk, a.k, a.k_ld, a.k_so, a.k_si, true) && rows(m.kn, a.k, a.k_ld, a.k_so, a.k_si, false) && rows(m.vk, a.v, a.v_ld, a.v_so, a.v_si, true) && rows(m.qk, a.q, a.q_ld, a.q_so, a.q_si, true) &&
                    rows(m.qn, a.q, a.q_ld, a.q_so, a.q_si, false) && rows(m.ok, a.g, a.g_ld, a.g_so, a.g_si, true) && rows(m.on, a.g, a.g_ld, a.g_so, a.g_si, false) &&
                    rows(m.dq, a.dq, a.d_ld, a.d_so, a.d_si, true) && rows(m.dk, a.dk, a.d_ld, a.d_so, a.d_si, true) && rows(m.dv, a.dv, a.d_ld, a.d_so, a.d_si, true),
                "window attention: strides beyond what TMA can address");
    if (p.tab) return a.D <= 32 ? run_bwd<32, true>(ctx, p, m) : run_bwd<64, true>(ctx, p, m);
    return a.D <= 32 ? run_bwd<32, false>(ctx, p, m) : run_bwd<64, false>(ctx, p, m);
}

}  // namespace gcb
