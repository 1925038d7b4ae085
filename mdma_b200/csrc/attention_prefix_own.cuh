// Single tokens behind shared prefixes, as streams of keys (bfloat16, pages of a multiple of 32 tokens, up to 16 query heads a kv
// head): every sequence's own keys with the join of its prefix's parts, and prefixes that few rows share.
//
// A block takes one (sequence, kv head): the query heads of the group are the rows of one 16-row tile on mma.sync, its warps take
// the key tiles in turn, each with a running maximum, sum and output of its own and with its next key tile on the way (TMA)
// while it multiplies with the values.  It is bound by memory: every key and value is read once.  The kernel of the prefixes
// runs beside it; only when the own keys are done does the block wait for that kernel, and joins the warps' sums, the
// prefix's parts (in their order) and the sink.  With `own_splits` > 1 a block takes a piece of the own keys and leaves its sums for
// the merge.  Without pieces (`pieces` 0) nothing is shared: a sequence's own keys are all it sees.
//
// SHARED: the same over a piece of a prefix, the 16 rows those of several members; every block leaves its sums.
#pragma once
#include "mma_tiles.cuh"
#include "prefix.cuh"
#include "ptx.cuh"

namespace mdma {

constexpr int kPoMaxPieces = 32;

template <int DMAX, int KB, int NW>
struct PoSmem {
    static constexpr int kTile = KB * DMAX * 2, kRow = DMAX + 8;                      // bytes of a tile; floats of a warp's row of sums
    static constexpr int kTiles = NW * 2 * kTile, kComb = NW * 16 * kRow * 4;
    static constexpr int kQ = kTiles > kComb ? kTiles : kComb, kBars = kQ + 16 * DMAX * 2, kTop = kBars + NW * 16 + 16;
    static constexpr int kBytes = kTop + (3 * NW + kPoMaxPieces + 3) * 16 * 4;
};

template <int DMAX, int KB, int NW, bool SHARED>
__global__ void __launch_bounds__(NW * 32, NW >= 8 ? 1 : NW == 4 ? 3 : NW == 3 ? 4 : 5)
prefix_stream_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, const PrefixParams p) {
    using L = PoSmem<DMAX, KB, NW>;
    constexpr int kChunks = DMAX / 8, kHalf = KB * 128;
    extern __shared__ __align__(1024) uint8_t smem[];
    const uint32_t s0 = (uint32_t)__cvta_generic_to_shared(smem);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t sK = s0 + warp * 2 * L::kTile, sV = sK + L::kTile, sQ = s0 + L::kQ;
    const uint32_t kbar = s0 + L::kBars + warp * 16, vbar = kbar + 8;
    volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + L::kBars + NW * 16);
    auto kv_offset = [](int row, int chunk) -> uint32_t {        // 16-byte chunk of a key row inside a tile
        return (uint32_t)((chunk >> 3) * kHalf + row * 128 + (((chunk & 7) ^ (row & 7)) << 4));
    };
    // (the kernel of the prefixes lets the next one start only when it has waited itself: that one counts on it)
    if (SHARED || p.pieces == 0) chain_wait();
    chain_release();
    if (threadIdx.x == 0) {
        for (int w = 0; w < NW; ++w) { ptx::mbar_init(s0 + L::kBars + w * 16, 1); ptx::mbar_init(s0 + L::kBars + w * 16 + 8, 1); }
        *abort_flag = (s0 & 1023u) ? 1 : 0;
        ptx::fence_mbar_init();
    }
    __syncthreads();
    const int kvh = blockIdx.x % p.n_kv_heads, split = blockIdx.x / p.n_kv_heads;
    const int D = p.head_dim, G = p.group, d_chunks = D / 8, halves = (D + 63) / 64;
    int seq, token = 0, skip = 0, lo, hi, rows = G;                                   // keys [lo, hi) for so many rows
    PrefixTile tile = {};
    if (SHARED) {
        if (!prefix_tile(p, blockIdx.y, 16 / G, tile)) return;
        const int keys = prefix_piece(tile.len, p.pieces, p.unit);
        seq = p.group_seq[tile.g]; lo = split * keys; hi = min(tile.len, lo + keys); rows = tile.count * G;
        if (lo >= hi) return;
    } else {
        seq = blockIdx.y;
        const int end = p.seq_pos0[seq] + 1;
        token = seq;                                             // (every sequence brings one)
        skip = p.pieces > 0 ? p.seq_skip[seq] : 0;
        own_piece(p, skip, end, split, KB, lo, hi);
    }
    const int* pages = p.page_table + (size_t)p.seq_slot[seq] * p.max_pages;
    // the token of a row of the tile
    auto token_of = [&](int r) { return SHARED ? p.toks[tile.first + r / G] : token; };
    const int b1 = hi > lo ? (hi - 1) / KB + 1 : 0;
    int blk = lo / KB + warp;
    auto load_tile = [&](const CUtensorMap* map, uint32_t dst, uint32_t bar, int at) {      // one lane
        const int key0 = at * KB, page = pages[key0 / p.page_size], row = key0 % p.page_size;
        ptx::fence_proxy_async_shared();
        ptx::mbar_expect_tx(bar, halves * kHalf);
        for (int h = 0; h < halves; ++h) ptx::tma_load_4d(dst + h * kHalf, map, bar, h * 64, kvh, row, page);
    };
    if (*abort_flag != 0) blk = b1;
    if (blk < b1 && lane == 0) { load_tile(&map_k, sK, kbar, blk); load_tile(&map_v, sV, vbar, blk); }
    const __nv_bfloat16* q = reinterpret_cast<const __nv_bfloat16*>(p.q);
    for (int i = threadIdx.x; i < 16 * kChunks; i += NW * 32) {  // query rows: zeros beyond the group and the head size
        const int r = i / kChunks, c = i % kChunks;
        const bool valid = r < rows && c < d_chunks;
        cp_async_16(sQ + tile_offset<DMAX>(r, c), valid ? q + (size_t)token_of(r) * p.q_stride + (size_t)(kvh * G + r % G) * D + c * 8 : q, valid);
    }
    cp_async_commit();
    cp_async_wait<0>();
    __syncthreads();
    uint32_t qf[DMAX / 16][4];
#pragma unroll
    for (int kd = 0; kd < DMAX / 16; ++kd)
        ldmatrix_x4(sQ + tile_offset<DMAX>(lane & 15, kd * 2 + (lane >> 4)), qf[kd][0], qf[kd][1], qf[kd][2], qf[kd][3]);
    float o[DMAX / 8][4];
#pragma unroll
    for (int n = 0; n < DMAX / 8; ++n) { o[n][0] = o[n][1] = o[n][2] = o[n][3] = 0.f; }
    float m_lo = -INFINITY, m_hi = -INFINITY, l_lo = 0.f, l_hi = 0.f;
    uint32_t phase = 0;
    for (; blk < b1; blk += NW, phase ^= 1u) {
        if (!__all_sync(0xffffffffu, ptx::mbar_wait(kbar, phase, abort_flag))) break;
        float s[KB / 8][4];
#pragma unroll
        for (int n = 0; n < KB / 8; ++n) { s[n][0] = s[n][1] = s[n][2] = s[n][3] = 0.f; }
#pragma unroll
        for (int kd = 0; kd < DMAX / 16; ++kd) {
            if (kd * 16 < D) {
#pragma unroll
                for (int n2 = 0; n2 < KB / 16; ++n2) {
                    uint32_t k0, k1, k2, k3;
                    const int krow = n2 * 16 + (lane & 7) + ((lane >> 4) << 3);
                    ldmatrix_x4(sK + kv_offset(krow, kd * 2 + ((lane >> 3) & 1)), k0, k1, k2, k3);
                    mma_16816(s[n2 * 2], qf[kd][0], qf[kd][1], qf[kd][2], qf[kd][3], k0, k1);
                    mma_16816(s[n2 * 2 + 1], qf[kd][0], qf[kd][1], qf[kd][2], qf[kd][3], k2, k3);
                }
            }
        }
        __syncwarp();
        const bool more = blk + NW < b1;
        if (more && lane == 0) load_tile(&map_k, sK, kbar, blk + NW);                 // the key buffer is free
        float mx_lo = m_lo, mx_hi = m_hi;
#pragma unroll
        for (int n = 0; n < KB / 8; ++n) {
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const int key = blk * KB + n * 8 + (lane & 3) * 2 + e;
                const bool seen = key >= lo && key < hi;
                s[n][e] = seen ? s[n][e] * p.scale_log2 : -INFINITY;
                s[n][2 + e] = seen ? s[n][2 + e] * p.scale_log2 : -INFINITY;
                mx_lo = fmaxf(mx_lo, s[n][e]); mx_hi = fmaxf(mx_hi, s[n][2 + e]);
            }
        }
        mx_lo = fmaxf(mx_lo, __shfl_xor_sync(0xffffffffu, mx_lo, 1)); mx_lo = fmaxf(mx_lo, __shfl_xor_sync(0xffffffffu, mx_lo, 2));
        mx_hi = fmaxf(mx_hi, __shfl_xor_sync(0xffffffffu, mx_hi, 1)); mx_hi = fmaxf(mx_hi, __shfl_xor_sync(0xffffffffu, mx_hi, 2));
        const float ref_lo = mx_lo == -INFINITY ? 0.f : mx_lo, ref_hi = mx_hi == -INFINITY ? 0.f : mx_hi;
        const float corr_lo = exp2f(m_lo - ref_lo), corr_hi = exp2f(m_hi - ref_hi);
        m_lo = mx_lo; m_hi = mx_hi;
        float sum_lo = 0.f, sum_hi = 0.f;
        uint32_t pa[KB / 16][4];                                 // the weights are rounded to bfloat16 for the second product
#pragma unroll
        for (int n = 0; n < KB / 8; ++n) {
            const float p0 = exp2f(s[n][0] - ref_lo), p1 = exp2f(s[n][1] - ref_lo), p2 = exp2f(s[n][2] - ref_hi), p3 = exp2f(s[n][3] - ref_hi);
            sum_lo += p0 + p1; sum_hi += p2 + p3;
            pa[n >> 1][(n & 1) * 2] = pack_bf16(p0, p1);
            pa[n >> 1][(n & 1) * 2 + 1] = pack_bf16(p2, p3);
        }
        l_lo = l_lo * corr_lo + sum_lo; l_hi = l_hi * corr_hi + sum_hi;
#pragma unroll
        for (int n = 0; n < DMAX / 8; ++n) { o[n][0] *= corr_lo; o[n][1] *= corr_lo; o[n][2] *= corr_hi; o[n][3] *= corr_hi; }
        if (!__all_sync(0xffffffffu, ptx::mbar_wait(vbar, phase, abort_flag))) break;
        {
            // a tile is fetched whole: value rows of keys outside [lo, hi) are cleared, they may not be finite (the first and the last tile)
            const int r_lo = lo - blk * KB, r_hi = hi - blk * KB;
            if (r_lo > 0 || r_hi < KB) {
                for (int i = lane; i < halves * KB * 8; i += 32) {
                    const int h = i / (KB * 8), r = (i >> 3) % KB, c = i & 7;
                    if (r < r_lo || r >= r_hi)
                        asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(sV + h * kHalf + r * 128 + c * 16), "r"(0u) : "memory");
                }
                __syncwarp();
            }
        }
#pragma unroll
        for (int kk = 0; kk < KB / 16; ++kk) {
#pragma unroll
            for (int n2 = 0; n2 < DMAX / 16; ++n2) {
                if (n2 * 16 < D) {
                    uint32_t v0, v1, v2, v3;
                    const int vrow = kk * 16 + (lane & 7) + (((lane >> 3) & 1) << 3);
                    ldmatrix_x4_trans(sV + kv_offset(vrow, n2 * 2 + (lane >> 4)), v0, v1, v2, v3);
                    mma_16816(o[n2 * 2], pa[kk][0], pa[kk][1], pa[kk][2], pa[kk][3], v0, v1);
                    mma_16816(o[n2 * 2 + 1], pa[kk][0], pa[kk][1], pa[kk][2], pa[kk][3], v2, v3);
                }
            }
        }
        __syncwarp();
        if (more && lane == 0) load_tile(&map_v, sV, vbar, blk + NW);
    }
    l_lo += __shfl_xor_sync(0xffffffffu, l_lo, 1); l_lo += __shfl_xor_sync(0xffffffffu, l_lo, 2);
    l_hi += __shfl_xor_sync(0xffffffffu, l_hi, 1); l_hi += __shfl_xor_sync(0xffffffffu, l_hi, 2);

    // ---- join: the warps in their order, then the prefix's parts in theirs and what the warps made behind them (as the merge
    // kernel joins them, so that it does not matter to a sequence which of the two does) -------------------------------
    __syncthreads();                                             // the tiles are read: their place takes the warps' sums
    float* comb = reinterpret_cast<float*>(smem);
    float* top = reinterpret_cast<float*>(smem + L::kTop);       // [NW][16] maxima, [NW][16] sums of the warps
    float* share = top + 2 * NW * 16;                            // [NW + pieces + 1][16] shares of the warps, of the prefix's parts and of the own keys
    float *row_m = share + (NW + kPoMaxPieces + 1) * 16, *row_l = row_m + 16;
    {
        float* mine = comb + (size_t)warp * 16 * L::kRow;
        const int r_lo = lane >> 2, r_hi = r_lo + 8;
#pragma unroll
        for (int n = 0; n < DMAX / 8; ++n) {
            const int d = n * 8 + (lane & 3) * 2;
            if (r_lo < rows) *reinterpret_cast<float2*>(mine + r_lo * L::kRow + d) = make_float2(o[n][0], o[n][1]);
            if (r_hi < rows) *reinterpret_cast<float2*>(mine + r_hi * L::kRow + d) = make_float2(o[n][2], o[n][3]);
        }
        if ((lane & 3) == 0) {
            top[warp * 16 + r_lo] = m_lo; top[(NW + warp) * 16 + r_lo] = l_lo;
            top[warp * 16 + r_hi] = m_hi; top[(NW + warp) * 16 + r_hi] = l_hi;
        }
    }
    const bool joins = !SHARED && p.own_splits == 1;
    const int used = joins && p.pieces > 0 ? prefix_pieces_used(skip, p.pieces, p.unit) : 0, slots = p.pieces + p.own_splits;
    auto row_of = [&](int r) { return (size_t)token_of(r) * p.n_heads + kvh * G + r % G; };
    if (!SHARED) chain_wait();                                   // the prefixes' parts are there, and all that was waited for before them
    __syncthreads();
    // a warp a row: the warps' maxima, shares and sum (a lane a warp), then those of the prefix's parts and the own keys (a lane a
    // contribution, up to two)
    for (int r = warp; r < rows; r += NW) {
        const float2* ml = reinterpret_cast<const float2*>(p.part_ml) + row_of(r) * slots;
        float2 part[2];
#pragma unroll
        for (int u = 0; u < 2; ++u) part[u] = u * 32 + lane < used ? __ldcg(ml + u * 32 + lane) : make_float2(-INFINITY, 0.f);
        const float2 mine = lane < NW ? make_float2(top[lane * 16 + r], top[(NW + lane) * 16 + r]) : make_float2(-INFINITY, 0.f);
        float m = warp_max(mine.x);
        const float f = prefix_share(mine, m);
        float l = warp_sum(prefix_joins(f) ? f * mine.y : 0.f);
        if (lane < NW) share[lane * 16 + r] = f;
        if (joins) {
            const float2 own = make_float2(m, l);
#pragma unroll
            for (int u = 0; u < 2; ++u) if (u * 32 + lane == used) part[u] = own;
            m = warp_max(fmaxf(part[0].x, part[1].x));
            l = 0.f;
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const float g = prefix_share(part[u], m);
                if (prefix_joins(g)) l += g * part[u].y;
                if (u * 32 + lane <= used) share[(NW + u * 32 + lane) * 16 + r] = g;
            }
            l = warp_sum(l);
            if (p.sinks) l += exp2f(p.sinks[kvh * G + r % G] * p.sink_rate - m);
        }
        if (lane == 0) { row_m[r] = m; row_l[r] = l; }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < rows * (D / 4); i += NW * 32) {
        const int r = i / (D / 4), d = 4 * (i - r * (D / 4));
        const float l = row_l[r];
        auto join = [&](float f, const float4& x, float4& acc) {
            if (prefix_joins(f)) { acc.x = fmaf(f, x.x, acc.x); acc.y = fmaf(f, x.y, acc.y); acc.z = fmaf(f, x.z, acc.z); acc.w = fmaf(f, x.w, acc.w); }
        };
        const size_t row = row_of(r);
        const float* part = p.part_o + row * slots * D + d;
        float4 x[8];
        auto fetch = [&](int s0) {                               // eight parts in flight
#pragma unroll
            for (int u = 0; u < 8; ++u) x[u] = __ldcg(reinterpret_cast<const float4*>(part + (size_t)min(s0 + u, used - 1) * D));
        };
        if (used > 0) fetch(0);
        float4 own = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < NW; ++w) join(share[w * 16 + r], *reinterpret_cast<const float4*>(comb + ((size_t)w * 16 + r) * L::kRow + d), own);
        if (joins) {
            float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
            for (int s0 = 0; s0 < used; s0 += 8) {
                if (s0 > 0) fetch(s0);
#pragma unroll
                for (int u = 0; u < 8; ++u) if (s0 + u < used) join(share[(NW + s0 + u) * 16 + r], x[u], acc);
            }
            join(share[(NW + used) * 16 + r], own, acc);
            __nv_bfloat162 y[2] = {__floats2bfloat162_rn(acc.x / l, acc.y / l), __floats2bfloat162_rn(acc.z / l, acc.w / l)};
            *reinterpret_cast<uint2*>(reinterpret_cast<__nv_bfloat16*>(p.out) + row * D + d) = *reinterpret_cast<const uint2*>(y);
        } else {
            const size_t slot = row * slots + (SHARED ? 0 : p.pieces) + split;
            *reinterpret_cast<float4*>(p.part_o + slot * D + d) = own;
            if (d == 0) *reinterpret_cast<float2*>(p.part_ml + slot * 2) = make_float2(row_m[r], l);
        }
    }
    if (threadIdx.x == 0 && *abort_flag && p.status) atomicExch(p.status, 8);
}

}  // namespace mdma
