// The tcgen05 kernel of attention over shared prefixes (bfloat16, pages of a multiple of 64 tokens).
//
// A block takes up to 256 query rows of one kv head, two tiles of 128 (token, query head of the group) rows whose tokens may be of
// several members of a group, and walks a list of key blocks of 128:
//     S = Q K^T    tcgen05.mma, M = N = 128, operands from shared memory (keys by TMA, 128-byte swizzle), S in tensor memory
//     softmax      128 threads a tile, a row a thread: the row out of tensor memory, mask, running maximum and sum in float, the
//                  weights rounded to bfloat16 and written back over S, 64 keys at a time
//     O += P V     tcgen05.mma, A = P from tensor memory, V as the cache holds it (MN-major), O in tensor memory; the first 64
//                  keys' product runs under the second's exponentials
// The two tiles take turns: while one is in its softmax the tensor pipe works for the other, and both use the same key and
// value blocks.  Tensor memory: S and P of the tiles in columns 0 and 128, O in 256 and 384.  One thread issues all products, a
// tile's P V and its next S one behind the other, so whoever sees S(j) complete knows that P(j-1) V(j-1) is, too, and the
// tiles' S are complete half a period apart.
// The weights are taken against a reference that moves only when a row's maximum has grown by more than 2^8 since; O is
// rescaled only then.
// Measured, cycles a block of 128 keys and both tiles (the tensor pipe's own: 2,048; the exponential unit's as many): 3,400,
// of which a tile's softmax and its products, one behind the other, are the chain.  What was slower or no faster: two threads a
// row (the issue slots of sixteen softmax warps are the bound then) 4,200; a warp that issues for each tile, both in step, 4,850;
// P V behind the whole softmax 3,450; steps of 64 keys with two places for S (products of N = 64 cost as much as of N = 128)
// 3,700; the first half's weights before the row's maximum is known 3,450; a quarter of the exponentials by a polynomial on the
// multiply-add units 3,400; the two tiles' exponentials in turns (a barrier for every pair of warps) 3,650; the next blocks asked into
// L2 ahead, 15% more where they come from memory.
// 8,960 rows a kv head over 8,000 keys, 32 heads of 128: 307 us, 1.04 PFLOP/s; 337 to 351 and 0.91 in long runs, at the power limit.
//
// The list: the prefix's blocks, which all rows see, and (`whole`) behind them the own blocks of every sequence with tokens in the
// tiles, which only that sequence's rows see: the others' lanes of O are left out of the product, so that what they are
// multiplied with does not reach them.  `pieces` blocks share a list; each then leaves its sums for the merge.
//
// The kernel takes all 512 columns of tensor memory and is launched programmatically, which is sound in the order that it
// keeps: it waits for the kernel before it, takes the columns, and only then lets the next one start.  So no block waits for columns
// beside a block that waits for it, and a block needs no other one to be placed.
#pragma once
#include "prefix.cuh"
#include "ptx.cuh"

namespace mdma {

constexpr int kPtRows = 128, kPtKeys = 128, kPtThreads = 320, kPtMaxTokens = 2 * kPtRows;
constexpr int kPtHalf = kPtRows * 128;                           // 128 rows (or keys) x 64 numbers
constexpr int kPtSlot = 2 * kPtHalf;
constexpr int kPtStage = 132;                                   // floats from row to row of results on their way out
constexpr int kPtSmemK = 2 * kPtSlot, kPtSmemV = kPtSmemK + 2 * kPtSlot, kPtSmemBars = kPtSmemV + 2 * kPtSlot;
struct PtSegment { int seq, key0, key1, tok0, toks, block0; };  // keys [key0, key1) for the tile's tokens [tok0, tok0 + toks); its first block
constexpr int kPtSmemSegs = kPtSmemBars + 256;
constexpr int kPtSmem = kPtSmemSegs + (kPtMaxTokens + 4) * (int)sizeof(PtSegment);

// Walks the blocks of a list; what the current segment says is kept in registers.
struct PtWalk {
    const PtSegment* segs;
    int seg, block, next0;                                       // the segment, the block of the list, the next segment's first block
    PtSegment s;
    int key;                                                     // the block's first key (of an own segment's first block: the multiple of 64 below its first key)
    int ra[2], rb[2];                                            // rows [ra, rb) of each tile see the block
    __device__ __forceinline__ PtWalk(const PtSegment* list, int first, int tt, int G) : segs(list), seg(0), block(first) {
        while (first >= segs[seg + 1].block0) ++seg;
        enter(tt, G);
        key += (block - s.block0) * kPtKeys;
    }
    __device__ __forceinline__ void enter(int tt, int G) {
        s = segs[seg];
        next0 = segs[seg + 1].block0;
        key = s.key0 & ~63;
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            ra[t] = max(s.tok0 - t * tt, 0) * G;
            rb[t] = max(min(s.tok0 + s.toks - t * tt, tt), 0) * G;
        }
    }
    __device__ __forceinline__ void next(int tt, int G) {
        key += kPtKeys;
        if (++block < next0) return;
        do ++seg; while (block >= segs[seg + 1].block0);
        enter(tt, G);
    }
    __device__ __forceinline__ bool active(int t) const { return ra[t] < rb[t]; }
    __device__ __forceinline__ int steps() const { return s.key1 - key > 64 ? 2 : 1; }        // of 64 keys
};

// Two products and sums, two sums at once.
__device__ __forceinline__ float2 fma_pair(float2 a, float2 b, float2 c) {
    float2 d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(reinterpret_cast<unsigned long long&>(d))
        : "l"(reinterpret_cast<unsigned long long&>(a)), "l"(reinterpret_cast<unsigned long long&>(b)), "l"(reinterpret_cast<unsigned long long&>(c)));
    return d;
}
__device__ __forceinline__ float2 add_pair(float2 a, float2 b) {
    float2 d;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(reinterpret_cast<unsigned long long&>(d))
        : "l"(reinterpret_cast<unsigned long long&>(a)), "l"(reinterpret_cast<unsigned long long&>(b)));
    return d;
}
__global__ void __launch_bounds__(kPtThreads, 1)
prefix_tc_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, const PrefixParams p) {
    extern __shared__ __align__(1024) uint8_t smem[];
    const uint32_t base = ptx::smem_addr(smem), bars = base + kPtSmemBars;
    auto k_full = [&](int s) { return bars + 8u * s; };
    auto k_empty = [&](int s) { return bars + 8u * (2 + s); };
    auto v_full = [&](int s) { return bars + 8u * (4 + s); };
    auto v_empty = [&](int s) { return bars + 8u * (6 + s); };
    auto s_full = [&](int t) { return bars + 8u * (8 + t); };
    auto p_ready = [&](int t, int half) { return bars + 8u * (10 + 2 * t + half); };
    const uint32_t q_full = bars + 8u * 14;
    volatile uint32_t* tmem_slot = reinterpret_cast<volatile uint32_t*>(smem + kPtSmemBars + 8 * 15);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + kPtSmemBars + 8 * 16);
    int* warp_starts = reinterpret_cast<int*>(smem + kPtSmemBars + 8 * 17);          // [9]
    PtSegment* segs = reinterpret_cast<PtSegment*>(smem + kPtSmemSegs);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int G = p.group, D = p.head_dim, kvh = blockIdx.x, split = blockIdx.z, tt = kPtRows / G;

    chain_wait();
    // ---- which rows, which keys ------------------------------------------------------------------------------------
    PrefixTile tile;
    if (!prefix_tile(p, blockIdx.y, 2 * tt, tile)) return;
    const int count = tile.count, len = tile.len;                // tokens of both tiles; the prefix
    int b0 = 0, b1 = 0;                                          // this block's part of the list
    if (!p.whole) {
        const int keys = prefix_piece(len, p.pieces, p.unit), lo = split * keys, hi = min(len, lo + keys);
        if (lo >= hi) return;
        if (threadIdx.x == 0) {
            segs[0] = {p.group_seq[tile.g], lo, hi, 0, count, 0};
            segs[1].block0 = 0x7fffffff;
        }
        b1 = (hi - lo + kPtKeys - 1) / kPtKeys;
    }
    if (threadIdx.x == 0) {
        for (int s = 0; s < 2; ++s) {
            ptx::mbar_init(k_full(s), 1); ptx::mbar_init(k_empty(s), 1);
            ptx::mbar_init(v_full(s), 1); ptx::mbar_init(v_empty(s), 1);
            ptx::mbar_init(s_full(s), 1);
            for (int h = 0; h < 2; ++h) ptx::mbar_init(p_ready(s, h), 4);        // a tile's four warps
        }
        ptx::mbar_init(q_full, 256);
        *abort_flag = (base & 1023u) ? 1 : 0;                    // the tiles need 1024-byte alignment
        ptx::fence_mbar_init();
    }
    if (warp == 9) { ptx::tmem_alloc(ptx::smem_addr((const void*)tmem_slot), 512); ptx::tmem_relinquish(); }
    ptx::tc_fence_before_sync();
    __syncthreads();
    ptx::tc_fence_after_sync();
    const uint32_t tmem = *tmem_slot;
    // only now: a kernel that starts early behind this one may count on what this one waited for, and finds the tensor memory taken
    chain_release();
    if (p.whole) {
        // a segment starts where the token's sequence differs from that of the token before
        const int t = threadIdx.x;
        int token = 0, seq = -1, before = -1;
        if (t < count) {
            token = p.toks[tile.first + t]; seq = p.tok_seq[token];
            before = t > 0 ? p.tok_seq[p.toks[tile.first + t - 1]] : -1;
        }
        const bool starts = t < count && seq != before;
        const uint32_t mask = __ballot_sync(0xffffffffu, starts);
        if (warp < 8 && lane == 0) warp_starts[warp] = __popc(mask);
        __syncthreads();
        const int shared = len > 0 ? 1 : 0;
        if (starts) {
            int at = shared + __popc(mask & ((1u << lane) - 1u));
            for (int w = 0; w < warp; ++w) at += warp_starts[w];
            const int first = p.seq_start[seq], n = min(p.seq_start[seq + 1] - token, count - t);
            segs[at] = {seq, p.seq_skip[seq], p.seq_pos0[seq] + token - first + n, t, n, 0};
        }
        if (threadIdx.x == 0 && shared) segs[0] = {p.group_seq[tile.g], 0, len, 0, count, 0};
        __syncthreads();
        if (threadIdx.x == 0) {
            int n_segs = shared, at = 0;
            for (int w = 0; w < 8; ++w) n_segs += warp_starts[w];
            for (int s = 0; s < n_segs; ++s) {
                segs[s].block0 = at;
                at += max(segs[s].key1 - (segs[s].key0 & ~63) + kPtKeys - 1, 0) / kPtKeys;
            }
            segs[n_segs].block0 = at;
            segs[n_segs + 1].block0 = 0x7fffffff;
            warp_starts[8] = at;
        }
        __syncthreads();
        const int blocks = warp_starts[8], per = (blocks + p.pieces - 1) / p.pieces;
        b0 = split * per; b1 = min(blocks, b0 + per);
    }
    const bool working = b0 < b1 && !(base & 1023u);
    const int halves = (D + 63) / 64;

    if (working && warp == 8 && lane == 0) {
        // ---- TMA producer: K(0) V(0) K(1) V(1) .. -----------------------------------------------------------------
        PtWalk w(segs, b0, tt, G);
        bool fine = true;
        for (int j = 0; fine && b0 + j < b1; ++j, w.next(tt, G)) {
            const int* pages = p.page_table + (size_t)p.seq_slot[w.s.seq] * p.max_pages;
            const int boxes = w.steps();                         // of 64 keys each
            int page[2], row[2];
            for (int b = 0; b < boxes; ++b) { page[b] = pages[(w.key + 64 * b) / p.page_size]; row[b] = (w.key + 64 * b) % p.page_size; }
            const int s = j & 1;
            const uint32_t phase = ((j >> 1) & 1) ^ 1;
            for (int which = 0; which < 2 && fine; ++which) {
                const uint32_t full = which ? v_full(s) : k_full(s);
                fine = ptx::mbar_wait(which ? v_empty(s) : k_empty(s), phase, abort_flag);
                if (!fine) break;
                ptx::mbar_expect_tx(full, boxes * halves * 64 * 128);
                for (int h = 0; h < halves; ++h)
                    for (int b = 0; b < boxes; ++b)
                        ptx::tma_load_4d(base + (which ? kPtSmemV : kPtSmemK) + s * kPtSlot + h * kPtHalf + b * 64 * 128, which ? &map_v : &map_k,
                                         full, h * 64, kvh, row[b], page[b]);
            }
        }
    } else if (working && warp == 9) {
        // ---- MMA issuer: the whole warp walks, one lane issues (what the instructions take then stays in uniform registers) ----
        const bool lead = ptx::elect_one();
        const uint32_t idesc_s = ptx::idesc_bf16_f32_ex(kPtRows, kPtKeys, 0), idesc_o = ptx::idesc_bf16_f32_ex(kPtRows, D, 1);
        const uint32_t tmem_u = __shfl_sync(0xffffffffu, tmem, 0);
        const int ksteps = D / 16;
        auto product_s = [&](int t, int s) {
            const uint64_t qd = ptx::smem_desc_sw128(base + t * kPtSlot), kd = ptx::smem_desc_sw128(base + kPtSmemK + s * kPtSlot);
            if (lead) {
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    if (i < ksteps) {
                        const uint32_t at = ((i >> 2) * kPtHalf + (i & 3) * 32) >> 4;
                        ptx::mma_bf16_ss(tmem_u + t * 128, qd + at, kd + at, idesc_s, i > 0);
                    }
                ptx::mma_commit(s_full(t));
            }
        };
        auto off_lanes = [](int a, int b, int word) -> uint32_t {             // bits of lanes outside [a, b)
            const int lo = max(a - word * 32, 0), hi = min(b - word * 32, 32);
            if (lo >= hi) return 0xffffffffu;
            const uint32_t on = (hi == 32 ? 0xffffffffu : (1u << hi) - 1u) & ~((1u << lo) - 1u);
            return ~on;
        };
        PtWalk w(segs, b0, tt, G);
        uint32_t done[2][2] = {{0, 0}, {0, 0}};                  // products of the weights of either half, a tile
        bool ok = ptx::mbar_wait(q_full, 0, abort_flag) && ptx::mbar_wait(k_full(0), 0, abort_flag);
        if (ok) {
            ptx::tc_fence_after_sync();
#pragma unroll
            for (int t = 0; t < 2; ++t) if (w.active(t)) product_s(t, 0);
            if (lead) ptx::mma_commit(k_empty(0));
        }
        for (int j = 0; b0 + j < b1 && ok; ++j) {
            const int s = j & 1, steps = w.steps();
            const bool more = b0 + j + 1 < b1;
            // (rows beyond the tiles' tokens take part in the products of what all rows see: nobody reads them)
            const bool all = w.seg == 0 && w.s.toks == count;
            const int ra[2] = {w.ra[0], w.ra[1]}, rb[2] = {w.rb[0], w.rb[1]};
            if (more) w.next(tt, G);
            ok = ptx::mbar_wait(v_full(s), (j >> 1) & 1, abort_flag);
            if (ok && more) ok = ptx::mbar_wait(k_full(s ^ 1), ((j + 1) >> 1) & 1, abort_flag);
            if (!ok) break;
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                if (ra[t] < rb[t]) {
                    const uint32_t o = tmem_u + 256 + t * 128;
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        if (h >= steps) break;
                        ok = ok && ptx::mbar_wait(p_ready(t, h), done[t][h] & 1, abort_flag);
                        if (!ok) break;
                        ++done[t][h];
                        ptx::tc_fence_after_sync();
                        const uint64_t vd = ptx::smem_desc_sw128_mn(base + kPtSmemV + s * kPtSlot + h * 64 * 128, kPtHalf);
                        const uint32_t pa = tmem_u + t * 128 + h * 32;
                        if (lead) {
                            if (all) {
#pragma unroll
                                for (int i = 0; i < 4; ++i) ptx::mma_bf16_ts(o, pa + i * 8, vd + ((i * 16 * 128) >> 4), idesc_o);
                            } else {
                                const uint4 off = make_uint4(off_lanes(ra[t], rb[t], 0), off_lanes(ra[t], rb[t], 1),
                                                             off_lanes(ra[t], rb[t], 2), off_lanes(ra[t], rb[t], 3));
#pragma unroll
                                for (int i = 0; i < 4; ++i) ptx::mma_bf16_ts(o, pa + i * 8, vd + ((i * 16 * 128) >> 4), idesc_o, off);
                            }
                        }
                    }
                    if (!ok) break;
                }
                if (more && w.active(t)) product_s(t, s ^ 1);
            }
            if (ok && lead) {
                ptx::mma_commit(v_empty(s));
                if (more) ptx::mma_commit(k_empty(s ^ 1));
            }
        }
        if (ok && lead) { ptx::mma_commit(s_full(0)); ptx::mma_commit(s_full(1)); }       // the last sums are complete
    } else if (working && warp < 8) {
        // ---- softmax: a row a thread --------------------------------------------------------------------------------
        const int t = warp >> 2, quad = warp & 3, r = quad * 32 + lane;
        const uint32_t lanes = (uint32_t)(quad * 32) << 16, tmem_s = tmem + t * 128 + lanes, tmem_o = tmem + 256 + t * 128 + lanes;
        const int tok = t * tt + r / G;                          // of the block's tokens
        const bool row_valid = r / G < tt && tok < count;
        const int token = row_valid ? p.toks[tile.first + tok] : -1;
        if (t == 0 || count > tt) {
            // the warp's queries into shared memory, 128-byte rows with the 128-byte swizzle, zeros beyond the tile's rows: half a
            // warp a row, all of it in flight (each lane has asked for its own row's token before)
            const __nv_bfloat16* q = reinterpret_cast<const __nv_bfloat16*>(p.q);
            const int c = lane & 15;
            uint4 x[16];
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const int from = 2 * i + (lane >> 4), of = __shfl_sync(0xffffffffu, token, from);
                x[i] = of >= 0 && c * 8 < D ? *reinterpret_cast<const uint4*>(q + (size_t)of * p.q_stride + (size_t)(kvh * G + (quad * 32 + from) % G) * D + c * 8)
                                            : make_uint4(0u, 0u, 0u, 0u);
            }
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const int to = quad * 32 + 2 * i + (lane >> 4);
                if (c < halves * 8) *reinterpret_cast<uint4*>(smem + t * kPtSlot + (c >> 3) * kPtHalf + to * 128 + (((c & 7) ^ (to & 7)) << 4)) = x[i];
            }
            ptx::fence_proxy_async_shared();
        }
        ptx::mbar_arrive(q_full);
        const int pos = p.whole && row_valid ? p.seq_pos0[p.tok_seq[token]] + token - p.seq_start[p.tok_seq[token]] : 0;
        float m_ref = -INFINITY, l = 0.f;
        {
            float zero[32];
#pragma unroll
            for (int j = 0; j < 32; ++j) zero[j] = 0.f;
#pragma unroll
            for (int c = 0; c < 4; ++c) if (c * 32 < D) ptx::tmem_store_32_nowait(tmem_o + c * 32, zero);
            ptx::tmem_store_wait();
        }
        PtWalk w(segs, b0, tt, G);
        uint32_t seen = 0;
        bool ok = true;
        const float2 rate = make_float2(p.scale_log2, p.scale_log2);
        for (int j = 0; b0 + j < b1 && ok; ++j, w.next(tt, G)) {
            const int ra = t == 0 ? w.ra[0] : w.ra[1], rb = t == 0 ? w.rb[0] : w.rb[1];
            if (ra >= rb) continue;
            const int end = w.s.key1 - w.key, steps = w.steps();                     // block rows beyond `end` belong to nobody
            const bool shared = w.seg == 0 && len > 0;
            int c0 = 0, c1 = end;                                // columns of the block that this row sees
            if (!shared) {
                c0 = w.s.key0 - w.key;
                c1 = r >= ra && r < rb ? min(end, pos - w.key + 1) : 0;
            }
            const bool masks = __any_sync(0xffffffffu, c0 > 0 || c1 < kPtKeys);
            const bool mine = shared || (rb > quad * 32 && ra < quad * 32 + 32);       // (a warp none of whose rows sees the block has nothing to do)
            ok = __all_sync(0xffffffffu, ptx::mbar_wait(s_full(t), seen & 1, abort_flag));
            if (!ok) break;
            ptx::tc_fence_after_sync();
            ++seen;
            if (end < steps * 64) {
                // such value rows are cleared before the product reads them: a weight of zero times what is not finite would not be
                // zero (each tile clears them for its own product, the other may be behind; and only now that its scores are
                // there: a tile that many blocks do not concern would otherwise take an earlier block's values for this one's)
                const int s = j & 1;
                ok = __all_sync(0xffffffffu, ptx::mbar_wait(v_full(s), (j >> 1) & 1, abort_flag));
                if (!ok) break;
                for (int e = threadIdx.x & 127; e < halves * kPtKeys * 8; e += 128) {
                    const int h = e / (kPtKeys * 8), kr = (e >> 3) % kPtKeys, c = e & 7;
                    if (kr >= end) *reinterpret_cast<uint4*>(smem + kPtSmemV + s * kPtSlot + h * kPtHalf + kr * 128 + c * 16) = make_uint4(0u, 0u, 0u, 0u);
                }
                ptx::fence_proxy_async_shared();
            }
            // twice over the row, 64 keys at a time (as straight code with the whole row in registers it spilled and was 2% slower)
            float2 sum = make_float2(0.f, 0.f), sum2 = make_float2(0.f, 0.f);
            float2 off = make_float2(0.f, 0.f);
            auto scores = [&](int h, float* sv) {                // the row's scores of 64 keys, unseen ones taken out
                ptx::tmem_load_32_nowait(tmem_s + h * 64, sv);
                ptx::tmem_load_32_nowait(tmem_s + h * 64 + 32, sv + 32);
                ptx::tmem_load_wait();
                if (masks) {
#pragma unroll
                    for (int i = 0; i < 64; ++i) if (h * 64 + i < c0 || h * 64 + i >= c1) sv[i] = -INFINITY;
                }
            };
            if (mine) {
                float mx = -INFINITY;
#pragma unroll 1
                for (int h = 0; h < steps; ++h) {
                    float sv[64];
                    scores(h, sv);
                    float m4[4] = {mx, sv[0], sv[1], sv[2]};
#pragma unroll
                    for (int i = 3; i < 59; i += 8) {
#pragma unroll
                        for (int q = 0; q < 4; ++q) m4[q] = fmaxf(fmaxf(m4[q], sv[i + 2 * q]), sv[i + 2 * q + 1]);
                    }
                    m4[0] = fmaxf(fmaxf(m4[0], sv[59]), sv[60]); m4[1] = fmaxf(fmaxf(m4[1], sv[61]), sv[62]);
                    m4[2] = fmaxf(m4[2], sv[63]);
                    mx = fmaxf(fmaxf(m4[0], m4[1]), fmaxf(m4[2], m4[3]));
                }
                mx *= p.scale_log2;                              // scale > 0
                float corr = 1.f;
                if (mx > m_ref + 8.f) {
                    corr = m_ref == -INFINITY ? 0.f : ptx::ex2_approx(m_ref - mx);
                    m_ref = mx;
                    l *= corr;
                }
                if (seen > 1 && __any_sync(0xffffffffu, corr != 1.f)) {              // rare: rescale these rows of O
#pragma unroll
                    for (int c = 0; c < 4; ++c) {
                        if (c * 32 < D) {
                            float v[32];
                            ptx::tmem_load_32_nowait(tmem_o + c * 32, v);
                            ptx::tmem_load_wait();
#pragma unroll
                            for (int i = 0; i < 32; ++i) v[i] *= corr;
                            ptx::tmem_store_32_nowait(tmem_o + c * 32, v);
                        }
                    }
                    ptx::tmem_store_wait();
                }
                const float ref = m_ref == -INFINITY ? 0.f : m_ref;
                off = make_float2(-ref, -ref);
            }
#pragma unroll 1
            for (int h = 0; h < steps; ++h) {
                if (mine) {
                    float sv[64];
                    scores(h, sv);
#pragma unroll
                    for (int u = 0; u < 2; ++u) {
                        uint32_t pk[16];
#pragma unroll
                        for (int i = 0; i < 16; ++i) {
                            const float2 x = fma_pair(make_float2(sv[u * 32 + 2 * i], sv[u * 32 + 2 * i + 1]), rate, off);
                            const float2 e = make_float2(ptx::ex2_approx(x.x), ptx::ex2_approx(x.y));
                            if (i & 1) sum = add_pair(sum, e); else sum2 = add_pair(sum2, e);
                            const __nv_bfloat162 b2 = __floats2bfloat162_rn(e.x, e.y);
                            pk[i] = *reinterpret_cast<const uint32_t*>(&b2);
                        }
                        // (over scores that have been read: 16 columns of weights for every 32 of scores)
                        ptx::tmem_store_16_nowait(tmem_s + h * 32 + u * 16, pk);
                    }
                    ptx::tmem_store_wait();
                }
                ptx::tc_fence_before_sync();
                __syncwarp();
                if (lane == 0) ptx::mbar_arrive(p_ready(t, h));
            }
            l += (sum.x + sum.y) + (sum2.x + sum2.y);
        }
        if (ok) ok = __all_sync(0xffffffffu, ptx::mbar_wait(s_full(t), seen & 1, abort_flag));
        if (ok) {
            ptx::tc_fence_after_sync();
            // Rows go out through shared memory (every product has read its operands): written by the thread that holds it, a
            // row's pieces of 16 bytes would lie 512 bytes and more apart from the next thread's.
            const bool final = p.whole && p.pieces == 1;
            const size_t row = (size_t)max(token, 0) * p.n_heads + kvh * G + r % G, at = row * (p.pieces + p.own_splits) + split;
            float inv = 1.0f;
            if (final) {
                if (p.sinks) l += exp2f(p.sinks[kvh * G + r % G] * p.sink_rate - m_ref);
                inv = 1.0f / l;
            } else if (row_valid) {
                *reinterpret_cast<float2*>(p.part_ml + at * 2) = make_float2(m_ref, l);
            }
            float* stage = reinterpret_cast<float*>(smem) + warp * 32 * kPtStage;
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                if (c * 32 < D) {
                    float v[32];
                    ptx::tmem_load_32_nowait(tmem_o + c * 32, v);
                    ptx::tmem_load_wait();
#pragma unroll
                    for (int q = 0; q < 8; ++q)
                        *reinterpret_cast<float4*>(stage + lane * kPtStage + c * 32 + q * 4) =
                            make_float4(v[4 * q] * inv, v[4 * q + 1] * inv, v[4 * q + 2] * inv, v[4 * q + 3] * inv);
                }
            }
            __syncwarp();
            const uint64_t mine = row_valid ? (final ? row : at) : ~0ull;
#pragma unroll 4
            for (int i = 0; i < 32; ++i) {
                const uint64_t to = __shfl_sync(0xffffffffu, mine, i);
                if (to == ~0ull || lane * 4 >= D) continue;
                const float4 x = *reinterpret_cast<const float4*>(stage + i * kPtStage + lane * 4);
                if (final) {
                    const __nv_bfloat162 y[2] = {__floats2bfloat162_rn(x.x, x.y), __floats2bfloat162_rn(x.z, x.w)};
                    *reinterpret_cast<uint2*>(reinterpret_cast<__nv_bfloat16*>(p.out) + to * D + lane * 4) = *reinterpret_cast<const uint2*>(y);
                } else {
                    *reinterpret_cast<float4*>(p.part_o + to * D + lane * 4) = x;
                }
            }
            ptx::tc_fence_before_sync();
        }
    } else if (!working && warp < 8) {
        // a piece without blocks: empty parts for the merge
        const int t = warp >> 2, r = (warp & 3) * 32 + lane, tok = t * tt + r / G;
        if (r / G < tt && tok < count && !(base & 1023u)) {
            const size_t at = ((size_t)p.toks[tile.first + tok] * p.n_heads + kvh * G + r % G) * (p.pieces + p.own_splits) + split;
            *reinterpret_cast<float2*>(p.part_ml + at * 2) = make_float2(-INFINITY, 0.f);
        }
    }
    ptx::tc_fence_before_sync();
    __syncthreads();
    if (warp == 9) { ptx::tc_fence_after_sync(); ptx::tmem_dealloc(tmem, 512); }
    if (threadIdx.x == 0 && *abort_flag && p.status) atomicExch(p.status, 8);
}

}  // namespace mdma
