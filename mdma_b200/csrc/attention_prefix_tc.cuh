// The tcgen05 kernel of attention over shared prefixes (bfloat16, pages of a multiple of 64 tokens).
//
// A block takes up to 256 query rows of one kv head, two tiles of 128 (token, query head of the group) rows whose tokens may be of
// several members of a group, and walks a list of key blocks of 128:
//     S = Q K^T    tcgen05.mma, M = N = 128, operands from shared memory (keys by TMA, 128-byte swizzle), S in tensor memory
//     softmax      128 threads a tile, a row a thread: the row out of tensor memory, mask, running maximum and sum in float, the
//                  weights rounded to bfloat16 and written back over S
//     O += P V     tcgen05.mma, A = P from tensor memory, V as the cache holds it (MN-major), O in tensor memory
// The two tiles take turns: while one is in its softmax the tensor pipe works for the other, and both use the same key and
// value blocks.  Tensor memory: S and P of the tiles in columns 0 and 128, O in 256 and 384.  The products of a tile are issued by one thread
// in the order S(0), P(0) V(0), S(1), .., so whoever sees S(j) complete knows that P(j-1) V(j-1) is, too.
// The weights are taken against a reference that moves only when a row's maximum has grown by more than 2^8 since; O is
// rescaled only then.
//
// The list: the prefix's blocks, which all rows see, and (`whole`) behind them the own blocks of every sequence with tokens in the
// tiles, which only that sequence's rows see: the others' lanes of O are left out of the product, so that what they are
// multiplied with does not reach them.  `pieces` blocks share a list; each then leaves its sums for the merge.
#pragma once
#include "prefix.cuh"
#include "ptx.cuh"

namespace mdma {

constexpr int kPtRows = 128, kPtKeys = 128, kPtThreads = 320, kPtMaxTokens = 2 * kPtRows;
constexpr int kPtHalf = kPtRows * 128;                           // 128 rows (or keys) x 64 numbers
constexpr int kPtSlot = 2 * kPtHalf;
constexpr int kPtSmemK = 2 * kPtSlot, kPtSmemV = kPtSmemK + 2 * kPtSlot, kPtSmemBars = kPtSmemV + 2 * kPtSlot;
struct PtSegment { int seq, key0, key1, tok0, toks, block0; };  // keys [key0, key1) for the tile's tokens [tok0, tok0 + toks); its first block
constexpr int kPtSmemSegs = kPtSmemBars + 256;
constexpr int kPtSmem = kPtSmemSegs + (kPtMaxTokens + 4) * (int)sizeof(PtSegment);

// Walks the blocks of a list.
struct PtWalk {
    const PtSegment* segs;
    int seg, block;
    __device__ __forceinline__ PtWalk(const PtSegment* s, int first) : segs(s), seg(0), block(first) {
        while (first >= segs[seg + 1].block0) ++seg;
    }
    __device__ __forceinline__ void next() {
        ++block;
        while (block >= segs[seg + 1].block0) ++seg;
    }
    __device__ __forceinline__ const PtSegment& s() const { return segs[seg]; }
    // (of an own segment the first block starts at the multiple of 64 below its first key)
    __device__ __forceinline__ int key() const { return (s().key0 & ~63) + (block - s().block0) * kPtKeys; }
    // rows [a, b) of tile `tile` that see this block
    __device__ __forceinline__ void rows(int tile, int tt, int G, int& a, int& b) const {
        a = max(s().tok0 - tile * tt, 0) * G;
        b = max(min(s().tok0 + s().toks - tile * tt, tt), 0) * G;
    }
    __device__ __forceinline__ bool active(int tile, int tt, int G) const {
        int a, b;
        rows(tile, tt, G, a, b);
        return a < b;
    }
};

__global__ void __launch_bounds__(kPtThreads, 1)
prefix_tc_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, const PrefixParams p) {
    extern __shared__ __align__(1024) uint8_t smem[];
    const uint32_t base = ptx::smem_addr(smem), bars = base + kPtSmemBars;
    auto k_full = [&](int s) { return bars + 8u * s; };
    auto k_empty = [&](int s) { return bars + 8u * (2 + s); };
    auto v_full = [&](int s) { return bars + 8u * (4 + s); };
    auto v_empty = [&](int s) { return bars + 8u * (6 + s); };
    auto s_full = [&](int t) { return bars + 8u * (8 + t); };
    auto p_ready = [&](int t) { return bars + 8u * (10 + t); };
    volatile uint32_t* tmem_slot = reinterpret_cast<volatile uint32_t*>(smem + kPtSmemBars + 8 * 12);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + kPtSmemBars + 8 * 13);
    int* warp_starts = reinterpret_cast<int*>(smem + kPtSmemBars + 8 * 14);          // [9]
    PtSegment* segs = reinterpret_cast<PtSegment*>(smem + kPtSmemSegs);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int G = p.group, D = p.head_dim, kvh = blockIdx.x, split = blockIdx.z, tt = kPtRows / G;

    chain_wait();
    PrefixTile tile;
    if (!prefix_tile(p, blockIdx.y, 2 * tt, tile)) return;
    if (threadIdx.x == 0) {
        for (int s = 0; s < 2; ++s) {
            ptx::mbar_init(k_full(s), 1); ptx::mbar_init(k_empty(s), 1);
            ptx::mbar_init(v_full(s), 1); ptx::mbar_init(v_empty(s), 1);
            ptx::mbar_init(s_full(s), 1); ptx::mbar_init(p_ready(s), 128);
        }
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

    // ---- which rows, which keys ------------------------------------------------------------------------------------
    const bool found = !(base & 1023u);
    const int count = tile.count;                                // tokens of both tiles
    int blocks = 0, b0 = 0, b1 = 0;
    if (found) {                                                 // (uniform over the block)
        const int len = p.group_len[tile.g];
        if (!p.whole) {
            const int keys = prefix_piece(len, p.pieces), lo = split * keys, hi = min(len, lo + keys);
            if (threadIdx.x == 0) {
                segs[0] = {p.group_seq[tile.g], lo, hi, 0, count, 0};
                segs[1].block0 = 0x7fffffff;
            }
            b1 = blocks = hi > lo ? (hi - lo + kPtKeys - 1) / kPtKeys : 0;
        } else {
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
            int n_segs = shared;
            for (int w = 0; w < 8; ++w) n_segs += warp_starts[w];
            if (threadIdx.x == 0) {
                int at = 0;
                for (int s = 0; s < n_segs; ++s) {
                    segs[s].block0 = at;
                    at += max(segs[s].key1 - (segs[s].key0 & ~63) + kPtKeys - 1, 0) / kPtKeys;
                }
                segs[n_segs].block0 = at;
                segs[n_segs + 1].block0 = 0x7fffffff;
                warp_starts[8] = at;
            }
            __syncthreads();
            blocks = warp_starts[8];
            const int per = (blocks + p.pieces - 1) / p.pieces;
            b0 = split * per; b1 = min(blocks, b0 + per);
        }
        // queries into shared memory, 128-byte rows with the 128-byte swizzle, zeros beyond the tiles' rows
        if (b0 < b1 && warp < 8) {
            const __nv_bfloat16* q = reinterpret_cast<const __nv_bfloat16*>(p.q);
            const int chunks = ((D + 63) / 64) * 8;
            for (int i = threadIdx.x; i < 2 * kPtRows * chunks; i += 256) {
                const int r = i / chunks, c = i % chunks, tr = r % kPtRows, t = r / kPtRows * tt + tr / G;
                uint4 x = make_uint4(0u, 0u, 0u, 0u);
                if (tr / G < tt && t < count && c * 8 < D)
                    x = *reinterpret_cast<const uint4*>(q + (size_t)p.toks[tile.first + t] * p.q_stride + (size_t)(kvh * G + tr % G) * D + c * 8);
                *reinterpret_cast<uint4*>(smem + r / kPtRows * kPtSlot + (c >> 3) * kPtHalf + tr * 128 + (((c & 7) ^ (tr & 7)) << 4)) = x;
            }
            ptx::fence_proxy_async_shared();
        }
    }
    __syncthreads();
    const bool working = b0 < b1;
    const int halves = (D + 63) / 64;

    if (working && warp == 8 && lane == 0) {
        // ---- TMA producer: K(0) V(0) K(1) V(1) .. -----------------------------------------------------------------
        PtWalk w(segs, b0);
        bool fine = true;
        for (int j = 0; fine && b0 + j < b1; ++j, w.next()) {
            const int* pages = p.page_table + (size_t)p.seq_slot[w.s().seq] * p.max_pages;
            const int key0 = w.key(), boxes = w.s().key1 - key0 > 64 ? 2 : 1;       // of 64 keys each
            int page[2], row[2];
            for (int b = 0; b < boxes; ++b) { page[b] = pages[(key0 + 64 * b) / p.page_size]; row[b] = (key0 + 64 * b) % p.page_size; }
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
    } else if (working && warp == 9 && lane == 0) {
        // ---- MMA issuer ---------------------------------------------------------------------------------------------
        const uint32_t idesc_s = ptx::idesc_bf16_f32_ex(kPtRows, kPtKeys, 0), idesc_o = ptx::idesc_bf16_f32_ex(kPtRows, D, 1);
        const int steps = D / 16;
        auto product_s = [&](int t, int s) {
            const uint64_t qd = ptx::smem_desc_sw128(base + t * kPtSlot), kd = ptx::smem_desc_sw128(base + kPtSmemK + s * kPtSlot);
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (i < steps) {
                    const uint32_t at = ((i >> 2) * kPtHalf + (i & 3) * 32) >> 4;
                    ptx::mma_bf16_ss(tmem + t * 128, qd + at, kd + at, idesc_s, i > 0);
                }
            ptx::mma_commit(s_full(t));
        };
        auto off_lanes = [](int a, int b, int word) -> uint32_t {             // bits of lanes outside [a, b)
            const int lo = max(a - word * 32, 0), hi = min(b - word * 32, 32);
            if (lo >= hi) return 0xffffffffu;
            const uint32_t on = (hi == 32 ? 0xffffffffu : (1u << hi) - 1u) & ~((1u << lo) - 1u);
            return ~on;
        };
        PtWalk w(segs, b0), ahead(segs, b0);
        uint32_t done[2] = {0, 0};
        bool ok = ptx::mbar_wait(k_full(0), 0, abort_flag);
        if (ok) {
            ptx::tc_fence_after_sync();
            for (int t = 0; t < 2; ++t) if (ahead.active(t, tt, G)) product_s(t, 0);
            ptx::mma_commit(k_empty(0));
        }
        const int n = b1 - b0;
        for (int j = 0; j < n && ok; ++j, w.next()) {
            const int s = j & 1;
            const bool more = j + 1 < n;
            ahead.next();
            ok = ptx::mbar_wait(v_full(s), (j >> 1) & 1, abort_flag);
            for (int t = 0; t < 2 && ok; ++t) {
                int a, b;
                w.rows(t, tt, G, a, b);
                if (a < b) {
                    ok = ptx::mbar_wait(p_ready(t), done[t] & 1, abort_flag);
                    if (!ok) break;
                    ++done[t];
                    ptx::tc_fence_after_sync();
                    // (rows beyond the tile's tokens take part in a prefix's products: nobody reads them)
                    const bool all = a == 0 && (w.seg == 0 && w.s().toks == count);
                    const uint4 off = all ? make_uint4(0u, 0u, 0u, 0u) : make_uint4(off_lanes(a, b, 0), off_lanes(a, b, 1), off_lanes(a, b, 2), off_lanes(a, b, 3));
                    const uint64_t vd = ptx::smem_desc_sw128_mn(base + kPtSmemV + s * kPtSlot, kPtHalf);
#pragma unroll
                    for (int i = 0; i < kPtKeys / 16; ++i)
                        ptx::mma_bf16_ts(tmem + 256 + t * 128, tmem + t * 128 + i * 8, vd + ((i * 16 * 128) >> 4), idesc_o, off);
                }
                if (more && ahead.active(t, tt, G)) {
                    ok = ptx::mbar_wait(k_full(s ^ 1), ((j + 1) >> 1) & 1, abort_flag);
                    if (!ok) break;
                    ptx::tc_fence_after_sync();
                    product_s(t, s ^ 1);
                }
            }
            if (!ok) break;
            ptx::mma_commit(v_empty(s));
            if (more) ptx::mma_commit(k_empty(s ^ 1));
        }
        if (ok) { ptx::mma_commit(s_full(0)); ptx::mma_commit(s_full(1)); }       // the last sums are complete
    } else if (working && warp < 8) {
        // ---- softmax: a row a thread --------------------------------------------------------------------------------
        const int t = warp >> 2, quad = warp & 3, r = quad * 32 + lane;
        const uint32_t lanes = (uint32_t)(quad * 32) << 16, tmem_s = tmem + t * 128 + lanes, tmem_o = tmem + 256 + t * 128 + lanes;
        const int tok = t * tt + r / G;                          // of the block's tokens
        const bool row_valid = r / G < tt && tok < count;
        const int token = row_valid ? p.toks[tile.first + tok] : -1;
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
        PtWalk w(segs, b0);
        uint32_t seen = 0;
        bool ok = true;
        for (int j = 0; b0 + j < b1 && ok; ++j, w.next()) {
            int ra, rb;
            w.rows(t, tt, G, ra, rb);
            const int key0 = w.key(), end = w.s().key1 - key0;   // block rows beyond `end` belong to nobody
            const bool shared = w.seg == 0 && w.s().toks == count && (!p.whole || p.group_len[tile.g] > 0);
            if (end < kPtKeys && (t == 0 ? ra < rb : !w.active(0, tt, G))) {
                // one tile's threads clear such value rows before the products read them: a weight of zero times what is not
                // finite would not be zero
                const int s = j & 1;
                ok = __all_sync(0xffffffffu, ptx::mbar_wait(v_full(s), (j >> 1) & 1, abort_flag));
                if (!ok) break;
                for (int e = threadIdx.x & 127; e < halves * kPtKeys * 8; e += 128) {
                    const int h = e / (kPtKeys * 8), kr = (e >> 3) % kPtKeys, c = e & 7;
                    if (kr >= end) *reinterpret_cast<uint4*>(smem + kPtSmemV + s * kPtSlot + h * kPtHalf + kr * 128 + c * 16) = make_uint4(0u, 0u, 0u, 0u);
                }
                ptx::fence_proxy_async_shared();
            }
            if (ra >= rb) continue;
            ok = __all_sync(0xffffffffu, ptx::mbar_wait(s_full(t), seen & 1, abort_flag));
            if (!ok) break;
            ++seen;
            ptx::tc_fence_after_sync();
            if (shared || (rb > quad * 32 && ra < quad * 32 + 32)) {        // (a warp none of whose rows sees the block has nothing to do)
                float sv[128];
#pragma unroll
                for (int c = 0; c < 4; ++c) ptx::tmem_load_32_nowait(tmem_s + c * 32, sv + c * 32);
                ptx::tmem_load_wait();
                int c0 = 0, c1 = min(end, kPtKeys);              // columns this row sees
                if (!shared) {
                    const bool mine = r >= ra && r < rb;
                    c0 = max(w.s().key0 - key0, 0);
                    c1 = mine ? min(c1, pos - key0 + 1) : 0;
                }
                if (__any_sync(0xffffffffu, c0 > 0 || c1 < kPtKeys)) {
#pragma unroll
                    for (int c = 0; c < 128; ++c) if (c < c0 || c >= c1) sv[c] = -INFINITY;
                }
                float m4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                for (int c = 0; c < 128; c += 2) m4[(c >> 1) & 3] = fmaxf(m4[(c >> 1) & 3], fmaxf(sv[c], sv[c + 1]));
                const float mx = fmaxf(fmaxf(m4[0], m4[1]), fmaxf(m4[2], m4[3])) * p.scale_log2;      // scale > 0
                float corr = 1.f;
                if (mx > m_ref + 8.f) {
                    corr = m_ref == -INFINITY ? 0.f : ptx::ex2_approx(m_ref - mx);
                    m_ref = mx;
                }
                const float ref = m_ref == -INFINITY ? 0.f : m_ref;
                float s4[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    uint32_t pk[16];
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        const float e0 = ptx::ex2_approx(fmaf(sv[c * 32 + 2 * i], p.scale_log2, -ref));
                        const float e1 = ptx::ex2_approx(fmaf(sv[c * 32 + 2 * i + 1], p.scale_log2, -ref));
                        s4[i & 3] += e0 + e1;
                        const __nv_bfloat162 b2 = __floats2bfloat162_rn(e0, e1);
                        pk[i] = *reinterpret_cast<const uint32_t*>(&b2);
                    }
                    ptx::tmem_store_16_nowait(tmem_s + c * 16, pk);
                }
                l = l * corr + ((s4[0] + s4[1]) + (s4[2] + s4[3]));
                if (__any_sync(0xffffffffu, corr != 1.f)) {      // rare: rescale these rows of O (P V of the block before is done)
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
                }
                ptx::tmem_store_wait();
            }
            ptx::tc_fence_before_sync();
            ptx::mbar_arrive(p_ready(t));
        }
        if (ok) ok = __all_sync(0xffffffffu, ptx::mbar_wait(s_full(t), seen & 1, abort_flag));
        if (ok) {
            ptx::tc_fence_after_sync();
            const size_t row = (size_t)(row_valid ? token : 0) * p.n_heads + kvh * G + r % G;
            if (p.whole && p.pieces == 1) {
                if (p.sinks) l += exp2f(p.sinks[kvh * G + r % G] * p.sink_rate - m_ref);
                const float inv = 1.0f / l;
                __nv_bfloat16* dst = reinterpret_cast<__nv_bfloat16*>(p.out) + row * D;
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    if (c * 32 < D) {
                        float v[32];
                        ptx::tmem_load_32_nowait(tmem_o + c * 32, v);
                        ptx::tmem_load_wait();
                        if (row_valid) {
#pragma unroll
                            for (int q = 0; q < 4; ++q)
                                if (c * 32 + q * 8 < D) {
                                    uint32_t x[4];
#pragma unroll
                                    for (int i = 0; i < 4; ++i) {
                                        const __nv_bfloat162 b2 = __floats2bfloat162_rn(v[q * 8 + 2 * i] * inv, v[q * 8 + 2 * i + 1] * inv);
                                        x[i] = *reinterpret_cast<const uint32_t*>(&b2);
                                    }
                                    *reinterpret_cast<uint4*>(dst + c * 32 + q * 8) = make_uint4(x[0], x[1], x[2], x[3]);
                                }
                        }
                    }
                }
            } else {
                const size_t at = row * (p.pieces + p.own_splits) + split;
                float* dst = p.part_o + at * D;
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    if (c * 32 < D) {
                        float v[32];
                        ptx::tmem_load_32_nowait(tmem_o + c * 32, v);
                        ptx::tmem_load_wait();
                        if (row_valid) {
#pragma unroll
                            for (int q = 0; q < 8; ++q)
                                if (c * 32 + q * 4 < D)
                                    *reinterpret_cast<float4*>(dst + c * 32 + q * 4) = make_float4(v[4 * q], v[4 * q + 1], v[4 * q + 2], v[4 * q + 3]);
                        }
                    }
                }
                if (row_valid) *reinterpret_cast<float2*>(p.part_ml + at * 2) = make_float2(m_ref, l);
            }
            ptx::tc_fence_before_sync();
        }
    } else if (!working && found && p.whole && warp < 8) {
        // a piece without blocks: empty parts for the merge
        const int t = warp >> 2, r = (warp & 3) * 32 + lane, tok = t * tt + r / G;
        if (r / G < tt && tok < count) {
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
