// Attention of a step whose sequences share prefixes: what the kernels of it have in common.
//
// Every sequence belongs to one group; a group's first `group_len` tokens lie in pages that its members' page tables share
// (the rows of a partly filled last page are the same in each member's copy), so one member's table row leads to them all.
// A query of a member sees the whole prefix and the keys [group_len, its position] of its own sequence.  With m the maximum
// of the scores and l the sum of their exponentials over a set of keys, o the weighted sum of the values, two disjoint sets A, B join as
//     m = max(mA, mB),  l = lA 2^(mA - m) + lB 2^(mB - m),  o = oA 2^(mA - m) + oB 2^(mB - m)
// (scores in powers of two).  So a prefix is read once for the query rows of all members, which fill the rows of one tile,
// every sequence's own keys are read by its own rows, and a last step joins the parts in a fixed order.
#pragma once
#include "common.cuh"

namespace mdma {

struct PrefixParams {
    const void* q; long q_stride;                    // rows of the projection; queries first
    const void* k_cache; const void* v_cache;        // [pages, page_size, kv_heads, head_dim]
    const int* seq_start; const int* seq_pos0; const int* seq_slot; const int* tok_seq;
    const int* page_table; int max_pages; int page_size; int n_pages;
    const int* group_len; const int* group_seq; const int* tok_first; const int* toks; const int* seq_skip;
    void* out;
    float* part_o; float* part_ml;                   // [token][head][slot][head_dim], [token][head][slot][2]
    int n_groups, n_seqs, n_tokens, max_new;
    int n_shared;                                    // groups that have a prefix, at most
    int n_heads, n_kv_heads, head_dim, group;
    int pieces, own_splits;                          // a prefix in `pieces` pieces at most, own keys in `own_splits`: slots of the parts
    int own_keys;                                    // keys of a piece of streamed own keys, the last takes the rest (0: equal pieces)
    int unit;                                        // a piece of a prefix is a multiple of so many keys
    int whole;                                       // own_splits 0: all keys of a row tile, prefix and own ones, are one list in `pieces` pieces
    float scale_log2;                                // scale * log2(e)
    const float* sinks; float sink_rate;             // sinks[head] * sink_rate is in powers of two; null: none
    int* status;
};

// Keys of a piece of a prefix of `len` tokens: a multiple of `unit` that follows from the prefix alone, so that a sequence's sums
// are cut at the same places whoever shares the step.
__host__ __device__ __forceinline__ int prefix_piece(int len, int pieces, int unit) {
    return ((len + pieces - 1) / pieces + unit - 1) / unit * unit;
}
__host__ __device__ __forceinline__ int prefix_pieces_used(int len, int pieces, int unit) {
    if (len <= 0) return 0;
    const int keys = prefix_piece(len, pieces, unit);
    return (len + keys - 1) / keys;
}

// Piece `split` of a sequence's own keys [skip, end), of the streaming kernel: keys [lo, hi), of a multiple of `unit`.  Pieces of a fixed length are the same
// whoever shares the step (only how many a step has room for follows from its longest sequence); most are empty beside one
// long sequence.
__device__ __forceinline__ void own_piece(const PrefixParams& p, int skip, int end, int split, int unit, int& lo, int& hi) {
    const int keys = p.own_keys > 0 ? p.own_keys : ((end - skip + p.own_splits - 1) / p.own_splits + unit - 1) / unit * unit;
    lo = skip + split * keys;
    hi = p.own_keys > 0 && split == p.own_splits - 1 ? end : min(end, lo + keys);
}

// Tile t of the prefixes' query rows, `tile_tokens` tokens each: which group, which of its tokens.  Groups without a prefix
// have no tiles (unless their own keys are walked, too).  False: there is no such tile.
// (A lane a group, thirty-two at a time: one round of loads finds the tile.)  All lanes of a warp call this together.
struct PrefixTile { int g, first, count, len; };     // toks[first .. first + count); the group's prefix
__device__ __forceinline__ bool prefix_tile(const PrefixParams& p, int t, int tile_tokens, PrefixTile& out) {
    const int lane = threadIdx.x & 31;
    for (int g0 = 0; g0 < p.n_groups; g0 += 32) {
        const int g = g0 + lane;
        int len = 0, a = 0, n = 0, tiles = 0;
        if (g < p.n_groups) {
            len = p.group_len[g]; a = p.tok_first[g]; n = p.tok_first[g + 1] - a;
            tiles = len > 0 || p.whole ? (n + tile_tokens - 1) / tile_tokens : 0;
        }
        int last = tiles;                            // tiles up to and with this lane's group
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int x = __shfl_up_sync(0xffffffffu, last, o);
            if (lane >= o) last += x;
        }
        const uint32_t behind = __ballot_sync(0xffffffffu, last > t);
        if (behind) {
            const int at = __ffs(behind) - 1;
            const int mine = t - (__shfl_sync(0xffffffffu, last, at) - __shfl_sync(0xffffffffu, tiles, at));
            out.g = g0 + at;
            out.first = __shfl_sync(0xffffffffu, a, at) + mine * tile_tokens;
            out.count = min(tile_tokens, __shfl_sync(0xffffffffu, n, at) - mine * tile_tokens);
            out.len = __shfl_sync(0xffffffffu, len, at);
            return true;
        }
        t -= __shfl_sync(0xffffffffu, last, 31);
    }
    return false;
}
// The most tiles a step can have: every group leaves one partly filled.  (Sequences that share nothing are groups, too, but have
// no tiles unless their own keys are walked: with a block for each, 8 sequences behind 2,048 tokens beside 56 that share
// nothing took 108 us on the tcgen05 kernel, whose blocks do not share an SM.)
static inline long prefix_tiles_bound(const PrefixParams& p, int tile_tokens) {
    return (long)p.n_tokens / tile_tokens + (p.whole ? p.n_groups : p.n_shared);
}

// A part's share of the whole, 2^(its maximum - m).  -1, no share: a part without keys leaves no maximum and no sum.  (The
// maximum passes over NaN: a part whose scores are all NaN leaves no maximum either, but a sum that is NaN, and joins.)
__device__ __forceinline__ float prefix_share(float2 ml, float m) { return ml.x == -INFINITY && ml.y == 0.f ? -1.f : exp2f(ml.x - m); }
__device__ __forceinline__ bool prefix_joins(float share) { return !(share < 0.f); }

// out[token, head] from its parts: those of its prefix in order, then those of its own keys.  One warp for 64 numbers of a row: a lane
// a part for the maxima, the sums and the shares (at most 64 parts), then all lanes over the parts' numbers, eight parts in flight.
template <typename T>
__global__ void __launch_bounds__(128)
prefix_merge_kernel(const PrefixParams p) {
    chain_release();
    chain_wait();
    const int lane = threadIdx.x & 31, D = p.head_dim, chunks = (D + 63) / 64;
    const long item = (long)blockIdx.x * 4 + (threadIdx.x >> 5), row = item / chunks;            // row: token * heads + head
    if (row >= (long)p.n_tokens * p.n_heads) return;
    const int slots = p.pieces + p.own_splits;
    const int used = p.whole || p.pieces == 0 ? p.pieces : prefix_pieces_used(p.seq_skip[p.tok_seq[row / p.n_heads]], p.pieces, p.unit), parts = used + p.own_splits;
    const float2* ml = reinterpret_cast<const float2*>(p.part_ml) + row * slots;
    auto slot_of = [&](int s) { return s < used ? s : p.pieces + s - used; };
    float2 mine[2];
#pragma unroll
    for (int u = 0; u < 2; ++u) mine[u] = u * 32 + lane < parts ? ml[slot_of(u * 32 + lane)] : make_float2(-INFINITY, 0.f);
    const float m = warp_max(fmaxf(mine[0].x, mine[1].x));
    float share[2], l = 0.f;
#pragma unroll
    for (int u = 0; u < 2; ++u) {
        share[u] = prefix_share(mine[u], m);
        if (prefix_joins(share[u])) l += share[u] * mine[u].y;
    }
    l = warp_sum(l);
    if (p.sinks) l += exp2f(p.sinks[row % p.n_heads] * p.sink_rate - m);
    const float* o = p.part_o + row * slots * D;
    T* to = reinterpret_cast<T*>(p.out) + row * D;
    {                                                // two numbers a lane, 32 apart
        const int d = (int)(item % chunks) * 64 + lane;
        const bool one = d < D, two = d + 32 < D;
        float a0 = 0.f, a1 = 0.f;
        for (int s0 = 0; s0 < parts; s0 += 8) {
            float x0[8], x1[8];
#pragma unroll
            for (int u = 0; u < 8; ++u) {
                const float* from = o + (size_t)slot_of(min(s0 + u, parts - 1)) * D + d;
                x0[u] = one ? __ldcg(from) : 0.f; x1[u] = two ? __ldcg(from + 32) : 0.f;
            }
#pragma unroll
            for (int u = 0; u < 8; ++u) {
                const int s = s0 + u;
                const float f = __shfl_sync(0xffffffffu, s < 32 ? share[0] : share[1], s & 31);
                if (s < parts && prefix_joins(f)) { a0 = fmaf(f, x0[u], a0); a1 = fmaf(f, x1[u], a1); }
            }
        }
        if (one) to[d] = from_float<T>(a0 / l);
        if (two) to[d + 32] = from_float<T>(a1 / l);
    }
}

static inline unsigned prefix_merge_blocks(const PrefixParams& p) {
    return (unsigned)(((long)p.n_tokens * p.n_heads * ((p.head_dim + 63) / 64) + 3) / 4);
}

// The arguments as one array of 64-bit words, in the order below (a step makes this call once a layer: converting thirty
// arguments one by one costs the host more than the launches).
static inline int prefix_params(const long long* w, int n_words, float scale, PrefixParams* out) {
    MDMA_REQUIRE(n_words == 34, "prefix_attention: %d argument words", n_words);
    PrefixParams& p = *out;
    int i = 0;
    auto ptr = [&]() { return (void*)(uintptr_t)w[i++]; };
    auto num = [&]() { return (int)w[i++]; };
    p.q = ptr(); p.q_stride = (long)w[i++];
    p.k_cache = ptr(); p.v_cache = ptr();
    p.seq_start = (const int*)ptr(); p.seq_pos0 = (const int*)ptr(); p.seq_slot = (const int*)ptr(); p.tok_seq = (const int*)ptr();
    p.page_table = (const int*)ptr(); p.max_pages = num(); p.page_size = num(); p.n_pages = num();
    p.group_len = (const int*)ptr(); p.group_seq = (const int*)ptr(); p.tok_first = (const int*)ptr(); p.toks = (const int*)ptr();
    p.seq_skip = (const int*)ptr();
    p.out = ptr();
    float* scratch = (float*)ptr();
    const long long floats = w[i++];
    p.n_groups = num(); p.n_shared = num(); p.n_seqs = num(); p.n_tokens = num(); p.max_new = num();
    p.n_heads = num(); p.n_kv_heads = num(); p.head_dim = num();
    p.pieces = num(); p.own_splits = num(); p.own_keys = num();
    p.sinks = (const float*)ptr();
    p.status = (int*)ptr();
    p.sink_rate = w[i++] ? 1.0f : 1.4426950408889634f;      // the sinks come times log2(e), or as they are
    p.scale_log2 = scale * 1.4426950408889634f;
    MDMA_REQUIRE(p.n_heads > 0 && p.n_kv_heads > 0 && p.n_heads % p.n_kv_heads == 0, "prefix_attention: %d heads over %d kv heads", p.n_heads, p.n_kv_heads);
    MDMA_REQUIRE(p.head_dim > 0 && p.head_dim <= 256, "prefix_attention: head_dim %d is beyond the limit of 256", p.head_dim);
    MDMA_REQUIRE(p.page_table && p.page_size > 0 && p.max_pages > 0, "prefix_attention: bad cache geometry");
    MDMA_REQUIRE(p.n_groups >= 0 && p.n_shared >= 0 && p.n_shared <= p.n_groups && p.n_seqs >= 0 && p.n_tokens >= 0 &&
                     (p.n_tokens == 0 || (p.max_new > 0 && p.n_groups > 0)),
                 "prefix_attention: %d tokens of %d sequences in %d groups, %d with a prefix, at most %d of one", p.n_tokens, p.n_seqs,
                 p.n_groups, p.n_shared, p.max_new);
    MDMA_REQUIRE(p.pieces >= 0 && p.own_splits >= 0 && p.own_keys >= 0 && p.pieces + p.own_splits > 0, "prefix_attention: bad pieces");
    MDMA_REQUIRE(p.pieces <= 32 && p.own_splits <= 32, "prefix_attention: %d and %d pieces are beyond the limit of 32", p.pieces, p.own_splits);
    MDMA_REQUIRE(scale > 0.f, "prefix_attention: the score scale must be positive");
    p.group = p.n_heads / p.n_kv_heads;
    p.whole = p.own_splits == 0; p.unit = 128;
    const long long slots = p.pieces + p.own_splits == 1 ? 0 : (long long)p.n_tokens * p.n_heads * (p.pieces + p.own_splits), need = slots ? slots * (p.head_dim + 2) + 4 : 0;
    MDMA_REQUIRE(need == 0 || (scratch && floats >= need), "prefix_attention: %lld floats of scratch are needed, %lld given", need, floats);
    MDMA_REQUIRE(((uintptr_t)scratch & 15) == 0, "prefix_attention: the scratch must be 16-byte aligned");
    // pairs first, so that they lie at multiples of 8 bytes and the sums behind them of 16, whatever the head size
    p.part_ml = scratch; p.part_o = scratch + (slots * 2 + 3) / 4 * 4;
    return 0;
}

}  // namespace mdma
