// Attention over shared prefixes on the CUDA cores: the true 32-bit engine's, and bfloat16 of any geometry (head sizes up to
// 256, any page size).  See prefix.cuh for the parts and how they join.
//
// A block takes a tile of 8, 32 or 64 query rows of one kv head, (token, query head of the group) pairs, and walks its keys 32
// at a time: keys and values are staged in shared memory as floats, the next 32 on their way while these are worked on; a
// thread holds the scores of a few rows x keys and as many rows' sums.  Rows of a prefix tile come from all members of a group,
// so a key row is read once for all of them; 64 rows make four rows x four keys a thread, which the multiply-add units need to
// be fed from shared memory; the own keys of a single token are worked on by eight rows of sixteen threads.  The prefixes' kernel
// and that of the own keys run side by side, a third one joins the parts.  16 sequences behind 2,048 tokens, 16/4 heads of 256: 60 us,
// in bfloat16, whose numbers are fetched two bytes at a time, 149 (1,824 and 1,904 where every sequence reads by itself).
#include "mma_tiles.cuh"
#include "prefix.cuh"

namespace mdma {

constexpr int kPsKeys = 32, kPsThreads = 128;

// RG groups of threads, RT rows each; the KG = 128 / RG threads of a group hold KT = 32 / KG keys and 4 of every 4 KG numbers of a head.
template <int RG, int RT, int DC>
struct PsShape {
    static constexpr int kRows = RG * RT, kKG = kPsThreads / RG, kKT = kPsKeys / kKG, kPitch = DC * 4 * kKG + 4;
    static constexpr int kFloats = (kRows + 4 * kPsKeys) * kPitch + kRows * (kPsKeys + 1);
};

template <typename T, int RG, int RT, int DC>        // DC: steps of 4 KG numbers that cover a head
__global__ void __launch_bounds__(kPsThreads)
prefix_simple_kernel(const PrefixParams p, int own_tiles, int wide) {
    using S = PsShape<RG, RT, DC>;
    constexpr int kRows = S::kRows, KG = S::kKG, KT = S::kKT, kPitch = S::kPitch, kWidth = DC * 4 * KG;
    extern __shared__ __align__(16) float ps_smem[];
    float* sq = ps_smem;                             // [rows][pitch]
    float* skv = sq + kRows * kPitch;                // [stage][keys, values][32][pitch]
    float* sp = skv + 4 * kPsKeys * kPitch;          // [rows][33]
    __shared__ int row_token[kRows], row_last[kRows];
    __shared__ long place[2][kPsKeys];

    const int G = p.group, D = p.head_dim, kvh = blockIdx.y, tt = kRows / G > 0 ? kRows / G : 1;
    const int parts = (G + kRows - 1) / kRows, heads_at = (int)blockIdx.z % parts * kRows;       // first head of the group in this tile
    const int heads = min(G - heads_at, kRows), split = blockIdx.z / parts;
    int lo, hi, slot, n_tok, seq;
    if (own_tiles == 0) {                            // prefixes
        chain_wait();
        chain_release();                             // (only now: the own keys' kernel counts on what this one waited for)
        PrefixTile t;
        if (!prefix_tile(p, blockIdx.x, tt, t)) return;
        const int keys = prefix_piece(t.len, p.pieces, p.unit);
        lo = split * keys; hi = min(t.len, lo + keys); slot = split; n_tok = t.count; seq = p.group_seq[t.g];
        if (lo >= hi) return;
        for (int r = threadIdx.x; r < kRows; r += kPsThreads) {
            row_token[r] = r / heads < n_tok ? p.toks[t.first + r / heads] : -1;
            row_last[r] = hi - 1;
        }
    } else {
        chain_release();
        seq = (int)blockIdx.x / own_tiles;
        const int tok0 = (int)blockIdx.x % own_tiles * tt, n_new = p.seq_start[seq + 1] - p.seq_start[seq];
        if (tok0 >= n_new) { chain_wait(); return; }
        n_tok = min(tt, n_new - tok0);
        const int skip = p.seq_skip[seq], end = p.seq_pos0[seq] + tok0 + n_tok;
        const int keys = ((end - skip + p.own_splits - 1) / p.own_splits + kPsKeys - 1) / kPsKeys * kPsKeys;
        lo = skip + split * keys; hi = min(end, lo + keys); slot = p.pieces + split;
        for (int r = threadIdx.x; r < kRows; r += kPsThreads) {
            row_token[r] = r / heads < n_tok ? p.seq_start[seq] + tok0 + r / heads : -1;
            row_last[r] = p.seq_pos0[seq] + tok0 + min(r / heads, n_tok - 1);
        }
    }
    const int* pages = p.page_table + (size_t)p.seq_slot[seq] * p.max_pages;
    const T* kc = reinterpret_cast<const T*>(p.k_cache);
    const T* vc = reinterpret_cast<const T*>(p.v_cache);
    // where the rows of a tile lie: looked up by a thread a row, one tile before the tile is fetched
    auto find = [&](int key0, int which) {
        const int key = key0 + (int)threadIdx.x;
        if ((int)threadIdx.x < kPsKeys)
            place[which][threadIdx.x] = key < hi ? (((long)pages[key / p.page_size] * p.page_size + key % p.page_size) * p.n_kv_heads + kvh) * D : -1;
    };
    auto load = [&](int stage) {
        float* dk = skv + stage * 2 * kPsKeys * kPitch;
        float* dv = dk + kPsKeys * kPitch;
        if (wide) {                                  // floats, 16 bytes at a time, asynchronously
            const int chunks = kWidth / 4;
#pragma unroll 4
            for (int i = threadIdx.x; i < kPsKeys * chunks; i += kPsThreads) {
                const int r = i / chunks, c = i % chunks;
                const bool valid = place[stage][r] >= 0 && c * 4 < D;      // rows beyond belong to nobody: zeros instead
                const long at = valid ? place[stage][r] + c * 4 : 0;
                cp_async_16((uint32_t)__cvta_generic_to_shared(dk + r * kPitch + c * 4), kc + at, valid);
                cp_async_16((uint32_t)__cvta_generic_to_shared(dv + r * kPitch + c * 4), vc + at, valid);
            }
        } else {
#pragma unroll 4
            for (int i = threadIdx.x; i < kPsKeys * kWidth; i += kPsThreads) {
                const int r = i / kWidth, d = i % kWidth;
                float k = 0.f, v = 0.f;
                if (place[stage][r] >= 0 && d < D) { k = to_float(kc[place[stage][r] + d]); v = to_float(vc[place[stage][r] + d]); }
                dk[r * kPitch + d] = k; dv[r * kPitch + d] = v;
            }
        }
        cp_async_commit();
    };
    find(lo, 0);
    find(lo + kPsKeys, 1);
    __syncthreads();                                 // the rows' tokens and the first keys' places are known
    if (lo < hi) load(0);
    const T* q = reinterpret_cast<const T*>(p.q);
    if (wide) {
        constexpr int chunks = kWidth / 4;
#pragma unroll 8
        for (int i = threadIdx.x; i < kRows * chunks; i += kPsThreads) {
            const int r = i / chunks, c = i % chunks, token = row_token[r];
            float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
            if (token >= 0 && c * 4 < D) x = *reinterpret_cast<const float4*>(q + token * p.q_stride + (long)(kvh * G + heads_at + r % heads) * D + c * 4);
            *reinterpret_cast<float4*>(sq + r * kPitch + c * 4) = make_float4(x.x * p.scale_log2, x.y * p.scale_log2, x.z * p.scale_log2, x.w * p.scale_log2);
        }
    } else
#pragma unroll 4
    for (int i = threadIdx.x; i < kRows * kWidth; i += kPsThreads) {
        const int r = i / kWidth, d = i % kWidth, token = row_token[r];
        sq[r * kPitch + d] = token >= 0 && d < D ? to_float(q[token * p.q_stride + (long)(kvh * G + heads_at + r % heads) * D + d]) * p.scale_log2 : 0.f;
    }
    const int ty = threadIdx.x / KG, tx = threadIdx.x % KG, r0 = ty * RT;
    float m[RT], l[RT], acc[RT][DC][4];
#pragma unroll
    for (int i = 0; i < RT; ++i) {
        m[i] = -INFINITY; l[i] = 0.f;
#pragma unroll
        for (int c = 0; c < DC; ++c) acc[i][c][0] = acc[i][c][1] = acc[i][c][2] = acc[i][c][3] = 0.f;
    }
    const bool working = r0 < n_tok * heads;         // (whole groups of threads)
    const uint32_t group = ((1u << KG) - 1u) << ((threadIdx.x & 31) / KG * KG);      // this group's lanes
    int stage = 0;
    for (int key0 = lo; key0 < hi; key0 += kPsKeys, stage ^= 1) {
        if (key0 + kPsKeys < hi) load(stage ^ 1); else cp_async_commit();
        cp_async_wait<1>();
        __syncthreads();
        find(key0 + 2 * kPsKeys, stage);             // (the places of the keys that are here have been used)
        const float* sk = skv + stage * 2 * kPsKeys * kPitch;
        const float* sv = sk + kPsKeys * kPitch;
        if (working) {
            float s[RT][KT];
#pragma unroll
            for (int i = 0; i < RT; ++i)
#pragma unroll
                for (int j = 0; j < KT; ++j) s[i][j] = 0.f;
#pragma unroll 4
            for (int d = 0; d < kWidth; d += 4) {
                float4 a[RT];
#pragma unroll
                for (int i = 0; i < RT; ++i) a[i] = *reinterpret_cast<const float4*>(sq + (r0 + i) * kPitch + d);
#pragma unroll
                for (int j = 0; j < KT; ++j) {
                    const float4 k = *reinterpret_cast<const float4*>(sk + (tx + KG * j) * kPitch + d);
#pragma unroll
                    for (int i = 0; i < RT; ++i) s[i][j] = fmaf(a[i].x, k.x, fmaf(a[i].y, k.y, fmaf(a[i].z, k.z, fmaf(a[i].w, k.w, s[i][j]))));
                }
            }
#pragma unroll
            for (int i = 0; i < RT; ++i) {
                const int last = min(row_last[r0 + i], hi - 1);
                float mx = m[i];
#pragma unroll
                for (int j = 0; j < KT; ++j) {
                    if (key0 + tx + KG * j > last) s[i][j] = -INFINITY;
                    mx = fmaxf(mx, s[i][j]);
                }
#pragma unroll
                for (int o = 1; o < KG; o <<= 1) mx = fmaxf(mx, __shfl_xor_sync(group, mx, o));
                const float ref = mx == -INFINITY ? 0.f : mx, corr = exp2f(m[i] - ref);
                m[i] = mx;
                float sum = 0.f;
#pragma unroll
                for (int j = 0; j < KT; ++j) {
                    const float e = exp2f(s[i][j] - ref);
                    sum += e;
                    sp[(r0 + i) * (kPsKeys + 1) + tx + KG * j] = e;
                }
                l[i] = l[i] * corr + sum;
#pragma unroll
                for (int c = 0; c < DC; ++c) { acc[i][c][0] *= corr; acc[i][c][1] *= corr; acc[i][c][2] *= corr; acc[i][c][3] *= corr; }
            }
        }
        __syncwarp();                                // a row's weights are written and read by threads of one warp
        if (working) {
#pragma unroll 2
            for (int j = 0; j < kPsKeys; ++j) {
                float e[RT];
#pragma unroll
                for (int i = 0; i < RT; ++i) e[i] = sp[(r0 + i) * (kPsKeys + 1) + j];
#pragma unroll
                for (int c = 0; c < DC; ++c) {
                    const float4 v = *reinterpret_cast<const float4*>(sv + j * kPitch + c * 4 * KG + tx * 4);
#pragma unroll
                    for (int i = 0; i < RT; ++i) {
                        acc[i][c][0] = fmaf(e[i], v.x, acc[i][c][0]); acc[i][c][1] = fmaf(e[i], v.y, acc[i][c][1]);
                        acc[i][c][2] = fmaf(e[i], v.z, acc[i][c][2]); acc[i][c][3] = fmaf(e[i], v.w, acc[i][c][3]);
                    }
                }
            }
        }
        __syncthreads();                             // the stage may be overwritten
    }
    cp_async_wait<0>();
    const int slots = p.pieces + p.own_splits;
#pragma unroll
    for (int i = 0; i < RT; ++i) {
#pragma unroll
        for (int o = 1; o < KG; o <<= 1) l[i] += __shfl_xor_sync(0xffffffffu, l[i], o);
        const int r = r0 + i;
        if (r >= n_tok * heads) continue;
        const size_t row = (size_t)row_token[r] * p.n_heads + kvh * G + heads_at + r % heads;
        float* to = p.part_o + (row * slots + slot) * D;
#pragma unroll
        for (int c = 0; c < DC; ++c) {
            const int d = c * 4 * KG + tx * 4;
            if (wide) {
                if (d < D) *reinterpret_cast<float4*>(to + d) = make_float4(acc[i][c][0], acc[i][c][1], acc[i][c][2], acc[i][c][3]);
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e) if (d + e < D) to[d + e] = acc[i][c][e];
            }
        }
        if (tx == 0) { p.part_ml[(row * slots + slot) * 2] = m[i]; p.part_ml[(row * slots + slot) * 2 + 1] = l[i]; }
    }
    if (own_tiles > 0) chain_wait();                 // whoever waits for this kernel has waited for the prefixes', too
}

template <typename T, int RG, int RT, int DC>
static int launch_prefix_simple_as(const PrefixParams& p, bool own, int wide, cudaStream_t stream) {
    using S = PsShape<RG, RT, DC>;
    const int G = p.group, tt = S::kRows / G > 0 ? S::kRows / G : 1, parts = (G + S::kRows - 1) / S::kRows;
    const int own_tiles = own ? (p.max_new + tt - 1) / tt : 0;
    const long tiles = own ? (long)own_tiles * p.n_seqs : prefix_tiles_bound(p, tt);
    const int splits = own ? p.own_splits : p.pieces;
    MDMA_REQUIRE(tiles <= 0x7fffffffl && p.n_kv_heads <= 65535 && splits * parts <= 65535, "prefix_attention: grid too large");
    auto kernel = prefix_simple_kernel<T, RG, RT, DC>;
    cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, S::kFloats * 4);
    const dim3 grid((unsigned)tiles, p.n_kv_heads, splits * parts);
    if (e == cudaSuccess) e = launch_chained(kernel, grid, dim3(kPsThreads), S::kFloats * 4, stream, p, own_tiles, wide);
    if (e != cudaSuccess) return fail("prefix_attention: launch failed: %s", cudaGetErrorString(e));
    return 0;
}
// `rows`: how many of them a block should take
template <typename T>
static int launch_prefix_simple_rows(const PrefixParams& p, bool own, int rows, int wide, cudaStream_t stream) {
    const int D = p.head_dim;
    if (rows <= 8)
        return D <= 64    ? launch_prefix_simple_as<T, 8, 1, 1>(p, own, wide, stream)
               : D <= 128 ? launch_prefix_simple_as<T, 8, 1, 2>(p, own, wide, stream)
                          : launch_prefix_simple_as<T, 8, 1, 4>(p, own, wide, stream);
    if (rows <= 32 || D > 128)
        return D <= 64    ? launch_prefix_simple_as<T, 16, 2, 2>(p, own, wide, stream)
               : D <= 96  ? launch_prefix_simple_as<T, 16, 2, 3>(p, own, wide, stream)
               : D <= 128 ? launch_prefix_simple_as<T, 16, 2, 4>(p, own, wide, stream)
                          : launch_prefix_simple_as<T, 16, 2, 8>(p, own, wide, stream);
    return D <= 64   ? launch_prefix_simple_as<T, 16, 4, 2>(p, own, wide, stream)
           : D <= 96 ? launch_prefix_simple_as<T, 16, 4, 3>(p, own, wide, stream)
                     : launch_prefix_simple_as<T, 16, 4, 4>(p, own, wide, stream);
}

template <typename T>
static int launch_prefix_simple(const PrefixParams& p, int prefix_rows, int own_rows, cudaStream_t stream) {
    const int wide = sizeof(T) == 4 && p.head_dim % 4 == 0 && p.q_stride % 4 == 0 &&
                     (((uintptr_t)p.k_cache | (uintptr_t)p.v_cache | (uintptr_t)p.q | (uintptr_t)p.part_o) & 15) == 0;
    if (int rc = launch_prefix_simple_rows<T>(p, false, prefix_rows, wide, stream)) return rc;
    if (int rc = launch_prefix_simple_rows<T>(p, true, own_rows, wide, stream)) return rc;
    const cudaError_t e = launch_chained(prefix_merge_kernel<T>, dim3(prefix_merge_blocks(p)), dim3(128), 0, stream, p);
    if (e != cudaSuccess) return fail("prefix_attention: launch failed: %s", cudaGetErrorString(e));
    return 0;
}

}  // namespace mdma

using namespace mdma;

extern "C" int mdma_prefix_attention_simple(const long long* words, int n_words, float scale, int dtype, int prefix_rows, int own_rows,
                                            cudaStream_t stream) {
    PrefixParams p;
    if (int rc = prefix_params(words, n_words, scale, &p)) return rc;
    p.unit = kPsKeys;
    MDMA_REQUIRE(!p.whole && p.pieces > 0, "prefix_attention: %d and %d pieces are none of this kernel's", p.pieces, p.own_splits);
    if (p.n_tokens == 0 || p.n_seqs == 0) return 0;
    MDMA_DISPATCH_DTYPE(dtype, T, return launch_prefix_simple<T>(p, prefix_rows, own_rows, stream));
    return 0;
}
