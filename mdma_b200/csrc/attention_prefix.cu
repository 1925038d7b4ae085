// Attention over shared prefixes on the tensor cores (bfloat16 in, float softmax and accumulation).  See prefix.cuh for the
// parts and how they join.
#include <mutex>

#include "attention_prefix_own.cuh"
#include "attention_prefix_tc.cuh"
#include "mma_tiles.cuh"
#include "prefix.cuh"

namespace mdma {

constexpr int kPrRows = 64, kPrKeys = 64, kPrThreads = 128;

// Any page size, any step: 64 query rows of one kv head, (token, query head of the group) pairs, against a run of keys in
// blocks of 64 (cp.async, looked up row by row, two blocks in flight), products by mma.sync.  The rows of a prefix tile come
// from all members of a group; those of an own tile are one sequence's.  Every tile leaves its sums, maxima and sums of weights for
// the merge.  16 sequences behind 2,048 tokens on pages of 16, 32/8 heads of 128: 48 us with own keys and merge (79 where every one
// reads by itself); lookups row by row and three dependent kernels at latency bound it.
template <int DMAX>
__global__ void __launch_bounds__(kPrThreads)
prefix_rows_kernel(const PrefixParams p, int own_tiles) {           // own_tiles: of a sequence; 0: the prefixes
    constexpr int kChunks = DMAX / 8, kTile = kPrRows * DMAX * 2;
    extern __shared__ __align__(1024) uint8_t smem[];
    __shared__ int row_token[kPrRows];
    const uint32_t sQ = (uint32_t)__cvta_generic_to_shared(smem), sK = sQ + kTile, sV = sK + 2 * kTile;

    chain_wait();
    // only now: a kernel that starts early behind this one may count on what this one waited for
    chain_release();
    const int G = p.group, D = p.head_dim, kvh = blockIdx.y, tt = kPrRows / G, split = blockIdx.z;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const bool prefix = own_tiles == 0;
    int lo, hi, slot, n_tok, seq, first_pos = 0;     // keys [lo, hi); the tile's tokens stand at first_pos, first_pos + 1, ..
    if (prefix) {
        PrefixTile t;
        if (!prefix_tile(p, blockIdx.x, tt, t)) return;
        const int len = p.group_len[t.g], keys = prefix_piece(len, p.pieces, p.unit);
        lo = split * keys; hi = min(len, lo + keys); slot = split; n_tok = t.count; seq = p.group_seq[t.g];
        if (lo >= hi) return;
        if ((int)threadIdx.x < kPrRows) row_token[threadIdx.x] = (int)threadIdx.x / G < n_tok ? p.toks[t.first + threadIdx.x / G] : -1;
    } else {
        seq = (int)blockIdx.x / own_tiles;
        const int tok0 = (int)blockIdx.x % own_tiles * tt, n_new = p.seq_start[seq + 1] - p.seq_start[seq];
        if (tok0 >= n_new) return;
        n_tok = min(tt, n_new - tok0);
        first_pos = p.seq_pos0[seq] + tok0;
        const int skip = p.seq_skip[seq], end = first_pos + n_tok;
        const int keys = ((end - skip + p.own_splits - 1) / p.own_splits + kPrKeys - 1) / kPrKeys * kPrKeys;
        lo = skip + split * keys; hi = min(end, lo + keys); slot = p.pieces + split;
        if ((int)threadIdx.x < kPrRows) row_token[threadIdx.x] = (int)threadIdx.x / G < n_tok ? p.seq_start[seq] + tok0 + (int)threadIdx.x / G : -1;
    }
    __syncthreads();
    const int* pages = p.page_table + (size_t)p.seq_slot[seq] * p.max_pages;
    const __nv_bfloat16* q = reinterpret_cast<const __nv_bfloat16*>(p.q);
    const __nv_bfloat16* kc = reinterpret_cast<const __nv_bfloat16*>(p.k_cache);
    const __nv_bfloat16* vc = reinterpret_cast<const __nv_bfloat16*>(p.v_cache);
    for (int i = threadIdx.x; i < kPrRows * kChunks; i += kPrThreads) {
        const int r = i / kChunks, c = i % kChunks, token = row_token[r];
        const bool valid = token >= 0 && c * 8 < D;
        cp_async_16(sQ + tile_offset<DMAX>(r, c), valid ? q + (size_t)token * p.q_stride + (size_t)(kvh * G + r % G) * D + c * 8 : q, valid);
    }
    auto load_kv = [&](int key0, int stage) {
        for (int i = threadIdx.x; i < kPrKeys * kChunks; i += kPrThreads) {
            const int r = i / kChunks, c = i % kChunks, key = key0 + r;
            const bool valid = key < hi && c * 8 < D;              // rows beyond belong to nobody: zeros instead
            size_t off = 0;
            if (valid) off = (((size_t)pages[key / p.page_size] * p.page_size + key % p.page_size) * p.n_kv_heads + kvh) * D + c * 8;
            cp_async_16(sK + stage * kTile + tile_offset<DMAX>(r, c), kc + off, valid);
            cp_async_16(sV + stage * kTile + tile_offset<DMAX>(r, c), vc + off, valid);
        }
    };
    if (lo < hi) load_kv(lo, 0);
    cp_async_commit();

    const int r_lo = warp * 16 + (lane >> 2), r_hi = r_lo + 8;
    const int last_lo = prefix ? hi - 1 : min(first_pos + min(r_lo / G, n_tok - 1), hi - 1);
    const int last_hi = prefix ? hi - 1 : min(first_pos + min(r_hi / G, n_tok - 1), hi - 1);
    float o[DMAX / 8][4];
#pragma unroll
    for (int n = 0; n < DMAX / 8; ++n) { o[n][0] = o[n][1] = o[n][2] = o[n][3] = 0.f; }
    float m_lo = -INFINITY, m_hi = -INFINITY, l_lo = 0.f, l_hi = 0.f;
    int stage = 0;
    for (int key0 = lo; key0 < hi; key0 += kPrKeys, stage ^= 1) {
        if (key0 + kPrKeys < hi) load_kv(key0 + kPrKeys, stage ^ 1);
        cp_async_commit();
        cp_async_wait<1>();
        __syncthreads();
        float s[kPrKeys / 8][4];
#pragma unroll
        for (int n = 0; n < kPrKeys / 8; ++n) { s[n][0] = s[n][1] = s[n][2] = s[n][3] = 0.f; }
#pragma unroll
        for (int kd = 0; kd < DMAX / 16; ++kd) {
            if (kd * 16 < D) {
                uint32_t a0, a1, a2, a3;
                ldmatrix_x4(sQ + tile_offset<DMAX>(warp * 16 + (lane & 15), kd * 2 + (lane >> 4)), a0, a1, a2, a3);
#pragma unroll
                for (int n2 = 0; n2 < kPrKeys / 16; ++n2) {
                    uint32_t k0, k1, k2, k3;
                    const int krow = n2 * 16 + (lane & 7) + ((lane >> 4) << 3);
                    ldmatrix_x4(sK + stage * kTile + tile_offset<DMAX>(krow, kd * 2 + ((lane >> 3) & 1)), k0, k1, k2, k3);
                    mma_16816(s[n2 * 2], a0, a1, a2, a3, k0, k1);
                    mma_16816(s[n2 * 2 + 1], a0, a1, a2, a3, k2, k3);
                }
            }
        }
        float mx_lo = m_lo, mx_hi = m_hi;
#pragma unroll
        for (int n = 0; n < kPrKeys / 8; ++n) {
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const int key = key0 + n * 8 + (lane & 3) * 2 + e;
                s[n][e] = key <= last_lo ? s[n][e] * p.scale_log2 : -INFINITY;
                s[n][2 + e] = key <= last_hi ? s[n][2 + e] * p.scale_log2 : -INFINITY;
                mx_lo = fmaxf(mx_lo, s[n][e]); mx_hi = fmaxf(mx_hi, s[n][2 + e]);
            }
        }
        mx_lo = fmaxf(mx_lo, __shfl_xor_sync(0xffffffffu, mx_lo, 1)); mx_lo = fmaxf(mx_lo, __shfl_xor_sync(0xffffffffu, mx_lo, 2));
        mx_hi = fmaxf(mx_hi, __shfl_xor_sync(0xffffffffu, mx_hi, 1)); mx_hi = fmaxf(mx_hi, __shfl_xor_sync(0xffffffffu, mx_hi, 2));
        const float ref_lo = mx_lo == -INFINITY ? 0.f : mx_lo, ref_hi = mx_hi == -INFINITY ? 0.f : mx_hi;
        const float corr_lo = exp2f(m_lo - ref_lo), corr_hi = exp2f(m_hi - ref_hi);
        m_lo = mx_lo; m_hi = mx_hi;
        float sum_lo = 0.f, sum_hi = 0.f;
        uint32_t pa[kPrKeys / 16][4];                  // the weights are rounded to bfloat16 for the second product
#pragma unroll
        for (int n = 0; n < kPrKeys / 8; ++n) {
            const float p0 = exp2f(s[n][0] - ref_lo), p1 = exp2f(s[n][1] - ref_lo), p2 = exp2f(s[n][2] - ref_hi), p3 = exp2f(s[n][3] - ref_hi);
            sum_lo += p0 + p1; sum_hi += p2 + p3;
            pa[n >> 1][(n & 1) * 2] = pack_bf16(p0, p1);
            pa[n >> 1][(n & 1) * 2 + 1] = pack_bf16(p2, p3);
        }
        l_lo = l_lo * corr_lo + sum_lo; l_hi = l_hi * corr_hi + sum_hi;
#pragma unroll
        for (int n = 0; n < DMAX / 8; ++n) { o[n][0] *= corr_lo; o[n][1] *= corr_lo; o[n][2] *= corr_hi; o[n][3] *= corr_hi; }
#pragma unroll
        for (int kk = 0; kk < kPrKeys / 16; ++kk) {
#pragma unroll
            for (int n2 = 0; n2 < DMAX / 16; ++n2) {
                if (n2 * 16 < D) {
                    uint32_t v0, v1, v2, v3;
                    const int vrow = kk * 16 + (lane & 7) + (((lane >> 3) & 1) << 3);
                    ldmatrix_x4_trans(sV + stage * kTile + tile_offset<DMAX>(vrow, n2 * 2 + (lane >> 4)), v0, v1, v2, v3);
                    mma_16816(o[n2 * 2], pa[kk][0], pa[kk][1], pa[kk][2], pa[kk][3], v0, v1);
                    mma_16816(o[n2 * 2 + 1], pa[kk][0], pa[kk][1], pa[kk][2], pa[kk][3], v2, v3);
                }
            }
        }
        __syncthreads();
    }
    cp_async_wait<0>();
    l_lo += __shfl_xor_sync(0xffffffffu, l_lo, 1); l_lo += __shfl_xor_sync(0xffffffffu, l_lo, 2);
    l_hi += __shfl_xor_sync(0xffffffffu, l_hi, 1); l_hi += __shfl_xor_sync(0xffffffffu, l_hi, 2);
    const int slots = p.pieces + p.own_splits;
#pragma unroll
    for (int half = 0; half < 2; ++half) {
        const int r = half ? r_hi : r_lo, token = row_token[r];
        if (token < 0) continue;
        const size_t at = ((size_t)token * p.n_heads + kvh * G + r % G) * slots + slot;
#pragma unroll
        for (int n = 0; n < DMAX / 8; ++n) {
            const int d = n * 8 + (lane & 3) * 2;
            if (d < D) *reinterpret_cast<float2*>(p.part_o + at * D + d) = make_float2(o[n][half * 2], o[n][half * 2 + 1]);
        }
        if ((lane & 3) == 0) *reinterpret_cast<float2*>(p.part_ml + at * 2) = make_float2(half ? m_hi : m_lo, half ? l_hi : l_lo);
    }
}

static int launch_prefix_merge(const PrefixParams& p, cudaStream_t stream) {
    const cudaError_t e = launch_chained(prefix_merge_kernel<__nv_bfloat16>, dim3(prefix_merge_blocks(p)), dim3(128), 0, stream, p);
    if (e != cudaSuccess) return fail("prefix_attention: launch failed: %s", cudaGetErrorString(e));
    return 0;
}

// The prefixes, or the sequences' own keys.
static int launch_prefix_rows(const PrefixParams& p, bool own, cudaStream_t stream) {
    const int tt = kPrRows / p.group, own_tiles = own ? (p.max_new + tt - 1) / tt : 0, splits = own ? p.own_splits : p.pieces;
    const long tiles = own ? (long)own_tiles * p.n_seqs : prefix_tiles_bound(p, tt);
    MDMA_REQUIRE(tiles <= 0x7fffffffl && p.n_kv_heads <= 65535 && splits <= 65535, "prefix_attention: grid too large");
    auto run = [&](auto kernel, int dmax) -> int {
        const int bytes = 5 * kPrRows * dmax * 2;
        cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
        if (e == cudaSuccess) e = launch_chained(kernel, dim3((unsigned)tiles, p.n_kv_heads, splits), dim3(kPrThreads), bytes, stream, p, own_tiles);
        if (e != cudaSuccess) return fail("prefix_attention: launch failed: %s", cudaGetErrorString(e));
        return 0;
    };
    return p.head_dim <= 64 ? run(prefix_rows_kernel<64>, 64) : run(prefix_rows_kernel<128>, 128);
}

// A tensor map over a cache [pages, page_size, kv_heads, head_dim] with boxes of 64 numbers x 1 head x `keys` keys x 1 page
// (128-byte swizzle).
typedef CUresult (*PrefixEncodeFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                                   const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                   CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
static int prefix_cache_map(CUtensorMap* out, const void* cache, const PrefixParams& p, int keys) {
    static PrefixEncodeFn fn = nullptr;
    static std::once_flag once;
    std::call_once(once, [] {
        void* sym = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &sym, cudaEnableDefault, &q) == cudaSuccess &&
            q == cudaDriverEntryPointSuccess)
            fn = reinterpret_cast<PrefixEncodeFn>(sym);
    });
    if (!fn) return fail("prefix_attention: the driver does not offer cuTensorMapEncodeTiled");
    const cuuint64_t row = (cuuint64_t)p.n_kv_heads * p.head_dim * 2;
    cuuint64_t dims[4] = {(cuuint64_t)p.head_dim, (cuuint64_t)p.n_kv_heads, (cuuint64_t)p.page_size, (cuuint64_t)p.n_pages};
    cuuint64_t strides[3] = {(cuuint64_t)p.head_dim * 2, row, row * p.page_size};
    cuuint32_t box[4] = {64, 1, (cuuint32_t)keys, 1}, elem[4] = {1, 1, 1, 1};
    const CUresult r = fn(out, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, const_cast<void*>(cache), dims, strides, box, elem,
                          CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                          CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) return fail("prefix_attention: cuTensorMapEncodeTiled failed with %d", (int)r);
    return 0;
}

static bool prefix_stream_fits(const PrefixParams& p) {
    return p.max_new == 1 && p.n_tokens == p.n_seqs && p.group <= 16 && p.page_size % 32 == 0 && p.pieces <= kPoMaxPieces && p.own_splits >= 1;
}
// The sequences' own keys, or the prefixes.
template <bool SHARED>
static int launch_prefix_stream(const PrefixParams& p, int sms, cudaStream_t stream) {
    const int kb = p.head_dim <= 64 && p.page_size % 64 == 0 ? 64 : 32;       // a tile of 8 KB either way
    const long items = SHARED ? prefix_tiles_bound(p, 16 / p.group) : p.n_seqs, splits = SHARED ? p.pieces : p.own_splits;
    // (those that have something to do, about: of a sequence's pieces one, so that its sums do not follow from how many there are)
    const long blocks = p.n_kv_heads * (SHARED ? splits * ((p.n_tokens * p.group + 15) / 16) : items);
    MDMA_REQUIRE(items <= 65535 && p.n_kv_heads * splits <= 0x7fffffffl, "prefix_attention: grid too large");
    CUtensorMap mk, mv;
    if (int rc = prefix_cache_map(&mk, p.k_cache, p, kb)) return rc;
    if (int rc = prefix_cache_map(&mv, p.v_cache, p, kb)) return rc;
    auto run = [&](auto kernel, int nw, int bytes) -> int {
        cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
        if (e == cudaSuccess) e = launch_chained(kernel, dim3((unsigned)(p.n_kv_heads * splits), (unsigned)items), dim3(nw * 32), bytes, stream, mk, mv, p);
        if (e != cudaSuccess) return fail("prefix_attention: launch failed: %s", cudaGetErrorString(e));
        return 0;
    };
    // as many warps a block as leave every block resident at once, two at least (51 sequences x 32 kv heads, own keys and prefixes:
    // 53 us in rounds of two-warp blocks, 56 with one warp, 67 with four; a sequence of 30,000 own keys in 8 pieces beside four
    // of 100, 8 kv heads: 61 us, with the warps for all pieces' blocks 98)
    const int nw = blocks <= sms ? 12 : blocks <= 3l * sms ? 4 : blocks <= 4l * sms ? 3 : 2;
#define MDMA_STREAM(DM, KB) (nw == 12 ? run(prefix_stream_kernel<DM, KB, 12, SHARED>, 12, PoSmem<DM, KB, 12>::kBytes) \
                           : nw == 4 ? run(prefix_stream_kernel<DM, KB, 4, SHARED>, 4, PoSmem<DM, KB, 4>::kBytes) \
                           : nw == 3 ? run(prefix_stream_kernel<DM, KB, 3, SHARED>, 3, PoSmem<DM, KB, 3>::kBytes) \
                                     : run(prefix_stream_kernel<DM, KB, 2, SHARED>, 2, PoSmem<DM, KB, 2>::kBytes))
    return kb == 64 ? MDMA_STREAM(64, 64) : p.head_dim <= 64 ? MDMA_STREAM(64, 32) : MDMA_STREAM(128, 32);
#undef MDMA_STREAM
}

static int launch_prefix_tc(const PrefixParams& p, cudaStream_t stream) {
    const long tiles = prefix_tiles_bound(p, 2 * (kPtRows / p.group));
    MDMA_REQUIRE(tiles <= 65535 && p.pieces <= 65535, "prefix_attention: grid too large");
    CUtensorMap mk, mv;
    if (int rc = prefix_cache_map(&mk, p.k_cache, p, 64)) return rc;
    if (int rc = prefix_cache_map(&mv, p.v_cache, p, 64)) return rc;
    cudaError_t e = cudaFuncSetAttribute(prefix_tc_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kPtSmem);
    if (e == cudaSuccess) e = launch_chained(prefix_tc_kernel, dim3(p.n_kv_heads, (unsigned)tiles, p.pieces), dim3(kPtThreads), kPtSmem, stream, mk, mv, p);
    if (e != cudaSuccess) return fail("prefix_attention: launch failed: %s", cudaGetErrorString(e));
    return 0;
}

}  // namespace mdma

using namespace mdma;

// `kind`: who does the prefixes: 0 the tcgen05 kernel (which also takes whole lists of keys), 1 the streaming one, 2 the one for
// any page size; the own keys of single tokens are streamed where the geometry allows.
extern "C" int mdma_prefix_attention(const long long* words, int n_words, float scale, int kind, cudaStream_t stream) {
    PrefixParams p;
    if (int rc = prefix_params(words, n_words, scale, &p)) return rc;
    MDMA_REQUIRE(p.head_dim % 16 == 0 && p.head_dim <= 128 && p.group <= kPrRows,
                 "prefix_attention: heads %d / kv heads %d / head_dim %d is outside its limits (head_dim a multiple of 16 up to 128, group up to 64)",
                 p.n_heads, p.n_kv_heads, p.head_dim);
    MDMA_REQUIRE(p.q_stride % 8 == 0 && (((uintptr_t)p.q | (uintptr_t)p.k_cache | (uintptr_t)p.v_cache) & 15) == 0, "prefix_attention: rows must be 16-byte aligned");
    MDMA_REQUIRE(((uintptr_t)p.out & 15) == 0, "prefix_attention: the results must be 16-byte aligned");
    MDMA_REQUIRE(kind >= 0 && kind <= 2 && (kind == 0 || !p.whole), "prefix_attention: no kernel %d for this step", kind);
    MDMA_REQUIRE(kind != 0 || p.page_size % 64 == 0, "prefix_attention: the tcgen05 kernel wants pages of a multiple of 64 tokens");
    MDMA_REQUIRE(kind != 1 || prefix_stream_fits(p),
                 "prefix_attention: the streaming kernel wants single tokens, pages of a multiple of 32 tokens and groups of up to 16 heads");
    MDMA_REQUIRE(p.pieces > 0 || prefix_stream_fits(p), "prefix_attention: prefixes in no pieces");
    if (p.n_tokens == 0 || p.n_seqs == 0) return 0;
    p.unit = kind == 0 ? kPtKeys : 64;
    int sms = 0, dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess)
        return fail("prefix_attention: no CUDA device");
    if (p.pieces > 0) {
        const int rc = kind == 0   ? launch_prefix_tc(p, stream)
                       : kind == 1 ? launch_prefix_stream<true>(p, sms, stream)
                                   : launch_prefix_rows(p, false, stream);
        if (rc) return rc;
        if (p.whole && p.pieces == 1) return 0;
    }
    if (!p.whole) {
        const bool stream_own = prefix_stream_fits(p);
        if (int rc = stream_own ? launch_prefix_stream<false>(p, sms, stream) : launch_prefix_rows(p, true, stream)) return rc;
        if (stream_own && p.own_splits == 1) return 0;
    }
    return launch_prefix_merge(p, stream);
}
