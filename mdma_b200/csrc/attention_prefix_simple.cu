// Attention over shared prefixes on the CUDA cores: the true 32-bit engine's, and bfloat16 of any geometry (head sizes up to
// 256, any page size).  See prefix.cuh for the parts and how they join.
//
// A block takes 32 query rows of one kv head, (token, query head of the group) pairs, and walks its keys in tiles of 32:
// keys and values staged in shared memory as floats, a thread holds the scores of 2 rows x 4 keys and the sums of 2 rows x
// head_dim / 8 numbers.  Rows of a prefix tile come from all members of a group, so a key row is read once for 32 rows.
#include "prefix.cuh"

namespace mdma {

constexpr int kPsRows = 32, kPsKeys = 32, kPsThreads = 128;

template <typename T, int DC>                        // DC: head_dim rounded up to a multiple of 32, over 32
__global__ void __launch_bounds__(kPsThreads)
prefix_simple_kernel(const PrefixParams p, int prefix_tiles, int own_tiles) {
    constexpr int kPitch = DC * 32 + 4;              // floats of a staged row
    extern __shared__ __align__(16) float ps_smem[];
    float* sq = ps_smem;                             // [rows][pitch]
    float* sk = sq + kPsRows * kPitch;
    float* sv = sk + kPsKeys * kPitch;
    float* sp = sv + kPsKeys * kPitch;               // [rows][keys + 1]
    __shared__ int row_token[kPsRows], row_last[kPsRows];

    chain_release();
    chain_wait();
    const int G = p.group, D = p.head_dim, kvh = blockIdx.y, tt = kPsRows / G > 0 ? kPsRows / G : 1;
    const bool prefix = (int)blockIdx.x < prefix_tiles;
    const int heads_at = G > kPsRows ? (int)blockIdx.z % ((G + kPsRows - 1) / kPsRows) * kPsRows : 0;     // first head of the group in this tile
    const int heads = min(G - heads_at, kPsRows), split = G > kPsRows ? (int)blockIdx.z / ((G + kPsRows - 1) / kPsRows) : blockIdx.z;
    int lo, hi, slot, n_tok, seq;
    if (prefix) {
        PrefixTile t;
        if (split >= p.pieces || !prefix_tile(p, blockIdx.x, tt, t)) return;
        const int len = p.group_len[t.g], keys = prefix_piece(len, p.pieces);
        lo = split * keys; hi = min(len, lo + keys); slot = split; n_tok = t.count; seq = p.group_seq[t.g];
        if (lo >= hi) return;
        if ((int)threadIdx.x < kPsRows) {
            const int r = threadIdx.x;
            row_token[r] = r / heads < n_tok ? p.toks[t.first + r / heads] : -1;
            row_last[r] = hi - 1;
        }
    } else {
        seq = ((int)blockIdx.x - prefix_tiles) / own_tiles;
        const int tok0 = ((int)blockIdx.x - prefix_tiles) % own_tiles * tt, n_new = p.seq_start[seq + 1] - p.seq_start[seq];
        if (split >= p.own_splits || tok0 >= n_new) return;
        n_tok = min(tt, n_new - tok0);
        const int skip = p.seq_skip[seq], end = p.seq_pos0[seq] + tok0 + n_tok;
        const int keys = ((end - skip + p.own_splits - 1) / p.own_splits + kPsKeys - 1) / kPsKeys * kPsKeys;
        lo = skip + split * keys; hi = min(end, lo + keys); slot = p.pieces + split;
        if ((int)threadIdx.x < kPsRows) {
            const int r = threadIdx.x;
            row_token[r] = r / heads < n_tok ? p.seq_start[seq] + tok0 + r / heads : -1;
            row_last[r] = p.seq_pos0[seq] + tok0 + min(r / heads, n_tok - 1);
        }
    }
    __syncthreads();
    const T* q = reinterpret_cast<const T*>(p.q);
    for (int i = threadIdx.x; i < kPsRows * kPitch; i += kPsThreads) {
        const int r = i / kPitch, d = i % kPitch, token = row_token[r];
        sq[i] = token >= 0 && d < D ? to_float(q[token * p.q_stride + (long)(kvh * G + heads_at + r % heads) * D + d]) * p.scale_log2 : 0.f;
    }
    const int* pages = p.page_table + (size_t)p.seq_slot[seq] * p.max_pages;
    const T* kc = reinterpret_cast<const T*>(p.k_cache);
    const T* vc = reinterpret_cast<const T*>(p.v_cache);
    const int ty = threadIdx.x >> 3, tx = threadIdx.x & 7, r0 = ty * 2;
    float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f}, acc[2][DC][4];
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int c = 0; c < DC; ++c) acc[i][c][0] = acc[i][c][1] = acc[i][c][2] = acc[i][c][3] = 0.f;
    const bool working = r0 < n_tok * heads;         // (whole groups of eight lanes)
    for (int key0 = lo; key0 < hi; key0 += kPsKeys) {
        __syncthreads();
        for (int i = threadIdx.x; i < kPsKeys * DC * 32; i += kPsThreads) {
            const int r = i / (DC * 32), d = i % (DC * 32), key = key0 + r;
            float k = 0.f, v = 0.f;                  // rows beyond the last key belong to nobody: never read
            if (key < hi && d < D) {
                const size_t at = (((size_t)pages[key / p.page_size] * p.page_size + key % p.page_size) * p.n_kv_heads + kvh) * D + d;
                k = to_float(kc[at]); v = to_float(vc[at]);
            }
            sk[r * kPitch + d] = k; sv[r * kPitch + d] = v;
        }
        __syncthreads();
        float s[2][4];
#pragma unroll
        for (int i = 0; i < 2; ++i) s[i][0] = s[i][1] = s[i][2] = s[i][3] = 0.f;
        if (working) {
#pragma unroll 4
            for (int d = 0; d < DC * 32; d += 4) {
                const float4 a = *reinterpret_cast<const float4*>(sq + r0 * kPitch + d), b = *reinterpret_cast<const float4*>(sq + (r0 + 1) * kPitch + d);
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const float4 k = *reinterpret_cast<const float4*>(sk + (tx + 8 * j) * kPitch + d);
                    s[0][j] = fmaf(a.x, k.x, fmaf(a.y, k.y, fmaf(a.z, k.z, fmaf(a.w, k.w, s[0][j]))));
                    s[1][j] = fmaf(b.x, k.x, fmaf(b.y, k.y, fmaf(b.z, k.z, fmaf(b.w, k.w, s[1][j]))));
                }
            }
        }
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int last = min(row_last[r0 + i], hi - 1);
            float mx = m[i];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                if (key0 + tx + 8 * j > last) s[i][j] = -INFINITY;
                mx = fmaxf(mx, s[i][j]);
            }
#pragma unroll
            for (int o = 1; o < 8; o <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
            const float ref = mx == -INFINITY ? 0.f : mx, corr = exp2f(m[i] - ref);
            m[i] = mx;
            float sum = 0.f;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float e = exp2f(s[i][j] - ref);
                sum += e;
                sp[(r0 + i) * (kPsKeys + 1) + tx + 8 * j] = e;
            }
            l[i] = l[i] * corr + sum;
#pragma unroll
            for (int c = 0; c < DC; ++c) { acc[i][c][0] *= corr; acc[i][c][1] *= corr; acc[i][c][2] *= corr; acc[i][c][3] *= corr; }
        }
        __syncwarp();                                // a row's weights are written and read by eight lanes of one warp
        if (working) {
#pragma unroll 2
            for (int j = 0; j < kPsKeys; ++j) {
                const float e0 = sp[r0 * (kPsKeys + 1) + j], e1 = sp[(r0 + 1) * (kPsKeys + 1) + j];
#pragma unroll
                for (int c = 0; c < DC; ++c) {
                    const float4 v = *reinterpret_cast<const float4*>(sv + j * kPitch + c * 32 + tx * 4);
                    acc[0][c][0] = fmaf(e0, v.x, acc[0][c][0]); acc[0][c][1] = fmaf(e0, v.y, acc[0][c][1]);
                    acc[0][c][2] = fmaf(e0, v.z, acc[0][c][2]); acc[0][c][3] = fmaf(e0, v.w, acc[0][c][3]);
                    acc[1][c][0] = fmaf(e1, v.x, acc[1][c][0]); acc[1][c][1] = fmaf(e1, v.y, acc[1][c][1]);
                    acc[1][c][2] = fmaf(e1, v.z, acc[1][c][2]); acc[1][c][3] = fmaf(e1, v.w, acc[1][c][3]);
                }
            }
        }
        __syncwarp();
    }
    const int slots = p.pieces + p.own_splits;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
#pragma unroll
        for (int o = 1; o < 8; o <<= 1) l[i] += __shfl_xor_sync(0xffffffffu, l[i], o);
        const int r = r0 + i;
        if (r >= n_tok * heads) continue;
        const size_t row = (size_t)row_token[r] * p.n_heads + kvh * G + heads_at + r % heads;
        float* to = p.part_o + (row * slots + slot) * D;
#pragma unroll
        for (int c = 0; c < DC; ++c)
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (c * 32 + tx * 4 + e < D) to[c * 32 + tx * 4 + e] = acc[i][c][e];
        if (tx == 0) { p.part_ml[(row * slots + slot) * 2] = m[i]; p.part_ml[(row * slots + slot) * 2 + 1] = l[i]; }
    }
}

template <typename T>
static int launch_prefix_simple(const PrefixParams& p, cudaStream_t stream) {
    const int G = p.group, tt = kPsRows / G > 0 ? kPsRows / G : 1, parts = (G + kPsRows - 1) / kPsRows;
    const int own_tiles = (p.max_new + tt - 1) / tt;
    const long prefix_tiles = prefix_tiles_bound(p, tt), tiles = prefix_tiles + (long)own_tiles * p.n_seqs;
    const int splits = p.pieces > p.own_splits ? p.pieces : p.own_splits;
    MDMA_REQUIRE(tiles <= 0x7fffffffl && p.n_kv_heads <= 65535 && splits * parts <= 65535, "prefix_attention: grid too large");
    const dim3 grid((unsigned)tiles, p.n_kv_heads, splits * parts);
    const int dc = (p.head_dim + 31) / 32;
    auto run = [&](auto kernel, int pitch_dc) -> int {
        const int pitch = pitch_dc * 32 + 4, bytes = ((kPsRows + 2 * kPsKeys) * pitch + kPsRows * (kPsKeys + 1)) * 4;
        cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
        if (e == cudaSuccess) e = launch_chained(kernel, grid, dim3(kPsThreads), bytes, stream, p, (int)prefix_tiles, own_tiles);
        if (e != cudaSuccess) return fail("prefix_attention: launch failed: %s", cudaGetErrorString(e));
        return 0;
    };
    const int rc = dc <= 2 ? run(prefix_simple_kernel<T, 2>, 2) : dc <= 4 ? run(prefix_simple_kernel<T, 4>, 4) : run(prefix_simple_kernel<T, 8>, 8);
    if (rc) return rc;
    const long rows = (long)p.n_tokens * p.n_heads;
    const cudaError_t e = launch_chained(prefix_merge_kernel<T>, dim3((unsigned)((rows + 3) / 4)), dim3(128), 0, stream, p);
    if (e != cudaSuccess) return fail("prefix_attention: launch failed: %s", cudaGetErrorString(e));
    return 0;
}

}  // namespace mdma

using namespace mdma;

extern "C" int mdma_prefix_attention_simple(const long long* words, int n_words, float scale, int dtype, cudaStream_t stream) {
    PrefixParams p;
    if (int rc = prefix_params(words, n_words, scale, &p)) return rc;
    if (p.n_tokens == 0 || p.n_seqs == 0) return 0;
    MDMA_DISPATCH_DTYPE(dtype, T, return launch_prefix_simple<T>(p, stream));
    return 0;
}
