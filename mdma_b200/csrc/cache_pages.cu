// Copies of cache pages: rows of pages (or whole ones) to other pages of the same pools, at every site, for keys and values
// alike, in one launch; also rows of per-sequence state (a slot is a page of one row).
//
// A pool is [sites][pages][page_size][...]; copy i brings the first rows[i] rows of page src[i] to page dst[i].  The list
// travels in the kernel's parameters: nothing is uploaded, the host does not wait, and a captured launch keeps its list.
// It is bound by memory: a block keeps 16 KB of a page in registers and writes them to every copy of that page in its run,
// so a page that many sequences fork from is read from memory once (runs of one page's copies are cut where there would be
// too few blocks; the second run's reads come from L2).
#include "common.cuh"

namespace mdma {

constexpr int kCopyThreads = 256, kCopyUnroll = 4, kCopyPools = 32;

struct CopyPools {
    char* base[kCopyPools];
    long page_bytes[kCopyPools], site_bytes[kCopyPools], row_bytes[kCopyPools];
    int first_site[kCopyPools + 1];          // sites of all pools in one count
    int n_pools;
};
template <int N>
struct CopyList {                            // copies of one page follow one another; run r: copies run[r] .. run[r + 1]
    int src[N], dst[N], rows[N];
    int run[N + 1];
};

template <typename V, int N>
__global__ void __launch_bounds__(kCopyThreads)
copy_pages_kernel(const __grid_constant__ CopyPools pools, const __grid_constant__ CopyList<N> list) {
    chain_wait();
    int pool = 0;
    while ((int)blockIdx.z >= pools.first_site[pool + 1]) ++pool;
    const int e0 = list.run[blockIdx.y], e1 = list.run[blockIdx.y + 1];
    const long n = list.rows[e0] * pools.row_bytes[pool] / (long)sizeof(V);
    const long at = (long)blockIdx.x * (kCopyThreads * kCopyUnroll) + threadIdx.x;
    if (at >= n) return;
    char* site = pools.base[pool] + (blockIdx.z - pools.first_site[pool]) * pools.site_bytes[pool];
    const V* from = reinterpret_cast<const V*>(site + list.src[e0] * pools.page_bytes[pool]);
    V r[kCopyUnroll];
#pragma unroll
    for (int u = 0; u < kCopyUnroll; ++u)
        if (at + u * kCopyThreads < n) r[u] = from[at + u * kCopyThreads];
    for (int e = e0; e < e1; ++e) {
        V* to = reinterpret_cast<V*>(site + list.dst[e] * pools.page_bytes[pool]);
#pragma unroll
        for (int u = 0; u < kCopyUnroll; ++u)
            if (at + u * kCopyThreads < n) to[at + u * kCopyThreads] = r[u];
    }
}

struct CopyItem { int src, dst, rows; };
static int copy_order(const void* a, const void* b) {
    const CopyItem *x = (const CopyItem*)a, *y = (const CopyItem*)b;
    if (x->src != y->src) return x->src < y->src ? -1 : 1;
    if (x->rows != y->rows) return x->rows > y->rows ? -1 : 1;
    return x->dst < y->dst ? -1 : x->dst > y->dst ? 1 : 0;
}

template <int N>
static int launch_copies(const CopyPools& pools, const CopyItem* items, int n, int vec, int sms, cudaStream_t stream) {
    CopyList<N> list;
    long most = 0;
    const int sites = pools.first_site[pools.n_pools];
    for (int i = 0; i < n; ++i) {
        list.src[i] = items[i].src; list.dst[i] = items[i].dst; list.rows[i] = items[i].rows;
        for (int q = 0; q < pools.n_pools; ++q) {
            const long bytes = items[i].rows * pools.row_bytes[q];
            most = bytes > most ? bytes : most;
        }
    }
    const long chunk = (long)kCopyThreads * kCopyUnroll * vec, chunks = (most + chunk - 1) / chunk;
    MDMA_REQUIRE(chunks <= 0x7fffffffl && sites <= 65535, "copy_pages: grid too large");
    // a run is as long as leaves eight blocks an SM, sixteen copies at most
    long longest = chunks * sites * n / (8l * sms);
    longest = longest < 1 ? 1 : longest > 16 ? 16 : longest;
    int runs = 0;
    for (int i = 0; i < n; ++i) {
        const bool same = i > 0 && items[i].src == items[i - 1].src && items[i].rows == items[i - 1].rows;
        if (!same || i - list.run[runs - 1] >= longest) list.run[runs++] = i;
    }
    list.run[runs] = n;
    const dim3 grid((unsigned)chunks, runs, sites);
    cudaError_t e = vec == 16 ? launch_chained(copy_pages_kernel<uint4, N>, grid, dim3(kCopyThreads), 0, stream, pools, list)
                  : vec == 4 ? launch_chained(copy_pages_kernel<uint32_t, N>, grid, dim3(kCopyThreads), 0, stream, pools, list)
                  : vec == 2 ? launch_chained(copy_pages_kernel<uint16_t, N>, grid, dim3(kCopyThreads), 0, stream, pools, list)
                             : launch_chained(copy_pages_kernel<uint8_t, N>, grid, dim3(kCopyThreads), 0, stream, pools, list);
    if (e != cudaSuccess) return fail("copy_pages: launch failed: %s", cudaGetErrorString(e));
    return 0;
}

}  // namespace mdma

using namespace mdma;

// words: number of pools, pages, rows a page, copies, addresses of the lists (source pages, destination pages, leading rows of each
// copy or null: whole pages), the number of launches (written here); then for every pool its address, bytes of a page, of a site
// and of a row, and its sites.
extern "C" int mdma_copy_pages(long long* words, cudaStream_t stream) {
    const int n_pools = (int)words[0], n_pages = (int)words[1], page_rows = (int)words[2], n = (int)words[3];
    const int *src = (const int*)(uintptr_t)words[4], *dst = (const int*)(uintptr_t)words[5], *rows = (const int*)(uintptr_t)words[6];
    long long *launches = words + 7;
    const long long* pool_words = words + 8;
    *launches = 0;
    MDMA_REQUIRE(n_pools > 0 && n_pages > 0 && page_rows > 0 && n >= 0, "copy_pages: %d pools of %d pages of %d rows", n_pools, n_pages, page_rows);
    if (n == 0) return 0;
    unsigned char* mark = (unsigned char*)calloc((size_t)n_pages, 1);
    CopyItem* items = (CopyItem*)malloc(sizeof(CopyItem) * (size_t)n);
    if (!mark || !items) { free(mark); free(items); return fail("copy_pages: no host memory for %d copies", n); }
    int rc = 0, kept = 0;
    bool apart = false;                      // whether copies of one page lie apart in the list
    for (int i = 0; i < n && !rc; ++i) {
        const int r = rows ? rows[i] : page_rows;
        if (src[i] < 0 || src[i] >= n_pages || dst[i] < 0 || dst[i] >= n_pages) rc = fail("copy_pages: page %d to page %d, the pools hold %d pages", src[i], dst[i], n_pages);
        else if (r < 0 || r > page_rows) rc = fail("copy_pages: %d rows of pages of %d", r, page_rows);
        else if (mark[dst[i]] & 1) rc = fail("copy_pages: page %d is written twice", dst[i]);
        else {
            if (r > 0) {
                apart = apart || ((mark[src[i]] & 4) && items[kept - 1].src != src[i]);
                mark[src[i]] |= 4;
                items[kept++] = {src[i], dst[i], r};
            }
            mark[dst[i]] |= 1; mark[src[i]] |= 2;
        }
    }
    for (int i = 0; i < n && !rc; ++i)
        if (mark[dst[i]] & 2) rc = fail("copy_pages: page %d is read and written in one call", dst[i]);
    free(mark);
    int dev = 0, sms = 148;
    if (!rc && (cudaGetDevice(&dev) != cudaSuccess || cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess))
        rc = fail("copy_pages: no CUDA device");
    // (sorting 482 pages that move cost the host 20 us of 44)
    if (!rc && apart) qsort(items, kept, sizeof(CopyItem), copy_order);
    for (int q0 = 0; q0 < n_pools && !rc; q0 += kCopyPools) {
        CopyPools pools = {};
        pools.n_pools = n_pools - q0 < kCopyPools ? n_pools - q0 : kCopyPools;
        unsigned long long align = 16;
        for (int q = 0; q < pools.n_pools; ++q) {
            const long long* w = pool_words + 5 * (q0 + q);
            pools.base[q] = (char*)(uintptr_t)w[0]; pools.page_bytes[q] = w[1]; pools.site_bytes[q] = w[2]; pools.row_bytes[q] = w[3];
            pools.first_site[q + 1] = pools.first_site[q] + (int)w[4];
            align |= (unsigned long long)w[0] | (unsigned long long)w[1] | (unsigned long long)w[2] | (unsigned long long)w[3];
        }
        const int vec = (align & 15) == 0 ? 16 : (align & 3) == 0 ? 4 : (align & 1) == 0 ? 2 : 1;
        for (int i = 0; i < kept && !rc;) {
            const int take = kept - i < 1000 ? kept - i : 1000;
            rc = take <= 16 ? launch_copies<16>(pools, items + i, take, vec, sms, stream) : take <= 128 ? launch_copies<128>(pools, items + i, take, vec, sms, stream)
                                                                                                : launch_copies<1000>(pools, items + i, take, vec, sms, stream);
            i += take;
            ++*launches;
        }
    }
    free(items);
    return rc;
}
