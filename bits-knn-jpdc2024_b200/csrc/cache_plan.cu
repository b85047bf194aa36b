// Paged 8-bit cache: argument checks shared by its entry points, and cache_plan (block tables and
// slot maps from request lengths).
#include <algorithm>

#include "cache.cuh"

namespace bitsknn
{

int check_cache(const bitsknn_cache_t* cache, cache::view* out)
{
    if (cache == nullptr || cache->d_keys == nullptr || cache->d_values == nullptr || cache->d_key_scales == nullptr ||
        cache->d_value_scales == nullptr)
    {
        return fail(BITSKNN_ERR_INVALID_ARGUMENT, "null pointer argument");
    }
    const int rc = dispatch_cache_dim(cache->dim, [](auto) { return BITSKNN_OK; });
    if (rc != BITSKNN_OK)
    {
        return rc;
    }
    const int rows = cache->page_rows;
    if (rows < 16 || rows > 256 || (rows & (rows - 1)) != 0)
    {
        return fail(BITSKNN_ERR_INVALID_ARGUMENT, "page_rows=%d: pages hold 16, 32, 64, 128 or 256 rows", rows);
    }
    if (cache->pages < 1 || cache->pages > 0x7fffffff || cache->heads < 1 || cache->heads > 65535)
    {
        return fail(BITSKNN_ERR_INVALID_ARGUMENT, "invalid cache sizes pages=%lld heads=%d",
                    static_cast<long long>(cache->pages), cache->heads);
    }
    const int64_t dense = static_cast<int64_t>(cache->heads) * rows * cache->dim;
    const int64_t stride = cache->page_stride == 0 ? dense : cache->page_stride;
    if (stride < dense || (stride & 15) != 0)
    {
        return fail(BITSKNN_ERR_INVALID_ARGUMENT, "page_stride=%lld: at least %lld codes and a multiple of 16",
                    static_cast<long long>(stride), static_cast<long long>(dense));
    }
    const auto codes = reinterpret_cast<uintptr_t>(cache->d_keys) | reinterpret_cast<uintptr_t>(cache->d_values);
    const auto scales =
        reinterpret_cast<uintptr_t>(cache->d_key_scales) | reinterpret_cast<uintptr_t>(cache->d_value_scales);
    if ((codes & 15) != 0 || (scales & 3) != 0)
    {
        return fail(BITSKNN_ERR_INVALID_ARGUMENT, "misaligned cache: codes need 16-byte, scales 4-byte alignment");
    }
    out->keys = static_cast<uint8_t*>(cache->d_keys);
    out->values = static_cast<uint8_t*>(cache->d_values);
    out->key_scales = cache->d_key_scales;
    out->value_scales = cache->d_value_scales;
    out->pages = cache->pages;
    out->page_stride = stride;
    out->heads = cache->heads;
    out->page_shift = 0;
    while ((1 << out->page_shift) < rows)
    {
        ++out->page_shift;
    }
    return BITSKNN_OK;
}

int check_cache_batch(const bitsknn_cache_batch_t* in, int page_rows, cache::batch* out)
{
    if (in == nullptr)
    {
        return fail(BITSKNN_ERR_INVALID_ARGUMENT, "null pointer argument");
    }
    if (in->requests < 0 || in->tokens < 0 || in->requests > cache::MOST_ROWS ||
        in->tokens > cache::MOST_ROWS)
    {
        return fail(BITSKNN_ERR_INVALID_ARGUMENT, "invalid batch sizes requests=%lld tokens=%lld",
                    static_cast<long long>(in->requests), static_cast<long long>(in->tokens));
    }
    if (in->requests > 0 && (in->d_table == nullptr || in->d_lengths == nullptr))
    {
        return fail(BITSKNN_ERR_INVALID_ARGUMENT, "null pointer argument");
    }
    if (in->table_pages < 0 || in->table_ld < in->table_pages)
    {
        return fail(BITSKNN_ERR_INVALID_ARGUMENT, "invalid table shape: table_pages=%lld table_ld=%lld",
                    static_cast<long long>(in->table_pages), static_cast<long long>(in->table_ld));
    }
    if (in->d_starts == nullptr && in->tokens != in->requests)
    {
        return fail(BITSKNN_ERR_INVALID_ARGUMENT,
                    "without d_starts every request has one token (tokens=%lld requests=%lld)",
                    static_cast<long long>(in->tokens), static_cast<long long>(in->requests));
    }
    out->table = in->d_table;
    out->table_ld = in->table_ld;
    // positions are int32 throughout, with room for one more block of them
    out->limit = std::min<int64_t>(in->table_pages * page_rows, 0x7fffffff - 65536);
    out->lengths = in->d_lengths;
    out->starts = in->d_starts;
    out->requests = static_cast<int>(in->requests);
    out->tokens = static_cast<int>(in->tokens);
    return BITSKNN_OK;
}

int check_apart(const extent* writes, int write_count, const extent* reads, int read_count)
{
    for (int i = 0; i < write_count; ++i)
    {
        for (int j = 0; j < i + read_count; ++j)
        {
            const extent& other = j < i ? writes[j] : reads[j - i];
            if (overlap(writes[i], other))
            {
                return fail(BITSKNN_ERR_INVALID_ARGUMENT, "%s overlaps %s: what the call writes has to lie apart",
                            writes[i].name, other.name);
            }
        }
    }
    return BITSKNN_OK;
}

int check_cache_queries(const void* d_queries, int dtype, int64_t* query_stride, int query_heads, int heads, int dim)
{
    if (dtype != BITSKNN_F16 && dtype != BITSKNN_BF16)
    {
        return fail(BITSKNN_ERR_UNSUPPORTED_MODE, "query dtype %d: only F16 and BF16", dtype);
    }
    if (query_heads < heads || query_heads % heads != 0 || query_heads / heads > 65535)
    {
        return fail(BITSKNN_ERR_INVALID_ARGUMENT, "query_heads=%d is not a multiple of the cache's %d heads",
                    query_heads, heads);
    }
    const int64_t dense = static_cast<int64_t>(query_heads) * dim;
    if (*query_stride == 0)
    {
        *query_stride = dense;
    }
    if (*query_stride < dense || (*query_stride & 7) != 0)
    {
        return fail(BITSKNN_ERR_INVALID_ARGUMENT, "stride %lld between tokens: at least %lld and a multiple of 8",
                    static_cast<long long>(*query_stride), static_cast<long long>(dense));
    }
    if (d_queries == nullptr)
    {
        return fail(BITSKNN_ERR_INVALID_ARGUMENT, "null pointer argument");
    }
    if ((reinterpret_cast<uintptr_t>(d_queries) & 15) != 0)
    {
        return fail(BITSKNN_ERR_INVALID_ARGUMENT, "misaligned vectors: 16-byte alignment needed");
    }
    return BITSKNN_OK;
}

namespace
{

constexpr int PLAN_THREADS = 512;
constexpr int PLAN_PER = 4;
constexpr int PLAN_CHUNK = PLAN_THREADS * PLAN_PER; // requests in shared memory at a time

struct plan_args
{
    const int32_t* lengths;
    const int32_t* added;
    int requests;
    int page_shift;
    const int32_t* free_pages;
    int64_t free_count;
    int32_t* table;
    int64_t table_ld;
    int64_t table_pages;
    int32_t* starts;
    int32_t* new_lengths;
    int64_t* slots;
    int64_t max_tokens;
    int32_t* counts;
};

// Pages of `rows` positions.  Unsigned: a length and its new tokens together may pass 2^31.
__device__ __forceinline__ int pages_of(int length, int added, int page_shift)
{
    const unsigned mask = (1U << page_shift) - 1;
    return static_cast<int>((static_cast<unsigned>(length) + static_cast<unsigned>(added) + mask) >> page_shift);
}

// Inclusive sums of a pair over the block; `totals` gets the block's sums.
__device__ __forceinline__ int2 block_scan(int2 v, int2* warp_sums, int2* totals)
{
    const int lane = threadIdx.x & 31;
    const int warp = threadIdx.x >> 5;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1)
    {
        const int x = __shfl_up_sync(FULL_MASK, v.x, o);
        const int y = __shfl_up_sync(FULL_MASK, v.y, o);
        if (lane >= o)
        {
            v.x += x;
            v.y += y;
        }
    }
    if (lane == 31)
    {
        warp_sums[warp] = v;
    }
    __syncthreads();
    int2 before = make_int2(0, 0);
    int2 all = make_int2(0, 0);
#pragma unroll
    for (int w = 0; w < PLAN_THREADS / 32; ++w)
    {
        const int2 s = warp_sums[w];
        before.x += w < warp ? s.x : 0;
        before.y += w < warp ? s.y : 0;
        all.x += s.x;
        all.y += s.y;
    }
    __syncthreads();
    *totals = all;
    return make_int2(v.x + before.x, v.y + before.y);
}

// Every block sums all requests by itself (8 bytes each, from L2) instead of waiting for another
// block, then fills its share of the slots: tiles of 512 tokens dealt round robin, each token
// finding its request by bisection in shared memory.  A token at row 0 of a page is the one that
// enters the page into the table, so no block reads what another one writes.  Bound by latency:
// one launch, about four dependent memory round trips (24 requests 3.8 us, 4096 requests with
// 302 K tokens 9.6 us).
__global__ void __launch_bounds__(PLAN_THREADS) cache_plan_kernel(const plan_args a)
{
    __shared__ int s_start[PLAN_CHUNK];  // first token
    __shared__ int s_length[PLAN_CHUNK]; // cached positions
    __shared__ int s_page[PLAN_CHUNK];   // first entry of the free list
    __shared__ int2 s_sums[PLAN_THREADS / 32];
    const int t = threadIdx.x;
    const int rows = 1 << a.page_shift;
    int2 carry = make_int2(0, 0); // tokens, pages of the chunks before
    int short_of = 0;             // block 0: tokens that got no place
    for (int base = 0; base < a.requests; base += PLAN_CHUNK)
    {
        const int count = min(PLAN_CHUNK, a.requests - base);
        int len[PLAN_PER];
        int add[PLAN_PER];
        int2 sum = make_int2(0, 0);
#pragma unroll
        for (int i = 0; i < PLAN_PER; ++i)
        {
            const int j = t * PLAN_PER + i;
            len[i] = j < count ? max(a.lengths[base + j], 0) : 0;
            add[i] = j < count ? max(a.added[base + j], 0) : 0;
            sum.x += add[i];
            sum.y += pages_of(len[i], add[i], a.page_shift) - pages_of(len[i], 0, a.page_shift);
        }
        int2 total;
        const int2 upto = block_scan(sum, s_sums, &total);
        int2 at = make_int2(carry.x + upto.x - sum.x, carry.y + upto.y - sum.y);
#pragma unroll
        for (int i = 0; i < PLAN_PER; ++i)
        {
            const int j = t * PLAN_PER + i;
            const int have = pages_of(len[i], 0, a.page_shift);
            const int need = pages_of(len[i], add[i], a.page_shift);
            const int64_t asked = static_cast<int64_t>(len[i]) + add[i];
            if (j < count)
            {
                s_start[j] = at.x;
                s_length[j] = len[i];
                s_page[j] = at.y;
                if (blockIdx.x == 0)
                {
                    a.starts[base + j] = at.x;
                    a.new_lengths[base + j] = static_cast<int>(min(asked, static_cast<int64_t>(0x7fffffff)));
                    // rows there is room for: pages held, plus those the free list still has, cut by the table
                    const int64_t left = max(static_cast<int64_t>(0), a.free_count - at.y);
                    const int64_t pages = min(have + min(static_cast<int64_t>(need - have), left), a.table_pages);
                    const int64_t room = max(pages << a.page_shift, static_cast<int64_t>(len[i]));
                    short_of += static_cast<int>(max(static_cast<int64_t>(0), asked - room));
                }
            }
            at.x += add[i];
            at.y += need - have;
        }
        __syncthreads();
        // tiles of this chunk that are this block's
        const int begin = carry.x;
        const int end = carry.x + total.x;
        int tile = begin / PLAN_THREADS;
        tile += (static_cast<int>(blockIdx.x) - tile % static_cast<int>(gridDim.x) + static_cast<int>(gridDim.x)) %
                static_cast<int>(gridDim.x);
        // sums beyond 2^31, which the caller must not ask for, wrap: nothing is placed then, see the bounds below
        for (int64_t token0 = static_cast<int64_t>(tile) * PLAN_THREADS; token0 < end;
             token0 += static_cast<int64_t>(gridDim.x) * PLAN_THREADS)
        {
            const int64_t token = token0 + t;
            if (token < begin || token >= end || token < 0)
            {
                continue;
            }
            int lo = 0;
            int hi = count;
            while (hi - lo > 1)
            {
                const int mid = (lo + hi) >> 1;
                if (s_start[mid] <= token)
                {
                    lo = mid;
                }
                else
                {
                    hi = mid;
                }
            }
            const int length = s_length[lo];
            const unsigned position = static_cast<unsigned>(length) + static_cast<unsigned>(token - s_start[lo]);
            const int column = static_cast<int>(position >> a.page_shift);
            const int fresh = column - pages_of(length, 0, a.page_shift); // which of the new pages
            const int row = static_cast<int>(position) & (rows - 1);
            int page = -1;
            if (column < a.table_pages)
            {
                int32_t* entry = a.table + (base + lo) * a.table_ld + column;
                if (fresh < 0)
                {
                    page = *entry;
                }
                else
                {
                    const int64_t f = static_cast<int64_t>(s_page[lo]) + fresh;
                    page = f >= 0 && f < a.free_count ? a.free_pages[f] : -1;
                    if (row == 0)
                    {
                        *entry = page;
                    }
                }
            }
            if (token < a.max_tokens)
            {
                a.slots[token] = page < 0 ? -1 : (static_cast<int64_t>(page) << a.page_shift) + row;
            }
        }
        carry.x += total.x;
        carry.y += total.y;
        __syncthreads();
    }
    for (int64_t token = max(carry.x, 0) + blockIdx.x * static_cast<int64_t>(PLAN_THREADS) + t; token < a.max_tokens;
         token += static_cast<int64_t>(gridDim.x) * PLAN_THREADS)
    {
        a.slots[token] = -1;
    }
    if (blockIdx.x == 0)
    {
        int2 all;
        block_scan(make_int2(short_of, 0), s_sums, &all);
        if (t == 0)
        {
            a.starts[a.requests] = carry.x;
            a.counts[0] = carry.x;
            a.counts[1] = carry.y;
            a.counts[2] = all.x;
        }
    }
}

} // namespace

} // namespace bitsknn

extern "C" int bitsknn_cache_plan(const int32_t* d_lengths, const int32_t* d_new, int64_t requests, int page_rows,
                                  const int32_t* d_free_pages, int64_t free_count, int32_t* d_table, int64_t table_ld,
                                  int64_t table_pages, int32_t* d_starts, int32_t* d_new_lengths, int64_t* d_slots,
                                  int64_t max_tokens, int32_t* d_counts, bitsknn_stream_t stream)
{
    using namespace bitsknn;
    if (requests < 0 || requests > cache::MOST_ROWS || free_count < 0 || max_tokens < 0)
    {
        return fail(BITSKNN_ERR_INVALID_ARGUMENT, "invalid plan sizes requests=%lld free_count=%lld max_tokens=%lld",
                    static_cast<long long>(requests), static_cast<long long>(free_count),
                    static_cast<long long>(max_tokens));
    }
    if (page_rows < 16 || page_rows > 256 || (page_rows & (page_rows - 1)) != 0)
    {
        return fail(BITSKNN_ERR_INVALID_ARGUMENT, "page_rows=%d: pages hold 16, 32, 64, 128 or 256 rows", page_rows);
    }
    if (table_pages < 0 || table_ld < table_pages)
    {
        return fail(BITSKNN_ERR_INVALID_ARGUMENT, "invalid table shape: table_pages=%lld table_ld=%lld",
                    static_cast<long long>(table_pages), static_cast<long long>(table_ld));
    }
    if (d_starts == nullptr || d_counts == nullptr || (max_tokens > 0 && d_slots == nullptr) ||
        (free_count > 0 && d_free_pages == nullptr) ||
        (requests > 0 && (d_lengths == nullptr || d_new == nullptr || d_table == nullptr || d_new_lengths == nullptr)))
    {
        return fail(BITSKNN_ERR_INVALID_ARGUMENT, "null pointer argument");
    }
    // every block reads all lengths and its own entries of the others, while other blocks write
    const extent writes[] = {dense_extent("d_starts", d_starts, (requests + 1) * 4),
                             dense_extent("d_new_lengths", d_new_lengths, requests * 4),
                             dense_extent("d_slots", d_slots, max_tokens * 8), dense_extent("d_counts", d_counts, 3 * 4),
                             {"d_table", d_table, requests, table_ld * 4, table_pages * 4}};
    const extent reads[] = {dense_extent("d_lengths", d_lengths, requests * 4), dense_extent("d_new", d_new, requests * 4),
                            dense_extent("d_free_pages", d_free_pages, free_count * 4)};
    const int rc = check_apart(writes, 5, reads, 3);
    if (rc != BITSKNN_OK)
    {
        return rc;
    }
    plan_args a{};
    a.lengths = d_lengths;
    a.added = d_new;
    a.requests = static_cast<int>(requests);
    while ((1 << a.page_shift) < page_rows)
    {
        ++a.page_shift;
    }
    a.free_pages = d_free_pages;
    a.free_count = free_count;
    a.table = d_table;
    a.table_ld = table_ld;
    a.table_pages = table_pages;
    a.starts = d_starts;
    a.new_lengths = d_new_lengths;
    a.slots = d_slots;
    a.max_tokens = max_tokens;
    a.counts = d_counts;
    const int64_t tiles = (std::max<int64_t>(max_tokens, requests) + PLAN_THREADS - 1) / PLAN_THREADS;
    const int blocks = static_cast<int>(std::min<int64_t>(std::max<int64_t>(tiles, 1), device_sm_count()));
    cache_plan_kernel<<<blocks, PLAN_THREADS, 0, static_cast<cudaStream_t>(stream)>>>(a);
    BITSKNN_CUDA_TRY(cudaGetLastError());
    return BITSKNN_OK;
}
