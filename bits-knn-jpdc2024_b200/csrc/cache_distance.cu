// cache_distance: the distance matrix of query tokens against the keys of a paged 8-bit cache.
#include <algorithm>

#include "cache.cuh"

namespace bitsknn
{

namespace
{

using namespace cache;

constexpr int DIST_STAGES = 6;

struct distance_args
{
    view c;
    batch b;
    const void* queries;
    int dtype;
    int64_t query_stride;
    int group;        // query heads per cache head
    float* dist;
    int64_t ld;
    int n;
    int chunk;        // columns per block, a multiple of TILE
    int chunks;
    int token_block;  // tokens per block
};

__device__ __forceinline__ float max_nan(float a, float b)
{
    float y;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
    return y;
}

template <int DIM, int NB>
struct distance_smem
{
    static constexpr int STAGE = SUB * PITCH<DIM, false>;
    static constexpr int SCRATCH = 8 * NB * (SUB + 1) * 4;
    static constexpr int IMAGE = NB * 16 * DIM; // 8 NB columns of DIM halves
    static constexpr int BYTES = IMAGE + 8 * NB * 4 + WARPS * (DIST_STAGES * STAGE + SCRATCH);
};

// One block = a few query tokens of one head against `chunk` cache positions; every warp streams
// its own 16-position subtiles (asynchronous copies, DIST_STAGES deep, no block barrier) and
// multiplies them with all columns at once on the tensor cores: keys are the 16 rows of the
// matrix step, the query heads of the tokens its columns, so a code is converted to a half once
// for all of them.  Products of a key code (4 significant bits) and a query half are exact; the sums
// are FP32.  Bound by the key bytes and the matrix it writes (HBM) while the columns are few: 16 requests of
// 2000 ... 60000 positions, 8 heads of 128, 294 MB in 60 us = 4.9 TB/s, 0.75 of the measured copy rate.
template <int DIM, int NB>
__global__ void __launch_bounds__(THREADS) cache_distance_kernel(const distance_args a)
{
    using smem = distance_smem<DIM, NB>;
    extern __shared__ __align__(16) unsigned char shared[];
    uint32_t* const image = reinterpret_cast<uint32_t*>(shared);
    float* const undo = reinterpret_cast<float*>(shared + smem::IMAGE);
    const int warp = threadIdx.x >> 5;
    const int lane = threadIdx.x & 31;
    unsigned char* const mine = shared + smem::IMAGE + 8 * NB * 4 + warp * (DIST_STAGES * smem::STAGE + smem::SCRATCH);
    float* const scratch = reinterpret_cast<float*>(mine + DIST_STAGES * smem::STAGE);

    const int chunk = static_cast<int>(blockIdx.x % static_cast<unsigned>(a.chunks));
    const int rest = static_cast<int>(blockIdx.x / static_cast<unsigned>(a.chunks));
    const int head = rest % a.c.heads;
    const int64_t token_end =
        min(static_cast<int64_t>(rest / a.c.heads + 1) * a.token_block, static_cast<int64_t>(a.b.tokens));
    int token = rest / a.c.heads * a.token_block;
    const int begin = chunk * a.chunk;
    const int end = min(begin + a.chunk, a.n);
    const int rows_mask = (1 << a.c.page_shift) - 1;

    while (token < token_end)
    {
        const int r = owner_of(a.b, token);
        if (r < 0)
        {
            ++token;
            continue;
        }
        const request q = request_of(a.b, r);
        const int many = max(static_cast<int>(min(token_end, static_cast<int64_t>(q.first) + q.count)) - token, 1);
        const int furthest = min(visible_of(a.b, q, token + many - 1 - q.first), a.n);
        const int64_t nearest = static_cast<int64_t>(q.length) - q.count + (token - q.first) + 1; // token i sees i more
        const int32_t* table = a.b.table + r * a.b.table_ld;
        const int columns = many * a.group;
        float* const only = a.dist + (static_cast<int64_t>(token) * a.c.heads + head) * a.ld;
        // columns that no token sees, but for those that share a subtile with some that one does
        const int unseen = max((furthest + SUB - 1) / SUB * SUB, begin);
        for (int i = 0; i < many; ++i)
        {
            float* const out = only + static_cast<int64_t>(i) * a.c.heads * a.ld;
            for (int col = unseen + static_cast<int>(threadIdx.x); col < end; col += THREADS)
            {
                out[col] = INFINITY;
            }
        }
        if (begin >= furthest)
        {
            token += many;
            continue;
        }
        // blocks of columns: one, unless a head has more query heads than a block has columns
        for (int col0 = 0; col0 < columns; col0 += 8 * NB)
        {
            __syncthreads();
            for (int col = warp; col < 8 * NB; col += WARPS)
            {
                const int g = col0 + col;
                const bool real = g < columns;
                const int64_t at = static_cast<int64_t>(token + g / a.group) * a.query_stride +
                                   static_cast<int64_t>(head * a.group + g % a.group) * DIM;
                const float f = pack_column<DIM, NB>(image, col, real ? a.queries : nullptr, at, a.dtype);
                if (lane == 0)
                {
                    undo[col] = f;
                }
            }
            __syncthreads();
            float factor[NB][2]; // of this thread's columns
#pragma unroll
            for (int nb = 0; nb < NB; ++nb)
            {
                factor[nb][0] = undo[nb * 8 + (lane & 3) * 2];
                factor[nb][1] = undo[nb * 8 + (lane & 3) * 2 + 1];
            }
            const int first = begin / SUB + warp;
            const int seen = min(end, furthest);
            const int count = seen > first * SUB ? ((seen - 1) / SUB - first) / WARPS + 1 : 0;
            // Where the warp's next 32 subtiles lie and their scales, one subtile per lane; looked up a batch
            // ahead.  A subtile lies within one page, so its rows are contiguous and share a scale.
            auto page_of = [&](int j) {
                const int p = j < count ? table[((first + j * WARPS) * SUB) >> a.c.page_shift] : -1;
                return p < a.c.pages ? p : -1;
            };
            auto offset_of = [&](int page, int j) -> int64_t {
                const int pos = (first + j * WARPS) * SUB;
                return page < 0 ? -1
                                : page * a.c.page_stride +
                                      ((static_cast<int64_t>(head) << a.c.page_shift) + (pos & rows_mask)) * DIM;
            };
            auto scale_of = [&](int page) { // 0 marks an absent page
                return page < 0 ? 0.0F : a.c.key_scales[static_cast<int64_t>(page) * a.c.heads + head];
            };
            int batch = 0; // first subtile of the batch the copies are in
            const int page_first = page_of(lane);
            int page_next = page_of(32 + lane);
            int64_t offset_now = offset_of(page_first, lane);
            float scale_now = scale_of(page_first);
            float scale_before = 0.0F;
            int slot_in = 0;
            int slot_out = 0;
            const uint32_t stage0 = ptx::smem_addr(mine);
            constexpr int PARTS = DIM / 16;
            auto issue = [&](int j) {
                if (j < count)
                {
                    if (j - batch == 32)
                    {
                        batch = j;
                        offset_now = offset_of(page_next, j + lane);
                        scale_before = scale_now;
                        scale_now = scale_of(page_next);
                        page_next = page_of(j + 32 + lane);
                    }
                    const int64_t offset = __shfl_sync(FULL_MASK, offset_now, j - batch);
                    const int there = offset < 0 ? 0 : min(SUB, furthest - (first + j * WARPS) * SUB);
                    const uint32_t dst = stage0 + slot_in * smem::STAGE;
                    const uint8_t* src = a.c.keys + max(offset, static_cast<int64_t>(0)) + lane * 16;
#pragma unroll
                    for (int x = 0; x < DIM / 32; ++x)
                    {
                        const int e = lane + x * 32;
                        const uint32_t to = dst + granule_byte<DIM, false>(e / PARTS, e % PARTS);
                        if (there == SUB)
                        {
                            copy16(to, src + x * 512);
                        }
                        else
                        {
                            copy16(to, src + x * 512, e / PARTS < there ? 16U : 0U);
                        }
                    }
                }
                copy_commit();
                slot_in = slot_in + 1 == DIST_STAGES ? 0 : slot_in + 1;
            };
#pragma unroll
            for (int j = 0; j < DIST_STAGES - 1; ++j)
            {
                issue(j);
            }
            // One token whose heads all are columns of this block: the maximum over them stays in registers.
            const bool simple = many == 1 && columns <= 8 * NB;
            const int row = lane & (SUB - 1);
            const int half = lane >> 4;
            const int cols = min(columns - col0, 8 * NB);
            for (int j = 0; j < count; ++j)
            {
                const int pos = (first + j * WARPS) * SUB;
                copy_wait<DIST_STAGES - 2>();
                __syncwarp();
                const unsigned char* const stage = mine + slot_out * smem::STAGE;
                slot_out = slot_out + 1 == DIST_STAGES ? 0 : slot_out + 1;
                const float ks = __shfl_sync(FULL_MASK, j < batch ? scale_before : scale_now, j & 31);
                float s[NB][4];
                score_rows<DIM, NB, false>(s, stage, reinterpret_cast<const uint2*>(image));
                if (simple)
                {
                    float lo = -INFINITY;
                    float hi = -INFINITY;
#pragma unroll
                    for (int nb = 0; nb < NB; ++nb)
                    {
                        const int c = nb * 8 + (lane & 3) * 2;
                        lo = max_nan(lo, c < columns ? s[nb][0] * factor[nb][0] : -INFINITY);
                        hi = max_nan(hi, c < columns ? s[nb][2] * factor[nb][0] : -INFINITY);
                        lo = max_nan(lo, c + 1 < columns ? s[nb][1] * factor[nb][1] : -INFINITY);
                        hi = max_nan(hi, c + 1 < columns ? s[nb][3] * factor[nb][1] : -INFINITY);
                    }
#pragma unroll
                    for (int o = 1; o < 4; o <<= 1)
                    {
                        lo = max_nan(lo, __shfl_xor_sync(FULL_MASK, lo, o));
                        hi = max_nan(hi, __shfl_xor_sync(FULL_MASK, hi, o));
                    }
                    // lanes 0 and 1 of a group of four write its rows row_order and 8 + row_order
                    const int at = pos + row_order<DIM, false>(lane >> 2) + (lane & 1) * 8;
                    if ((lane & 2) == 0 && at < end)
                    {
                        only[at] = ks != 0.0F && at < furthest ? -(((lane & 1) == 0 ? lo : hi) * ks) : INFINITY;
                    }
                    __syncwarp();
                    issue(j + DIST_STAGES - 1);
                    continue;
                }
                {
#pragma unroll
                    for (int nb = 0; nb < NB; ++nb)
                    {
                        float* out = scratch + (nb * 8 + (lane & 3) * 2) * (SUB + 1) + row_order<DIM, false>(lane >> 2);
                        out[0] = s[nb][0] * factor[nb][0];
                        out[SUB + 1] = s[nb][1] * factor[nb][1];
                        out[8] = s[nb][2] * factor[nb][0];
                        out[SUB + 1 + 8] = s[nb][3] * factor[nb][1];
                    }
                }
                __syncwarp();
                if (many == 1)
                {
                    // all columns are one token's: the two halves of the warp share them
                    float best = half < cols ? scratch[half * (SUB + 1) + row] : -INFINITY;
#pragma unroll 4
                    for (int g = half + 2; g < cols; g += 2)
                    {
                        best = max_nan(best, scratch[g * (SUB + 1) + row]);
                    }
                    best = max_nan(best, __shfl_xor_sync(FULL_MASK, best, 16));
                    float d = ks != 0.0F && pos + row < furthest ? -(best * ks) : INFINITY;
                    if (half == 0 && pos + row < end)
                    {
                        if (col0 > 0) // the head's first columns were in an earlier block
                        {
                            d = -max_nan(-d, -only[pos + row]);
                        }
                        only[pos + row] = d;
                    }
                }
                else
                {
                    for (int i = col0 / a.group + half; i * a.group < col0 + cols; i += 2)
                    {
                        const int g0 = max(i * a.group, col0) - col0;
                        const int g1 = min((i + 1) * a.group - col0, cols);
                        float best = scratch[g0 * (SUB + 1) + row];
                        for (int g = g0 + 1; g < g1; ++g)
                        {
                            best = max_nan(best, scratch[g * (SUB + 1) + row]);
                        }
                        float d = ks != 0.0F && pos + row < nearest + i ? -(best * ks) : INFINITY;
                        if (pos + row < end)
                        {
                            float* out = only + static_cast<int64_t>(i) * a.c.heads * a.ld + pos + row;
                            if (g0 + col0 != i * a.group)
                            {
                                d = -max_nan(-d, -*out);
                            }
                            *out = d;
                        }
                    }
                }
                __syncwarp();
                issue(j + DIST_STAGES - 1);
            }
            copy_wait<0>();
        }
        token += many;
    }
}

template <int DIM, int NB>
int launch_distance(const distance_args& a, int64_t blocks, cudaStream_t stream)
{
    constexpr int bytes = distance_smem<DIM, NB>::BYTES;
    static_assert(bytes <= 227 * 1024, "shared memory");
    static cache::device_set prepared;
    if (!prepared.contains_current())
    {
        BITSKNN_CUDA_TRY(
            cudaFuncSetAttribute(cache_distance_kernel<DIM, NB>, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes));
        prepared.add_current();
    }
    {
        kernel_scope scope("cache_distance_kernel", stream);
        cache_distance_kernel<DIM, NB><<<static_cast<unsigned>(blocks), THREADS, bytes, stream>>>(a);
    }
    BITSKNN_CUDA_TRY(cudaGetLastError());
    return BITSKNN_OK;
}

} // namespace

} // namespace bitsknn

extern "C" int bitsknn_cache_distance(const bitsknn_cache_t* cache, const bitsknn_cache_batch_t* batch,
                                      const void* d_queries, int dtype, int64_t query_stride, int query_heads,
                                      float* d_dist, int64_t ld, int64_t n, bitsknn_stream_t stream)
{
    using namespace bitsknn;
    distance_args a{};
    int rc = check_cache(cache, &a.c);
    if (rc != BITSKNN_OK || (rc = check_cache_batch(batch, cache->page_rows, &a.b)) != BITSKNN_OK)
    {
        return rc;
    }
    if (batch->tokens > 0 || d_queries != nullptr)
    {
        rc = check_cache_queries(d_queries, dtype, &query_stride, query_heads, cache->heads, cache->dim);
        if (rc != BITSKNN_OK)
        {
            return rc;
        }
    }
    if (n < 0 || ld < n || n > 0x7fffffff - 65536)
    {
        return fail(BITSKNN_ERR_INVALID_ARGUMENT, "invalid matrix shape: n=%lld ld=%lld", static_cast<long long>(n),
                    static_cast<long long>(ld));
    }
    if (batch->tokens == 0 || batch->requests == 0 || n == 0)
    {
        return BITSKNN_OK;
    }
    if (d_dist == nullptr)
    {
        return fail(BITSKNN_ERR_INVALID_ARGUMENT, "null pointer argument");
    }
    if ((reinterpret_cast<uintptr_t>(d_dist) & 3) != 0)
    {
        return fail(BITSKNN_ERR_INVALID_ARGUMENT, "misaligned matrix: 4-byte alignment needed");
    }
    const extent write = {"d_dist", d_dist, batch->tokens * cache->heads, ld * 4, n * 4};
    const extent read = {"d_queries", d_queries, batch->tokens, query_stride * 2,
                         static_cast<int64_t>(query_heads) * cache->dim * 2};
    rc = check_apart(&write, 1, &read, 1);
    if (rc != BITSKNN_OK)
    {
        return rc;
    }
    a.queries = d_queries;
    a.dtype = dtype;
    a.query_stride = query_stride;
    a.group = query_heads / cache->heads;
    a.dist = d_dist;
    a.ld = ld;
    a.n = static_cast<int>(n);
    // columns a pass over the keys can serve: the query heads of the tokens a request has on average
    const int64_t per_request = batch->d_starts == nullptr ? 1 : (batch->tokens + batch->requests - 1) / batch->requests;
    const int64_t want = a.group * per_request;
    const int nb = want <= 8 ? 1 : want <= 16 ? 2 : 4;
    a.token_block = per_request == 1 ? 1 : std::max(1, 8 * nb / a.group);
    const int64_t items = (batch->tokens + a.token_block - 1) / a.token_block * cache->heads;
    // some twelve blocks per SM, of 256 to 4096 columns
    const int64_t target = static_cast<int64_t>(device_sm_count()) * 12;
    const int64_t chunk = (items * n / target + cache::TILE - 1) / cache::TILE * cache::TILE;
    a.chunk = static_cast<int>(std::min<int64_t>(std::max<int64_t>(chunk, 256), 4096));
    a.chunks = static_cast<int>((n + a.chunk - 1) / a.chunk);
    const int64_t blocks = items * a.chunks;
    if (blocks > 0x7fffffff)
    {
        return fail(BITSKNN_ERR_INVALID_ARGUMENT, "tokens=%lld x n=%lld exceeds the grid limit",
                    static_cast<long long>(batch->tokens), static_cast<long long>(n));
    }
    return dispatch_cache_dim(cache->dim, [&](auto dim) {
        constexpr int DIM = decltype(dim)::value;
        auto s = static_cast<cudaStream_t>(stream);
        return nb == 1   ? launch_distance<DIM, 1>(a, blocks, s)
               : nb == 2 ? launch_distance<DIM, 2>(a, blocks, s)
                         : launch_distance<DIM, 4>(a, blocks, s);
    });
}
