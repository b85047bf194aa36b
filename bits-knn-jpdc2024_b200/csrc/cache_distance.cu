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
    static constexpr int STAGE = SUB * PITCH<DIM> + SUB * 4;
    static constexpr int SCRATCH = 8 * NB * (SUB + 1) * 4;
    static constexpr int IMAGE = NB * 16 * DIM; // 8 NB columns of DIM halves
    static constexpr int BYTES = IMAGE + 8 * NB * 4 + WARPS * (DIST_STAGES * STAGE + SCRATCH);
};

// One block = a few query tokens of one head against `chunk` cache positions; every warp streams
// its own 16-position subtiles (asynchronous copies, DIST_STAGES deep, no block barrier) and
// multiplies them with all columns at once on the tensor cores: keys are the 16 rows of the
// matrix step, the query heads of the tokens its columns, so a code is converted to a half once
// for all of them.  Products of a key code (4 significant bits) and a query half are exact; the sums
// are FP32.  Bound by the key bytes and the matrix it writes (HBM) while the columns are few.
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
        const int32_t* table = a.b.table + r * a.b.table_ld;
        const int columns = many * a.group;
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
            const int first = begin / SUB + warp;
            const int count = end > first * SUB ? ((end - 1) / SUB - first) / WARPS + 1 : 0;
            const int loaded = furthest > first * SUB ? min(count, ((furthest - 1) / SUB - first) / WARPS + 1) : 0;
            auto page_of = [&](int j) { // page of subtile j of this warp
                const int p = j < loaded ? table[((first + j * WARPS) * SUB) >> a.c.page_shift] : -1;
                return p < a.c.pages ? p : -1;
            };
            int next_page = page_of(0);
            auto issue = [&](int j) {
                if (j < loaded)
                {
                    const int page = next_page;
                    next_page = page_of(j + 1);
                    const int pos = (first + j * WARPS) * SUB;
                    const int there = page < 0 ? 0 : min(SUB, furthest - pos);
                    const uint32_t dst = ptx::smem_addr(mine + (j % DIST_STAGES) * smem::STAGE);
                    const int safe = max(page, 0);
                    const uint8_t* src = a.c.keys + safe * a.c.page_stride +
                                         ((static_cast<int64_t>(head) << a.c.page_shift) + (pos & rows_mask)) * DIM;
                    constexpr int PARTS = DIM / 16;
#pragma unroll
                    for (int x = 0; x < DIM / 32; ++x)
                    {
                        const int e = lane + x * 32;
                        const int row = e / PARTS;
                        copy16(dst + row * PITCH<DIM> + (e % PARTS) * 16, src + e * 16, row < there ? 16U : 0U);
                    }
                    if (lane < SUB)
                    {
                        copy4(dst + SUB * PITCH<DIM> + lane * 4,
                              a.c.key_scales + static_cast<int64_t>(safe) * a.c.heads + head, lane < there ? 4U : 0U);
                    }
                }
                copy_commit();
            };
#pragma unroll
            for (int j = 0; j < DIST_STAGES - 1; ++j)
            {
                issue(j);
            }
            for (int j = 0; j < count; ++j)
            {
                const int pos = (first + j * WARPS) * SUB;
                copy_wait<DIST_STAGES - 2>();
                __syncwarp();
                if (j < loaded)
                {
                    const unsigned char* stage = mine + (j % DIST_STAGES) * smem::STAGE;
                    float s[NB][4];
                    score_rows<DIM, NB>(s, stage, reinterpret_cast<const uint2*>(image));
                    const int row = row_order(lane >> 2);
                    const int c = (lane & 3) * 2;
#pragma unroll
                    for (int nb = 0; nb < NB; ++nb)
                    {
                        float* out = scratch + (nb * 8 + c) * (SUB + 1) + row;
                        out[0] = s[nb][0] * undo[nb * 8 + c];
                        out[SUB + 1] = s[nb][1] * undo[nb * 8 + c + 1];
                        out[8] = s[nb][2] * undo[nb * 8 + c];
                        out[SUB + 1 + 8] = s[nb][3] * undo[nb * 8 + c + 1];
                    }
                }
                __syncwarp();
                const int row = lane & (SUB - 1);
                // the scale of an absent position was copied as zero
                const float ks = j < loaded ? reinterpret_cast<const float*>(mine + (j % DIST_STAGES) * smem::STAGE +
                                                                             SUB * PITCH<DIM>)[row]
                                            : 0.0F;
                const int last = (min(columns, col0 + 8 * NB) - 1) / a.group;
                for (int i = col0 / a.group + (lane >> 4); i <= last; i += 2)
                {
                    const int g0 = max(i * a.group, col0);
                    const int g1 = min((i + 1) * a.group, min(columns, col0 + 8 * NB));
                    float d = INFINITY;
                    if (j < loaded && ks != 0.0F && pos + row < visible_of(a.b, q, token + i - q.first))
                    {
                        float best = scratch[(g0 - col0) * (SUB + 1) + row];
                        for (int g = g0 + 1; g < g1; ++g)
                        {
                            best = max_nan(best, scratch[(g - col0) * (SUB + 1) + row]);
                        }
                        d = -(best * ks);
                    }
                    if (pos + row < end)
                    {
                        float* out = a.dist + (static_cast<int64_t>(token + i) * a.c.heads + head) * a.ld + pos + row;
                        if (g0 != i * a.group) // the head's first columns were in an earlier block
                        {
                            d = -max_nan(-d, -*out);
                        }
                        *out = d;
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
    BITSKNN_CUDA_TRY(cudaFuncSetAttribute(cache_distance_kernel<DIM, NB>, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes));
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
