// cache_append: new keys and values are quantised into the paged 8-bit cache.
#include <algorithm>

#include "cache.cuh"

namespace bitsknn
{

namespace
{

constexpr int APPEND_THREADS = 128;

struct append_args
{
    cache::view c;
    const void* src[2]; // keys, values
    int64_t stride[2];  // elements between tokens
    const int64_t* slots;
    int tokens;
    int window;         // tokens per block
    int dim;
    int dtype;
};

// Eight numbers as they lie in memory (one 16-byte word, two for FP32), and as floats.
template <int DTYPE>
struct raw8
{
    uint4 w[DTYPE == BITSKNN_F32 ? 2 : 1];
};

template <int DTYPE>
__device__ __forceinline__ raw8<DTYPE> load8(const void* src, int64_t at)
{
    raw8<DTYPE> r;
    if constexpr (DTYPE == BITSKNN_F32)
    {
        const uint4* p = reinterpret_cast<const uint4*>(static_cast<const float*>(src) + at);
        r.w[0] = __ldg(p);
        r.w[1] = __ldg(p + 1);
    }
    else
    {
        r.w[0] = __ldg(reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(src) + at));
    }
    return r;
}

__device__ __forceinline__ void prefetch_l2(const void* src, int64_t at, int bytes)
{
    asm volatile("prefetch.global.L2 [%0];" ::"l"(static_cast<const char*>(src) + at * bytes));
}

// Vectors of eight numbers a thread keeps between the two passes over a run.
template <int DTYPE>
constexpr int HELD = DTYPE == BITSKNN_F32 ? 4 : 8;

template <int DTYPE>
__device__ __forceinline__ void floats_of(const raw8<DTYPE>& r, float (&v)[8])
{
#pragma unroll
    for (int i = 0; i < (DTYPE == BITSKNN_F32 ? 2 : 1); ++i)
    {
        const uint32_t w[4] = {r.w[i].x, r.w[i].y, r.w[i].z, r.w[i].w};
#pragma unroll
        for (int j = 0; j < 4; ++j)
        {
            if constexpr (DTYPE == BITSKNN_F32)
            {
                v[4 * i + j] = __uint_as_float(w[j]);
            }
            else if constexpr (DTYPE == BITSKNN_BF16)
            {
                v[2 * j] = __uint_as_float(w[j] << 16);
                v[2 * j + 1] = __uint_as_float(w[j] & 0xffff0000U);
            }
            else
            {
                const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[j]));
                v[2 * j] = f.x;
                v[2 * j + 1] = f.y;
            }
        }
    }
}

// The largest size among the numbers of `r` and `acc`: two packed 16-bit numbers, or one float's bits.  NaN
// counts for nothing, infinities count.
template <int DTYPE>
__device__ __forceinline__ uint32_t larger(uint32_t acc, const raw8<DTYPE>& r)
{
#pragma unroll
    for (int i = 0; i < (DTYPE == BITSKNN_F32 ? 2 : 1); ++i)
    {
        const uint32_t w[4] = {r.w[i].x, r.w[i].y, r.w[i].z, r.w[i].w};
#pragma unroll
        for (int j = 0; j < 4; ++j)
        {
            if constexpr (DTYPE == BITSKNN_F32)
            {
                acc = __float_as_uint(fmaxf(__uint_as_float(acc), fabsf(__uint_as_float(w[j]))));
            }
            else if constexpr (DTYPE == BITSKNN_BF16)
            {
                const __nv_bfloat162 m = __hmax2(*reinterpret_cast<const __nv_bfloat162*>(&acc),
                                                 __habs2(*reinterpret_cast<const __nv_bfloat162*>(&w[j])));
                acc = *reinterpret_cast<const uint32_t*>(&m);
            }
            else
            {
                const __half2 m =
                    __hmax2(*reinterpret_cast<const __half2*>(&acc), __habs2(*reinterpret_cast<const __half2*>(&w[j])));
                acc = *reinterpret_cast<const uint32_t*>(&m);
            }
        }
    }
    return acc;
}

template <int DTYPE>
__device__ __forceinline__ float size_of(uint32_t acc)
{
    if constexpr (DTYPE == BITSKNN_F32)
    {
        return __uint_as_float(acc);
    }
    else if constexpr (DTYPE == BITSKNN_BF16)
    {
        return fmaxf(__uint_as_float(acc << 16), __uint_as_float(acc & 0xffff0000U));
    }
    else
    {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&acc));
        return fmaxf(f.x, f.y);
    }
}

// Smallest power of two s in [2^E_MIN, 2^E_MAX] with amax <= 448 s.  448 = 1.75 * 2^8, so the
// exponent is that of amax less 8, and one more if its fraction is above 1.75.
__device__ __forceinline__ float scale_of(float amax)
{
    const uint32_t bits = __float_as_uint(amax);
    const int e = static_cast<int>(bits >> 23) - 127 - 8 + ((bits & 0x7fffffU) > 0x600000U ? 1 : 0);
    return cache::pow2_int(min(max(e, cache::E_MIN), cache::E_MAX)); // subnormal amax: far below the border
}

// A team of threads (a warp or a block) = one window of tokens, one head, keys or values (gridDim = windows
// x heads x 2).  It serves the pages whose first token lies in its window, run after run: a run is the longest
// stretch of tokens of one page with ascending rows.  Two passes over a run: the largest finite
// entry (the team's maximum), then rounding; what fits into HELD vectors per thread stays in
// registers between them (a block: 64 rows of 128 halves, 32 of 128 floats; a warp a quarter of that), the
// rest is read again from L2.  Where pages are small the teams are warps: four runs are then under way where a
// block has one.
// A page has one scale per head, which is why a run belongs to one team and why a later token
// that needs a larger scale re-rounds the rows in front of it: with powers of two that only
// costs bits at the subnormal end, code * 2^(old - new) is exact for every other code.
//
// Bound by HBM (numbers in, codes out) for prompts: 27392 tokens x 8 heads x 128 halves in pages of 64 rows,
// 169 MB, in 37 us = 4.6 TB/s, 0.70 of the measured copy rate; a decode step is one launch of 4 us.
template <int DTYPE, int TEAM>
__global__ void __launch_bounds__(APPEND_THREADS, 8) cache_append_kernel(const append_args a)
{
    constexpr int KEPT = HELD<DTYPE>;
    __shared__ float s_top[APPEND_THREADS / 32];
    __shared__ int s_first[APPEND_THREADS / 32];
    const int t = threadIdx.x % TEAM;
    const int lane = t & 31;
    const int head = blockIdx.y;
    const int which = blockIdx.z;
    const void* src = which == 0 ? a.src[0] : a.src[1];
    const int64_t stride = which == 0 ? a.stride[0] : a.stride[1];
    uint8_t* const codes = which == 0 ? a.c.keys : a.c.values;
    float* const scales = which == 0 ? a.c.key_scales : a.c.value_scales;
    // a thread serves one vector of eight numbers of every row_step-th row
    const int vecs = a.dim >> 3;
    const int row_step = TEAM / vecs;
    const int row0 = t < row_step * vecs ? t / vecs : 1 << 20;
    const int at_vec = t % vecs * 8;
    const int rows_mask = (1 << a.c.page_shift) - 1;
    const int64_t window_begin =
        (static_cast<int64_t>(blockIdx.x) * (APPEND_THREADS / TEAM) + threadIdx.x / TEAM) * a.window;
    if (window_begin >= a.tokens)
    {
        return; // a warp of the last block (blocks as teams have a window each)
    }
    const int first_token = static_cast<int>(window_begin);
    int end_token = min(first_token + a.window, a.tokens);
    auto page_of = [&](int64_t slot) -> int64_t {
        const int64_t p = slot < 0 ? -1 : slot >> a.c.page_shift;
        return p < a.c.pages ? p : -1;
    };
    // first token in [from, limit) that has a place on a page other than `but`, else `limit`; every
    // warp looks for itself, 128 slots at a time
    auto find = [&](int from, int limit, int64_t but) {
        for (; from < limit; from += 128)
        {
            int64_t s[4];
#pragma unroll
            for (int x = 0; x < 4; ++x)
            {
                const int j = from + x * 32 + lane;
                s[x] = j < limit ? a.slots[j] : -1;
            }
#pragma unroll
            for (int x = 0; x < 4; ++x)
            {
                const int64_t p = page_of(s[x]);
                const unsigned hit = __ballot_sync(FULL_MASK, p >= 0 && p != but);
                if (hit != 0)
                {
                    return from + x * 32 + __ffs(hit) - 1;
                }
            }
        }
        return limit;
    };
    auto team_sync = [] {
        if constexpr (TEAM > 32)
        {
            __syncthreads();
        }
        else
        {
            __syncwarp();
        }
    };
    // the same up to the last token.  The padding of a batch may lie there, so the whole team looks
    // when nothing is near, 512 (a warp: 256) slots at a time.
    auto find_far = [&](int from) {
        constexpr int LOOKS = TEAM > 32 ? 4 : 8;
        const int close = min(from + 128, a.tokens);
        int first = find(from, close, -1);
        for (from = close; first == close && from < a.tokens; from += LOOKS * TEAM)
        {
            first = a.tokens;
#pragma unroll
            for (int x = LOOKS - 1; x >= 0; --x)
            {
                const int j = from + x * TEAM + t;
                first = page_of(j < a.tokens ? a.slots[j] : -1) >= 0 ? j : first;
            }
            first = __reduce_min_sync(FULL_MASK, first);
            if constexpr (TEAM > 32)
            {
                if (lane == 0)
                {
                    s_first[t >> 5] = first;
                }
                __syncthreads();
#pragma unroll
                for (int w = 0; w < TEAM / 32; ++w)
                {
                    first = min(first, s_first[w]);
                }
                __syncthreads();
            }
            if (first < a.tokens)
            {
                return first;
            }
            first = close; // go on
        }
        return first == close ? a.tokens : first;
    };
    int i = find(first_token, end_token, -1);
    if (i < end_token && first_token > 0)
    {
        // a page whose tokens reach into the window from the left is served by an earlier block
        int64_t before = -1;
        for (int j = first_token - 1; j >= 0 && before < 0; j -= 32)
        {
            const int64_t p = j - lane >= 0 ? page_of(a.slots[j - lane]) : -1;
            const unsigned hit = __ballot_sync(FULL_MASK, p >= 0);
            before = hit != 0 ? __shfl_sync(FULL_MASK, p, __ffs(hit) - 1) : -1;
        }
        i = find(i, end_token, before);
    }
    while (i < end_token)
    {
        const int64_t slot0 = a.slots[i];
        const int64_t page = page_of(slot0);
        // length of the run: every warp finds it for itself
        int64_t last = slot0;
        int run = 1;
        bool more = true;
        while (more)
        {
            const int j = i + run + lane;
            const int64_t s = j < a.tokens ? a.slots[j] : -1;
            int64_t left = __shfl_up_sync(FULL_MASK, s, 1);
            left = lane == 0 ? last : left;
            const unsigned stop = __ballot_sync(FULL_MASK, page_of(s) != page || s <= left);
            const int n = stop == 0 ? 32 : __ffs(stop) - 1;
            last = __shfl_sync(FULL_MASK, s, 31);
            run += n;
            more = stop == 0;
        }
        const int offset0 = static_cast<int>(slot0) & rows_mask;
        const int64_t base = page * a.c.page_stride + (static_cast<int64_t>(head) << a.c.page_shift) * a.dim;
        // rows of the page one after the other, as they are unless a caller leaves some out
        const bool dense = a.slots[i + run - 1] - slot0 == run - 1;
        const int64_t from = (i + row0) * stride + static_cast<int64_t>(head) * a.dim + at_vec;
        raw8<DTYPE> held[KEPT];
        auto fetch = [&](int h) { return load8<DTYPE>(src, from + h * row_step * stride); };
        uint32_t acc = 0;
        // the whole page at once: every thread has all its vectors, and nothing is asked for each of them
        const bool full = run >= KEPT * row_step && row_step * vecs == TEAM;
        if (full)
        {
#pragma unroll
            for (int h = 0; h < KEPT; ++h)
            {
                held[h] = fetch(h);
            }
#pragma unroll
            for (int h = 0; h < KEPT; ++h)
            {
                acc = larger<DTYPE>(acc, held[h]);
            }
            if constexpr (TEAM > 32)
            {
                // the next run's numbers set out for L2 while this one is finished, one lane per 128 bytes
                // (27392 tokens in pages of 64 rows: 40 -> 36 us; runs of warps are too short for it)
                if ((t & (DTYPE == BITSKNN_F32 ? 3 : 7)) == 0)
                {
#pragma unroll
                    for (int h = 0; h < KEPT; ++h)
                    {
                        if (i + run + row0 + h * row_step < end_token)
                        {
                            prefetch_l2(src, from + (run + h * row_step) * stride, DTYPE == BITSKNN_F32 ? 4 : 2);
                        }
                    }
                }
            }
        }
        else
        {
#pragma unroll
            for (int h = 0; h < KEPT; ++h)
            {
                if (row0 + h * row_step < run)
                {
                    held[h] = fetch(h);
                    acc = larger<DTYPE>(acc, held[h]);
                }
            }
        }
        for (int h = KEPT; row0 + h * row_step < run; ++h)
        {
            acc = larger<DTYPE>(acc, fetch(h));
        }
        float top = size_of<DTYPE>(acc);
        if (top == INFINITY)
        {
            // infinities set no scale: the largest finite number of this thread
            top = 0.0F;
            for (int h = 0; row0 + h * row_step < run; ++h)
            {
                float f[8];
                floats_of<DTYPE>(fetch(h), f);
#pragma unroll
                for (int e = 0; e < 8; ++e)
                {
                    top = fabsf(f[e]) < INFINITY ? fmaxf(top, fabsf(f[e])) : top;
                }
            }
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1)
        {
            top = fmaxf(top, __shfl_xor_sync(FULL_MASK, top, o));
        }
        float* const scale_at = scales + page * a.c.heads + head;
        const float stored = offset0 == 0 ? 0.0F : *scale_at;
        if constexpr (TEAM > 32)
        {
            if (lane == 0)
            {
                s_top[t >> 5] = top;
            }
            __syncthreads();
#pragma unroll
            for (int w = 0; w < TEAM / 32; ++w)
            {
                top = fmaxf(top, s_top[w]);
            }
        }
        // a page that is begun forgets the scale of its former owner; one that is continued keeps
        // at least its own (anything but a positive number in range counts as the smallest)
        const float old =
            stored > 0.0F && stored <= cache::pow2_int(cache::E_MAX) ? stored : cache::pow2_int(cache::E_MIN);
        const float scale = fmaxf(scale_of(top), old);
        const float inverse = 1.0F / scale;
        uint8_t* const to = codes + base + at_vec;
        auto store = [&](int h, const raw8<DTYPE>& x, bool in_order) {
            float f[8];
            floats_of<DTYPE>(x, f);
            const int row = row0 + h * row_step;
            const int offset = in_order ? offset0 + row : static_cast<int>(a.slots[i + row]) & rows_mask;
            uint2 out;
            out.x = cache::codes_of_floats(f[0] * inverse, f[1] * inverse) |
                    cache::codes_of_floats(f[2] * inverse, f[3] * inverse) << 16;
            out.y = cache::codes_of_floats(f[4] * inverse, f[5] * inverse) |
                    cache::codes_of_floats(f[6] * inverse, f[7] * inverse) << 16;
            *reinterpret_cast<uint2*>(to + offset * a.dim) = out;
        };
        if (full && dense)
        {
#pragma unroll
            for (int h = 0; h < KEPT; ++h)
            {
                store(h, held[h], true);
            }
        }
        else
        {
#pragma unroll
            for (int h = 0; h < KEPT; ++h)
            {
                if (row0 + h * row_step < run)
                {
                    store(h, held[h], dense);
                }
            }
        }
        for (int h = KEPT; row0 + h * row_step < run; ++h)
        {
            store(h, fetch(h), dense);
        }
        if (offset0 > 0 && scale > old)
        {
            const float shrink = old / scale;
            const int granules = offset0 * a.dim >> 4;
            auto shrunk = [&](uint32_t c) {
                uint32_t lo, hi;
                cache::halves_of_codes(c, lo, hi);
                const float2 x = __half22float2(*reinterpret_cast<const __half2*>(&lo));
                const float2 y = __half22float2(*reinterpret_cast<const __half2*>(&hi));
                return cache::codes_of_floats(x.x * shrink, x.y * shrink) |
                       cache::codes_of_floats(y.x * shrink, y.y * shrink) << 16;
            };
            for (int g = t; g < granules; g += TEAM)
            {
                uint4* const p = reinterpret_cast<uint4*>(codes + base) + g;
                const uint4 c = *p;
                *p = make_uint4(shrunk(c.x), shrunk(c.y), shrunk(c.z), shrunk(c.w));
            }
        }
        team_sync(); // the next run may continue this page
        if (t == 0)
        {
            *scale_at = scale;
        }
        team_sync();
        i += run;
        if (i < end_token)
        {
            i = find(i, end_token, -1);
        }
        if (i >= end_token)
        {
            // the page may go on behind the window, with rows that do not ascend
            i = find_far(i);
            if (i == a.tokens || page_of(a.slots[i]) != page)
            {
                return;
            }
            end_token = i + 1;
        }
    }
}

template <int DTYPE, int TEAM>
int launch_append_teams(append_args a, cudaStream_t stream)
{
    constexpr int TEAMS = APPEND_THREADS / TEAM;
    // Few tokens: one team for each, so that the runs of a decode step (one token long) run side by side;
    // many: windows, as many as run at once (27392 tokens, 8 heads of 128: 8 blocks per SM 37 us, 16 and 32 40).
    const int64_t target =
        std::max<int64_t>(1, static_cast<int64_t>(device_sm_count()) * 8 * TEAMS / (2 * a.c.heads));
    a.window = static_cast<int>((a.tokens + target - 1) / target);
    const int64_t windows = (static_cast<int64_t>(a.tokens) + a.window - 1) / a.window;
    const dim3 grid(static_cast<unsigned>((windows + TEAMS - 1) / TEAMS), static_cast<unsigned>(a.c.heads), 2U);
    {
        kernel_scope scope("cache_append_kernel", stream);
        cache_append_kernel<DTYPE, TEAM><<<grid, APPEND_THREADS, 0, stream>>>(a);
    }
    BITSKNN_CUDA_TRY(cudaGetLastError());
    return BITSKNN_OK;
}

template <int DTYPE>
int launch_append(const append_args& a, int page_rows, cudaStream_t stream)
{
    // Warps for pages of up to twice what they keep (8192 tokens, 8 heads of 128: pages of 16 rows 9.5 us, blocks
    // 24; of 32 rows 11.6 and 18), blocks for larger ones (27392 tokens, 64 rows: 37 us, warps 62).
    return page_rows * a.dim <= 2 * 32 * HELD<DTYPE> * 8 ? launch_append_teams<DTYPE, 32>(a, stream)
                                                         : launch_append_teams<DTYPE, APPEND_THREADS>(a, stream);
}

} // namespace

} // namespace bitsknn

extern "C" int bitsknn_cache_append(const bitsknn_cache_t* cache, const void* d_new_keys, const void* d_new_values,
                                    int dtype, int64_t key_stride, int64_t value_stride, const int64_t* d_slots,
                                    int64_t tokens, bitsknn_stream_t stream)
{
    using namespace bitsknn;
    append_args a{};
    const int rc = check_cache(cache, &a.c);
    if (rc != BITSKNN_OK)
    {
        return rc;
    }
    if (dtype != BITSKNN_F32 && dtype != BITSKNN_F16 && dtype != BITSKNN_BF16)
    {
        return fail(BITSKNN_ERR_UNSUPPORTED_MODE, "dtype %d: only F32, F16 and BF16", dtype);
    }
    if (tokens < 0 || tokens > cache::MOST_ROWS)
    {
        return fail(BITSKNN_ERR_INVALID_ARGUMENT, "invalid token count %lld", static_cast<long long>(tokens));
    }
    const int64_t dense = static_cast<int64_t>(cache->heads) * cache->dim;
    key_stride = key_stride == 0 ? dense : key_stride;
    value_stride = value_stride == 0 ? dense : value_stride;
    const int64_t unit = dtype == BITSKNN_F32 ? 4 : 8; // elements in 16 bytes
    if (key_stride < dense || value_stride < dense || key_stride % unit != 0 || value_stride % unit != 0)
    {
        return fail(BITSKNN_ERR_INVALID_ARGUMENT,
                    "strides %lld and %lld between tokens: at least %lld and a multiple of %lld",
                    static_cast<long long>(key_stride), static_cast<long long>(value_stride),
                    static_cast<long long>(dense), static_cast<long long>(unit));
    }
    if (tokens == 0)
    {
        return BITSKNN_OK;
    }
    if (d_new_keys == nullptr || d_new_values == nullptr || d_slots == nullptr)
    {
        return fail(BITSKNN_ERR_INVALID_ARGUMENT, "null pointer argument");
    }
    if (((reinterpret_cast<uintptr_t>(d_new_keys) | reinterpret_cast<uintptr_t>(d_new_values)) & 15) != 0)
    {
        return fail(BITSKNN_ERR_INVALID_ARGUMENT, "misaligned vectors: 16-byte alignment needed");
    }
    a.src[0] = d_new_keys;
    a.src[1] = d_new_values;
    a.stride[0] = key_stride;
    a.stride[1] = value_stride;
    a.slots = d_slots;
    a.tokens = static_cast<int>(tokens);
    a.dim = cache->dim;
    a.dtype = dtype;
    auto s = static_cast<cudaStream_t>(stream);
    return dtype == BITSKNN_F32   ? launch_append<BITSKNN_F32>(a, cache->page_rows, s)
           : dtype == BITSKNN_F16 ? launch_append<BITSKNN_F16>(a, cache->page_rows, s)
                                  : launch_append<BITSKNN_BF16>(a, cache->page_rows, s);
}
