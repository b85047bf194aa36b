// What the attention kernels over the paged 8-bit cache share: arguments, the division of the work
// among blocks, and the join of items that several blocks worked on.
//
// Mathematics.  For a query column with logits (base 2) t_j = scale * log2(e) * <q, code_j> * ks_j,
// the weights are w_j = 2^(t_j + log2(vs_j) - m): the value scale rides on the logit, so that the
// second product multiplies weights with bare codes, and m is the running maximum of t_j + log2(vs_j).
// The denominator sums w_j / vs_j = 2^(t_j - m), in the same units, so out = sum w_j code_j / sum w_j / vs_j
// needs no scale at all.  One pass: when m grows, what was summed is multiplied by 2^(m_old - m_new).
// Logits, maxima and sums are FP32.  Weights are rounded to halves (11 bits, the codes are exact
// halves): the reference point m is kept 7 binary orders below the half range's 2^7 ... 2^15, so a
// weight of 2^-31 of the largest is still not lost, which 10^5 positions of little weight need.
//
// Largest means the largest of p_j vs_j.  Where value scales lie far apart that is not the largest p_j:
// a page of a scale 2^30 times the others' would take the halves of all other positions to zero,
// though it may hold a single number, and the outputs of the dimensions it has none in would be lost.  So
// positions whose scale is below 2^-SCALE_SPREAD of the largest one so far get their weights as sums of two
// BF16 numbers (17 bits, the range of floats) and their codes as BF16 (exact).  For the others a half, off by at most
// 2^-25 where the largest p vs has 2^7 or more, is off by 2^(SCALE_SPREAD - 32) = 2^-28 of the largest p.  The BF16
// weights end at the smallest float: p vs below 2^-133 of the largest counts as zero.
#pragma once

#include "cache.cuh"

namespace bitsknn::cache
{

struct attend_args
{
    view c;
    batch b;
    const void* queries;
    int dtype;
    int64_t query_stride;
    int group;
    float scale;      // times log2(e)
    void* out;
    int64_t out_stride;
    float* lse;
    const int32_t* idx; // selected: lists
    int64_t ld_idx;
    int k;
    float* part_o;    // [2 * blocks][columns][DIM]
    float2* part_ml;  // [2 * blocks][columns]
    int4* joins;      // [blocks]
    int* join_end;    // [blocks]
    int cluster;        // > 0: an item to every cluster of so many blocks, which joins by itself
};

// What the stream of a block works on: one block of query columns of a request and head.
struct item
{
    int request;
    int first_token; // packed token of column 0 of the request (selected: the token)
    int head;
    int column0;
    int columns;     // columns of the request (selected: of the token) in total
    int64_t begin;   // where it lies on the axis of the work
    int64_t end;
};

} // namespace bitsknn::cache

namespace bitsknn
{

namespace
{

using namespace cache;

constexpr float WEIGHT_BIAS = 7.0F;  // the weight of the reference point is 2^7
constexpr float WEIGHT_SLACK = 8.0F; // a logit may pass the reference point by 8 (weight 2^15) before it moves
constexpr uint32_t SCALE_SPREAD = 4;  // binary orders of value scales that halves can serve together
constexpr float LOG2_E = 1.4426950408889634F;
constexpr float LN_2 = 0.6931471805599453F;

__device__ __forceinline__ void store_out(void* out, int64_t at, float v, int dtype)
{
    if (dtype == BITSKNN_F16)
    {
        static_cast<__half*>(out)[at] = __float2half_rn(v);
    }
    else
    {
        static_cast<__nv_bfloat16*>(out)[at] = __float2bfloat16_rn(v);
    }
}

// ---- shares of the work ----------------------------------------------------------------------
// All items lie on one axis: requests in order, within a request heads, within a head blocks of
// SHAPE::COLS columns.  An item covers SHAPE::COST units for its beginning and end (packing the
// queries, filling the pipeline, joining the sums) and one unit for each of its tiles of
// SHAPE::ROWS positions.  Block c of the grid takes the c-th equal share of the axis, so a long
// request is spread over many blocks and short ones fill up the others.
template <class SHAPE>
__device__ __forceinline__ int units_of_block(const attend_args& a, const request& q, int column0)
{
    const int last = min(column0 + SHAPE::COLS, q.count * a.group) - 1;
    return (visible_of(a.b, q, last / a.group) + SHAPE::ROWS - 1) / SHAPE::ROWS + SHAPE::COST;
}

template <class SHAPE>
__device__ __forceinline__ int64_t units_of_head(const attend_args& a, const request& q)
{
    int64_t sum = 0;
    for (int col = 0; col < q.count * a.group; col += SHAPE::COLS)
    {
        sum += units_of_block<SHAPE>(a, q, col);
    }
    return sum;
}

template <int WARPS>
__device__ __forceinline__ int64_t block_sum(int64_t v, int64_t* words)
{
#pragma unroll
    for (int o = 16; o > 0; o >>= 1)
    {
        v += __shfl_xor_sync(FULL_MASK, v, o);
    }
    __syncthreads();
    if ((threadIdx.x & 31) == 0)
    {
        words[threadIdx.x >> 5] = v;
    }
    __syncthreads();
    int64_t sum = 0;
#pragma unroll
    for (int w = 0; w < WARPS; ++w)
    {
        sum += words[w];
    }
    return sum;
}

// The request that holds unit `at`, and the first unit of that request.
template <class SHAPE, int WARPS>
__device__ __forceinline__ int find_request(const attend_args& a, int64_t at, int64_t* first, int64_t* words, int* found)
{
    int64_t before = 0;
    for (int base = 0; base < a.b.requests; base += WARPS * 32)
    {
        const int r = base + threadIdx.x;
        const int64_t mine = r < a.b.requests ? units_of_head<SHAPE>(a, request_of(a.b, r)) * a.c.heads : 0;
        int64_t upto = mine;
        const int lane = threadIdx.x & 31;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1)
        {
            const int64_t x = __shfl_up_sync(FULL_MASK, upto, o);
            upto += lane >= o ? x : 0;
        }
        __syncthreads();
        if (lane == 31)
        {
            words[threadIdx.x >> 5] = upto;
        }
        if (threadIdx.x == 0)
        {
            *found = -1;
        }
        __syncthreads();
        int64_t all = 0;
#pragma unroll
        for (int w = 0; w < WARPS; ++w)
        {
            upto += w < static_cast<int>(threadIdx.x >> 5) ? words[w] : 0;
            all += words[w];
        }
        const int64_t start = before + upto - mine;
        __syncthreads();
        if (at >= start && at < start + mine)
        {
            *found = r;
            words[0] = start;
        }
        __syncthreads();
        if (*found >= 0)
        {
            *first = words[0];
            return *found;
        }
        before += all;
    }
    return -1; // not reached: `at` lies below the total
}

// Joins the parts of items that several blocks worked on: block c looks after the item that begins
// in block c of the main kernel and ends in a later one, whose parts are part 1 of block c and
// part 0 of the blocks up to its last.  Always in that order, so results do not depend on timing.
// SPLIT warps share the parts of a column when there are many (few columns of a long request that decodes); few
// parts are a warp's work, so that most of the grid has nothing to do (64 requests 115 -> 114
// us, 32 requests with lists 43 -> 41).  Launched while the main kernel still runs
// (griddepcontrol), so that its own launch takes no time.
constexpr int JOIN_WARPS = 8;

template <int DIM, int COLS>
constexpr int JOIN_SPLIT = COLS <= 32 ? JOIN_WARPS : 1;

template <int DIM, int COLS>
__global__ void __launch_bounds__(JOIN_WARPS * 32) cache_join_kernel(const attend_args a)
{
    constexpr int SPLIT = JOIN_SPLIT<DIM, COLS>;
    constexpr int PER = DIM / 32;
    constexpr int VEC = PER % 4 == 0 ? 4 : PER % 2 == 0 ? 2 : 1; // numbers per load
    struct alignas(4 * VEC) vec
    {
        float v[VEC];
    };
    __shared__ float s_sum[SPLIT > 1 ? SPLIT : 1][DIM];
    __shared__ float2 s_ml[SPLIT > 1 ? SPLIT : 1];
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int4 join = a.joins[blockIdx.x];
    const int warp = threadIdx.x >> 5;
    const int lane = threadIdx.x & 31;
    const int all = a.join_end[blockIdx.x] - static_cast<int>(blockIdx.x) + 1; // of no meaning without a join
    constexpr int FEW = 4;
    const bool alone = SPLIT == 1 || all <= FEW; // a column is one warp's work
    const int col = static_cast<int>(blockIdx.y) * (alone ? JOIN_WARPS : 1) + (alone ? warp : 0);
    if (col >= min(join.w - join.z, COLS))
    {
        return; // the whole block when warps share a column
    }
    const int64_t first = 2 * static_cast<int64_t>(blockIdx.x) + 1;
    auto part = [&](int i) { return (first + (i == 0 ? 0 : 2 * i - 1)) * COLS + col; };
    // this warp's parts, a run of them so that the order of the sums is that of the positions
    const int begin = alone ? 0 : warp * all / SPLIT;
    const int parts = alone ? all : (warp + 1) * all / SPLIT - begin;
    float top = -INFINITY;
    float sum[PER];
#pragma unroll
    for (int x = 0; x < PER; ++x)
    {
        sum[x] = 0.0F;
    }
    float den = 0.0F;
    if (alone && parts <= FEW)
    {
        // the usual case of prompts and of batches: everything is loaded at once, and every lane weighs for itself
        float2 ml[FEW];
        vec w[FEW][PER / VEC];
#pragma unroll
        for (int i = 0; i < FEW; ++i)
        {
            ml[i] = make_float2(-INFINITY, 0.0F);
            if (i < parts)
            {
                ml[i] = a.part_ml[part(i)];
                const vec* from = reinterpret_cast<const vec*>(a.part_o + part(i) * DIM) + lane;
#pragma unroll
                for (int x = 0; x < PER / VEC; ++x)
                {
                    w[i][x] = from[x * 32];
                }
            }
        }
#pragma unroll
        for (int i = 0; i < FEW; ++i)
        {
            top = fmaxf(top, ml[i].x);
        }
#pragma unroll
        for (int i = 0; i < FEW; ++i)
        {
            if (i < parts)
            {
                const float keep = ml[i].x == -INFINITY ? 1.0F : exp2_fast(ml[i].x - top);
                den = fmaf(keep, ml[i].y, den);
#pragma unroll
                for (int x = 0; x < PER; ++x)
                {
                    sum[x] = fmaf(keep, w[i][x / VEC].v[x % VEC], sum[x]);
                }
            }
        }
    }
    else
    {
        for (int i = lane; i < parts; i += 32)
        {
            top = fmaxf(top, a.part_ml[part(begin + i)].x);
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1)
        {
            top = fmaxf(top, __shfl_xor_sync(FULL_MASK, top, o));
        }
        for (int base = 0; base < parts; base += 32)
        {
            float keep = 0.0F;
            if (base + lane < parts)
            {
                const float2 ml = a.part_ml[part(begin + base + lane)];
                keep = ml.x == -INFINITY ? 1.0F : exp2_fast(ml.x - top);
                den = fmaf(keep, ml.y, den);
            }
            const int here = min(parts - base, 32);
#pragma unroll 8
            for (int i = 0; i < here; ++i)
            {
                const float f = __shfl_sync(FULL_MASK, keep, i);
                const vec* from = reinterpret_cast<const vec*>(a.part_o + part(begin + base + i) * DIM) + lane;
#pragma unroll
                for (int x = 0; x < PER / VEC; ++x)
                {
                    const vec w = from[x * 32];
#pragma unroll
                    for (int y = 0; y < VEC; ++y)
                    {
                        sum[x * VEC + y] = fmaf(f, w.v[y], sum[x * VEC + y]);
                    }
                }
            }
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1)
        {
            den += __shfl_xor_sync(FULL_MASK, den, o);
        }
    }
    if (!alone)
    {
#pragma unroll
        for (int x = 0; x < PER; ++x)
        {
            s_sum[warp][(x / VEC * 32 + lane) * VEC + x % VEC] = sum[x];
        }
        if (lane == 0)
        {
            s_ml[warp] = make_float2(top, den);
        }
        __syncthreads();
        if (warp > 0)
        {
            return;
        }
#pragma unroll
        for (int w = 0; w < SPLIT; ++w)
        {
            top = fmaxf(top, s_ml[w].x);
        }
        den = 0.0F;
#pragma unroll
        for (int x = 0; x < PER; ++x)
        {
            sum[x] = 0.0F;
        }
#pragma unroll
        for (int w = 0; w < SPLIT; ++w)
        {
            const float2 ml = s_ml[w];
            const float keep = ml.x == -INFINITY ? 1.0F : exp2_fast(ml.x - top);
            den = fmaf(keep, ml.y, den);
#pragma unroll
            for (int x = 0; x < PER; ++x)
            {
                sum[x] = fmaf(keep, s_sum[w][(x / VEC * 32 + lane) * VEC + x % VEC], sum[x]);
            }
        }
    }
    const int g = join.z + col;
    const int64_t token = join.x + g / a.group;
    const int qhead = join.y * a.group + g % a.group;
#pragma unroll
    for (int x = 0; x < PER; ++x)
    {
        const int d = (x / VEC * 32 + lane) * VEC + x % VEC;
        store_out(a.out, token * a.out_stride + static_cast<int64_t>(qhead) * DIM + d,
                  den == 0.0F ? 0.0F : sum[x] / den, a.dtype);
    }
    if (lane == 0 && a.lse != nullptr)
    {
        a.lse[token * a.group * a.c.heads + qhead] = den == 0.0F ? -INFINITY : (top - WEIGHT_BIAS + log2f(den)) * LN_2;
    }
}

constexpr size_t JOIN_BYTES = sizeof(int4) + sizeof(int);

// Workspace of a launch of `blocks` blocks: two parts per block and its join.
template <int DIM, int COLS>
size_t parts_bytes(int blocks)
{
    return static_cast<size_t>(blocks) * (2 * COLS * (DIM * sizeof(float) + sizeof(float2)) + JOIN_BYTES) + 256;
}

// Checks the workspace and the arrays of a call (none of its writes may lie where it reads) and places the parts.
template <int DIM, int COLS>
int place_parts(attend_args& a, int blocks, void* workspace, size_t workspace_bytes)
{
    if (workspace_bytes < parts_bytes<DIM, COLS>(blocks))
    {
        return fail(BITSKNN_ERR_WORKSPACE, "workspace of %zu bytes is smaller than the %zu needed", workspace_bytes,
                    parts_bytes<DIM, COLS>(blocks));
    }
    // other blocks still read when the first ones write
    const int64_t heads = static_cast<int64_t>(a.group) * a.c.heads;
    const extent writes[] = {{"d_out", a.out, a.b.tokens, a.out_stride * 2, heads * DIM * 2},
                             dense_extent("d_lse", a.lse, a.b.tokens * heads * 4),
                             dense_extent("the workspace", workspace, static_cast<int64_t>(parts_bytes<DIM, COLS>(blocks)))};
    const extent reads[] = {{"d_queries", a.queries, a.b.tokens, a.query_stride * 2, heads * DIM * 2},
                            {"d_idx", a.idx, static_cast<int64_t>(a.b.tokens) * a.c.heads, a.ld_idx * 4, a.k * 4LL}};
    const int rc = check_apart(writes, 3, reads, 2);
    if (rc != BITSKNN_OK)
    {
        return rc;
    }
    a.part_o = static_cast<float*>(workspace);
    a.joins = reinterpret_cast<int4*>(a.part_o + static_cast<size_t>(blocks) * 2 * COLS * DIM);
    a.part_ml = reinterpret_cast<float2*>(a.joins + blocks);
    a.join_end = reinterpret_cast<int*>(a.part_ml + static_cast<size_t>(blocks) * 2 * COLS);
    return BITSKNN_OK;
}

// The join, launched while the main kernel of `blocks` blocks runs.
template <int DIM, int COLS>
int launch_join(const attend_args& a, int blocks, cudaStream_t stream)
{
    cudaLaunchAttribute early{};
    early.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    early.val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t config{};
    config.gridDim = dim3(static_cast<unsigned>(blocks), COLS * JOIN_SPLIT<DIM, COLS> / JOIN_WARPS);
    config.blockDim = dim3(JOIN_WARPS * 32);
    config.stream = stream;
    config.attrs = &early;
    config.numAttrs = 1;
    BITSKNN_CUDA_TRY(cudaLaunchKernelEx(&config, cache_join_kernel<DIM, COLS>, a));
    return BITSKNN_OK;
}

} // namespace

// Attention of many query columns per request and head through tensor memory (cache_attend_tc.cu).
size_t attend_tc_workspace_bytes(int dim);
int launch_attend_tc(int dim, const cache::attend_args& a, void* workspace, size_t workspace_bytes, cudaStream_t stream);

} // namespace bitsknn
