// cache_attend for many query columns per request and head (prompts, chunks of prompts): both
// products on the fifth-generation tensor cores, scores and sums in tensor memory.
#include <algorithm>

#include "cache_attend.cuh"
#include "tc.cuh"

namespace bitsknn
{

namespace
{

constexpr int TC_GROUPS = 4;  // scale slots: positions in flight between a conversion and its softmax
constexpr int TC_THREADS = 14 * 32;
constexpr int CONVERTERS = 128;

// One block: NQ tiles of 128 query rows against tiles of ROWS positions.  Rows of 192 and 256 numbers
// leave tensor memory (512 columns: scores + sums) for one query tile only, and shared memory for tiles
// of 64 positions.
template <int DIM>
struct tc_shape
{
    static constexpr int NQ = DIM <= 128 ? 2 : 1;
    static constexpr int COLS = 128 * NQ;
    static constexpr int ROWS = DIM <= 128 ? 128 : 64;
    static constexpr int COST = 2;               // an item's beginning and end, in tiles
    static constexpr int BLK = (DIM + 63) / 64;  // 128-byte blocks of 64 halves per row
    static constexpr int Q_BYTES = BLK * 128 * 128;
    static constexpr int KV_BYTES = BLK * ROWS * 128;
    static constexpr int GROUPS = ROWS / 16;
    static constexpr int O_COL = NQ * ROWS;      // tensor memory: scores of the query tiles, then their sums
    static constexpr int USED_COLS = O_COL + NQ * DIM;
    static constexpr int TMEM_COLS = USED_COLS <= 128 ? 128 : USED_COLS <= 256 ? 256 : 512;
    static constexpr int TAIL = TC_GROUPS * GROUPS * 16 + DIM * 4 + 15 * 8 + 8; // scales, first NaN, barriers, tmem slot
    static constexpr int BYTES = NQ * Q_BYTES + 4 * KV_BYTES + TAIL + 1024;
    static_assert(USED_COLS <= 512, "tensor memory");
    static_assert(BYTES <= 227 * 1024, "shared memory");
};

// D[tmem] (+)= A[tmem] * B[smem], halves, FP32 sums; issued by one thread.
__device__ __forceinline__ void mma_ts(uint32_t d_tmem, uint32_t a_tmem, uint64_t b_desc, uint32_t idesc, bool accumulate)
{
    asm volatile("{\n"
                 ".reg .pred p;\n"
                 "setp.ne.b32 p, %4, 0;\n"
                 "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n"
                 "}\n" ::"r"(d_tmem),
                 "r"(a_tmem), "l"(b_desc), "r"(idesc), "r"(accumulate ? 1U : 0U)
                 : "memory");
}

__device__ __forceinline__ void tmem_st_16(uint32_t taddr, const uint32_t (&v)[16])
{
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
                 "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(taddr),
                 "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]),
                 "r"(v[9]), "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15])
                 : "memory");
}

__device__ __forceinline__ void tmem_st_32(uint32_t taddr, const uint32_t (&v)[32])
{
    asm volatile("tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
                 "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, "
                 "%17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};" ::"r"(taddr),
                 "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]),
                 "r"(v[9]), "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15]), "r"(v[16]),
                 "r"(v[17]), "r"(v[18]), "r"(v[19]), "r"(v[20]), "r"(v[21]), "r"(v[22]), "r"(v[23]), "r"(v[24]),
                 "r"(v[25]), "r"(v[26]), "r"(v[27]), "r"(v[28]), "r"(v[29]), "r"(v[30]), "r"(v[31])
                 : "memory");
}

__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// Descriptor of the values as second operand of the second product: rows are positions (the
// contraction), each 128-byte row holds 64 dims of one position, so the tile is contiguous along
// its outputs.  8-row groups are 1024 bytes apart (stride offset), blocks of 64 dims `block_bytes`
// (leading offset).  Same bytes in shared memory as a K-major tile of positions x dims.
__device__ __forceinline__ uint64_t values_desc(const void* tile, uint32_t block_bytes)
{
    const uint64_t addr = (ptx::smem_addr(tile) & 0x3FFFFU) >> 4;
    return addr | static_cast<uint64_t>(block_bytes >> 4) << 16 | static_cast<uint64_t>(1024 >> 4) << 32 |
           static_cast<uint64_t>(1) << 46 | static_cast<uint64_t>(2) << 61;
}

// Shared-memory byte of halves [8 * chunk, 8 * chunk + 8) of row `row` of a tile with `rows` rows in
// blocks of 64 halves, 128-byte swizzle.
__device__ __forceinline__ uint32_t tile_byte(int row, int chunk, int rows)
{
    return static_cast<uint32_t>((chunk >> 3) * rows * 128 + row * 128 + (((chunk & 7) ^ (row & 7)) << 4));
}

__device__ __forceinline__ void st_shared16(uint32_t addr, uint32_t a, uint32_t b, uint32_t c, uint32_t d)
{
    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}

__device__ __forceinline__ void fence_async_proxy() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

// A wait of a whole warp: its threads go on, or give up, together.
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity)
{
    return __all_sync(FULL_MASK, ptx::mbar_wait_bounded_spin(bar, parity)) != 0;
}

// Warps 0-3 and 4-7: softmax of query tile 0 and 1, one thread per row.  Warps 8-11: converters, codes
// to halves.  Warps 12 and 13: one thread each issues the products of a query tile.
//
// A tile of ROWS positions goes round like this.  The converters bring 16 codes per thread and load
// from the cache a tile ahead, turn them into halves and store them in the swizzled layout the tensor
// cores read (two stages each of keys and values).  S = Q K^T lands in tensor memory; a softmax thread
// reads its row twice (maximum, then weights; the row's 128 scores would not fit its registers) and
// writes the weights as halves over the scores; O += P V takes them from there as its first
// operand, and the values as they lie, contiguous along the outputs.  While one query tile is with its
// softmax warps the tensor cores work for the other one.  The two issuing threads do not wait for one
// another (a thread is held while its products run).  O stays in tensor memory; it is touched
// only when a row's reference point has to move by more than 2^8 (rarely after the first tile).
//
// Bound by the exponentials (16 per clock and SM: 2048 clocks for 256 rows x 128 positions) and the
// tensor cores (4 products of 128 x 128 x 128: about 2300 clocks) alike.
template <int DIM>
__global__ void __launch_bounds__(TC_THREADS, 1) cache_attend_tc_kernel(const attend_args a, int* status)
{
    using shape = tc_shape<DIM>;
    constexpr int NQ = shape::NQ;
    constexpr int ROWS = shape::ROWS;
    constexpr int GROUPS = shape::GROUPS;
    constexpr int PARTS = DIM / 16;                        // 16-code pieces per row
    constexpr int PIECES = ROWS * PARTS / CONVERTERS;      // per converter thread and tile
    static_assert(ROWS * PARTS % CONVERTERS == 0, "pieces");
    extern __shared__ unsigned char raw[];
    unsigned char* const base = raw + ((1024U - (ptx::smem_addr(raw) & 1023U)) & 1023U);
    unsigned char* const q_tiles = base;
    unsigned char* const k_tiles = base + NQ * shape::Q_BYTES;
    unsigned char* const v_tiles = k_tiles + 2 * shape::KV_BYTES;
    float4* const scales = reinterpret_cast<float4*>(v_tiles + 2 * shape::KV_BYTES); // [TC_GROUPS][GROUPS]: ks, lv, 1 / vs
    int* const first_nan = reinterpret_cast<int*>(scales + TC_GROUPS * GROUPS);      // [DIM]
    uint64_t* const bars = reinterpret_cast<uint64_t*>(first_nan + DIM);
    uint64_t* const k_full = bars;        // [2]
    uint64_t* const k_empty = bars + 2;   // [2]
    uint64_t* const v_full = bars + 4;    // [2]
    uint64_t* const v_empty = bars + 6;   // [2]
    uint64_t* const s_full = bars + 8;    // [2] per query tile
    uint64_t* const p_full = bars + 10;   // [2]
    uint64_t* const o_done = bars + 12;   // [2]
    uint32_t* const tmem_slot = reinterpret_cast<uint32_t*>(bars + 14);
    __shared__ int64_t s_words[TC_THREADS / 32];
    __shared__ int s_found;
    const int t = threadIdx.x;
    const int warp = t >> 5;
    const int lane = t & 31;
    const int rows_mask = (1 << a.c.page_shift) - 1;

    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    if (t == 0)
    {
        a.joins[blockIdx.x] = make_int4(0, 0, 0, 0);
        for (int i = 0; i < 2; ++i)
        {
            ptx::mbar_init(&k_full[i], CONVERTERS);
            ptx::mbar_init(&v_full[i], CONVERTERS);
            ptx::mbar_init(&k_empty[i], NQ);
            ptx::mbar_init(&v_empty[i], NQ);
            ptx::mbar_init(&s_full[i], 2); // the products' commit, and the issuing thread itself: what it has
            ptx::mbar_init(&p_full[i], 128);
            ptx::mbar_init(&o_done[i], 2); // seen of the converters (scales, NaN) is then seen by the softmax
        }
        ptx::mbar_init_fence();
    }
    if (warp == 0)
    {
        tc::tmem_alloc(tmem_slot, shape::TMEM_COLS);
    }
    tc::fence_before_sync();
    __syncthreads();
    tc::fence_after_sync();
    const uint32_t tmem = *tmem_slot;

    int64_t sum = 0;
    for (int r = t; r < a.b.requests; r += TC_THREADS)
    {
        sum += units_of_head<shape>(a, request_of(a.b, r)) * a.c.heads;
    }
    const int64_t total = block_sum<TC_THREADS / 32>(sum, s_words);
    const int64_t blocks = min(static_cast<int64_t>(gridDim.x), total);
    bool fine = true; // no wait of this thread has expired
    if (blockIdx.x < blocks)
    {
        int64_t at = blockIdx.x * total / blocks;
        const int64_t share_end = (blockIdx.x + 1) * total / blocks;
        item it{};
        int64_t first = 0;
        it.request = find_request<shape, TC_THREADS / 32>(a, at, &first, s_words, &s_found);
        request q = request_of(a.b, it.request);
        const int64_t per_head = units_of_head<shape>(a, q);
        it.head = static_cast<int>((at - first) / per_head);
        it.begin = first + it.head * per_head;
        it.first_token = q.first;
        it.columns = q.count * a.group;
        it.end = it.begin + units_of_block<shape>(a, q, 0);
        while (at >= it.end)
        {
            it.column0 += shape::COLS;
            it.begin = it.end;
            it.end += units_of_block<shape>(a, q, it.column0);
        }
        uint32_t kv_tiles = 0; // tiles of keys and values this block has gone through
        uint32_t s_tiles = 0;  // and those of this warp's query tile
        while (true)
        {
            const int64_t seg_end = min(it.end, share_end);
            const int first_tile = max(static_cast<int>(at - it.begin) - shape::COST, 0);
            const int count = max(static_cast<int>(seg_end - it.begin) - shape::COST, 0) - first_tile;
            const int last_col = min(it.column0 + shape::COLS, it.columns) - 1;
            const int furthest = visible_of(a.b, q, last_col / a.group);
            const int nearest = visible_of(a.b, q, it.column0 / a.group);
            const bool whole = at == it.begin && seg_end == it.end;
            const int64_t part = 2 * static_cast<int64_t>(blockIdx.x) + (at == it.begin ? 1 : 0);
            const int tiles = it.columns - it.column0 > 128 ? NQ : 1; // query tiles with real rows
            const int my_tile = warp < 8 ? warp >> 2 : warp - 12;     // softmax warps and issuers
            // ---- query rows: one softmax thread each ----
            const int col = it.column0 + t; // of softmax threads
            const bool softmax = warp < 8 && my_tile < tiles;
            const bool real = softmax && col < it.columns;
            const int token = col / a.group;
            const int qhead = it.head * a.group + col % a.group;
            float factor = 0.0F;
            int see = 0;
            if (softmax)
            {
                const uint32_t to = ptx::smem_addr(q_tiles + my_tile * shape::Q_BYTES);
                const int row = t & 127;
                uint4 v[DIM / 8];
                float top = 0.0F;
                const uint4* from = reinterpret_cast<const uint4*>(
                    static_cast<const uint16_t*>(a.queries) +
                    (real ? static_cast<int64_t>(it.first_token + token) * a.query_stride + static_cast<int64_t>(qhead) * DIM
                          : 0));
                auto floats = [&](uint32_t w) {
                    if (a.dtype == BITSKNN_BF16)
                    {
                        return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000U));
                    }
                    return __half22float2(*reinterpret_cast<const __half2*>(&w));
                };
#pragma unroll
                for (int i = 0; i < DIM / 8; ++i)
                {
                    v[i] = real ? __ldg(from + i) : make_uint4(0U, 0U, 0U, 0U);
                }
#pragma unroll
                for (int i = 0; i < DIM / 8; ++i)
                {
                    const uint32_t w[4] = {v[i].x, v[i].y, v[i].z, v[i].w};
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                    {
                        const float2 f = floats(w[j]);
                        top = fabsf(f.x) < INFINITY ? fmaxf(top, fabsf(f.x)) : top;
                        top = fabsf(f.y) < INFINITY ? fmaxf(top, fabsf(f.y)) : top;
                    }
                }
                // the same scaling as pack_column: a power of two that puts the largest entry into
                // [2^14, 2^15); the sign of the scale goes with the query
                const int e = max(static_cast<int>(__float_as_uint(top) >> 23), 1) - 127;
                const int shift = top > 0.0F ? min(max(14 - e, -126), 126) : 0;
                const float up = a.scale < 0.0F ? -pow2_int(shift) : pow2_int(shift);
                factor = pow2_int(-shift) * fabsf(a.scale);
#pragma unroll
                for (int i = 0; i < DIM / 8; ++i)
                {
                    const uint32_t w[4] = {v[i].x, v[i].y, v[i].z, v[i].w};
                    uint32_t h[4];
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                    {
                        const float2 f = floats(w[j]);
                        h[j] = pack_half2(f.x * up, f.y * up);
                    }
                    st_shared16(to + tile_byte(row, i, 128), h[0], h[1], h[2], h[3]);
                }
                see = real ? visible_of(a.b, q, token) : 0;
                fence_async_proxy();
            }
            for (int d = t; d < DIM; d += TC_THREADS)
            {
                first_nan[d] = 0x7fffffff;
            }
            __syncthreads();

            if (warp < 8)
            {
                // ================= softmax =================
                const uint32_t lane_base = static_cast<uint32_t>((warp & 3) * 32) << 16;
                const uint32_t s_addr = tmem + lane_base + my_tile * ROWS;
                const uint32_t o_addr = tmem + lane_base + shape::O_COL + my_tile * DIM;
                const int tile_nearest = visible_of(a.b, q, min(it.column0 + my_tile * 128, last_col) / a.group);
                float m = -INFINITY;
                float l = 0.0F;
                for (int j = 0; j < count && softmax && fine; ++j)
                {
                    const uint32_t n = kv_tiles + j;
                    fine = warp_wait(&s_full[my_tile], s_tiles & 1U);
                    if (!fine)
                    {
                        break;
                    }
                    ++s_tiles;
                    tc::fence_after_sync();
                    const int pos = (first_tile + j) * ROWS;
                    const float4* const sc = scales + (n % TC_GROUPS) * GROUPS;
                    const bool cut = pos + ROWS > tile_nearest;
                    float top = -INFINITY;
#pragma unroll
                    for (int c = 0; c < ROWS; c += 32)
                    {
                        uint32_t s[32];
                        tc::tmem_ld_32x32(s_addr + c, s);
                        tc::tmem_ld_wait();
#pragma unroll
                        for (int g = 0; g < 2; ++g)
                        {
                            const float4 k = sc[c / 16 + g];
                            float most = -INFINITY;
                            if (!cut)
                            {
#pragma unroll
                                for (int i = 0; i < 16; ++i)
                                {
                                    most = fmaxf(most, __uint_as_float(s[g * 16 + i]));
                                }
                            }
                            else
                            {
#pragma unroll
                                for (int i = 0; i < 16; ++i)
                                {
                                    most = pos + c + g * 16 + i < see ? fmaxf(most, __uint_as_float(s[g * 16 + i])) : most;
                                }
                            }
                            // an absent page has lv = -inf
                            top = fmaxf(top, most == -INFINITY ? most : fmaf(most, factor * k.x, k.y));
                        }
                    }
                    if (__any_sync(FULL_MASK, top > m + WEIGHT_SLACK))
                    {
                        const float raised = fmaxf(top, m);
                        const float keep = m == -INFINITY ? 0.0F : exp2_fast(m - raised);
                        m = raised;
                        l *= keep;
                        if (j > 0)
                        {
                            // the product before this one has to be through with the sums
                            fine = warp_wait(&o_done[my_tile], s_tiles & 1U);
                            if (!fine)
                            {
                                break;
                            }
                            tc::fence_after_sync();
#pragma unroll 1
                            for (int c = 0; c < DIM; c += 32)
                            {
                                uint32_t o[32];
                                tc::tmem_ld_32x32(o_addr + c, o);
                                tc::tmem_ld_wait();
#pragma unroll
                                for (int i = 0; i < 32; ++i)
                                {
                                    o[i] = __float_as_uint(__uint_as_float(o[i]) * keep);
                                }
                                tmem_st_32(o_addr + c, o);
                            }
                        }
                    }
                    const float bias = WEIGHT_BIAS - (m == -INFINITY ? 0.0F : m);
#pragma unroll
                    for (int c = 0; c < ROWS; c += 32)
                    {
                        uint32_t s[32];
                        tc::tmem_ld_32x32(s_addr + c, s);
                        tc::tmem_ld_wait();
                        uint32_t p[16];
#pragma unroll
                        for (int g = 0; g < 2; ++g)
                        {
                            const float4 k = sc[c / 16 + g];
                            const float f = factor * k.x;
                            const float add = k.y + bias;
                            float part_sum = 0.0F;
#pragma unroll
                            for (int i = 0; i < 16; i += 2)
                            {
                                float x = exp2_fast(fmaf(__uint_as_float(s[g * 16 + i]), f, add));
                                float y = exp2_fast(fmaf(__uint_as_float(s[g * 16 + i + 1]), f, add));
                                if (cut)
                                {
                                    x = pos + c + g * 16 + i < see ? x : 0.0F;
                                    y = pos + c + g * 16 + i + 1 < see ? y : 0.0F;
                                }
                                part_sum += x + y;
                                p[g * 8 + i / 2] = pack_half2(x, y);
                            }
                            l = fmaf(part_sum, k.z, l);
                        }
                        // weights of columns c ... c + 31 take the place of scores c / 2 ..., read before
                        tmem_st_16(s_addr + c / 2, p);
                    }
                    tmem_st_wait();
                    tc::fence_before_sync();
                    tc::mbar_arrive(&p_full[my_tile]);
                }
                // ---- results of the rows ----
                if (softmax && fine && count > 0)
                {
                    fine = warp_wait(&o_done[my_tile], (s_tiles - 1) & 1U);
                    tc::fence_after_sync();
                }
                if (softmax && fine)
                {
                    const float inverse = l == 0.0F ? 0.0F : 1.0F / l;
                    const int64_t row_token = it.first_token + token;
                    const int64_t out_at = row_token * a.out_stride + static_cast<int64_t>(qhead) * DIM;
                    const bool aligned = ((reinterpret_cast<uintptr_t>(a.out) | static_cast<uintptr_t>(a.out_stride * 2)) & 15) == 0;
                    float* const part_row = a.part_o + (part * shape::COLS + t) * DIM;
#pragma unroll 1
                    for (int c = 0; c < DIM; c += 32)
                    {
                        uint32_t o[32];
                        __syncwarp();
                        if (count > 0)
                        {
                            tc::tmem_ld_32x32(o_addr + c, o);
                            tc::tmem_ld_wait();
                        }
                        if (!real)
                        {
                            continue;
                        }
                        float v[32];
#pragma unroll
                        for (int i = 0; i < 32; ++i)
                        {
                            v[i] = count > 0 ? __uint_as_float(o[i]) : 0.0F;
                            v[i] = first_nan[c + i] < see ? NAN : v[i];
                        }
                        if (!whole)
                        {
#pragma unroll
                            for (int i = 0; i < 32; i += 4)
                            {
                                *reinterpret_cast<float4*>(part_row + c + i) = make_float4(v[i], v[i + 1], v[i + 2], v[i + 3]);
                            }
                            continue;
                        }
                        // l = 0: nothing was seen; NaN in l makes the row NaN
                        auto result = [&](float x) { return l == 0.0F ? 0.0F : x * inverse; };
                        auto pair = [&](float x, float y) {
                            if (a.dtype == BITSKNN_BF16)
                            {
                                const __nv_bfloat162 b = __floats2bfloat162_rn(result(x), result(y));
                                return *reinterpret_cast<const uint32_t*>(&b);
                            }
                            return pack_half2(result(x), result(y));
                        };
                        uint16_t* const out = static_cast<uint16_t*>(a.out) + out_at + c;
#pragma unroll
                        for (int i = 0; i < 32; i += 8)
                        {
                            const uint4 w = make_uint4(pair(v[i], v[i + 1]), pair(v[i + 2], v[i + 3]),
                                                       pair(v[i + 4], v[i + 5]), pair(v[i + 6], v[i + 7]));
                            if (aligned)
                            {
                                *reinterpret_cast<uint4*>(out + i) = w;
                            }
                            else
                            {
                                const uint32_t x[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
                                for (int y = 0; y < 8; ++y)
                                {
                                    out[i + y] = static_cast<uint16_t>(x[y >> 1] >> (16 * (y & 1)));
                                }
                            }
                        }
                    }
                    if (real && !whole)
                    {
                        a.part_ml[part * shape::COLS + t] = make_float2(m, l);
                    }
                    if (real && whole && a.lse != nullptr)
                    {
                        a.lse[row_token * a.group * a.c.heads + qhead] =
                            l == 0.0F ? -INFINITY : (m - WEIGHT_BIAS + log2f(l)) * LN_2;
                    }
                    tc::fence_before_sync();
                }
            }
            else if (warp < 12)
            {
                // ================= converters =================
                const int me = t - 8 * 32;
                const int32_t* const table = a.b.table + it.request * a.b.table_ld;
                auto page_of = [&](int j) { // page of this lane's 16 positions of tile j
                    const int pos = (first_tile + j) * ROWS + lane * 16;
                    const int p = lane < GROUPS && j < count && pos < furthest ? table[pos >> a.c.page_shift] : -1;
                    return p < a.c.pages ? p : -1;
                };
                auto load = [&](uint4 (&r)[PIECES], const uint8_t* codes, int j, int page) {
#pragma unroll
                    for (int i = 0; i < PIECES; ++i)
                    {
                        const int e = me + i * CONVERTERS;
                        const int row = e / PARTS;
                        const int p = __shfl_sync(FULL_MASK, page, row >> 4);
                        const int pos = (first_tile + j) * ROWS + row;
                        r[i] = make_uint4(0U, 0U, 0U, 0U);
                        if (p >= 0 && pos < furthest)
                        {
                            r[i] = __ldg(reinterpret_cast<const uint4*>(
                                codes + p * a.c.page_stride +
                                ((static_cast<int64_t>(it.head) << a.c.page_shift) + (pos & rows_mask)) * DIM +
                                (e % PARTS) * 16));
                        }
                    }
                };
                auto store = [&](const uint4 (&r)[PIECES], unsigned char* tile) {
                    const uint32_t to = ptx::smem_addr(tile);
#pragma unroll
                    for (int i = 0; i < PIECES; ++i)
                    {
                        const int e = me + i * CONVERTERS;
                        const int row = e / PARTS;
                        const int chunk = (e % PARTS) * 2;
                        uint32_t h[8];
                        halves_of_codes(r[i].x, h[0], h[1]);
                        halves_of_codes(r[i].y, h[2], h[3]);
                        halves_of_codes(r[i].z, h[4], h[5]);
                        halves_of_codes(r[i].w, h[6], h[7]);
                        // lanes whose block of 64 halves is odd store their second half first: the eight
                        // lanes of a phase then reach eight different granules
                        const bool turn = ((chunk >> 3) & 1) != 0;
                        st_shared16(to + tile_byte(row, chunk + (turn ? 1 : 0), ROWS), turn ? h[4] : h[0], turn ? h[5] : h[1],
                                    turn ? h[6] : h[2], turn ? h[7] : h[3]);
                        st_shared16(to + tile_byte(row, chunk + (turn ? 0 : 1), ROWS), turn ? h[0] : h[4], turn ? h[1] : h[5],
                                    turn ? h[2] : h[6], turn ? h[3] : h[7]);
                    }
                };
                // A NaN code times a weight of zero would spoil the rows that do not see its position.  In
                // tiles that only some rows see wholly the NaN are taken out of the values and the first
                // position of each dimension that had one is kept: a row is NaN there if it sees it.
                auto clean = [&](uint4 (&r)[PIECES], int j) {
#pragma unroll
                    for (int i = 0; i < PIECES; ++i)
                    {
                        uint32_t* const w = reinterpret_cast<uint32_t*>(&r[i]);
#pragma unroll
                        for (int x = 0; x < 4; ++x)
                        {
                            const uint32_t hit = ((w[x] & 0x7f7f7f7fU) + 0x01010101U) & 0x80808080U;
                            if (hit != 0)
                            {
                                const int e = me + i * CONVERTERS;
                                for (int y = 0; y < 4; ++y)
                                {
                                    if ((hit >> (8 * y + 7)) & 1U)
                                    {
                                        atomicMin(&first_nan[(e % PARTS) * 16 + x * 4 + y],
                                                  (first_tile + j) * ROWS + e / PARTS);
                                        w[x] &= ~(0xffU << (8 * y));
                                    }
                                }
                            }
                        }
                    }
                };
                uint4 rk[PIECES];
                uint4 rv[PIECES];
                int page = page_of(0);
                int next = page_of(1);
                load(rk, a.c.keys, 0, page);
                load(rv, a.c.values, 0, page);
                for (int j = 0; j < count; ++j)
                {
                    const uint32_t n = kv_tiles + j;
                    const uint32_t stage = n & 1;
                    const uint32_t phase = (n >> 1) & 1U;
                    float ks = 0.0F;
                    float vs = 1.0F;
                    if (warp == 8 && page >= 0)
                    {
                        ks = a.c.key_scales[static_cast<int64_t>(page) * a.c.heads + it.head];
                        vs = a.c.value_scales[static_cast<int64_t>(page) * a.c.heads + it.head];
                    }
                    fine = warp_wait(&k_empty[stage], phase ^ 1U);
                    if (!fine)
                    {
                        break;
                    }
                    store(rk, k_tiles + stage * shape::KV_BYTES);
                    if (warp == 8 && lane < GROUPS)
                    {
                        vs = fminf(fmaxf(vs, pow2_int(E_MIN)), pow2_int(E_MAX));
                        scales[(n % TC_GROUPS) * GROUPS + lane] =
                            make_float4(ks, ks == 0.0F ? -INFINITY : log2_fast(vs), __fdividef(1.0F, vs), 0.0F);
                    }
                    fence_async_proxy();
                    tc::mbar_arrive(&k_full[stage]);
                    load(rk, a.c.keys, j + 1, next);
                    fine = warp_wait(&v_empty[stage], phase ^ 1U);
                    if (!fine)
                    {
                        break;
                    }
                    if (nearest < furthest && (first_tile + j + 1) * ROWS > nearest)
                    {
                        clean(rv, j);
                    }
                    store(rv, v_tiles + stage * shape::KV_BYTES);
                    fence_async_proxy();
                    tc::mbar_arrive(&v_full[stage]);
                    load(rv, a.c.values, j + 1, next);
                    page = next;
                    next = page_of(j + 2);
                }
            }
            else if (my_tile < NQ && lane == 0)
            {
                // ================= issue of the products =================
                constexpr uint32_t s_idesc = tc::instr_desc(0U, 128U, ROWS);
                constexpr uint32_t o_idesc = tc::instr_desc(0U, 128U, DIM) | (1U << 16); // second operand along its outputs
                const uint32_t s_addr = tmem + my_tile * ROWS;
                const uint32_t o_addr = tmem + shape::O_COL + my_tile * DIM;
                const uint64_t q_desc = tc::smem_desc_sw128(q_tiles + my_tile * shape::Q_BYTES);
                for (int j = 0; j < count; ++j)
                {
                    const uint32_t n = kv_tiles + j;
                    const uint32_t stage = n & 1;
                    const uint32_t phase = (n >> 1) & 1U;
                    fine = ptx::mbar_wait_bounded_spin(&k_full[stage], phase);
                    // the weights that lie over the scores have to be read before
                    if (fine && my_tile < tiles && j > 0)
                    {
                        fine = ptx::mbar_wait_bounded_spin(&o_done[my_tile], (s_tiles - 1) & 1U);
                    }
                    if (!fine)
                    {
                        break;
                    }
                    if (my_tile >= tiles) // no rows in this query tile: give the stages back
                    {
                        tc::mbar_arrive(&k_empty[stage]);
                        fine = ptx::mbar_wait_bounded_spin(&v_full[stage], phase);
                        if (!fine)
                        {
                            break;
                        }
                        tc::mbar_arrive(&v_empty[stage]);
                        continue;
                    }
                    tc::fence_after_sync();
                    const uint64_t k_desc = tc::smem_desc_sw128(k_tiles + stage * shape::KV_BYTES);
#pragma unroll
                    for (int k = 0; k < DIM / 16; ++k)
                    {
                        tc::mma<true>(s_addr, q_desc + (k >> 2) * (128 * 128 >> 4) + (k & 3) * 2,
                                      k_desc + (k >> 2) * (ROWS * 128 >> 4) + (k & 3) * 2, s_idesc, k != 0);
                    }
                    tc::mbar_arrive(&s_full[my_tile]);
                    tc::mma_commit(&s_full[my_tile]);
                    tc::mma_commit(&k_empty[stage]);
                    fine = ptx::mbar_wait_bounded_spin(&v_full[stage], phase) &&
                           ptx::mbar_wait_bounded_spin(&p_full[my_tile], s_tiles & 1U);
                    if (!fine)
                    {
                        break;
                    }
                    ++s_tiles;
                    tc::fence_after_sync();
                    const uint64_t v_desc = values_desc(v_tiles + stage * shape::KV_BYTES, ROWS * 128);
#pragma unroll
                    for (int k = 0; k < ROWS / 16; ++k)
                    {
                        mma_ts(o_addr, s_addr + k * 8, v_desc + k * (16 * 128 >> 4), o_idesc, j != 0 || k != 0);
                    }
                    tc::mbar_arrive(&o_done[my_tile]);
                    tc::mma_commit(&o_done[my_tile]);
                    tc::mma_commit(&v_empty[stage]);
                }
            }
            kv_tiles += count;
            if (at == it.begin && !whole && t == 0)
            {
                a.joins[blockIdx.x] = make_int4(it.first_token, it.head, it.column0, it.columns);
                a.join_end[blockIdx.x] = static_cast<int>(((it.end * blocks) - 1) / total);
            }
            // all of the block leaves together when a wait has expired
            if (__syncthreads_or(fine ? 0 : 1) != 0)
            {
                if (!fine)
                {
                    atomicOr(status, DEVICE_STATUS_TIMEOUT);
                }
                break;
            }
            tc::fence_after_sync();
            at = seg_end;
            if (at >= share_end)
            {
                break;
            }
            it.begin = it.end;
            it.column0 += shape::COLS;
            if (it.column0 >= it.columns)
            {
                it.column0 = 0;
                if (++it.head == a.c.heads)
                {
                    it.head = 0;
                    do
                    {
                        ++it.request; // requests without tokens have no units; `at` < total, so one follows
                        q = request_of(a.b, it.request);
                    } while (q.count == 0);
                    it.first_token = q.first;
                    it.columns = q.count * a.group;
                }
            }
            it.end = it.begin + units_of_block<shape>(a, q, it.column0);
        }
    }
    tc::fence_before_sync();
    __syncthreads();
    if (warp == 0)
    {
        tc::tmem_dealloc(tmem, shape::TMEM_COLS);
    }
}

template <int DIM>
int launch_tc(attend_args a, void* workspace, size_t workspace_bytes, cudaStream_t stream)
{
    using shape = tc_shape<DIM>;
    const int blocks = device_sm_count();
    const int rc = place_parts<DIM, shape::COLS>(a, blocks, workspace, workspace_bytes);
    if (rc != BITSKNN_OK)
    {
        return rc;
    }
    int* status = device_status_word();
    if (status == nullptr)
    {
        return fail(BITSKNN_ERR_CUDA, "CUDA error. cannot resolve the device status word");
    }
    static cache::device_set prepared;
    if (!prepared.contains_current())
    {
        BITSKNN_CUDA_TRY(
            cudaFuncSetAttribute(cache_attend_tc_kernel<DIM>, cudaFuncAttributeMaxDynamicSharedMemorySize, shape::BYTES));
        prepared.add_current();
    }
    {
        kernel_scope scope("cache_attend_kernel", stream);
        cache_attend_tc_kernel<DIM><<<blocks, TC_THREADS, shape::BYTES, stream>>>(a, status);
    }
    BITSKNN_CUDA_TRY(cudaGetLastError());
    return launch_join<DIM, shape::COLS>(a, blocks, stream);
}

} // namespace

size_t attend_tc_workspace_bytes(int dim)
{
    size_t bytes = 0;
    dispatch_cache_dim(dim, [&](auto d) {
        constexpr int DIM = decltype(d)::value;
        bytes = parts_bytes<DIM, tc_shape<DIM>::COLS>(device_sm_count());
        return BITSKNN_OK;
    });
    return bytes;
}

int launch_attend_tc(int dim, const cache::attend_args& a, void* workspace, size_t workspace_bytes, cudaStream_t stream)
{
    return dispatch_cache_dim(
        dim, [&](auto d) { return launch_tc<decltype(d)::value>(a, workspace, workspace_bytes, stream); });
}

} // namespace bitsknn
