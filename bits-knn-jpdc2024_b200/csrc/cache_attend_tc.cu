// cache_attend for many query columns per request and head (prompts, chunks of prompts): both
// products on the fifth-generation tensor cores, scores and sums in tensor memory.
#include <algorithm>

#include "cache_attend.cuh"
#include "tc.cuh"

namespace bitsknn
{

namespace
{

constexpr int TC_THREADS = 16 * 32;
constexpr int CONVERTERS = 128;
constexpr int RING = 8;             // scale slots (tiles) and first-NaN slots (items): see cache_attend_tc_kernel
constexpr int BARRIERS = 32;        // of a pass over the share
// Registers of a thread after the split of the 512 x 128 the block is launched with: two warpgroups of
// softmax, one of converters, one of issuers: 256 * 168 + 128 * 112 + 128 * 56 = 64512 of 65536.
constexpr int SOFTMAX_REGISTERS = 168;
constexpr int CONVERT_REGISTERS = 112;
constexpr int ISSUE_REGISTERS = 56;

// One block: NQ tiles of 128 query rows against tiles of 64 positions.  Tensor memory (512 columns)
// holds two score tiles per query tile, so that the next scores are computed while a softmax runs, and
// the sums; rows of 192 and 256 numbers leave room for one query tile only.
template <int DIM>
struct tc_shape
{
    static constexpr int NQ = DIM <= 128 ? 2 : 1;
    static constexpr int COLS = 128 * NQ;
    static constexpr int ROWS = 64;
    // an item's beginning and end, in tiles (rows of 128: 4 375 us, 6 370, 8 367, 10 365; other rows not measured)
    static constexpr int COST = 10;
    static constexpr int BLK = (DIM + 63) / 64;  // 128-byte blocks of 64 halves per row
    static constexpr int Q_BYTES = BLK * 128 * 128;
    static constexpr int KV_BYTES = BLK * ROWS * 128;
    static constexpr int STAGES = DIM <= 128 ? 4 : DIM <= 192 ? 3 : 2; // of keys, and of values
    static constexpr int GROUPS = ROWS / 16;
    static constexpr int O_COL = NQ * 2 * ROWS;  // tensor memory: two score tiles per query tile, then the sums
    static constexpr int USED_COLS = O_COL + NQ * DIM;
    static constexpr int TMEM_COLS = USED_COLS <= 256 ? 256 : 512;
    static constexpr int NANS = DIM + 4; // words of a first-NaN slot: the dimensions, their largest, the first position
    static constexpr int TAIL = RING * GROUPS * 16 + RING * NANS * 4 + 2 * BARRIERS * 8; // scales, first NaN, barriers
    static constexpr int BYTES = NQ * Q_BYTES + 2 * STAGES * KV_BYTES + TAIL + 1024;
    static_assert(USED_COLS <= 512, "tensor memory");
    static_assert(BYTES <= 227 * 1024, "shared memory");
    static_assert(RING >= STAGES + 2, "scale slots");
};

// D[tmem] (+)= A[smem] * B[smem] and D[tmem] (+)= A[tmem] * B[smem], halves, FP32 sums; issued by one thread.
// Descriptors come as their low words (start address, leading offset) and the high word they all share.
template <bool ACCUMULATE>
__device__ __forceinline__ void mma_ss(uint32_t d_tmem, uint32_t a_lo, uint32_t b_lo, uint32_t hi, uint32_t idesc)
{
    asm volatile("{\n"
                 ".reg .pred p;\n"
                 ".reg .b64 da, db;\n"
                 "setp.ne.b32 p, %5, 0;\n"
                 "mov.b64 da, {%1, %3};\n"
                 "mov.b64 db, {%2, %3};\n"
                 "tcgen05.mma.cta_group::1.kind::f16 [%0], da, db, %4, p;\n"
                 "}\n" ::"r"(d_tmem),
                 "r"(a_lo), "r"(b_lo), "r"(hi), "r"(idesc), "n"(ACCUMULATE ? 1 : 0)
                 : "memory");
}

__device__ __forceinline__ void mma_ts(uint32_t d_tmem, uint32_t a_tmem, uint32_t b_lo, uint32_t hi, uint32_t idesc,
                                       bool accumulate)
{
    asm volatile("{\n"
                 ".reg .pred p;\n"
                 ".reg .b64 db;\n"
                 "setp.ne.b32 p, %5, 0;\n"
                 "mov.b64 db, {%2, %3};\n"
                 "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], db, %4, p;\n"
                 "}\n" ::"r"(d_tmem),
                 "r"(a_tmem), "r"(b_lo), "r"(hi), "r"(idesc), "r"(accumulate ? 1U : 0U)
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

__device__ __forceinline__ void tmem_st_16(uint32_t taddr, const uint32_t (&v)[16])
{
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
                 "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(taddr),
                 "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]),
                 "r"(v[9]), "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15])
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

__device__ __forceinline__ uint4 ld_shared16(uint32_t addr)
{
    uint4 v;
    asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
                 : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
                 : "r"(addr)
                 : "memory");
    return v;
}

__device__ __forceinline__ void fence_async_proxy() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

// Waits for this thread's loads from tensor memory.  The registers pass through the wait, so that nothing
// that uses them can be moved in front of it.
__device__ __forceinline__ void tmem_ld_wait(uint32_t (&v)[32])
{
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(v[0]), "+r"(v[1]), "+r"(v[2]), "+r"(v[3]), "+r"(v[4]), "+r"(v[5]), "+r"(v[6]), "+r"(v[7]),
                 "+r"(v[8]), "+r"(v[9]), "+r"(v[10]), "+r"(v[11]), "+r"(v[12]), "+r"(v[13]), "+r"(v[14]), "+r"(v[15]),
                 "+r"(v[16]), "+r"(v[17]), "+r"(v[18]), "+r"(v[19]), "+r"(v[20]), "+r"(v[21]), "+r"(v[22]), "+r"(v[23]),
                 "+r"(v[24]), "+r"(v[25]), "+r"(v[26]), "+r"(v[27]), "+r"(v[28]), "+r"(v[29]), "+r"(v[30]), "+r"(v[31])
                 :
                 : "memory");
}

__device__ __forceinline__ void tmem_ld_wait(uint32_t (&v)[16])
{
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(v[0]), "+r"(v[1]), "+r"(v[2]), "+r"(v[3]), "+r"(v[4]), "+r"(v[5]), "+r"(v[6]), "+r"(v[7]),
                   "+r"(v[8]), "+r"(v[9]), "+r"(v[10]), "+r"(v[11]), "+r"(v[12]), "+r"(v[13]), "+r"(v[14]), "+r"(v[15])
                 :
                 : "memory");
}

// Two FP32 numbers in a register pair.
__device__ __forceinline__ uint64_t pair_of(float x, float y)
{
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(x), "f"(y));
    return r;
}

__device__ __forceinline__ float2 floats_of_pair(uint64_t r)
{
    float2 f;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(f.x), "=f"(f.y) : "l"(r));
    return f;
}

__device__ __forceinline__ uint64_t fma_pair(uint64_t a, uint64_t b, uint64_t c)
{
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}

__device__ __forceinline__ uint64_t add_pair(uint64_t a, uint64_t b)
{
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}

// Largest logit of a row of 64 scores, 16 scores to a scale; with CUT only columns below `limit` count.
template <bool CUT>
__device__ __forceinline__ float row_top(const uint32_t (&s)[2][32], const float4* scales, float factor, int limit)
{
    float top = -INFINITY;
#pragma unroll
    for (int g = 0; g < 4; ++g)
    {
        const float4 k = scales[g];
        float v[16];
#pragma unroll
        for (int i = 0; i < 16; ++i)
        {
            v[i] = __uint_as_float(s[g / 2][g % 2 * 16 + i]);
            if constexpr (CUT)
            {
                v[i] = g * 16 + i < limit ? v[i] : -INFINITY;
            }
        }
        float a = fmaxf(fmaxf(v[0], v[1]), v[2]);
        float b = fmaxf(fmaxf(v[3], v[4]), v[5]);
        a = fmaxf(fmaxf(a, v[6]), v[7]);
        b = fmaxf(fmaxf(b, v[8]), v[9]);
        a = fmaxf(fmaxf(a, v[10]), v[11]);
        b = fmaxf(fmaxf(b, v[12]), v[13]);
        const float most = fmaxf(fmaxf(fmaxf(a, b), v[14]), v[15]);
        // an absent page has the logarithm -inf
        top = fmaxf(top, most == -INFINITY ? most : fmaf(most, factor * k.x, k.y));
    }
    return top;
}

// Scores to weights 2^(logit + bias) as halves.  x: sum of the weights, y: sum of the weights over their
// value scales (the row's share of the denominator).
template <bool CUT>
__device__ __forceinline__ float2 row_weights(const uint32_t (&s)[2][32], uint32_t (&p)[32], const float4* scales,
                                              float factor, float bias, int limit)
{
    float2 sums = make_float2(0.0F, 0.0F);
#pragma unroll
    for (int g = 0; g < 4; ++g)
    {
        const float4 k = scales[g];
        const float f = factor * k.x;
        const float add = k.y + bias;
        const uint64_t ff = pair_of(f, f);
        const uint64_t aa = pair_of(add, add);
        uint64_t sum = 0;
#pragma unroll
        for (int i = 0; i < 16; i += 2)
        {
            float2 x = floats_of_pair(fma_pair(pair_of(__uint_as_float(s[g / 2][g % 2 * 16 + i]),
                                                       __uint_as_float(s[g / 2][g % 2 * 16 + i + 1])),
                                               ff, aa));
            x.x = exp2_fast(x.x);
            x.y = exp2_fast(x.y);
            if constexpr (CUT)
            {
                x.x = g * 16 + i < limit ? x.x : 0.0F;
                x.y = g * 16 + i + 1 < limit ? x.y : 0.0F;
            }
            sum = i == 0 ? pair_of(x.x, x.y) : add_pair(sum, pair_of(x.x, x.y));
            p[g * 8 + i / 2] = pack_half2(x.x, x.y);
        }
        const float2 total = floats_of_pair(sum);
        sums.x += total.x + total.y;
        sums.y = fmaf(total.x + total.y, k.z, sums.y);
    }
    return sums;
}

template <int N>
__device__ __forceinline__ void more_registers()
{
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N));
}

template <int N>
__device__ __forceinline__ void fewer_registers()
{
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N));
}

// One arrival for a whole warp, after all its threads have come here (arrivals of single threads on one
// barrier are served one after the other: 512 of them per tile took a third of the shared-memory pipe).
__device__ __forceinline__ void warp_arrive(uint64_t* bar)
{
    __syncwarp();
    if ((threadIdx.x & 31) == 0)
    {
        tc::mbar_arrive(bar);
    }
}

// A wait of a whole warp: its threads go on, or give up, together.
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity)
{
    return __all_sync(FULL_MASK, ptx::mbar_wait_bounded_spin(bar, parity)) != 0;
}

// A row's step of the softmax over a tile whose weights become the sums of two BF16 numbers each: of every 16 words, 8
// for the upper numbers of 16 positions and 8 for the lower ones, over their scores.  Rare, so it is kept out of the way
// of the others: group after group, maxima first.  Returns the reference point and the sum, which is -inf if the wait for
// the product before (`done`, if there is one) ran out.
template <int DIM>
__device__ __forceinline__ float2 far_tile(uint32_t s_addr, uint32_t o_addr, const float4* scales, float factor, int limit,
                                           float m, float l, uint64_t* done, uint32_t phase)
{
    uint32_t s[16];
    float top = -INFINITY;
#pragma unroll 1
    for (int g = 0; g < 4; ++g)
    {
        tc::tmem_ld_32x16(s_addr + g * 16, s);
        tmem_ld_wait(s);
        float most = -INFINITY;
#pragma unroll
        for (int i = 0; i < 16; ++i)
        {
            most = g * 16 + i < limit ? fmaxf(most, __uint_as_float(s[i])) : most;
        }
        top = fmaxf(top, most == -INFINITY ? most : fmaf(most, factor * scales[g].x, scales[g].y));
    }
    if (__any_sync(FULL_MASK, m == -INFINITY || top > m + WEIGHT_SLACK))
    {
        top = fmaxf(top, m);
        const float keep = m == -INFINITY ? 0.0F : exp2_fast(m - top);
        m = top;
        l *= keep;
        if (done != nullptr)
        {
            if (!warp_wait(done, phase))
            {
                return make_float2(m, -INFINITY);
            }
            tc::fence_after_sync();
#pragma unroll 1
            for (int c = 0; c < DIM; c += 16)
            {
                tc::tmem_ld_32x16(o_addr + c, s);
                tmem_ld_wait(s);
#pragma unroll
                for (int i = 0; i < 16; ++i)
                {
                    s[i] = __float_as_uint(__uint_as_float(s[i]) * keep);
                }
                tmem_st_16(o_addr + c, s);
            }
        }
    }
    const float bias = WEIGHT_BIAS - (m == -INFINITY ? 0.0F : m);
#pragma unroll 1
    for (int g = 0; g < 4; ++g)
    {
        tc::tmem_ld_32x16(s_addr + g * 16, s);
        tmem_ld_wait(s);
        const float4 k = scales[g];
        float sum = 0.0F;
        uint32_t p[16];
#pragma unroll
        for (int i = 0; i < 16; i += 2)
        {
            float x = exp2_fast(fmaf(__uint_as_float(s[i]), factor * k.x, k.y + bias));
            float y = exp2_fast(fmaf(__uint_as_float(s[i + 1]), factor * k.x, k.y + bias));
            x = g * 16 + i < limit ? x : 0.0F;
            y = g * 16 + i + 1 < limit ? y : 0.0F;
            sum += x + y;
            split_bf16(x, y, p[i / 2], p[8 + i / 2]);
        }
        l = fmaf(sum, k.z, l);
        tmem_st_16(s_addr + g * 16, p);
    }
    return make_float2(m, l);
}

// First position of a dimension with a NaN among the tiles that only some rows of item number `items`
// see wholly, as an offset (below 1024: a block's columns span at most 256 tokens) from the first
// of these tiles.  The key grows with the item and towards earlier positions, so a maximum keeps
// the first one and what an item before has left needs no clearing.
__device__ __forceinline__ uint32_t nan_key(uint32_t items, int offset) { return (items + 1) << 10 | (1023U - offset); }

// A block's walk over its share: every role goes through the same items for itself.
template <class SHAPE>
struct walk
{
    item it;
    request q;
    int64_t at;        // of the axis
    int64_t share_end;

    __device__ __forceinline__ int64_t segment_end() const { return min(it.end, share_end); }
    __device__ __forceinline__ int first_tile() const { return max(static_cast<int>(at - it.begin) - SHAPE::COST, 0); }
    // tiles of the share; none if it ends within the units of the item's beginning
    __device__ __forceinline__ int count() const
    {
        return max(static_cast<int>(segment_end() - it.begin) - SHAPE::COST, 0) - first_tile();
    }
    __device__ __forceinline__ int query_tiles() const { return it.columns - it.column0 > 128 ? SHAPE::NQ : 1; }
    __device__ __forceinline__ int last_column() const { return min(it.column0 + SHAPE::COLS, it.columns) - 1; }
    __device__ __forceinline__ bool next(const attend_args& a)
    {
        at = segment_end();
        if (at >= share_end)
        {
            return false;
        }
        it.begin = it.end;
        it.column0 += SHAPE::COLS;
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
        it.end = it.begin + units_of_block<SHAPE>(a, q, it.column0);
        return true;
    }
};

// Barriers and buffers of a block in shared memory.
struct tc_state
{
    unsigned char* q_tiles;
    unsigned char* k_tiles;
    unsigned char* v_tiles;
    float4* scales;     // [RING][GROUPS]: key scale, log2 of the value scale, its inverse, 1 if the tile is BF16 (else 0)
    uint32_t* first_nan; // [RING][NANS]: nan_key; behind them the first position of the item's share that is there
    uint64_t* k_full;   // [STAGES]
    uint64_t* k_empty;
    uint64_t* v_full;
    uint64_t* v_empty;
    uint64_t* s_full;   // [query tile][score tile]
    uint64_t* p_full;   // [query tile][score tile]
    uint64_t* o_done;   // [query tile][score tile]
    uint64_t* q_full;   // [query tile]
    uint64_t* row_done; // [query tile]: the item's rows are written
};

// Where things lie in shared memory; the barriers of either pass over a share (cache_attend_tc_kernel).
template <int DIM>
__device__ __forceinline__ tc_state state_of(unsigned char* raw, int pass)
{
    using shape = tc_shape<DIM>;
    tc_state st;
    st.q_tiles = raw + ((1024U - (ptx::smem_addr(raw) & 1023U)) & 1023U);
    st.k_tiles = st.q_tiles + shape::NQ * shape::Q_BYTES;
    st.v_tiles = st.k_tiles + shape::STAGES * shape::KV_BYTES;
    st.scales = reinterpret_cast<float4*>(st.v_tiles + shape::STAGES * shape::KV_BYTES);
    st.first_nan = reinterpret_cast<uint32_t*>(st.scales + RING * shape::GROUPS);
    st.k_full = reinterpret_cast<uint64_t*>(st.first_nan + RING * shape::NANS) + pass * BARRIERS;
    st.k_empty = st.k_full + 4;
    st.v_full = st.k_full + 8;
    st.v_empty = st.k_full + 12;
    st.s_full = st.k_full + 16;
    st.p_full = st.k_full + 20;
    st.o_done = st.k_full + 24;
    st.q_full = st.k_full + 28;
    st.row_done = st.k_full + 30;
    return st;
}

// ================= softmax: one thread per query row =================
template <int DIM, bool FAR>
__device__ __forceinline__ bool softmax_role(const attend_args& a, const tc_state& st, walk<tc_shape<DIM>> w,
                                             uint32_t tmem)
{
    using shape = tc_shape<DIM>;
    const int t = threadIdx.x;
    const int lane = t & 31;
    const int my_tile = t >> 7;
    const uint32_t lane_base = static_cast<uint32_t>(((t >> 5) & 3) * 32) << 16;
    const uint32_t s_base = tmem + lane_base + my_tile * 2 * shape::ROWS;
    const uint32_t o_addr = tmem + lane_base + shape::O_COL + my_tile * DIM;
    uint32_t kv_tiles = 0; // tiles of the block so far
    uint32_t s_tiles = 0;  // and those of this query tile
    uint32_t items = 0;    // items with tiles
    do
    {
        const int count = w.count();
        if (my_tile < w.query_tiles())
        {
            const int col = w.it.column0 + t;
            const bool real = col < w.it.columns;
            const int token = col / a.group;
            const int qhead = w.it.head * a.group + col % a.group;
            const int64_t row_token = w.it.first_token + token;
            const int see = real ? visible_of(a.b, w.q, token) : 0;
            float factor = 0.0F;
            if (count > 0)
            {
                // The products that read the query tile's rows before are done: o_done was waited for.  A warp
                // packs its 32 rows together, G lanes to a row, so that its loads and stores are whole lines, and
                // in short loops, because what runs once an item comes from beyond the instruction cache (8400
                // clocks an item; a row to a thread 13500, all 16 steps unrolled 19000).
                constexpr int CHUNKS = DIM / 8; // of 16 bytes in a row
                constexpr int G = CHUNKS <= 4 ? 4 : CHUNKS <= 8 ? 8 : CHUNKS <= 16 ? 16 : 32;
                constexpr int TOGETHER = 32 / G;  // rows of a load
                const uint32_t to = ptx::smem_addr(st.q_tiles + my_tile * shape::Q_BYTES);
                const int chunk = lane % G;
                const int64_t mine = real ? row_token * a.query_stride + static_cast<int64_t>(qhead) * DIM : -1;
                auto floats = [&](uint32_t x) {
                    if (a.dtype == BITSKNN_BF16)
                    {
                        return make_float2(__uint_as_float(x << 16), __uint_as_float(x & 0xffff0000U));
                    }
                    return __half22float2(*reinterpret_cast<const __half2*>(&x));
                };
                // The same scaling as pack_column: a power of two that puts the largest entry into [2^14, 2^15).
                auto shift_of = [&](uint32_t most) {
                    const float top = floats(most).x;
                    const int e = max(static_cast<int>(__float_as_uint(top) >> 23), 1) - 127;
                    return top > 0.0F ? min(max(14 - e, -126), 126) : 0;
                };
                const uint32_t infinite = a.dtype == BITSKNN_BF16 ? 0x7f80U : 0x7c00U;
                // all rows are asked for at once, as they are, and converted where they come to lie
#pragma unroll 4
                for (int b = 0; b < G; ++b)
                {
                    const int64_t from = __shfl_sync(FULL_MASK, mine, b * TOGETHER + lane / G);
                    if (chunk < CHUNKS)
                    {
                        const int row = (t & 96) + b * TOGETHER + lane / G;
                        copy16(to + tile_byte(row, chunk, 128),
                               static_cast<const uint16_t*>(a.queries) + max(from, static_cast<int64_t>(0)) + chunk * 8,
                               from >= 0 ? 16U : 0U);
                    }
                }
                copy_commit();
                uint32_t row_most = 0; // of this thread's row
                copy_wait<0>();
                constexpr int BATCH = 4; // rows a lane has under way: the steps of one wait for each other
#pragma unroll 1
                for (int b = 0; b < G; b += BATCH)
                {
                    uint32_t x[BATCH][4];
                    uint32_t most[BATCH];
                    uint32_t at[BATCH];
                    uint32_t top = 0;
#pragma unroll
                    for (int i = 0; i < BATCH; ++i)
                    {
                        at[i] = to + tile_byte((t & 96) + (b + i) * TOGETHER + lane / G, chunk, 128);
                        const uint4 v = chunk < CHUNKS ? ld_shared16(at[i]) : make_uint4(0U, 0U, 0U, 0U);
                        x[i][0] = v.x;
                        x[i][1] = v.y;
                        x[i][2] = v.z;
                        x[i][3] = v.w;
                        // both 16-bit types order like their bits once the sign is gone
                        const uint32_t m = __vmaxu2(__vmaxu2(v.x & 0x7fff7fffU, v.y & 0x7fff7fffU),
                                                    __vmaxu2(v.z & 0x7fff7fffU, v.w & 0x7fff7fffU));
                        most[i] = max(m & 0xffffU, m >> 16);
                        top = max(top, most[i]);
                    }
                    if (__any_sync(FULL_MASK, top >= infinite))
                    {
                        // infinities and NaN set no scale: the largest finite entry
#pragma unroll
                        for (int i = 0; i < BATCH; ++i)
                        {
                            most[i] = 0;
#pragma unroll
                            for (int y = 0; y < 8; ++y)
                            {
                                const uint32_t one = x[i][y >> 1] >> (16 * (y & 1)) & 0x7fffU;
                                most[i] = one < infinite ? max(most[i], one) : most[i];
                            }
                        }
                    }
#pragma unroll
                    for (int o = 1; o < G; o <<= 1)
                    {
#pragma unroll
                        for (int i = 0; i < BATCH; ++i)
                        {
                            most[i] = max(most[i], __shfl_xor_sync(FULL_MASK, most[i], o));
                        }
                    }
#pragma unroll
                    for (int i = 0; i < BATCH; ++i)
                    {
                        const uint32_t got = __shfl_sync(FULL_MASK, most[i], lane % TOGETHER * G);
                        row_most = lane / TOGETHER == b + i ? got : row_most;
                        // the sign of the scale goes with the query
                        const float up = a.scale < 0.0F ? -pow2_int(shift_of(most[i])) : pow2_int(shift_of(most[i]));
                        uint32_t h[4];
#pragma unroll
                        for (int y = 0; y < 4; ++y)
                        {
                            const float2 f = floats(x[i][y]);
                            h[y] = pack_half2(f.x * up, f.y * up);
                        }
                        if (chunk < CHUNKS)
                        {
                            st_shared16(at[i], h[0], h[1], h[2], h[3]);
                        }
                    }
                }
                factor = pow2_int(-shift_of(row_most)) * fabsf(a.scale);
                fence_async_proxy();
                warp_arrive(&st.q_full[my_tile]);
            }
            const int nearest = visible_of(a.b, w.q, min(w.it.column0 + my_tile * 128, w.last_column()) / a.group);
            float m = -INFINITY;
            float l = 0.0F;
            for (int j = 0; j < count; ++j, ++s_tiles)
            {
                const uint32_t buffer = s_tiles & 1;
                const uint32_t phase = (s_tiles >> 1) & 1U;
                const uint32_t s_addr = s_base + buffer * shape::ROWS;
                if (!warp_wait(&st.s_full[my_tile * 2 + buffer], phase))
                {
                    return false;
                }
                tc::fence_after_sync();
                const int pos = (w.first_tile() + j) * shape::ROWS;
                const float4* const scales = st.scales + ((kv_tiles + j) % RING) * shape::GROUPS;
                const bool cut = pos + shape::ROWS > nearest;
                uint32_t s[2][32];
                tc::tmem_ld_32x32(s_addr, s[0]);
                tc::tmem_ld_32x32(s_addr + 32, s[1]);
                tmem_ld_wait(s[0]);
                tmem_ld_wait(s[1]);
                bool far = false;
                if constexpr (FAR)
                {
                    far = __any_sync(FULL_MASK, scales->w != 0.0F) != 0;
                }
                if (far)
                {
                    const float2 now = far_tile<DIM>(s_addr, o_addr, scales, factor, cut ? see - pos : shape::ROWS, m, l,
                                                     j > 0 ? &st.o_done[my_tile * 2 + ((s_tiles - 1) & 1)] : nullptr,
                                                     ((s_tiles - 1) >> 1) & 1U);
                    m = now.x;
                    l = now.y;
                    if (l == -INFINITY)
                    {
                        return false;
                    }
                }
                else
                {
                    // Weights against the reference point as it stands.  They are positive, so a sum of at most
                    // 2^15 says that none is too large for a half and nothing has to be compared; only when the
                    // sum is larger (or NaN, or there is no reference point yet) is the maximum looked for.
                    uint32_t p[32];
                    auto weigh = [&] {
                        const float bias = WEIGHT_BIAS - (m == -INFINITY ? 0.0F : m);
                        return cut ? row_weights<true>(s, p, scales, factor, bias, see - pos)
                                   : row_weights<false>(s, p, scales, factor, bias, 0);
                    };
                    float2 sums = weigh();
                    if (__any_sync(FULL_MASK, m == -INFINITY || !(sums.x <= 32768.0F)))
                    {
                        tc::tmem_ld_32x32(s_addr, s[0]);
                        tc::tmem_ld_32x32(s_addr + 32, s[1]);
                        tmem_ld_wait(s[0]);
                        tmem_ld_wait(s[1]);
                        const float raised = fmaxf(
                            cut ? row_top<true>(s, scales, factor, see - pos) : row_top<false>(s, scales, factor, 0), m);
                        const float keep = m == -INFINITY ? 0.0F : exp2_fast(m - raised);
                        m = raised;
                        l *= keep;
                        if (j > 0)
                        {
                            // the product before this one has to be through with the sums
                            if (!warp_wait(&st.o_done[my_tile * 2 + ((s_tiles - 1) & 1)], ((s_tiles - 1) >> 1) & 1U))
                            {
                                return false;
                            }
                            tc::fence_after_sync();
#pragma unroll 1
                            for (int c = 0; c < DIM; c += 32)
                            {
                                uint32_t o[32];
                                tc::tmem_ld_32x32(o_addr + c, o);
                                tmem_ld_wait(o);
#pragma unroll
                                for (int i = 0; i < 32; ++i)
                                {
                                    o[i] = __float_as_uint(__uint_as_float(o[i]) * keep);
                                }
                                tmem_st_32(o_addr + c, o);
                            }
                        }
                        sums = weigh();
                    }
                    l += sums.y;
                    tmem_st_32(s_addr, p); // over the scores
                }
                tmem_st_wait();
                tc::fence_before_sync();
                warp_arrive(&st.p_full[my_tile * 2 + buffer]);
            }
            // ---- the row's result ----
            if (count > 0 && !warp_wait(&st.o_done[my_tile * 2 + ((s_tiles - 1) & 1)], ((s_tiles - 1) >> 1) & 1U))
            {
                return false;
            }
            tc::fence_after_sync();
            const bool whole = w.at == w.it.begin && w.segment_end() == w.it.end;
            const int64_t part = 2 * static_cast<int64_t>(blockIdx.x) + (w.at == w.it.begin ? 1 : 0);
            const uint32_t* const first_nan = st.first_nan + (items % RING) * shape::NANS;
            // a key of this item at least as large stands for a position below `see`
            const int cut_base = visible_of(a.b, w.q, w.it.column0 / a.group) / shape::ROWS * shape::ROWS;
            const uint32_t seen_nan = see > cut_base ? nan_key(items, see - 1 - cut_base) : 0xffffffffU;
            const bool nan_here = count > 0 && first_nan[DIM] >= seen_nan;
            if (count > 0 && see <= static_cast<int>(first_nan[DIM + 1]))
            {
                // Nothing there was seen.  Positions of absent pages have weight 2^-inf, but for a query that is not finite
                // their scores, 0 times infinity, are NaN.
                m = -INFINITY;
                l = 0.0F;
            }
            const float inverse = l == 0.0F ? 1.0F : 1.0F / l; // l = 0: nothing was seen; a NaN makes the row NaN
            const bool aligned =
                ((reinterpret_cast<uintptr_t>(a.out) | static_cast<uintptr_t>(a.out_stride * 2)) & 15) == 0;
            // Through shared memory, 32 numbers of each of the warp's rows at a time, so that its stores are
            // whole lines too (6500 clocks an item; a row to a thread 9200).  The rows' queries have been read.
            const uint32_t rows_at = ptx::smem_addr(st.q_tiles + my_tile * shape::Q_BYTES + (t & 96) * 128);
            const int64_t mine = real ? row_token * a.out_stride + static_cast<int64_t>(qhead) * DIM : -1;
            float* const part_rows = a.part_o + (part * shape::COLS + (t & ~31)) * DIM;
            auto granule = [&](int row, int g) { return rows_at + row * 128 + ((g ^ (row & 7)) << 4); };
#pragma unroll 1
            for (int c = 0; c < DIM; c += 32)
            {
                uint32_t o[32];
                __syncwarp();
                if (count > 0)
                {
                    tc::tmem_ld_32x32(o_addr + c, o);
                    tmem_ld_wait(o);
                }
                if (l == 0.0F || nan_here)
                {
#pragma unroll
                    for (int i = 0; i < 32; ++i)
                    {
                        o[i] = l != 0.0F ? (first_nan[c + i] >= seen_nan ? 0x7fc00000U : o[i]) : 0U;
                    }
                }
                if (!whole)
                {
#pragma unroll
                    for (int g = 0; g < 8; ++g)
                    {
                        st_shared16(granule(lane, g), o[g * 4], o[g * 4 + 1], o[g * 4 + 2], o[g * 4 + 3]);
                    }
                    __syncwarp();
#pragma unroll
                    for (int i = 0; i < 8; ++i)
                    {
                        const int row = i * 4 + (lane >> 3);
                        const uint4 x = ld_shared16(granule(row, lane & 7));
                        if (__shfl_sync(FULL_MASK, real ? 1 : 0, row) != 0)
                        {
                            *reinterpret_cast<uint4*>(part_rows + row * DIM + c + (lane & 7) * 4) = x;
                        }
                    }
                    continue;
                }
                auto result = [&](uint32_t x) { return __uint_as_float(x) * inverse; };
                auto pair = [&](uint32_t x, uint32_t y) {
                    if (a.dtype == BITSKNN_BF16)
                    {
                        const __nv_bfloat162 b = __floats2bfloat162_rn(result(x), result(y));
                        return *reinterpret_cast<const uint32_t*>(&b);
                    }
                    return pack_half2(result(x), result(y));
                };
#pragma unroll
                for (int g = 0; g < 4; ++g)
                {
                    st_shared16(granule(lane, g), pair(o[g * 8], o[g * 8 + 1]), pair(o[g * 8 + 2], o[g * 8 + 3]),
                                pair(o[g * 8 + 4], o[g * 8 + 5]), pair(o[g * 8 + 6], o[g * 8 + 7]));
                }
                __syncwarp();
#pragma unroll
                for (int i = 0; i < 4; ++i)
                {
                    const int row = i * 8 + (lane >> 2);
                    const uint4 v = ld_shared16(granule(row, lane & 3));
                    const int64_t to = __shfl_sync(FULL_MASK, mine, row);
                    if (to < 0)
                    {
                        continue;
                    }
                    uint16_t* const out = static_cast<uint16_t*>(a.out) + to + c + (lane & 3) * 8;
                    if (aligned)
                    {
                        *reinterpret_cast<uint4*>(out) = v;
                    }
                    else
                    {
                        const uint32_t x[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
                        for (int y = 0; y < 8; ++y)
                        {
                            out[y] = static_cast<uint16_t>(x[y >> 1] >> (16 * (y & 1)));
                        }
                    }
                }
            }
            __syncwarp();
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
            if (count > 0)
            {
                warp_arrive(&st.row_done[my_tile]);
            }
        }
        kv_tiles += count;
        items += count > 0 ? 1 : 0;
    } while (w.next(a));
    return true;
}

// Scales of a page (-1: absent) and head; a key scale of 0 stands for an absent page.
__device__ __forceinline__ void scales_of(const view& c, int page, int head, float& ks, float& vs)
{
    const bool there = page >= 0;
    ks = there ? c.key_scales[static_cast<int64_t>(page) * c.heads + head] : 0.0F;
    vs = there ? c.value_scales[static_cast<int64_t>(page) * c.heads + head] : 1.0F;
}

// A thread's codes of a tile, PIECES of 16, to halves or to BF16 numbers in shared memory (both exact).
template <bool AS_BF16, int ROWS, int BLK, int PIECES>
__device__ __forceinline__ void store_codes(const uint4 (&r)[PIECES], unsigned char* tile, uint32_t first_half,
                                            uint32_t second_half)
{
    const uint32_t to = ptx::smem_addr(tile);
#pragma unroll
    for (int i = 0; i < PIECES; ++i)
    {
        const uint4 x = r[i];
        const uint32_t at_row = to + i % BLK * ROWS * 128 + i / BLK * 32 * 128;
        uint32_t h[8];
        halves_of_codes(x.x, h[0], h[1]);
        halves_of_codes(x.y, h[2], h[3]);
        halves_of_codes(x.z, h[4], h[5]);
        halves_of_codes(x.w, h[6], h[7]);
        if constexpr (AS_BF16)
        {
#pragma unroll
            for (int y = 0; y < 8; ++y)
            {
                h[y] = bf16_of_halves(h[y]);
            }
        }
        st_shared16(at_row + first_half, h[0], h[1], h[2], h[3]);
        st_shared16(at_row + second_half, h[4], h[5], h[6], h[7]);
    }
}

// ================= converters: codes from the cache to halves in shared memory =================
template <int DIM, bool FAR>
__device__ __forceinline__ bool convert_role(const attend_args& a, const tc_state& st, walk<tc_shape<DIM>> w, int* verdict)
{
    using shape = tc_shape<DIM>;
    constexpr int BLK = shape::BLK;
    constexpr int ROWS = shape::ROWS;
    constexpr int SLABS = ROWS / 32;     // rows a thread serves: one of every 32
    constexpr int PIECES = SLABS * BLK;  // 16-code pieces of a thread and tile
    constexpr int AHEAD = 32 / shape::GROUPS; // tiles whose pages a warp looks up at a time, one lane per 16 positions
    const int lane = threadIdx.x & 31;
    const int warp = (threadIdx.x >> 5) - 8;
    const int rows_mask = (1 << a.c.page_shift) - 1;
    // A warp's load covers 8 rows of 4 pieces (64 codes): its 8 rows lie within one page, and its
    // two 16-byte stores per piece reach eight different granules in every phase (two rows, four even or
    // four odd chunks, moved apart by the swizzle).
    const int piece = lane & 3;
    const int row0 = warp * 8 + (lane >> 2);
    const uint32_t first_half = tile_byte(row0, piece * 2, ROWS);
    const uint32_t second_half = tile_byte(row0, piece * 2 + 1, ROWS);
    uint32_t n = 0; // tiles so far
    uint32_t items = 0;
    uint32_t far_apart = 0;
    do
    {
        const int count = w.count();
        if (count == 0)
        {
            continue;
        }
        const int first_tile = w.first_tile();
        const int furthest = visible_of(a.b, w.q, w.last_column() / a.group);
        const int nearest = visible_of(a.b, w.q, w.it.column0 / a.group);
        const int32_t* const table = a.b.table + w.it.request * a.b.table_ld;
        uint32_t* const first_nan = st.first_nan + (items % RING) * shape::NANS;
        const int cut_base = nearest / ROWS * ROWS;
        // AHEAD tiles from tile j on, this lane's 16 positions: their page, and where their first row lies
        auto pages_from = [&](int j) {
            const int pos = (first_tile + j) * ROWS + lane * 16;
            const int p = j < count && pos < furthest ? table[pos >> a.c.page_shift] : -1;
            return p < a.c.pages ? p : -1;
        };
        auto offset_of = [&](int page, int j) -> int64_t {
            const int pos = (first_tile + j) * ROWS + lane * 16;
            return page < 0 ? -1
                            : page * a.c.page_stride +
                                  ((static_cast<int64_t>(w.it.head) << a.c.page_shift) + (pos & rows_mask)) * DIM;
        };
        const int page_first = pages_from(0);
        int page_next = pages_from(AHEAD);
        int64_t offset_now = offset_of(page_first, 0);
        float ks_now = 0.0F, vs_now = 1.0F, ks_next = 0.0F, vs_next = 1.0F;
        const bool scaling = FAR || warp == 0; // this warp looks the scales up
        if (scaling)
        {
            scales_of(a.c, page_first, w.it.head, ks_now, vs_now);
        }
        // Groups of 16 positions of the tiles looked up whose value scale is far below the largest one up to them
        // (cache_attend.cuh); the values of their tiles become BF16.  The scales are first touched here, long after
        // their loads (touched when they are loaded, 172 -> 182 us for rows of 256 numbers).
        uint32_t vs_least = 0; // the largest one over 2^SCALE_SPREAD; positive floats order like their bits
        uint32_t far_groups = 0;
        auto compare_scales = [&] {
            vs_now = fminf(fmaxf(vs_now, pow2_int(E_MIN)), pow2_int(E_MAX));
            const uint32_t bits = __float_as_uint(vs_now);
            const uint32_t most = __reduce_max_sync(FULL_MASK, ks_now != 0.0F ? bits : 0U);
            vs_least = max(vs_least, most - min(most, SCALE_SPREAD << 23));
            far_groups = __ballot_sync(FULL_MASK, ks_now != 0.0F && bits < vs_least);
            far_apart |= far_groups;
        };
        // the first position that is there, kept by the warp that looks the scales up in any case
        int first_there = 0x7fffffff;
        auto look_for_first = [&](int j) {
            const uint32_t there = __ballot_sync(FULL_MASK, ks_now != 0.0F);
            first_there = there != 0 ? (first_tile + j) * ROWS + (__ffs(there) - 1) * 16 : first_there;
            if (lane == 0)
            {
                first_nan[DIM + 1] = static_cast<uint32_t>(first_there);
            }
        };
        int base = 0; // first tile of offset_now
        const int whole_tiles = furthest / ROWS - first_tile; // tiles before this one have all their rows
        int64_t from[SLABS]; // of the tile loaded next, this thread's pieces; -1: absent
        bool all_there = false; // all pieces of the warp's tile exist
        auto locate = [&](int j) {
            if (j - base == AHEAD)
            {
                base = j;
                offset_now = offset_of(page_next, j);
                ks_now = ks_next;
                vs_now = vs_next;
                if (scaling)
                {
                    compare_scales();
                }
                if (warp == 0 && first_there == 0x7fffffff)
                {
                    look_for_first(j);
                }
                page_next = pages_from(j + AHEAD);
            }
            bool absent = false;
#pragma unroll
            for (int i = 0; i < SLABS; ++i)
            {
                const int64_t o =
                    __shfl_sync(FULL_MASK, offset_now, (j - base) * shape::GROUPS + i * 2 + (warp >> 1));
                const bool there = o >= 0 && j < count &&
                                   (j < whole_tiles || (first_tile + j) * ROWS + i * 32 + row0 < furthest);
                from[i] = there ? o + (row0 & 15) * DIM + piece * 16 : -1;
                absent |= !there;
            }
            all_there = DIM % 64 == 0 && !__any_sync(FULL_MASK, absent);
        };
        auto load = [&](uint4 (&r)[PIECES], const uint8_t* codes) {
            if (all_there)
            {
#pragma unroll
                for (int i = 0; i < SLABS; ++i)
                {
#pragma unroll
                    for (int b = 0; b < BLK; ++b)
                    {
                        r[i * BLK + b] = __ldg(reinterpret_cast<const uint4*>(codes + from[i] + b * 64));
                    }
                }
                return;
            }
#pragma unroll
            for (int i = 0; i < SLABS; ++i)
            {
#pragma unroll
                for (int b = 0; b < BLK; ++b)
                {
                    r[i * BLK + b] = make_uint4(0U, 0U, 0U, 0U);
                    if (from[i] >= 0 && (DIM % 64 == 0 || b * 64 + piece * 16 < DIM))
                    {
                        r[i * BLK + b] = __ldg(reinterpret_cast<const uint4*>(codes + from[i] + b * 64));
                    }
                }
            }
        };
        // A NaN code times a weight of zero would spoil the rows that do not see its position.  In
        // tiles that only some rows see wholly the NaN are taken out of the values and the first position
        // of each dimension that had one is kept: a row is NaN there if it sees it.
        auto clean = [&](uint4 (&r)[PIECES], int j) {
#pragma unroll
            for (int i = 0; i < PIECES; ++i)
            {
                uint32_t x[4] = {r[i].x, r[i].y, r[i].z, r[i].w};
#pragma unroll
                for (int y = 0; y < 4; ++y)
                {
                    const uint32_t hit = ((x[y] & 0x7f7f7f7fU) + 0x01010101U) & 0x80808080U;
                    if (hit != 0)
                    {
                        const int d = i % BLK * 64 + piece * 16 + y * 4;
                        const int pos = (first_tile + j) * ROWS + i / BLK * 32 + row0;
#pragma unroll 1
                        for (int z = 0; z < 4; ++z)
                        {
                            if ((hit >> (8 * z + 7)) & 1U)
                            {
                                atomicMax(&first_nan[d + z], nan_key(items, pos - cut_base));
                                atomicMax(&first_nan[DIM], nan_key(items, pos - cut_base));
                                x[y] &= ~(0xffU << (8 * z));
                            }
                        }
                    }
                }
                r[i] = make_uint4(x[0], x[1], x[2], x[3]);
            }
        };
        uint4 rk[PIECES];
        uint4 rv[PIECES];
        locate(0);
        load(rk, a.c.keys);
        load(rv, a.c.values);
        if (scaling) // behind the first loads, which would wait for the scales otherwise
        {
            compare_scales();
        }
        if (warp == 0)
        {
            look_for_first(0);
        }
        for (int j = 0; j < count; ++j, ++n)
        {
            const uint32_t stage = n % shape::STAGES;
            const uint32_t phase = (n / shape::STAGES) & 1U;
            if (!warp_wait(&st.k_empty[stage], phase ^ 1U))
            {
                return false;
            }
            store_codes<false, ROWS, BLK>(rk, st.k_tiles + stage * shape::KV_BYTES, first_half, second_half);
            const bool as_bf16 = FAR && (far_groups >> ((j - base) * shape::GROUPS) & ((1U << shape::GROUPS) - 1)) != 0;
            if (warp == 0 && lane / shape::GROUPS == j - base)
            {
                st.scales[(n % RING) * shape::GROUPS + lane % shape::GROUPS] =
                    make_float4(ks_now, ks_now == 0.0F ? -INFINITY : log2_fast(vs_now), __fdividef(1.0F, vs_now),
                                as_bf16 ? 1.0F : 0.0F);
            }
            if (scaling && j - base == AHEAD / 2)
            {
                scales_of(a.c, page_next, w.it.head, ks_next, vs_next);
            }
            fence_async_proxy();
            warp_arrive(&st.k_full[stage]);
            locate(j + 1);
            load(rk, a.c.keys);
            if (!warp_wait(&st.v_empty[stage], phase ^ 1U))
            {
                return false;
            }
            if (nearest < furthest && (first_tile + j + 1) * ROWS > nearest)
            {
                clean(rv, j);
            }
            if (as_bf16)
            {
                store_codes<true, ROWS, BLK>(rv, st.v_tiles + stage * shape::KV_BYTES, first_half, second_half);
            }
            else
            {
                store_codes<false, ROWS, BLK>(rv, st.v_tiles + stage * shape::KV_BYTES, first_half, second_half);
            }
            fence_async_proxy();
            warp_arrive(&st.v_full[stage]);
            load(rv, a.c.values);
        }
        ++items;
    } while (w.next(a));
    // the commits of the last tiles arrive before the block gives its shared memory back
    for (uint32_t i = n < shape::STAGES ? 0 : n - shape::STAGES; i < n; ++i)
    {
        const uint32_t phase = (i / shape::STAGES) & 1U;
        if (!warp_wait(&st.k_empty[i % shape::STAGES], phase) || !warp_wait(&st.v_empty[i % shape::STAGES], phase))
        {
            return false;
        }
    }
    if (!FAR && warp == 0 && lane == 0 && far_apart != 0)
    {
        verdict[0] = 1;
    }
    return true;
}

// ================= issue of the products of a query tile: one thread for each of the two =================
// A thread is held while its products run, and what it does between them -- waits, commits, address
// arithmetic -- adds up to as much again; so the scores and the sums of either query tile have a thread of
// their own, which only meet at barriers.
template <int DIM>
__device__ __forceinline__ bool scores_role(const attend_args& a, const tc_state& st, walk<tc_shape<DIM>> w,
                                            uint32_t tmem, int my_tile)
{
    using shape = tc_shape<DIM>;
    constexpr uint32_t idesc = tc::instr_desc(0U, 128U, shape::ROWS);
    const uint32_t s_base = tmem + my_tile * 2 * shape::ROWS;
    const uint64_t q_desc = tc::smem_desc_sw128(st.q_tiles + my_tile * shape::Q_BYTES);
    const uint32_t q_lo = static_cast<uint32_t>(q_desc);
    const uint32_t hi = static_cast<uint32_t>(q_desc >> 32);
    const uint32_t k_lo0 = static_cast<uint32_t>(tc::smem_desc_sw128(st.k_tiles));
    uint32_t stage = 0;
    uint32_t phase = 0;
    uint32_t s = 0; // score tiles of this query tile so far
    uint32_t q_items = 0;
    do
    {
        const int count = w.count();
        const bool active = my_tile < w.query_tiles(); // else no rows: give the stages back
        if (active && count > 0)
        {
            if (!ptx::mbar_wait_bounded_spin(&st.q_full[my_tile], q_items & 1U))
            {
                return false;
            }
            ++q_items;
        }
        for (int j = 0; j < count; ++j)
        {
            if (!ptx::mbar_wait_bounded_spin(&st.k_full[stage], phase))
            {
                return false;
            }
            if (active)
            {
                // the product before last has read the weights that lie over this score tile
                if (s >= 2 && !ptx::mbar_wait_bounded_spin(&st.o_done[my_tile * 2 + (s & 1)], ((s >> 1) - 1) & 1U))
                {
                    return false;
                }
                tc::fence_after_sync();
                const uint32_t s_addr = s_base + (s & 1) * shape::ROWS;
                const uint32_t k_lo = k_lo0 + stage * (shape::KV_BYTES >> 4);
                mma_ss<false>(s_addr, q_lo, k_lo, hi, idesc);
#pragma unroll
                for (int k = 1; k < DIM / 16; ++k)
                {
                    mma_ss<true>(s_addr, q_lo + (k >> 2) * (128 * 128 >> 4) + (k & 3) * 2,
                                 k_lo + (k >> 2) * (shape::ROWS * 128 >> 4) + (k & 3) * 2, hi, idesc);
                }
                tc::mma_commit(&st.s_full[my_tile * 2 + (s & 1)]);
                tc::mma_commit(&st.k_empty[stage]);
                tc::mbar_arrive(&st.s_full[my_tile * 2 + (s & 1)]);
                ++s;
            }
            else
            {
                tc::mbar_arrive(&st.k_empty[stage]);
            }
            if (++stage == shape::STAGES)
            {
                stage = 0;
                phase ^= 1U;
            }
        }
    } while (w.next(a));
    return true;
}

template <int DIM, bool FAR>
__device__ __forceinline__ bool sums_role(const attend_args& a, const tc_state& st, walk<tc_shape<DIM>> w,
                                          uint32_t tmem, int my_tile)
{
    using shape = tc_shape<DIM>;
    constexpr uint32_t along = 1U << 16; // second operand along its outputs
    constexpr uint32_t idesc = tc::instr_desc(0U, 128U, DIM) | along;
    constexpr uint32_t idesc_bf16 = tc::instr_desc(1U, 128U, DIM) | along;
    const uint32_t s_base = tmem + my_tile * 2 * shape::ROWS;
    const uint32_t o_addr = tmem + shape::O_COL + my_tile * DIM;
    const uint64_t v_desc = values_desc(st.v_tiles, shape::ROWS * 128);
    const uint32_t hi = static_cast<uint32_t>(v_desc >> 32);
    uint32_t stage = 0;
    uint32_t phase = 0;
    uint32_t n = 0; // tiles so far
    uint32_t s = 0; // products of this query tile so far
    uint32_t written = 0; // items of this query tile whose rows have to be written
    do
    {
        const int count = w.count();
        const bool active = my_tile < w.query_tiles();
        // Items without rows here could go by while the softmax still reads the first NaN of the last one that
        // had some, and take its slot.
        if (!active && count > 0 && written > 0 &&
            !ptx::mbar_wait_bounded_spin(&st.row_done[my_tile], (written - 1) & 1U))
        {
            return false;
        }
        written += active && count > 0 ? 1 : 0;
        for (int j = 0; j < count; ++j, ++n)
        {
            if (!ptx::mbar_wait_bounded_spin(&st.v_full[stage], phase))
            {
                return false;
            }
            if (active)
            {
                const bool as_bf16 = FAR && st.scales[(n % RING) * shape::GROUPS].w != 0.0F;
                if (!ptx::mbar_wait_bounded_spin(&st.p_full[my_tile * 2 + (s & 1)], (s >> 1) & 1U))
                {
                    return false;
                }
                tc::fence_after_sync();
                const uint32_t p_addr = s_base + (s & 1) * shape::ROWS;
                const uint32_t v_lo = static_cast<uint32_t>(v_desc) + stage * (shape::KV_BYTES >> 4);
                // the weights of 16 positions: 8 words of halves, or 8 of their upper parts and 8 of the lower ones
                const uint32_t words = as_bf16 ? 16U : 8U;
                const uint32_t form = as_bf16 ? idesc_bf16 : idesc;
#pragma unroll
                for (int k = 0; k < shape::ROWS / 16; ++k)
                {
                    mma_ts(o_addr, p_addr + k * words, v_lo + k * (16 * 128 >> 4), hi, form, j != 0 || k != 0);
                }
                if (as_bf16)
                {
#pragma unroll
                    for (int k = 0; k < shape::ROWS / 16; ++k)
                    {
                        mma_ts(o_addr, p_addr + 8 + k * words, v_lo + k * (16 * 128 >> 4), hi, form, true);
                    }
                }
                tc::mma_commit(&st.o_done[my_tile * 2 + (s & 1)]);
                tc::mma_commit(&st.v_empty[stage]);
                tc::mbar_arrive(&st.o_done[my_tile * 2 + (s & 1)]);
                ++s;
            }
            else
            {
                tc::mbar_arrive(&st.v_empty[stage]);
            }
            if (++stage == shape::STAGES)
            {
                stage = 0;
                phase ^= 1U;
            }
        }
    } while (w.next(a));
    return true;
}

// Where the roles meet after their way over the share: whether all of them have to go over it again.
template <class SHAPE>
__device__ __forceinline__ bool once_more(uint32_t* first_nan, int* verdict, bool fine)
{
    if (!fine)
    {
        verdict[1] = 1;
    }
    __syncwarp();
    tc::fence_before_sync();
    asm volatile("bar.sync 1, %0;" ::"n"(TC_THREADS) : "memory");
    if (verdict[0] == 0 || verdict[1] != 0)
    {
        return false;
    }
    for (int d = threadIdx.x; d < RING * SHAPE::NANS; d += TC_THREADS)
    {
        first_nan[d] = 0U;
    }
    asm volatile("bar.sync 1, %0;" ::"n"(TC_THREADS) : "memory");
    tc::fence_after_sync();
    return true;
}

// Warps 0-3 and 4-7: softmax of query tile 0 and 1, one thread per row.  Warps 8-11: converters, codes
// to halves.  Warps 12 ... 15: one thread each issues the scores (12, 13) or the sums (14, 15) of a query tile.
//
// A tile of 64 positions goes round like this.  The converters bring 16 codes per thread and load from
// the cache a tile ahead, turn them into halves and store them in the swizzled layout the tensor cores
// read (STAGES tiles each of keys and values).  S = Q K^T lands in one of a query tile's two score tiles
// in tensor memory; a softmax thread takes its row, and writes the weights as halves over the scores;
// O += P V takes them from there as its first operand, and the values as they lie, contiguous
// along the outputs.  The next scores are computed while the softmax runs.  O stays in tensor memory;
// it is touched only when a row's reference point has to move by more than 2^8 (rarely after the first
// tile).  The roles meet at mbarriers alone, also from one item to the next, so the next item's first
// tiles are converted while the last one is being written.
//   Rings: the converters are at most STAGES tiles ahead of the scores, and scores need the product
// before last, whose weights their softmax has written: a slot of RING >= STAGES + 2 is read before it is
// written again.  The first-NaN slots go by items of at least one tile, so the same holds for them while both
// query tiles have rows; an item without rows for one of them waits until that one's last rows are written.
//   Score tiles, weights and products have a barrier per score tile: a role may be a tile ahead of the one
// that waits, and a wait by parity can tell a phase from the next one only while it is at most one phase
// of the same barrier away.
//   Barriers that one role completes and another reads the fruits of (scales, NaN) carry an arrival of
// the issuing thread beside the products' commit: what it has seen of the converters is then seen too.
//
// Value scales far apart (cache_attend.cuh) take weights and values as BF16 numbers.  What that needs in addition cost
// the loops of the usual case 14 ... 100 us of 376 wherever it stood in them, taken or not.  So the converters only note
// that the share has such scales, and then the block goes over it again with roles of their own (FAR) and barriers of
// their own (1000 us; a kernel of its own for this pass cost each call 5 us).
//
// What bounds it: per 256 rows x 64 positions the exponentials need 1024 clocks (16 per clock and SM), the
// products about 1500 (the 8 + 4 of one query tile hold their threads for 516 + 234 clocks when it is alone in
// its block), their operands and the converters' stores about 1300 of shared-memory time; a tile takes some
// 2180, because the steps of one tile depend on one another and a warp's 64 weights alone take 1170 with the
// other warp of its scheduler doing the same; an item's beginning and end take 17000.  3 requests of 1500 ...
// 8000 cached and 700 ... 2100 new positions, 8 heads of 4 queries of 128: 309 GFLOP in 376 us = 0.82 PFLOP/s,
// 0.49 of the measured dense rate.  Steps on the way: tiles of 128 positions with one score tile 620 us; two
// score tiles of 64 511; packed arithmetic and offsets per 16 rows 444; a thread for each kind of product 405;
// rows packed and written in whole lines 365 (376 by now, with inputs that take turns).  Tried and slower: two
// threads per row (520), other register splits (403 ... 417), the weights' code shared by both paths in a loop (580:
// the scores then live on across it), one product of 128 positions for both score tiles of a query tile (502: the
// 516 clocks serve twice as much, but the softmax then waits 900 of them every time).
// Spills (-Xptxas -v: 0.5 KB stored, 0.8 KB loaded per thread) lie in the softmax: without it 16 bytes are left.
template <int DIM>
__global__ void __launch_bounds__(TC_THREADS, 1) cache_attend_tc_kernel(const attend_args a, int* status)
{
    using shape = tc_shape<DIM>;
    constexpr int WARPS_HERE = TC_THREADS / 32;
    extern __shared__ unsigned char raw[];
    __shared__ int64_t s_words[WARPS_HERE];
    __shared__ int s_found;
    __shared__ uint32_t s_tmem;
    __shared__ walk<shape> s_walk;
    __shared__ int s_verdict[2];
    const int t = threadIdx.x;
    const int warp = t >> 5;
    const int lane = t & 31;
    const tc_state st = state_of<DIM>(raw, 0);

    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    if (t == 0)
    {
        a.joins[blockIdx.x] = make_int4(0, 0, 0, 0);
        s_verdict[0] = s_verdict[1] = 0;
        for (int pass = 0; pass < 2; ++pass)
        {
            const tc_state set = state_of<DIM>(raw, pass);
            for (int i = 0; i < shape::STAGES; ++i)
            {
                ptx::mbar_init(&set.k_full[i], CONVERTERS / 32);
                ptx::mbar_init(&set.v_full[i], CONVERTERS / 32);
                ptx::mbar_init(&set.k_empty[i], shape::NQ);
                ptx::mbar_init(&set.v_empty[i], shape::NQ);
            }
            for (int i = 0; i < 4; ++i)
            {
                ptx::mbar_init(&set.s_full[i], 2);
                ptx::mbar_init(&set.p_full[i], 4);
                ptx::mbar_init(&set.o_done[i], 2);
            }
            for (int i = 0; i < 2; ++i)
            {
                ptx::mbar_init(&set.q_full[i], 4);
                ptx::mbar_init(&set.row_done[i], 4);
            }
        }
        ptx::mbar_init_fence();
    }
    for (int d = t; d < RING * shape::NANS; d += TC_THREADS)
    {
        st.first_nan[d] = 0U;
    }
    if (warp == 0)
    {
        tc::tmem_alloc(&s_tmem, shape::TMEM_COLS);
    }
    tc::fence_before_sync();
    __syncthreads();
    tc::fence_after_sync();
    const uint32_t tmem = s_tmem;

    int64_t sum = 0;
    for (int r = t; r < a.b.requests; r += TC_THREADS)
    {
        sum += units_of_head<shape>(a, request_of(a.b, r)) * a.c.heads;
    }
    const int64_t total = block_sum<WARPS_HERE>(sum, s_words);
    const int64_t blocks = min(static_cast<int64_t>(gridDim.x), total);
    if (blockIdx.x < blocks)
    {
        walk<shape> w{};
        w.at = blockIdx.x * total / blocks;
        w.share_end = (blockIdx.x + 1) * total / blocks;
        int64_t first = 0;
        w.it.request = find_request<shape, WARPS_HERE>(a, w.at, &first, s_words, &s_found);
        w.q = request_of(a.b, w.it.request);
        const int64_t per_head = units_of_head<shape>(a, w.q);
        w.it.head = static_cast<int>((w.at - first) / per_head);
        w.it.begin = first + w.it.head * per_head;
        w.it.first_token = w.q.first;
        w.it.columns = w.q.count * a.group;
        w.it.end = w.it.begin + units_of_block<shape>(a, w.q, 0);
        while (w.at >= w.it.end)
        {
            w.it.column0 += shape::COLS;
            w.it.begin = w.it.end;
            w.it.end += units_of_block<shape>(a, w.q, w.it.column0);
        }
        if (t == 0)
        {
            s_walk = w;
        }
        bool fine = true;
        if (warp < 8)
        {
            more_registers<SOFTMAX_REGISTERS>();
            const bool active = shape::NQ == 2 || warp < 4;
            if (active)
            {
                fine = softmax_role<DIM, false>(a, st, w, tmem);
            }
            if (once_more<shape>(st.first_nan, s_verdict, fine) && active)
            {
                fine = softmax_role<DIM, true>(a, state_of<DIM>(raw, 1), s_walk, tmem);
            }
        }
        else if (warp < 12)
        {
            fewer_registers<CONVERT_REGISTERS>();
            fine = convert_role<DIM, false>(a, st, w, s_verdict);
            if (once_more<shape>(st.first_nan, s_verdict, fine))
            {
                fine = convert_role<DIM, true>(a, state_of<DIM>(raw, 1), s_walk, s_verdict);
            }
        }
        else
        {
            fewer_registers<ISSUE_REGISTERS>();
            const int issuer = warp - 12; // 0, 1: scores of query tile 0, 1; 2, 3: sums
            const bool active = lane == 0 && (issuer & 1) < shape::NQ;
            if (active)
            {
                fine = issuer < 2 ? scores_role<DIM>(a, st, w, tmem, issuer & 1)
                                  : sums_role<DIM, false>(a, st, w, tmem, issuer & 1);
            }
            else if (warp == TC_THREADS / 32 - 1 && lane == 1)
            {
                // the item that begins here and ends in a later block, if there is one: the last of the share
                while (w.segment_end() < w.share_end)
                {
                    w.next(a);
                }
                if (w.at == w.it.begin && w.it.end > w.share_end)
                {
                    a.joins[blockIdx.x] = make_int4(w.it.first_token, w.it.head, w.it.column0, w.it.columns);
                    a.join_end[blockIdx.x] = static_cast<int>((w.it.end * blocks - 1) / total);
                }
            }
            if (once_more<shape>(st.first_nan, s_verdict, fine) && active)
            {
                const tc_state again = state_of<DIM>(raw, 1);
                fine = issuer < 2 ? scores_role<DIM>(a, again, s_walk, tmem, issuer & 1)
                                  : sums_role<DIM, true>(a, again, s_walk, tmem, issuer & 1);
            }
        }
        if (!fine)
        {
            atomicOr(status, DEVICE_STATUS_TIMEOUT);
        }
        __syncwarp();
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
