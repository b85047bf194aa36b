// cache_attend, cache_attend_selected: attention over a paged 8-bit cache, over all positions a token
// sees or over a list of them.
#include <algorithm>

#include "cache_attend.cuh"

namespace bitsknn
{

namespace
{

template <int DIM, int NB>
struct attend_smem
{
    static constexpr int COLS = 8 * NB;
    static constexpr int ROWS = TILE;
    // An item's beginning and end in tiles (ragged decode batch of 64 requests, 150 ... 24000 positions, rows of
    // 128: 141 us with 1, 131 with 3, 121 with 5 and with 8; other rows not measured).  Lists are all of one length;
    // there it only costs.
    static constexpr int COST = 6;
    static constexpr int LIST_COST = 1;
    static constexpr int SCALES = 2 * SUB * PITCH<DIM, true>; // offset of the scales in a stage
    static constexpr int STAGE = SCALES + 2 * SUB * 4;
    static constexpr int IMAGE = NB * 16 * DIM;
    static constexpr int SMALL = COLS * (4 + 4 + WARPS * 8 + 8); // undo, visible, (m, l) of warps and block
    // as many stages as three blocks per SM leave room for
    static constexpr int FIT = 18432 / STAGE;
    static constexpr int LEAST = NB > 3 ? NB : 3;
    static constexpr int STAGES = FIT < LEAST ? LEAST : FIT > 8 ? 8 : FIT;
    static constexpr int BYTES = IMAGE + SMALL + WARPS * STAGES * STAGE;
    static constexpr int BY_SMEM = 227 * 1024 / (BYTES + 1024);
    static constexpr int BY_REGS = NB * DIM <= 128 ? 4 : NB * DIM <= 256 ? 3 : 2;
    static constexpr int BLOCKS = BY_SMEM < BY_REGS ? BY_SMEM : BY_REGS; // per SM
    static_assert(BLOCKS >= 1, "shared memory");
    static_assert(WARPS * STAGES * STAGE >= WARPS * COLS * DIM * 4, "the stages hold the warps' sums at the end");
};

// ---- the kernel ------------------------------------------------------------------------------------
// Four warps, each streaming its own 16-position subtiles (position tile * 64 + warp * 16)
// through shared memory with asynchronous copies, without a block barrier in the loop: cached
// rows are the 16 rows of the matrix step, query columns its 8 columns, so eight query heads cost
// one conversion and one product, and scores come out with two positions of two columns per
// thread, which the 8 x 8 transposition turns into the operand of the second product.
//   scores  S^T = K Q^T   rows = positions  (operand: key codes as halves)
//   output  O^T = V^T P^T rows = dims       (operand: value codes, read transposed as pairs of
//                                            dims; the pairs are split when they become halves)
// The four warps' sums are joined in shared memory when an item ends, those of several blocks by
// cache_join_kernel, or, for few short items, those of a cluster's blocks through their shared memory.
//
// Bound by the bytes of the cache (HBM) while the columns are few.  One request with 250001 positions, 8 heads of 128
// (512 MB): 92 us = 5.6 TB/s, 0.85 of the measured copy rate, and 10 us for the join; 64 requests with 150 ... 24000
// positions (625 MB): 117 us, 0.82 and 7 us; 2048 listed positions of 32 requests (137 MB in gathers of 128 bytes):
// 41 us, 0.51 -- more copies in flight do not help there; whether single rows or the look-ups of entries and pages in
// front of them are the reason has not been told apart.
// Three stages and three blocks per SM (four stages: 97 us for the long request, two: 92).
template <int DIM, int NB, bool SELECTED, bool CLUSTER>
__global__ void __launch_bounds__(THREADS, attend_smem<DIM, NB>::BLOCKS) cache_attend_kernel(const attend_args a)
{
    using smem = attend_smem<DIM, NB>;
    constexpr int COLS = smem::COLS;
    constexpr int STAGES = smem::STAGES;
    extern __shared__ __align__(16) unsigned char shared[];
    __shared__ int64_t s_words[WARPS];
    __shared__ int s_found;
    uint32_t* const image = reinterpret_cast<uint32_t*>(shared);
    float* const undo = reinterpret_cast<float*>(shared + smem::IMAGE);
    int* const visible = reinterpret_cast<int*>(undo + COLS);
    float2* const warp_ml = reinterpret_cast<float2*>(visible + COLS);
    float2* const block_ml = warp_ml + WARPS * COLS; // of a cluster's block
    unsigned char* const stages = shared + smem::IMAGE + smem::SMALL;
    const int warp = threadIdx.x >> 5;
    const int lane = threadIdx.x & 31;
    unsigned char* const mine = stages + warp * STAGES * smem::STAGE;
    const int rows_mask = (1 << a.c.page_shift) - 1;
    const int c = (lane & 3) * 2;             // this thread's columns: c, c + 1 of every block of 8
    const int row_lo = row_order<DIM, true>(lane >> 2);  // its rows: row_lo, row_lo + 8

    // this block's share, and the item it begins in
    constexpr int COST = SELECTED ? smem::LIST_COST : smem::COST;
    const int list_units = SELECTED ? (a.k + TILE - 1) / TILE + COST : 0;
    const int list_blocks = SELECTED ? (a.group + COLS - 1) / COLS : 0;
    int64_t total;
    if constexpr (CLUSTER)
    {
        total = 0; // no shares
    }
    else if constexpr (SELECTED)
    {
        total = static_cast<int64_t>(a.b.tokens) * a.c.heads * list_blocks * list_units;
    }
    else
    {
        int64_t sum = 0;
        for (int r = threadIdx.x; r < a.b.requests; r += THREADS)
        {
            sum += units_of_head<smem>(a, request_of(a.b, r)) * a.c.heads;
        }
        total = block_sum<WARPS>(sum, s_words);
    }
    int64_t blocks = 0;
    int64_t at = 0;
    int64_t share_end = 0;
    item it{};
    if constexpr (CLUSTER)
    {
        // one token per request (or a list per token): the items are known without a look at the lengths
        const int column_blocks = (a.group + COLS - 1) / COLS;
        const int n = static_cast<int>(blockIdx.x) / a.cluster;
        it.column0 = n % column_blocks * COLS;
        it.head = n / column_blocks % a.c.heads;
        it.first_token = n / column_blocks / a.c.heads;
        it.request = it.first_token;
        it.columns = a.group;
        it.end = share_end = 1;
    }
    else
    {
        asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
        if (threadIdx.x == 0)
        {
            a.joins[blockIdx.x] = make_int4(0, 0, 0, 0);
        }
        blocks = min(static_cast<int64_t>(gridDim.x), total); // those that get a share at all
        if (blockIdx.x >= blocks)
        {
            return;
        }
        at = blockIdx.x * total / blocks;
        share_end = (blockIdx.x + 1) * total / blocks;
        if constexpr (SELECTED)
        {
            const int64_t n = at / list_units;
            it.begin = n * list_units;
            it.end = it.begin + list_units;
            it.column0 = static_cast<int>(n % list_blocks) * COLS;
            it.head = static_cast<int>(n / list_blocks % a.c.heads);
            it.first_token = static_cast<int>(n / list_blocks / a.c.heads);
            it.columns = a.group;
        }
        else
        {
            int64_t first = 0;
            it.request = find_request<smem, WARPS>(a, at, &first, s_words, &s_found);
            const request q = request_of(a.b, it.request);
            const int64_t per_head = units_of_head<smem>(a, q);
            it.head = static_cast<int>((at - first) / per_head);
            it.begin = first + it.head * per_head;
            it.first_token = q.first;
            it.columns = q.count * a.group;
            it.end = it.begin + units_of_block<smem>(a, q, 0);
            while (at >= it.end)
            {
                it.column0 += COLS;
                it.begin = it.end;
                it.end += units_of_block<smem>(a, q, it.column0);
            }
        }
    }

    while (true)
    {
        const int64_t seg_end = min(it.end, share_end);
        bool live = true;
        request q;
        if constexpr (SELECTED)
        {
            it.request = owner_of(a.b, it.first_token);
            live = it.request >= 0; // tokens behind the last request are not touched
        }
        if (live)
        {
            q = request_of(a.b, it.request);
            __syncthreads(); // the sums of the item before, which lie over the stages, have been read
            // columns of a block see ever more positions
            const int last = min(it.column0 + COLS, it.columns) - 1;
            const int furthest = visible_of(a.b, q, SELECTED ? it.first_token - q.first : last / a.group);
            const int nearest = SELECTED ? furthest : visible_of(a.b, q, it.column0 / a.group);
            const int32_t* const table = a.b.table + it.request * a.b.table_ld;
            const int32_t* list = nullptr;
            if constexpr (SELECTED)
            {
                list = a.idx + (static_cast<int64_t>(it.first_token) * a.c.heads + it.head) * a.ld_idx;
            }
            // tiles of the share; none if it ends within the units of the item's beginning
            int first_tile = max(static_cast<int>(at - it.begin) - COST, 0);
            int count = max(static_cast<int>(seg_end - it.begin) - COST, 0) - first_tile;
            if constexpr (CLUSTER)
            {
                const int tiles = ((SELECTED ? a.k : furthest) + TILE - 1) / TILE;
                const int rank = static_cast<int>(blockIdx.x) % a.cluster;
                first_tile = rank * tiles / a.cluster;
                count = (rank + 1) * tiles / a.cluster - first_tile;
            }
            const int row_end = SELECTED ? a.k : furthest; // rows behind it are zero
            auto row_of = [&](int j) { return (first_tile + j) * TILE + warp * SUB; };

            // ---- the stream ----
            constexpr int PARTS = DIM / 16;
            int slot_in = 0;
            int slot_out = 0;
            const uint32_t stage0 = ptx::smem_addr(mine);
            auto page_at = [&](int pos) {
                const int p = pos >= 0 ? table[pos >> a.c.page_shift] : -1;
                return p < a.c.pages ? p : -1;
            };
            // All positions: a subtile lies within one page, so its rows are contiguous and share their
            // scales; the page is looked up one subtile ahead of the copies.  (Pages of 32 subtiles looked up
            // at a time, one per lane, cost a ragged batch 7 us of 121: items end before it pays.)
            auto position = [&](int j) { return j < count && row_of(j) < furthest ? row_of(j) : -1; };
            // A list: the entries and pages of two subtiles at a time, one row per lane, entries two and
            // pages one such pair ahead.
            auto entry = [&](int j) {
                const int e = row_of(j + (lane >> 4)) + (lane & 15);
                const int p = j + (lane >> 4) < count && e < a.k ? list[e] : -1;
                return p < furthest ? p : -1;
            };
            int pos_next = SELECTED ? entry(0) : position(0);
            int page_next = page_at(pos_next);
            int pos_later = 0;
            int page_now = -1;
            int64_t offset_now = -1;
            if constexpr (SELECTED)
            {
                pos_later = entry(2);
            }
            auto issue = [&](int j) {
                if (j < count)
                {
                    const uint32_t dst = stage0 + slot_in * smem::STAGE;
                    if constexpr (SELECTED)
                    {
                        if ((j & 1) == 0)
                        {
                            page_now = page_next;
                            offset_now = -1;
                            if (page_now >= 0)
                            {
                                offset_now = page_now * a.c.page_stride +
                                             ((static_cast<int64_t>(it.head) << a.c.page_shift) + (pos_next & rows_mask)) * DIM;
                            }
                            pos_next = pos_later;
                            page_next = page_at(pos_next);
                            pos_later = entry(j + 4);
                        }
#pragma unroll
                        for (int x = 0; x < DIM / 32; ++x)
                        {
                            const int e = lane + x * 32;
                            const int row = e / PARTS;
                            const int64_t f = __shfl_sync(FULL_MASK, offset_now, (j & 1) * SUB + row);
                            const int64_t g = max(f, static_cast<int64_t>(0)) + (e % PARTS) * 16;
                            const uint32_t to = dst + row * PITCH<DIM, true> + (e % PARTS) * 16;
                            copy16(to, a.c.keys + g, f >= 0 ? 16U : 0U);
                            copy16(to + SUB * PITCH<DIM, true>, a.c.values + g, f >= 0 ? 16U : 0U);
                        }
                        if ((lane >> 4) == (j & 1)) // the scales of each row go with the rows
                        {
                            const int64_t at_scale = static_cast<int64_t>(max(page_now, 0)) * a.c.heads + it.head;
                            const uint32_t to = dst + smem::SCALES + (lane & 15) * 4;
                            copy4(to, a.c.key_scales + at_scale, page_now >= 0 ? 4U : 0U);
                            copy4(to + SUB * 4, a.c.value_scales + at_scale, page_now >= 0 ? 4U : 0U);
                        }
                    }
                    else
                    {
                        const int page = page_next;
                        const int safe = max(page, 0);
                        const int pos = row_of(j);
                        const int there = page < 0 ? 0 : min(SUB, furthest - pos);
                        page_next = page_at(position(j + 1));
                        const int64_t from = safe * a.c.page_stride + lane * 16 +
                                             ((static_cast<int64_t>(it.head) << a.c.page_shift) + (pos & rows_mask)) * DIM;
                        const uint8_t* const k_from = a.c.keys + from;
                        const uint8_t* const v_from = a.c.values + from;
                        if (there == SUB)
                        {
#pragma unroll
                            for (int x = 0; x < DIM / 32; ++x)
                            {
                                const int e = lane + x * 32;
                                const uint32_t to = dst + e / PARTS * PITCH<DIM, true> + (e % PARTS) * 16;
                                copy16(to, k_from + x * 512);
                                copy16(to + SUB * PITCH<DIM, true>, v_from + x * 512);
                            }
                        }
                        else
                        {
#pragma unroll
                            for (int x = 0; x < DIM / 32; ++x)
                            {
                                const int e = lane + x * 32;
                                const int row = e / PARTS;
                                const uint32_t to = dst + row * PITCH<DIM, true> + (e % PARTS) * 16;
                                copy16(to, k_from + x * 512, row < there ? 16U : 0U);
                                copy16(to + SUB * PITCH<DIM, true>, v_from + x * 512, row < there ? 16U : 0U);
                            }
                        }
                        if (lane < 2)
                        {
                            const float* scales = lane == 0 ? a.c.key_scales : a.c.value_scales;
                            copy4(dst + smem::SCALES + lane * 4, scales + static_cast<int64_t>(safe) * a.c.heads + it.head,
                                  page < 0 ? 0U : 4U);
                        }
                    }
                }
                copy_commit();
                slot_in = slot_in + 1 == STAGES ? 0 : slot_in + 1;
            };
#pragma unroll
            for (int j = 0; j < STAGES - 1; ++j)
            {
                issue(j);
            }
            // ---- the columns, while the first copies are under way ----
            for (int col = warp; col < COLS; col += WARPS)
            {
                const int g = it.column0 + col;
                const bool real = g < it.columns;
                const int i = g / a.group;
                const int64_t from = static_cast<int64_t>(it.first_token + i) * a.query_stride +
                                     static_cast<int64_t>(it.head * a.group + g % a.group) * DIM;
                const float f = pack_column<DIM, NB>(image, col, real ? a.queries : nullptr, from, a.dtype);
                if (lane == 0)
                {
                    undo[col] = f * a.scale;
                    const int token = SELECTED ? it.first_token - q.first : i;
                    visible[col] = real ? visible_of(a.b, q, token) : 0;
                }
            }
            __syncthreads();
            float o[DIM / 16][NB][4];
            float m[NB][2];
            float l[NB][2];
            float f[NB][2];
            int see[NB][2];
            uint32_t vs_least = 0; // bits of the largest value scale of the warp's rows so far over 2^SCALE_SPREAD
#pragma unroll
            for (int nb = 0; nb < NB; ++nb)
            {
#pragma unroll
                for (int x = 0; x < 2; ++x)
                {
                    m[nb][x] = -INFINITY;
                    l[nb][x] = 0.0F;
                    f[nb][x] = undo[nb * 8 + c + x];
                    see[nb][x] = SELECTED ? 0x7fffffff : visible[nb * 8 + c + x];
                }
#pragma unroll
                for (int g = 0; g < DIM / 16; ++g)
                {
                    o[g][nb][0] = o[g][nb][1] = o[g][nb][2] = o[g][nb][3] = 0.0F;
                }
            }
            for (int j = 0; j < count; ++j)
            {
                copy_wait<STAGES - 2>();
                __syncwarp();
                const int pos = row_of(j);
                if (pos < row_end)
                {
                    const unsigned char* const stage = mine + slot_out * smem::STAGE;
                    float s[NB][4];
                    score_rows<DIM, NB, true>(s, stage, reinterpret_cast<const uint2*>(image));
                    const float* const scales = reinterpret_cast<const float*>(stage + smem::SCALES);
                    const float ks_lo = SELECTED ? scales[row_lo] : scales[0];
                    const float ks_hi = SELECTED ? scales[row_lo + 8] : ks_lo;
                    float vs_lo = SELECTED ? scales[SUB + row_lo] : scales[1];
                    float vs_hi = SELECTED ? scales[SUB + row_lo + 8] : vs_lo;
                    // value scales at the border of their range and beyond would leave that of the sums
                    vs_lo = fminf(fmaxf(vs_lo, pow2_int(E_MIN)), pow2_int(E_MAX));
                    vs_hi = SELECTED ? fminf(fmaxf(vs_hi, pow2_int(E_MIN)), pow2_int(E_MAX)) : vs_lo;
                    const float lv_lo = log2_fast(vs_lo);
                    const float lv_hi = SELECTED ? log2_fast(vs_hi) : lv_lo;
                    const float iv_lo = __fdividef(1.0F, vs_lo);
                    const float iv_hi = SELECTED ? __fdividef(1.0F, vs_hi) : iv_lo;
                    // absent rows were copied as zeros, scale included; others are seen below `see`
                    const int at_lo = ks_lo != 0.0F ? pos + row_lo : 0x7fffffff;
                    const int at_hi = ks_hi != 0.0F ? pos + row_lo + 8 : 0x7fffffff;
#pragma unroll
                    for (int nb = 0; nb < NB; ++nb)
                    {
                        s[nb][0] = fmaf(s[nb][0], f[nb][0] * ks_lo, lv_lo);
                        s[nb][1] = fmaf(s[nb][1], f[nb][1] * ks_lo, lv_lo);
                        s[nb][2] = fmaf(s[nb][2], f[nb][0] * ks_hi, lv_hi);
                        s[nb][3] = fmaf(s[nb][3], f[nb][1] * ks_hi, lv_hi);
                    }
                    if (SELECTED || ks_lo == 0.0F || pos + SUB > nearest)
                    {
#pragma unroll
                        for (int nb = 0; nb < NB; ++nb)
                        {
                            s[nb][0] = at_lo < see[nb][0] ? s[nb][0] : -INFINITY;
                            s[nb][1] = at_lo < see[nb][1] ? s[nb][1] : -INFINITY;
                            s[nb][2] = at_hi < see[nb][0] ? s[nb][2] : -INFINITY;
                            s[nb][3] = at_hi < see[nb][1] ? s[nb][3] : -INFINITY;
                        }
                    }
                    bool raise = false;
#pragma unroll
                    for (int nb = 0; nb < NB; ++nb)
                    {
                        raise |= fmaxf(s[nb][0], s[nb][2]) > m[nb][0] + WEIGHT_SLACK;
                        raise |= fmaxf(s[nb][1], s[nb][3]) > m[nb][1] + WEIGHT_SLACK;
                    }
                    // a value scale above the largest one so far or far below it; positive floats order like their bits
                    auto apart = [&](float vs) { return __float_as_uint(vs) - vs_least > SCALE_SPREAD << 23; };
                    bool careful = false; // weights do not do as halves (cache_attend.cuh), or there is a NaN
                    if (__any_sync(FULL_MASK, raise || apart(vs_lo) || (SELECTED && apart(vs_hi))))
                    {
                        const uint32_t most_lo = ks_lo != 0.0F ? __float_as_uint(vs_lo) : 0U; // of rows that are there
                        const uint32_t most_hi = SELECTED && ks_hi != 0.0F ? __float_as_uint(vs_hi) : most_lo;
                        const uint32_t most = SELECTED ? __reduce_max_sync(FULL_MASK, max(most_lo, most_hi)) : most_lo;
                        vs_least = max(vs_least, most - min(most, SCALE_SPREAD << 23));
                        auto far = [&](float ks, float vs) { return ks != 0.0F && __float_as_uint(vs) < vs_least; };
                        careful = __any_sync(FULL_MASK, far(ks_lo, vs_lo) || (SELECTED && far(ks_hi, vs_hi))) != 0;
                        if (__any_sync(FULL_MASK, raise))
                        {
#pragma unroll
                            for (int nb = 0; nb < NB; ++nb)
                            {
#pragma unroll
                                for (int x = 0; x < 2; ++x)
                                {
                                    float top = fmaxf(s[nb][x], s[nb][2 + x]);
#pragma unroll
                                    for (int w = 4; w < 32; w <<= 1)
                                    {
                                        top = fmaxf(top, __shfl_xor_sync(FULL_MASK, top, w));
                                    }
                                    top = fmaxf(top, m[nb][x]);
                                    const float keep = m[nb][x] == -INFINITY ? 0.0F : exp2_fast(m[nb][x] - top);
                                    m[nb][x] = top;
                                    l[nb][x] *= keep;
#pragma unroll
                                    for (int g = 0; g < DIM / 16; ++g)
                                    {
                                        o[g][nb][x] *= keep;
                                        o[g][nb][2 + x] *= keep;
                                    }
                                }
                            }
                        }
                    }
                    auto weigh = [&](int nb, float (&p)[4]) { // rows lo, lo, hi, hi
                        const float b0 = WEIGHT_BIAS - (m[nb][0] == -INFINITY ? 0.0F : m[nb][0]);
                        const float b1 = WEIGHT_BIAS - (m[nb][1] == -INFINITY ? 0.0F : m[nb][1]);
                        p[0] = exp2_fast(s[nb][0] + b0);
                        p[1] = exp2_fast(s[nb][1] + b1);
                        p[2] = exp2_fast(s[nb][2] + b0);
                        p[3] = exp2_fast(s[nb][3] + b1);
                    };
                    uint32_t w_lo[NB];
                    uint32_t w_hi[NB];
#pragma unroll
                    for (int nb = 0; nb < NB; ++nb)
                    {
                        float p[4];
                        weigh(nb, p);
                        if constexpr (SELECTED)
                        {
                            l[nb][0] = fmaf(p[0], iv_lo, fmaf(p[2], iv_hi, l[nb][0]));
                            l[nb][1] = fmaf(p[1], iv_lo, fmaf(p[3], iv_hi, l[nb][1]));
                        }
                        else
                        {
                            l[nb][0] = fmaf(p[0] + p[2], iv_lo, l[nb][0]);
                            l[nb][1] = fmaf(p[1] + p[3], iv_lo, l[nb][1]);
                        }
                        w_lo[nb] = transpose_8x8(pack_half2(p[0], p[1]));
                        w_hi[nb] = transpose_8x8(pack_half2(p[2], p[3]));
                    }
                    // A NaN code times a weight of zero would spoil the columns that do not see its row.
                    // Only rows that some columns see and others do not can do that (rows nobody sees
                    // were copied as zeros); if such a subtile holds one, the codes are cleaned, and a
                    // product of indicators finds the outputs that the NaN belongs to.
                    const unsigned char* const vrows = stage + SUB * PITCH<DIM, true>;
                    bool nan_here = false;
                    if (!SELECTED && nearest < furthest && pos + SUB > nearest)
                    {
                        for (int e = lane; e < SUB * DIM / 4; e += 32)
                        {
                            const uint32_t w =
                                *reinterpret_cast<const uint32_t*>(vrows + (e * 4 / DIM) * PITCH<DIM, true> + e * 4 % DIM);
                            nan_here |= (((w & 0x7f7f7f7fU) + 0x01010101U) & 0x80808080U) != 0;
                        }
                        careful |= __any_sync(FULL_MASK, nan_here) != 0;
                    }
                    const uint32_t vaddr = ptx::smem_addr(vrows) +
                                           (((lane >> 3) & 1) * 8 + row_order<DIM, true>(lane & 7)) * PITCH<DIM, true> +
                                           (lane >> 4) * 16;
                    if (!careful)
                    {
#pragma unroll
                        for (int g = 0; g < DIM / 16; g += 2)
                        {
                            uint32_t r[4];
                            ldmatrix_x4_trans(r, vaddr + g * 16);
#pragma unroll
                            for (int x = 0; x < 2; ++x)
                            {
                                const uint32_t u = __byte_perm(r[2 * x], 0, 0x3120);
                                const uint32_t v = __byte_perm(r[2 * x + 1], 0, 0x3120);
                                uint32_t a0, a1, a2, a3;
                                halves_of_codes(u, a0, a1);
                                halves_of_codes(v, a2, a3);
#pragma unroll
                                for (int nb = 0; nb < NB; ++nb)
                                {
                                    mma_16816(o[g + x][nb], a0, a1, a2, a3, w_lo[nb], w_hi[nb]);
                                }
                            }
                        }
                    }
                    else
                    {
                        uint32_t one_lo[NB];
                        uint32_t one_hi[NB];
                        uint32_t w_lo[NB][2]; // the weights once more, each the sum of two BF16 numbers
                        uint32_t w_hi[NB][2];
#pragma unroll
                        for (int nb = 0; nb < NB; ++nb)
                        {
                            float p[4];
                            weigh(nb, p);
                            split_bf16(p[0], p[1], w_lo[nb][0], w_lo[nb][1]);
                            split_bf16(p[2], p[3], w_hi[nb][0], w_hi[nb][1]);
#pragma unroll
                            for (int y = 0; y < 2; ++y)
                            {
                                w_lo[nb][y] = transpose_8x8(w_lo[nb][y]);
                                w_hi[nb][y] = transpose_8x8(w_hi[nb][y]);
                            }
                            if constexpr (!SELECTED) // there everyone sees all rows
                            {
                                one_lo[nb] = transpose_8x8(
                                    pack_half2(at_lo < see[nb][0] ? 1.0F : 0.0F, at_lo < see[nb][1] ? 1.0F : 0.0F));
                                one_hi[nb] = transpose_8x8(
                                    pack_half2(at_hi < see[nb][0] ? 1.0F : 0.0F, at_hi < see[nb][1] ? 1.0F : 0.0F));
                            }
                        }
#pragma unroll
                        for (int g = 0; g < DIM / 16; g += 2)
                        {
                            uint32_t r[4];
                            ldmatrix_x4_trans(r, vaddr + g * 16);
#pragma unroll
                            for (int x = 0; x < 2; ++x)
                            {
                                const uint32_t u = __byte_perm(r[2 * x], 0, 0x3120);
                                const uint32_t v = __byte_perm(r[2 * x + 1], 0, 0x3120);
                                uint32_t h[4];
                                halves_of_codes(u, h[0], h[1]);
                                halves_of_codes(v, h[2], h[3]);
                                uint32_t is[4];
#pragma unroll
                                for (int y = 0; y < 4; ++y)
                                {
                                    // a half is NaN above 0x7c00 (codes give no infinities)
                                    const uint32_t low = (h[y] & 0x7fffU) > 0x7c00U ? 0xffffU : 0U;
                                    const uint32_t high = (h[y] & 0x7fff0000U) > 0x7c000000U ? 0xffff0000U : 0U;
                                    is[y] = (low | high) & 0x3c003c00U; // ones
                                    h[y] = bf16_of_halves(SELECTED ? h[y] : h[y] & ~(low | high));
                                }
#pragma unroll
                                for (int nb = 0; nb < NB; ++nb)
                                {
#pragma unroll
                                    for (int y = 0; y < 2; ++y)
                                    {
                                        mma_16816_bf16(o[g + x][nb], h[0], h[1], h[2], h[3], w_lo[nb][y], w_hi[nb][y]);
                                    }
                                    if constexpr (!SELECTED)
                                    {
                                        float hits[4] = {0.0F, 0.0F, 0.0F, 0.0F};
                                        mma_16816(hits, is[0], is[1], is[2], is[3], one_lo[nb], one_hi[nb]);
#pragma unroll
                                        for (int y = 0; y < 4; ++y)
                                        {
                                            o[g + x][nb][y] = hits[y] > 0.0F ? NAN : o[g + x][nb][y];
                                        }
                                    }
                                }
                            }
                        }
                    }
                }
                __syncwarp();
                slot_out = slot_out + 1 == STAGES ? 0 : slot_out + 1;
                issue(j + STAGES - 1);
            }
            copy_wait<0>();

            // ---- the four warps' sums ----
#pragma unroll
            for (int nb = 0; nb < NB; ++nb)
            {
#pragma unroll
                for (int x = 0; x < 2; ++x)
                {
#pragma unroll
                    for (int w = 4; w < 32; w <<= 1)
                    {
                        l[nb][x] += __shfl_xor_sync(FULL_MASK, l[nb][x], w);
                    }
                    if (lane < 4)
                    {
                        warp_ml[warp * COLS + nb * 8 + c + x] = make_float2(m[nb][x], l[nb][x]);
                    }
                }
            }
            __syncthreads(); // every warp's stream has ended: the stages are free
            float* const sums = reinterpret_cast<float*>(stages);
#pragma unroll
            for (int nb = 0; nb < NB; ++nb)
            {
#pragma unroll
                for (int x = 0; x < 2; ++x)
                {
                    const int col = nb * 8 + c + x;
                    float top = warp_ml[col].x;
#pragma unroll
                    for (int w = 1; w < WARPS; ++w)
                    {
                        top = fmaxf(top, warp_ml[w * COLS + col].x);
                    }
                    const float keep = m[nb][x] == -INFINITY ? (l[nb][x] == 0.0F ? 0.0F : 1.0F) : exp2_fast(m[nb][x] - top);
                    float* const to = sums + (warp * COLS + col) * DIM + (lane >> 2) * 2;
#pragma unroll
                    for (int g = 0; g < DIM / 16; ++g)
                    {
                        *reinterpret_cast<float2*>(to + g * 16) = make_float2(o[g][nb][x] * keep, o[g][nb][2 + x] * keep);
                    }
                }
            }
            __syncthreads();
            const bool whole = (!CLUSTER || a.cluster == 1) && at == it.begin && seg_end == it.end;
            // part 1 of a block: an item that begins in it and ends in another one; part 0: one that began before
            const int64_t part = 2 * static_cast<int64_t>(blockIdx.x) + (at == it.begin ? 1 : 0);
            for (int e = threadIdx.x; e < COLS * DIM; e += THREADS)
            {
                const int col = e / DIM;
                const int d = e % DIM;
                const int g = it.column0 + col;
                if (g >= it.columns)
                {
                    break;
                }
                float top = warp_ml[col].x;
#pragma unroll
                for (int w = 1; w < WARPS; ++w)
                {
                    top = fmaxf(top, warp_ml[w * COLS + col].x);
                }
                float sum = 0.0F;
                float den = 0.0F;
#pragma unroll
                for (int w = 0; w < WARPS; ++w)
                {
                    const float2 ml = warp_ml[w * COLS + col];
                    sum += sums[(w * COLS + col) * DIM + d];
                    den += ml.x == -INFINITY ? ml.y : ml.y * exp2_fast(ml.x - top);
                }
                if (CLUSTER && a.cluster > 1)
                {
                    // over the first warp's sum, which no other thread reads
                    sums[e] = sum;
                    if (d == 0)
                    {
                        block_ml[col] = make_float2(top, den);
                    }
                }
                else if (whole)
                {
                    const int64_t token = it.first_token + g / a.group;
                    const int qhead = it.head * a.group + g % a.group;
                    store_out(a.out, token * a.out_stride + static_cast<int64_t>(qhead) * DIM + d,
                              den == 0.0F ? 0.0F : sum / den, a.dtype);
                    if (d == 0 && a.lse != nullptr)
                    {
                        a.lse[token * a.group * a.c.heads + qhead] =
                            den == 0.0F ? -INFINITY : (top - WEIGHT_BIAS + log2f(den)) * LN_2;
                    }
                }
                else
                {
                    a.part_o[(part * COLS + col) * DIM + d] = sum;
                    if (d == 0)
                    {
                        a.part_ml[part * COLS + col] = make_float2(top, den);
                    }
                }
            }
            if (CLUSTER && a.cluster > 1)
            {
                // the blocks of the cluster have the same item: each joins its part of the numbers
                cluster_sync();
                const int rank = static_cast<int>(blockIdx.x) % a.cluster;
                for (int e = rank * THREADS + static_cast<int>(threadIdx.x); e < COLS * DIM; e += a.cluster * THREADS)
                {
                    const int col = e / DIM;
                    const int d = e % DIM;
                    const int g = it.column0 + col;
                    if (g >= it.columns)
                    {
                        break;
                    }
                    float top = -INFINITY;
                    for (int b = 0; b < a.cluster; ++b)
                    {
                        top = fmaxf(top, cluster_load(&block_ml[col].x, b));
                    }
                    float sum = 0.0F;
                    float den = 0.0F;
                    for (int b = 0; b < a.cluster; ++b)
                    {
                        const float m_b = cluster_load(&block_ml[col].x, b);
                        const float keep = m_b == -INFINITY ? 1.0F : exp2_fast(m_b - top);
                        sum = fmaf(keep, cluster_load(&sums[e], b), sum);
                        den = fmaf(keep, cluster_load(&block_ml[col].y, b), den);
                    }
                    const int64_t token = it.first_token + g / a.group;
                    const int qhead = it.head * a.group + g % a.group;
                    store_out(a.out, token * a.out_stride + static_cast<int64_t>(qhead) * DIM + d,
                              den == 0.0F ? 0.0F : sum / den, a.dtype);
                    if (d == 0 && a.lse != nullptr)
                    {
                        a.lse[token * a.group * a.c.heads + qhead] =
                            den == 0.0F ? -INFINITY : (top - WEIGHT_BIAS + log2f(den)) * LN_2;
                    }
                }
                cluster_sync(); // nobody leaves while its numbers are being read
            }
            else if (!CLUSTER && at == it.begin && !whole && threadIdx.x == 0)
            {
                // the block of the item's last unit: blocks begin at floor(c * total / blocks)
                a.joins[blockIdx.x] = make_int4(it.first_token, it.head, it.column0, it.columns);
                a.join_end[blockIdx.x] = static_cast<int>(((it.end * blocks) - 1) / total);
            }
        }
        if constexpr (CLUSTER)
        {
            return;
        }
        // ---- the next item ----
        at = seg_end;
        if (at >= share_end)
        {
            return;
        }
        it.begin = it.end;
        it.column0 += COLS;
        if constexpr (SELECTED)
        {
            it.end += list_units;
            if (it.column0 >= it.columns)
            {
                it.column0 = 0;
                if (++it.head == a.c.heads)
                {
                    it.head = 0;
                    ++it.first_token;
                }
            }
        }
        else
        {
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
            it.end = it.begin + units_of_block<smem>(a, q, it.column0);
        }
    }
}

template <int DIM, int NB>
int blocks_of()
{
    return device_sm_count() * attend_smem<DIM, NB>::BLOCKS;
}

// Most columns a block can take: the sums of 8 NB columns take NB * DIM / 4 registers of a thread.
constexpr int most_columns(int dim) { return dim <= 128 ? 4 : 2; }

template <int DIM, int NB, bool SELECTED>
int launch_attend(attend_args a, void* workspace, size_t workspace_bytes, cudaStream_t stream)
{
    using smem = attend_smem<DIM, NB>;
    int blocks = blocks_of<DIM, NB>();
    if (SELECTED || a.b.starts == nullptr)
    {
        // Few short items: each goes to a cluster of blocks of its own, which joins through its shared
        // memory, so that there is no second kernel and no search for shares.  Taken while the clusters
        // all run at once and a block has at most eight tiles; the table's width bounds the lengths, which the host does
        // not see (one request of 778 positions: 7.6 us, with starts or under a table of 131072 positions 12.4).
        const int64_t items = static_cast<int64_t>(a.b.tokens) * a.c.heads * ((a.group + smem::COLS - 1) / smem::COLS);
        const int64_t most = ((SELECTED ? a.k : a.b.limit) + TILE - 1) / TILE;
        int cluster = 1;
        while (cluster < 8 && cluster < most && items * cluster * 2 <= blocks)
        {
            cluster *= 2;
        }
        if (items * cluster <= blocks && most <= 8 * cluster)
        {
            a.cluster = cluster;
            blocks = static_cast<int>(items) * cluster;
        }
    }
    const int rc = place_parts<DIM, smem::COLS>(a, blocks_of<DIM, NB>(), workspace, workspace_bytes);
    if (rc != BITSKNN_OK)
    {
        return rc;
    }
    auto kernel =
        a.cluster > 0 ? cache_attend_kernel<DIM, NB, SELECTED, true> : cache_attend_kernel<DIM, NB, SELECTED, false>;
    static cache::device_set prepared[2];
    cache::device_set& ready = prepared[a.cluster > 0 ? 1 : 0];
    if (!ready.contains_current())
    {
        BITSKNN_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem::BYTES));
        ready.add_current();
    }
    {
        kernel_scope scope("cache_attend_kernel", stream);
        if (a.cluster > 1)
        {
            cudaLaunchAttribute shape{};
            shape.id = cudaLaunchAttributeClusterDimension;
            shape.val.clusterDim.x = static_cast<unsigned>(a.cluster);
            shape.val.clusterDim.y = 1;
            shape.val.clusterDim.z = 1;
            cudaLaunchConfig_t config{};
            config.gridDim = dim3(static_cast<unsigned>(blocks));
            config.blockDim = dim3(THREADS);
            config.dynamicSmemBytes = smem::BYTES;
            config.stream = stream;
            config.attrs = &shape;
            config.numAttrs = 1;
            BITSKNN_CUDA_TRY(cudaLaunchKernelEx(&config, kernel, a));
            return BITSKNN_OK;
        }
        kernel<<<blocks, THREADS, smem::BYTES, stream>>>(a);
    }
    BITSKNN_CUDA_TRY(cudaGetLastError());
    if (a.cluster > 0)
    {
        return BITSKNN_OK;
    }
    return launch_join<DIM, smem::COLS>(a, blocks, stream);
}

int attend(const bitsknn_cache_t* cache, const bitsknn_cache_batch_t* batch, const void* d_queries, int dtype,
           int64_t query_stride, int query_heads, bool selected, const int32_t* d_idx, int64_t ld_idx, int k, float scale,
           void* d_out, int64_t out_stride, float* d_lse, void* d_workspace, size_t workspace_bytes,
           bitsknn_stream_t stream)
{
    attend_args a{};
    int rc = check_cache(cache, &a.c);
    if (rc != BITSKNN_OK || (rc = check_cache_batch(batch, cache->page_rows, &a.b)) != BITSKNN_OK)
    {
        return rc;
    }
    if (selected && (k < 1 || k > (1 << 30))) // list positions are int32, with room for a block of them
    {
        return fail(BITSKNN_ERR_UNSUPPORTED_K, "Unsupported k value: %d", k);
    }
    if (selected && ld_idx < k)
    {
        return fail(BITSKNN_ERR_INVALID_ARGUMENT, "ld_idx=%lld is smaller than k=%d", static_cast<long long>(ld_idx), k);
    }
    const bool empty = batch->tokens == 0 || batch->requests == 0;
    rc = check_cache_queries(empty && d_queries == nullptr ? cache->d_keys : d_queries, dtype, &query_stride, query_heads,
                             cache->heads, cache->dim);
    if (rc != BITSKNN_OK)
    {
        return rc;
    }
    const int64_t dense = static_cast<int64_t>(query_heads) * cache->dim;
    out_stride = out_stride == 0 ? dense : out_stride;
    if (out_stride < dense)
    {
        return fail(BITSKNN_ERR_INVALID_ARGUMENT, "out_stride=%lld: at least %lld", static_cast<long long>(out_stride),
                    static_cast<long long>(dense));
    }
    if (empty)
    {
        return BITSKNN_OK;
    }
    if (d_out == nullptr || (selected && d_idx == nullptr) || d_workspace == nullptr)
    {
        return fail(d_workspace == nullptr && d_out != nullptr ? BITSKNN_ERR_WORKSPACE : BITSKNN_ERR_INVALID_ARGUMENT,
                    "null pointer argument");
    }
    if ((reinterpret_cast<uintptr_t>(d_workspace) & 255) != 0 || (reinterpret_cast<uintptr_t>(d_out) & 1) != 0 ||
        ((reinterpret_cast<uintptr_t>(d_lse) | reinterpret_cast<uintptr_t>(d_idx)) & 3) != 0)
    {
        return fail(BITSKNN_ERR_INVALID_ARGUMENT, "misaligned pointer (workspace 256 bytes, out 2, lse and idx 4)");
    }
    a.queries = d_queries;
    a.dtype = dtype;
    a.query_stride = query_stride;
    a.group = query_heads / cache->heads;
    a.scale = scale * LOG2_E;
    a.out = d_out;
    a.out_stride = out_stride;
    a.lse = d_lse;
    a.idx = d_idx;
    a.ld_idx = ld_idx;
    a.k = k;
    // columns that share a stream of the cache: the query heads of a token, times the tokens a request
    // has on average when the whole cache is attended to
    const int64_t per_request = selected ? 1 : (batch->tokens + batch->requests - 1) / batch->requests;
    const int64_t want = a.group * per_request;
    auto s = static_cast<cudaStream_t>(stream);
    // More columns than one stream of the cache can serve: the tensor-memory kernel takes over (16 requests
    // of 6000 positions, 8 heads of 128: 32 columns 109 us here and 129 there, 48 columns 169 and 130, 128
    // columns 324 and 134; heads of 256: 16 columns 113 and 165, 24 columns 187 and 167; by now the kernel taken
    // needs 100, 135, 140, 108 and 172).
    if (!selected && want > 8 * most_columns(cache->dim))
    {
        return launch_attend_tc(cache->dim, a, d_workspace, workspace_bytes, s);
    }
    return dispatch_cache_dim(cache->dim, [&](auto dim) {
        constexpr int DIM = decltype(dim)::value;
        if constexpr (most_columns(DIM) == 4)
        {
            if (want > 16)
            {
                return selected ? launch_attend<DIM, 4, true>(a, d_workspace, workspace_bytes, s)
                                : launch_attend<DIM, 4, false>(a, d_workspace, workspace_bytes, s);
            }
        }
        if (want > 8)
        {
            return selected ? launch_attend<DIM, 2, true>(a, d_workspace, workspace_bytes, s)
                            : launch_attend<DIM, 2, false>(a, d_workspace, workspace_bytes, s);
        }
        return selected ? launch_attend<DIM, 1, true>(a, d_workspace, workspace_bytes, s)
                        : launch_attend<DIM, 1, false>(a, d_workspace, workspace_bytes, s);
    });
}

} // namespace

} // namespace bitsknn

extern "C" size_t bitsknn_cache_attend_workspace_bytes(const bitsknn_cache_t* cache, int query_heads)
{
    using namespace bitsknn;
    cache::view v;
    if (check_cache(cache, &v) != BITSKNN_OK || query_heads < 1)
    {
        return 0;
    }
    size_t bytes = 0;
    dispatch_cache_dim(cache->dim, [&](auto dim) {
        constexpr int DIM = decltype(dim)::value;
        constexpr int MOST = most_columns(DIM);
        bytes = std::max({parts_bytes<DIM, 8>(blocks_of<DIM, 1>()), parts_bytes<DIM, 16>(blocks_of<DIM, 2>()),
                          parts_bytes<DIM, 8 * MOST>(blocks_of<DIM, MOST>()), attend_tc_workspace_bytes(DIM)});
        return BITSKNN_OK;
    });
    return bytes;
}

extern "C" int bitsknn_cache_attend(const bitsknn_cache_t* cache, const bitsknn_cache_batch_t* batch,
                                    const void* d_queries, int dtype, int64_t query_stride, int query_heads, float scale,
                                    void* d_out, int64_t out_stride, float* d_lse, void* d_workspace,
                                    size_t workspace_bytes, bitsknn_stream_t stream)
{
    return bitsknn::attend(cache, batch, d_queries, dtype, query_stride, query_heads, false, nullptr, 0, 0, scale, d_out,
                           out_stride, d_lse, d_workspace, workspace_bytes, stream);
}

extern "C" int bitsknn_cache_attend_selected(const bitsknn_cache_t* cache, const bitsknn_cache_batch_t* batch,
                                             const void* d_queries, int dtype, int64_t query_stride, int query_heads,
                                             const int32_t* d_idx, int64_t ld_idx, int k, float scale, void* d_out,
                                             int64_t out_stride, float* d_lse, void* d_workspace, size_t workspace_bytes,
                                             bitsknn_stream_t stream)
{
    return bitsknn::attend(cache, batch, d_queries, dtype, query_stride, query_heads, true, d_idx, ld_idx, k, scale, d_out,
                           out_stride, d_lse, d_workspace, workspace_bytes, stream);
}
