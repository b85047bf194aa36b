// Shared pieces of the paged 8-bit cache operators: the device view of a cache and of a batch of
// requests, e4m3 conversions, and the warp-level stream that brings 16 cached rows at a time into
// shared memory and multiplies them with a block of query columns.
//
// A cached number is code * scale: an e4m3 code (sign, 4 exponent bits with bias 7, 3 fraction
// bits, no infinities, 0x7f / 0xff = NaN) times the scale of its page and head.
#pragma once

#include <atomic>
#include <cstdint>
#include <type_traits>

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include "common.cuh"
#include "ptx.cuh"

namespace bitsknn::cache
{

constexpr int WARPS = 4;             // warps of a streaming block
constexpr int THREADS = WARPS * 32;
constexpr int SUB = 16;              // cached rows a warp handles at a time
constexpr int TILE = WARPS * SUB;    // cached rows a block handles at a time
constexpr int E_MIN = -60;           // exponents of the scales the append kernel writes
constexpr int E_MAX = 60;
constexpr int MOST_ROWS = 1 << 30;   // requests, tokens: their numbers plus a block of them stay below 2^31

// Devices on which a kernel's attributes have been set (they hold for the life of the context; a
// device beyond the 64th is set up at every call).
struct device_set
{
    std::atomic<uint64_t> bits{0};

    bool contains_current() const
    {
        int device = 64;
        return cudaGetDevice(&device) == cudaSuccess && device < 64 && ((bits.load() >> device) & 1) != 0;
    }
    void add_current()
    {
        int device = 64;
        if (cudaGetDevice(&device) == cudaSuccess && device < 64)
        {
            bits.fetch_or(1ULL << device);
        }
    }
};

// Device view of bitsknn_cache_t (strides resolved).
struct view
{
    uint8_t* keys;
    uint8_t* values;
    float* key_scales;
    float* value_scales;
    int64_t pages;
    int64_t page_stride; // codes from one page to the next
    int heads;
    int page_shift;      // log2(rows of a page)
};

// Device view of bitsknn_cache_batch_t.
struct batch
{
    const int32_t* table;
    int64_t table_ld;
    int64_t limit;       // positions a table row covers
    const int32_t* lengths;
    const int32_t* starts; // nullptr: one token per request
    int requests;
    int tokens;
};

// Request r: its tokens [first, first + count) of the packed rows and its cached length.
struct request
{
    int first;
    int count;
    int length;
};

__device__ __forceinline__ request request_of(const batch& b, int r)
{
    request q;
    q.first = r;
    q.count = 1;
    q.length = max(b.lengths[r], 0);
    if (b.starts != nullptr)
    {
        const int end = b.starts[r + 1];
        q.first = min(max(b.starts[r], 0), b.tokens);
        q.count = min(max(end, q.first), b.tokens) - q.first;
        // a request whose tokens the arrays hold in part: the others' positions lie behind all that these see
        q.length -= max(end - b.tokens, 0);
    }
    return q;
}

// Positions that token i of a request sees: its own and everything before it.
__device__ __forceinline__ int visible_of(const batch& b, const request& q, int i)
{
    const int64_t v = static_cast<int64_t>(q.length) - q.count + i + 1;
    return static_cast<int>(min(max(v, static_cast<int64_t>(0)), b.limit));
}

// Request a packed token belongs to (the last r with starts[r] <= token), -1 behind the last one.
__device__ __forceinline__ int owner_of(const batch& b, int token)
{
    if (b.starts == nullptr)
    {
        return token < b.requests ? token : -1;
    }
    if (token < b.starts[0] || token >= b.starts[b.requests])
    {
        return -1;
    }
    int lo = 0;
    int hi = b.requests; // starts[lo] <= token < starts[hi]
    while (hi - lo > 1)
    {
        const int mid = (lo + hi) >> 1;
        if (b.starts[mid] <= token)
        {
            lo = mid;
        }
        else
        {
            hi = mid;
        }
    }
    return lo;
}

// ---- number formats ------------------------------------------------------------------------
// The four codes of a word to halves, bytes 0, 1 to `lo` and bytes 2, 3 to `hi`; exact, every e4m3
// number is a half.
__device__ __forceinline__ void halves_of_codes(uint32_t w, uint32_t& lo, uint32_t& hi)
{
    asm("{\n.reg .b16 l, h;\nmov.b32 {l, h}, %2;\ncvt.rn.f16x2.e4m3x2 %0, l;\ncvt.rn.f16x2.e4m3x2 %1, h;\n}\n"
        : "=r"(lo), "=r"(hi)
        : "r"(w));
}

// Two floats to two codes (`lo` in the low byte): nearest, ties to even, saturating at 448; NaN -> 0x7f.
__device__ __forceinline__ uint32_t codes_of_floats(float lo, float hi)
{
    uint32_t out;
    asm("{\n.reg .b16 t;\ncvt.rn.satfinite.e4m3x2.f32 t, %2, %1;\ncvt.u32.u16 %0, t;\n}\n"
        : "=r"(out)
        : "f"(lo), "f"(hi));
    return out;
}

__device__ __forceinline__ float exp2_fast(float x)
{
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

__device__ __forceinline__ float log2_fast(float x)
{
    float y;
    asm("lg2.approx.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

__device__ __forceinline__ float pow2_int(int e) { return __int_as_float((e + 127) << 23); }

__device__ __forceinline__ float load_float(const void* p, int64_t i, int dtype)
{
    return dtype == BITSKNN_F16    ? __half2float(static_cast<const __half*>(p)[i])
           : dtype == BITSKNN_BF16 ? __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i])
                                   : static_cast<const float*>(p)[i];
}

// ---- asynchronous copies ---------------------------------------------------------------------
// 16 bytes global -> shared past L1; `bytes` = 0 writes zeros and reads nothing.
__device__ __forceinline__ void copy16(uint32_t dst, const void* src, uint32_t bytes)
{
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}

__device__ __forceinline__ void copy16(uint32_t dst, const void* src)
{
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}

__device__ __forceinline__ void copy4(uint32_t dst, const void* src, uint32_t bytes)
{
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}

__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }

template <int PENDING>
__device__ __forceinline__ void copy_wait()
{
    asm volatile("cp.async.wait_group %0;" ::"n"(PENDING) : "memory");
}

// ---- thread-block clusters ----------------------------------------------------------------------
__device__ __forceinline__ void cluster_sync()
{
    asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// A float of the shared memory of block `rank` of the cluster, at the place `mine` has in this block.
__device__ __forceinline__ float cluster_load(const float* mine, int rank)
{
    float v;
    asm volatile("{\n.reg .b32 a;\nmapa.shared::cluster.u32 a, %1, %2;\nld.shared::cluster.f32 %0, [a];\n}\n"
                 : "=f"(v)
                 : "r"(ptx::smem_addr(mine)), "r"(rank)
                 : "memory");
    return v;
}

// ---- warp matrix steps -------------------------------------------------------------------------
__device__ __forceinline__ void mma_16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                          uint32_t b0, uint32_t b1)
{
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
                 "{%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// The same with operands of BF16.
__device__ __forceinline__ void mma_16816_bf16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                               uint32_t b0, uint32_t b1)
{
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
                 "{%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

__device__ __forceinline__ void ldmatrix_x4_trans(uint32_t (&r)[4], uint32_t addr)
{
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}

// Transposes an 8 x 8 matrix of halves held two to a thread.
__device__ __forceinline__ uint32_t transpose_8x8(uint32_t x)
{
    uint32_t y;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}

__device__ __forceinline__ uint32_t pack_half2(float lo, float hi)
{
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
}

__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi)
{
    const __nv_bfloat162 b = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&b);
}

// Two halves that hold e4m3 numbers to two BF16 numbers; exact.
__device__ __forceinline__ uint32_t bf16_of_halves(uint32_t h)
{
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h));
    return pack_bf16(f.x, f.y);
}

// Two floats, each as the sum of two BF16 numbers (17 significant bits over the range of floats).
__device__ __forceinline__ void split_bf16(float x, float y, uint32_t& high, uint32_t& low)
{
    high = pack_bf16(x, y);
    low = pack_bf16(x - __uint_as_float(high << 16), y - __uint_as_float(high & 0xffff0000U));
}

// Staged rows in shared memory, DIM / 16 granules of 16 bytes each.  Eight rows at the same granule have to
// lie on eight different bank groups.  Padded: a granule is added to every row, which makes the pitch an odd
// number of them.  Swapped (where DIM is a power of two): the granules of a row change places by the row
// number.  The attention kernels pad (one long request: 88 us, swapped 103: the addresses of two operands
// cost more than the space is worth), the distance kernel swaps (74 us, padded 83).
template <int DIM, bool PADDED>
constexpr bool SWAPPED = !PADDED && (DIM & (DIM - 1)) == 0;

template <int DIM, bool PADDED>
constexpr int PITCH = SWAPPED<DIM, PADDED> ? DIM : DIM + 16; // bytes between staged rows

template <int DIM, bool PADDED>
__device__ __forceinline__ int granule_swap(int row)
{
    if constexpr (!SWAPPED<DIM, PADDED>)
    {
        return 0;
    }
    return DIM >= 128 ? row & 7 : DIM == 64 ? (row >> 1) & 3 : (row >> 2) & 1;
}

template <int DIM, bool PADDED>
__device__ __forceinline__ int granule_byte(int row, int granule)
{
    return row * PITCH<DIM, PADDED> + ((granule ^ granule_swap<DIM, PADDED>(row)) << 4);
}

// Row of a 16-row subtile that matrix row r (0 ... 7) stands for.  The eight lanes of a phase of a 128-bit
// load read four granules of two neighbouring matrix rows; unless 32 or 64 numbers are swapped these have
// to lie four rows apart (order 0 4 1 5 2 6 3 7) to fall on eight different bank groups.
template <int DIM, bool PADDED>
__device__ __forceinline__ int row_order(int r)
{
    return SWAPPED<DIM, PADDED> && DIM <= 64 ? r : (r >> 1) | ((r & 1) << 2);
}

// Query columns of a block as halves in the order the matrix step wants them: word pair
// [kstep][column block][lane] holds, for column lane / 4, the dims base + 0, 1 and base + 2, 3.
// Dims are permuted along the contraction so that a lane's share of a cached row is contiguous:
// units of 64 dims (32 for what is left) give each of the four lanes of a row 16 (8) bytes.
//
// Writes one query column into the packed image.  Halves hold 11 significant bits, more than the
// 8 of BF16, but far fewer exponents: the column is scaled by a power of two that puts its
// largest finite entry into [2^14, 2^15), so only entries 2^-28 times smaller and less lose bits.
// Returns the power that undoes the scaling.  One warp per column; `src` == nullptr writes zeros.
template <int DIM, int NB>
__device__ __forceinline__ float pack_column(uint32_t* image, int col, const void* src, int64_t offset, int dtype)
{
    constexpr int PER = DIM / 32;
    const int lane = threadIdx.x & 31;
    float v[PER];
    float top = 0.0F;
#pragma unroll
    for (int i = 0; i < PER; ++i)
    {
        // lane's dims PER * lane ...: whole pairs for every DIM but 32, which stores single halves
        v[i] = src != nullptr ? load_float(src, offset + lane * PER + i, dtype) : 0.0F;
        const float a = fabsf(v[i]);
        top = a < INFINITY ? fmaxf(top, a) : top;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1)
    {
        top = fmaxf(top, __shfl_xor_sync(FULL_MASK, top, o));
    }
    // exponent field of top; subnormal BF16 inputs get the smallest normal one
    const int e = max(static_cast<int>(__float_as_uint(top) >> 23), 1) - 127;
    const int shift = top > 0.0F ? min(max(14 - e, -126), 126) : 0;
    const float up = pow2_int(shift);
    __half* out = reinterpret_cast<__half*>(image);
#pragma unroll
    for (int i = 0; i < PER; ++i)
    {
        const int d = lane * PER + i;
        constexpr int FULL = DIM / 64;
        const int unit = d >> 6;
        const bool wide = unit < FULL;
        const int within = wide ? (d & 63) : d - FULL * 64;
        const int c = wide ? within >> 4 : within >> 3;
        const int kstep = wide ? unit * 4 + ((within & 15) >> 2) : FULL * 4 + ((within & 7) >> 2);
        const int ln = (col & 7) * 4 + c;
        const int word = ((kstep * NB + (col >> 3)) * 32 + ln) * 2 + ((d & 3) >> 1);
        out[word * 2 + (d & 1)] = __float2half_rn(v[i] * up);
    }
    return pow2_int(-shift);
}

// Scores of 16 staged rows against NB blocks of 8 query columns: s[nb] = rows x columns, where
// thread (r = lane / 4, c = lane % 4) gets rows row_order(r) and 8 + row_order(r) of columns
// 8 nb + 2 c and 2 c + 1.  `image` is the packed query image (shared memory).
template <int DIM, int NB, bool PADDED>
__device__ __forceinline__ void score_rows(float (&s)[NB][4], const unsigned char* rows, const uint2* image)
{
    constexpr int FULL = DIM / 64;
    const int lane = threadIdx.x & 31;
    const int c = lane & 3;
    // this lane's granules: c of every unit of four, moved by the row's swap (rows r and r + 8 share it)
    const int row = row_order<DIM, PADDED>(lane >> 2);
    const int swap = granule_swap<DIM, PADDED>(row);
    const unsigned char* low = rows + row * PITCH<DIM, PADDED> + ((c ^ (swap & 3)) << 4);
    const int unit_swap = (swap >> 2) * 64;
    // two sums, for even and odd steps, so that a step does not wait for the one before it
    float odd[NB][4];
#pragma unroll
    for (int nb = 0; nb < NB; ++nb)
    {
        s[nb][0] = s[nb][1] = s[nb][2] = s[nb][3] = 0.0F;
        odd[nb][0] = odd[nb][1] = odd[nb][2] = odd[nb][3] = 0.0F;
    }
    auto step = [&](int kstep, uint32_t a, uint32_t b) {
        uint32_t a0, a1, a2, a3;
        halves_of_codes(a, a0, a2);
        halves_of_codes(b, a1, a3);
#pragma unroll
        for (int nb = 0; nb < NB; ++nb)
        {
            const uint2 q = image[(kstep * NB + nb) * 32 + lane];
            mma_16816((kstep & 1) != 0 ? odd[nb] : s[nb], a0, a1, a2, a3, q.x, q.y);
        }
    };
#pragma unroll
    for (int u = 0; u < FULL; ++u)
    {
        const uint4 x = *reinterpret_cast<const uint4*>(low + ((u * 64) ^ unit_swap));
        const uint4 y = *reinterpret_cast<const uint4*>(low + ((u * 64) ^ unit_swap) + 8 * PITCH<DIM, PADDED>);
        step(u * 4 + 0, x.x, y.x);
        step(u * 4 + 1, x.y, y.y);
        step(u * 4 + 2, x.z, y.z);
        step(u * 4 + 3, x.w, y.w);
    }
    if constexpr (DIM % 64 != 0)
    {
        const unsigned char* tail = rows + granule_byte<DIM, PADDED>(row, FULL * 4 + (c >> 1)) + (c & 1) * 8;
        const uint2 x = *reinterpret_cast<const uint2*>(tail);
        const uint2 y = *reinterpret_cast<const uint2*>(tail + 8 * PITCH<DIM, PADDED>);
        step(FULL * 4 + 0, x.x, y.x);
        step(FULL * 4 + 1, x.y, y.y);
    }
#pragma unroll
    for (int nb = 0; nb < NB; ++nb)
    {
#pragma unroll
        for (int i = 0; i < 4; ++i)
        {
            s[nb][i] += odd[nb][i];
        }
    }
}

} // namespace bitsknn::cache

namespace bitsknn
{

// Checks shared by the cache entry points; fill the device views.  Defined in cache_plan.cu.
int check_cache(const bitsknn_cache_t* cache, cache::view* out);
int check_cache_batch(const bitsknn_cache_batch_t* in, int page_rows, cache::batch* out);
int check_cache_queries(const void* d_queries, int dtype, int64_t* query_stride, int query_heads, int heads, int dim);

// Rows of an array in memory, for the checks of what a call reads against what it writes.
struct extent
{
    const char* name;
    const void* data;
    int64_t rows;
    int64_t stride; // bytes between rows
    int64_t width;  // bytes of a row
};

inline extent dense_extent(const char* name, const void* data, int64_t bytes) { return {name, data, 1, bytes, bytes}; }

// Whether the first row of the array that begins later lies in rows of the other one.  For arrays of one stride that
// is whether they share memory; arrays that take turns in the rows of a wider one do not.
inline bool overlap(const extent& x, const extent& y)
{
    if (x.data == nullptr || y.data == nullptr || x.rows < 1 || y.rows < 1 || x.width < 1 || y.width < 1)
    {
        return false;
    }
    const bool ordered = reinterpret_cast<uintptr_t>(x.data) <= reinterpret_cast<uintptr_t>(y.data);
    const extent& a = ordered ? x : y;
    const extent& b = ordered ? y : x;
    const uint64_t apart = reinterpret_cast<uintptr_t>(b.data) - reinterpret_cast<uintptr_t>(a.data);
    const uint64_t stride = static_cast<uint64_t>(a.stride);
    const uint64_t last = static_cast<uint64_t>(a.rows) - 1;
    if (apart >= last * stride + static_cast<uint64_t>(a.width))
    {
        return false; // behind all of it: the usual case
    }
    const uint64_t row = apart / stride;
    return (row <= last && apart % stride < static_cast<uint64_t>(a.width)) ||
           (row < last && stride - apart % stride < static_cast<uint64_t>(b.width));
}

// Refuses arrays a call writes that share memory with one another or with those it reads.
int check_apart(const extent* writes, int write_count, const extent* reads, int read_count);

// Calls fn with std::integral_constant<int, DIM> for a supported row length (checked before).
template <typename F>
int dispatch_cache_dim(int dim, F&& fn)
{
    switch (dim)
    {
    case 32: return fn(std::integral_constant<int, 32>{});
    case 64: return fn(std::integral_constant<int, 64>{});
    case 96: return fn(std::integral_constant<int, 96>{});
    case 128: return fn(std::integral_constant<int, 128>{});
    case 192: return fn(std::integral_constant<int, 192>{});
    case 256: return fn(std::integral_constant<int, 256>{});
    default: return fail(BITSKNN_ERR_UNSUPPORTED_DIM, "Unsupported cache dim value: %d", dim);
    }
}

} // namespace bitsknn
