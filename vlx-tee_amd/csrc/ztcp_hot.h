// ztcp_hot.h -- what the operators on hot pages share (append, attention,
// page weights, eviction): argument checks on the host, page addressing and
// wave reductions on the device.
#pragma once

#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>

#include "../../include/ztcp.h"
#include "ztcp_device.h"
#include "ztcp_layout.h"

namespace ztcp {

// Sets the message ztcp_last_error returns (ztcp_abi.hip) and returns rc.
int arg_result(int rc, const char* why);

// ---- host ------------------------------------------------------------------

inline bool hot_aligned(const void* p) { return ((uintptr_t)p & 15u) == 0; }

// Whether two arrays of rows share a byte.  a: an rows of ab bytes, as_ bytes
// apart; b likewise.  Rows of one stride are compared modulo it, so that
// views side by side in one buffer do not count; otherwise by their extents.
inline bool rows_overlap(const void* a, int64_t an, int64_t ab, int64_t as_, const void* b, int64_t bn, int64_t bb,
                         int64_t bs) {
    if (!a || !b || an <= 0 || bn <= 0 || ab <= 0 || bb <= 0) return false;
    const uintptr_t a0 = (uintptr_t)a, b0 = (uintptr_t)b;
    const uintptr_t ae = a0 + (uintptr_t)((an - 1) * as_ + ab), be = b0 + (uintptr_t)((bn - 1) * bs + bb);
    if (!(a0 < be && b0 < ae)) return false;
    if (as_ != bs || as_ < ab || bs < bb) return true;
    const uint64_t d = b0 >= a0 ? (uint64_t)(b0 - a0) % (uint64_t)as_
                                : ((uint64_t)as_ - (uint64_t)(a0 - b0) % (uint64_t)as_) % (uint64_t)as_;
    return d < (uint64_t)ab || (uint64_t)as_ - d < (uint64_t)bb;
}

inline bool bytes_overlap(const void* a, int64_t an, const void* b, int64_t bn) {
    return rows_overlap(a, 1, an, an, b, 1, bn, bn);
}

// Division of 0 <= x < 2^31 by a page's tokens (1 <= d < 2^31):
// floor(x / d) = (x * mul) >> shift with mul = floor(2^shift / d) + 1,
// shift = 31 + ceil(log2 d): the product's excess over x * 2^shift / d is below
// x * d / d <= 2^31 <= 2^shift / d, too little to reach the next whole number.
struct DivBy {
    uint32_t mul;
    uint32_t shift;
};
inline DivBy div_by(uint32_t d) {
    uint32_t s = 0;
    while (((uint64_t)1 << s) < d) ++s;
    return DivBy{(uint32_t)(((uint64_t)1 << (31 + s)) / d + 1), 31 + s};
}

// Launches `blocks` workgroups.  A launch takes fewer than 2^32 threads, so more workgroups than that come in parts, each
// with its first one's number in p.first_block.
template <class Params, class... More>
inline void launch_blocks(void (*kernel)(Params, More...), uint64_t blocks, uint32_t threads, size_t lds, hipStream_t stream,
                          Params p, More... more) {
    const uint64_t most = 0xFFFFFFFFull / threads;
    for (uint64_t first = 0; first < blocks; first += most) {
        p.first_block = (uint32_t)first;
        const uint64_t n = blocks - first < most ? blocks - first : most;
        hipLaunchKernelGGL(kernel, dim3((uint32_t)n), dim3(threads), lds, stream, p, more...);
    }
}

// Bytes that a call which could do with less keeps between its kernels at most: beyond, it works in parts that use the same
// memory again.
constexpr int64_t kMostBetween = (int64_t)1 << 30;

// Compute units of the current device.
inline int cu_count(int& cus) {
    int dev = 0;
    return hipGetDevice(&dev) == hipSuccess &&
                   hipDeviceGetAttribute(&cus, hipDeviceAttributeMultiprocessorCount, dev) == hipSuccess && cus > 0
               ? ZTCP_OK
               : ZTCP_EHIP;
}

// What is wrong with a pool and its geometry, or nullptr.
inline const char* check_pool(const ztcp_page_pool* pool, const ztcp_geometry* g, int64_t max_head_dim) {
    if (!pool || !g) return "pool and geometry must not be NULL";
    if (!(g->num_tokens > 0 && g->num_heads > 0 && g->head_dim >= 16 && g->head_dim % 16 == 0))
        return "num_tokens, num_heads must be positive, head_dim a positive multiple of 16";
    if (g->head_dim > max_head_dim) return max_head_dim > 256 ? "head_dim must be at most 1024" : "head_dim must be at most 256";
    if (!(g->rope_dim >= 0 && g->rope_dim <= g->head_dim && g->rope_dim % 16 == 0)) return "Invalid rope_dim";
    if (g->hot_dtype != ZTCP_HOT_FP16 && g->hot_dtype != ZTCP_HOT_BF16)
        return "hot_dtype must be ZTCP_HOT_FP16 or ZTCP_HOT_BF16";
    const int64_t limit = (int64_t)1 << 30;
    if (g->num_tokens >= limit || g->num_heads >= limit || g->num_tokens * g->num_heads >= limit ||
        g->num_tokens * g->num_heads * g->head_dim >= limit)
        return "page too large (num_tokens * num_heads * head_dim must be below 2^30)";
    const int64_t page = g->num_tokens * g->num_heads * g->head_dim;
    if (pool->n_pages < 1 || pool->n_pages > (int64_t)0x7FFFFFFF) return "n_pages must be 1 .. 2^31 - 1";
    if (!pool->k) return "the pool's k must not be NULL";
    if (pool->n_pages > 1 && (pool->k_stride < page || (pool->v && pool->v_stride < page)))
        return "page strides must cover a page";
    if (!hot_aligned(pool->k) || !hot_aligned(pool->v) || (pool->k_stride | pool->v_stride) % 8 != 0)
        return "pages must be 16-byte aligned";
    return nullptr;
}

// A batch of sequences over a pool, as the kernels take it.
struct PagedView {
    const int32_t* table;
    const int32_t* lens;
    const int32_t* starts;
    int64_t table_stride;
    int32_t n_seqs, n_rows, n_pages;
    int32_t max_tokens;          // max_pages * page tokens
    int32_t page_tokens;
    DivBy page_div;
};

// What is wrong with a batch, or nullptr; fills `view`.
inline const char* check_batch(const ztcp_paged_batch* b, const ztcp_page_pool* pool, const ztcp_geometry* g,
                               int64_t q_heads, PagedView& view) {
    if (!b) return "batch must not be NULL";
    const int64_t most = (int64_t)1 << 31;
    if (b->n_seqs < 0 || b->n_seqs >= (int64_t)1 << 24 || b->n_rows < 0 || b->n_rows >= most || b->max_q_len < 0)
        return "n_seqs must be 0 .. 2^24 - 1, n_rows 0 .. 2^31 - 1, max_q_len not negative";
    if (q_heads < 1 || q_heads > 65536 || q_heads % g->num_heads != 0)
        return "q_heads must be a positive multiple of num_heads, at most 65536";
    if (b->max_pages < 1 || b->max_pages > (most - 1024) / g->num_tokens)
        return "max_pages must be positive, max_pages * num_tokens below 2^31 - 1024";
    if (b->n_rows * q_heads > most - 1024)   // blocks of up to 128 rows are counted beyond the last one
        return "too many query heads in one call (n_rows * q_heads must be at most 2^31 - 1024)";
    if (b->n_seqs > 0 && (!b->page_table || !b->kv_lens || !b->q_starts))
        return "page_table, kv_lens and q_starts must not be NULL";
    if (b->n_seqs > 1 && b->table_stride < b->max_pages) return "table_stride must cover max_pages";
    view = PagedView{b->page_table, b->kv_lens, b->q_starts, b->table_stride, (int32_t)b->n_seqs, (int32_t)b->n_rows,
                     (int32_t)pool->n_pages, (int32_t)(b->max_pages * g->num_tokens), (int32_t)g->num_tokens,
                     div_by((uint32_t)g->num_tokens)};
    return nullptr;
}

// ---- device ----------------------------------------------------------------

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

// A value that every lane of the wave has, in a scalar register.
__device__ __forceinline__ int uniform(int x) { return __builtin_amdgcn_readfirstlane(x); }
template <class T>
__device__ __forceinline__ T* uniform(T* p) {
    const uint64_t x = (uint64_t)p;
    return (T*)((uint64_t)(uint32_t)uniform((int)(uint32_t)x) | (uint64_t)(uint32_t)uniform((int)(uint32_t)(x >> 32)) << 32);
}

__device__ __forceinline__ int div_page(int x, DivBy d) { return (int)(((uint64_t)(uint32_t)x * d.mul) >> d.shift); }

// A sequence of the batch; whatever the arrays hold, its rows are rows of q and
// its tokens have table entries.
struct Seq {
    int row0, n_new, len;
    const int32_t* table;
    // Of global memory: the compiler, which has lost sight of that, would take a load that may be of LDS too, and a wait
    // for any LDS read behind it would wait for the entry, and for the loads in front of it.
    __device__ __forceinline__ int entry(int at) const { return ((const __attribute__((address_space(1))) int32_t*)table)[at]; }
};
__device__ __forceinline__ Seq uniform(Seq q) {
    return Seq{uniform(q.row0), uniform(q.n_new), uniform(q.len), uniform(q.table)};
}
__device__ __forceinline__ Seq seq_of(const PagedView& v, int s) {
    const int a = v.starts[s], b = v.starts[s + 1], len = v.lens[s];
    Seq q;
    q.row0 = min(max(a, 0), v.n_rows);
    q.n_new = min(max(b, q.row0), v.n_rows) - q.row0;
    q.len = min(max(len, 0), v.max_tokens);
    q.table = v.table + s * v.table_stride;
    return q;
}

// Work laid out sequence behind sequence, tiles(q) units of each: all of it, and
// what lies before sequence s.  Every lane of the wave takes part and gets the answer.
template <class F>
__device__ __forceinline__ int count_tiles(const PagedView& v, int s, int& before, F&& tiles) {
    const int lane = (int)threadIdx.x & 63;
    int total = 0;
    before = 0;
    for (int base = 0; base < v.n_seqs; base += 64) {
        int n = base + lane < v.n_seqs ? tiles(seq_of(v, base + lane)) : 0;
        int first = base + lane < s ? n : 0;
        for (int m = 1; m < 64; m <<= 1) {
            n += __shfl_xor(n, m);
            first += __shfl_xor(first, m);
        }
        total += n;
        before += first;
    }
    return total;
}

// The sequence that has unit `tile`, which becomes its number there; v.n_seqs if there are fewer units.
template <class F>
__device__ __forceinline__ int find_tile(const PagedView& v, int& tile, F&& tiles) {
    const int lane = (int)threadIdx.x & 63;
    for (int base = 0; base < v.n_seqs; base += 64) {
        const int n = base + lane < v.n_seqs ? tiles(seq_of(v, base + lane)) : 0;
        int upto = n;
        for (int m = 1; m < 64; m <<= 1) {
            const int y = __shfl_up(upto, m);
            upto += lane >= m ? y : 0;
        }
        const uint64_t past = __ballot(upto > tile);
        if (past) {
            const int at = __ffsll((unsigned long long)past) - 1;
            tile -= __shfl(upto, at) - __shfl(n, at);
            return base + at;
        }
        tile -= __shfl(upto, 63);
    }
    return v.n_seqs;
}

// The first of n ascending ends that is above x, n if none is; every lane of the wave asks for the same x.
__device__ __forceinline__ int find_above(const int32_t* ends, int n, int x) {
    const int lane = (int)threadIdx.x & 63;
    int low = 0, high = n;                                    // it is in low .. high
    while (low < high) {
        const int step = (high - low - 1) / 64 + 1, at = low + (lane + 1) * step - 1;
        const uint64_t past = __ballot(at >= high || ends[at] > x);
        if (past == 0) return high;
        const int first = __ffsll((unsigned long long)past) - 1;
        high = min(low + (first + 1) * step - 1, high);
        low += first * step;
    }
    return low;
}

// Where token `key` (below `stop`) is: its page, -1 if there is none, and its row in the page.
struct Place {
    int page, row;
};
__device__ __forceinline__ Place place_of(const PagedView& v, const Seq& q, int key, int stop) {
    Place p{-1, 0};
    if (key < stop) {
        const int at = div_page(key, v.page_div);
        const int id = q.table[at];
        if (id >= 0 && id < v.n_pages) p.page = id;
        p.row = key - at * v.page_tokens;
    }
    return p;
}

// 64 pieces of 16 bytes from global memory to LDS, a wave's piece i to lds + 16 i, without passing through registers;
// done once vmcnt says so.  Written in asm because the compiler, which cannot tell two buffers apart, would wait for
// the next tile's loads before this tile's reads.  It has no output that the load writes.  What the compiler does not
// add inside asm: a load to LDS needs one wait state behind the write of m0 that it uses, and five behind a vector
// instruction (readfirstlane) that wrote its scalar base; a scalar copy of the base, which waits for that by itself, is
// both.  m0 is reserved: it cannot be listed as overwritten, and the compiler keeps nothing in it; nothing else in
// these kernels' code uses it, which tests/test_hot_lds_loads.py checks.  The second form takes a base of the wave and
// each lane's offset.
__device__ __forceinline__ void load_lds16(const uint8_t* src, uint32_t lds) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(uniform((int)lds)), "v"(src) : "memory");
}
__device__ __forceinline__ void load_lds16(const uint8_t* base, uint32_t offset, uint32_t lds) {
    uint64_t copy;
    asm volatile("s_mov_b32 m0, %1\n\ts_mov_b64 %0, %3\n\tglobal_load_lds_dwordx4 %2, %0"
                 : "=&s"(copy) : "s"(uniform((int)lds)), "v"(offset), "s"(uniform(base)) : "memory");
}
__device__ __forceinline__ uint32_t lds_address(const void* p) {
    return (uint32_t)(uintptr_t)(const __attribute__((address_space(3))) void*)p;
}

// A load of what is read once and by whole lines (one that takes half a line would fetch it again for the other half).
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
__device__ __forceinline__ uint4 ldg16_once(const uint8_t* p) {
    const u32x4 x = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(p));
    return make_uint4(x.x, x.y, x.z, x.w);
}

// MFMA operands and results.
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

// Products of 16-bit operands in fp32.  Lane l holds eight numbers of row (A)
// or column (B) l % 16 (32), at depths (l / 16) * 8 + 0..7 ((l / 32) * 8 + 0..7);
// the result has column l % 16 (32) and rows (l / 16) * 4 + i
// (8 * (i / 4) + 4 * (l / 32) + i % 4).
template <int DT>
__device__ __forceinline__ f32x4 mfma16(uint4 a, uint4 b, f32x4 c) {
    if constexpr (DT == kHotBf16)
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}
template <int DT>
__device__ __forceinline__ f32x16 mfma32(uint4 a, uint4 b, f32x16 c) {
    if constexpr (DT == kHotBf16)
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

template <int DT>
__device__ __forceinline__ bool not_finite16(uint32_t h) {
    constexpr uint32_t e = DT == kHotBf16 ? 0x7F80u : 0x7C00u;
    return (h & e) == e;
}
// Sets those of eight numbers to 0 that are no finite numbers; whether there was one.
template <int DT>
__device__ __forceinline__ bool drop_not_finite(uint4& x) {
    uint32_t w[4] = {x.x, x.y, x.z, x.w};
    bool any = false;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if (not_finite16<DT>(w[i])) w[i] &= 0xFFFF0000u, any = true;
        if (not_finite16<DT>(w[i] >> 16)) w[i] &= 0x0000FFFFu, any = true;
    }
    if (any) x = make_uint4(w[0], w[1], w[2], w[3]);
    return any;
}

// Transposing LDS read of 16-bit numbers: the 16 lanes of a group give the
// addresses of four rows of 16 numbers (lane i: row i / 4, numbers (i % 4) * 4
// + 0..3), and lane i receives number i of the four rows.
typedef short s16x4 __attribute__((ext_vector_type(4)));
__device__ __forceinline__ uint2 lds_read_transposed(const uint8_t* p) {
    return __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)p));
}

// The larger, and the sum, of a lane's number and that of the lane 32 further on.
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
__device__ __forceinline__ float max_halves(float x) {
    const u32x2 r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return fmaxf(__uint_as_float(r.x), __uint_as_float(r.y));
}
__device__ __forceinline__ float sum_halves(float x) {
    const u32x2 r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return __uint_as_float(r.x) + __uint_as_float(r.y);
}

__device__ __forceinline__ float xor_sum(float x, int width) {  // over aligned groups of `width` lanes
    for (int m = 1; m < width; m <<= 1) x += __shfl_xor(x, m);
    return x;
}

}  // namespace ztcp
