// ztcp_evict.hip -- which pages of a sequence go cold: those with the least
// accumulated attention weight.
#include "ztcp_hot.h"

using namespace ztcp;

namespace {

constexpr int kDigitBits = 11;
constexpr int kBins = 1 << kDigitBits;
constexpr int kFew = 256;           // so many keys are ranked by counting
constexpr int kKeysInLds = 16384;   // 128 KiB of keys; longer tables sum their accounts again on every pass

struct EvictParams {
    const float* mass;
    const int32_t* table;
    int64_t table_stride;
    const int32_t* lens;
    int32_t heads, max_pages, page_tokens;
    int64_t budget, sink, recent;
    int32_t* out_table;
    int64_t out_table_stride;
    float* out_mass;
    int32_t* out_lens;
    int32_t* evicted;
    int32_t* n_evicted;
    uint32_t first_block;               // of this launch
};

// A number's place among all doubles as an unsigned whole number; the two
// zeros are one place, and every NaN is above infinity.
__device__ __forceinline__ uint64_t order_of(double x) {
    if (x != x) return ~0ull;
    const uint64_t b = (uint64_t)__double_as_longlong(x + 0.0);   // -0 + 0 = 0
    return (b >> 63) ? ~b : b | (1ull << 63);
}

// A page's key: its accounts added up in the order of the heads, in 64 bits.
__device__ __forceinline__ uint64_t key_from_accounts(const EvictParams& p, const float* mass, int page) {
    double t = 0.0;
    for (int h0 = 0; h0 < p.heads; h0 += 8) {   // eight loads in flight
        float m[8];
#pragma unroll
        for (int h = 0; h < 8; ++h) m[h] = h0 + h < p.heads ? mass[(int64_t)(h0 + h) * p.max_pages + page] : 0.f;
#pragma unroll
        for (int h = 0; h < 8; ++h) t += (double)m[h];
    }
    return order_of(t);
}

// Sum over the block's waves of each wave's value, and the sum before this wave.
template <int WAVES>
__device__ __forceinline__ int block_before(int of_wave, int* lds, int& total) {
    const int wave = (int)threadIdx.x / 64;
    __syncthreads();
    if ((threadIdx.x & 63u) == 0) lds[wave] = of_wave;
    __syncthreads();
    int before = 0;
    total = 0;
#pragma unroll
    for (int i = 0; i < WAVES; ++i) {
        const int x = lds[i];
        before += i < wave ? x : 0;
        total += x;
    }
    return before;
}

__device__ __forceinline__ int pages_of(const EvictParams& p, int32_t len) {
    const int64_t want = ((int64_t)(len < 0 ? 0 : len) + p.page_tokens - 1) / p.page_tokens;
    return (int)(want < p.max_pages ? want : p.max_pages);
}

// One workgroup per sequence.  What goes is found by closing in: of the keys
// from low to high, which hold the count-th smallest, the least and the greatest
// are found (equal ones are done), their span is cut into 2048 bins, and low and
// high become the bin's in which the count runs out; the last 256 keys are
// ranked by counting.  Sums of 32-bit accounts seldom need more than two rounds,
// also where a third of the pages has none.  Below low all go, and of those from
// low to high the first ones.  Then one walk in page order closes the gaps: a
// page moves down by the number of pages gone before it, so that a part that has
// been read whole may be written over itself.
//
// It is bound by latencies: what one compute unit has in flight brings about 16
// bytes a nanosecond.  8 sequences of 256 pages and 8 heads: 9.2 us by 256
// threads (13.4 by 1024, whose barriers and redundant scans cost more).  128
// sequences of up to 8,192 pages: 52 us a pass, 47.4 of them the kernel's (the
// profiler's time), of which the keys take 16, finding what goes 9, the walk 20
// with two pages a thread (51 with one; four spill); as three kernels, with keys
// and accounts moved by all compute units, 50.5 beside 47.6.
template <int THREADS, bool IN_LDS>
__global__ __launch_bounds__(THREADS) void evict_kernel(EvictParams p) {
    constexpr int kWaves = THREADS / 64, kOwn = kBins / THREADS, kOwnPages = THREADS == 1024 ? 2 : 1;
    extern __shared__ uint64_t keys[];
    __shared__ int bins[kBins];
    __shared__ int scan[kWaves];
    __shared__ uint64_t ends[2][kWaves];
    __shared__ uint64_t few[kFew];
    __shared__ int found[3], n_few;
    const int64_t s = (int64_t)p.first_block + blockIdx.x;
    const int tid = (int)threadIdx.x, lane = tid & 63;
    const float* mass = p.mass + s * p.heads * p.max_pages;
    const int32_t* table = p.table + s * p.table_stride;
    const int32_t raw_len = p.lens[s];
    const int n = pages_of(p, raw_len);
    const int first = (int)(p.sink < n ? p.sink : n);
    const int last = (int)(n - p.recent > first ? n - p.recent : first);   // candidates are first .. last - 1
    const int64_t over = (int64_t)n - p.budget;
    const int count = (int)(over < 0 ? 0 : over < last - first ? over : last - first);
    auto key_of = [&](int page) {
        if constexpr (IN_LDS) return keys[page];
        else return key_from_accounts(p, mass, page);
    };

    uint64_t low = 0, high = ~0ull;   // the keys below low go, and the first `left` of those from low to high
    int left = count, inside = last - first;
    for (bool summed = false; left > 0; summed = true) {
        if (summed && inside <= kFew) {   // a thread for each, which counts those below it
            for (int i = first + tid; i < last; i += THREADS) {
                const uint64_t k = key_of(i);
                if (k >= low && k <= high) few[atomicAdd(&n_few, 1)] = k;
            }
            __syncthreads();
            if (tid < inside) {
                const uint64_t mine = few[tid];
                int less = 0, same = 0;
#pragma unroll 8
                for (int j = 0; j < inside; ++j) less += few[j] < mine, same += few[j] == mine;
                if (less < left && left <= less + same) ends[0][0] = mine, found[0] = less;
            }
            __syncthreads();
            low = high = ends[0][0];
            left -= found[0];
            break;
        }
        uint64_t least = ~0ull, most = 0;
#pragma unroll 1
        for (int i = first + tid; i < last; i += THREADS) {
            const uint64_t k = summed ? key_of(i) : key_from_accounts(p, mass, i);
            if (IN_LDS && !summed) keys[i] = k;
            if (k >= low && k <= high) least = k < least ? k : least, most = k > most ? k : most;
        }
        for (int m = 1; m < 64; m <<= 1) {
            const uint64_t a = (uint64_t)__shfl_xor((unsigned long long)least, m);
            const uint64_t b = (uint64_t)__shfl_xor((unsigned long long)most, m);
            least = a < least ? a : least, most = b > most ? b : most;
        }
        if (lane == 0) ends[0][tid / 64] = least, ends[1][tid / 64] = most;
        for (int i = tid; i < kBins; i += THREADS) bins[i] = 0;
        if (tid == 0) n_few = 0;
        __syncthreads();
        low = ends[0][0], high = ends[1][0];
#pragma unroll
        for (int w = 1; w < kWaves; ++w) {
            low = ends[0][w] < low ? ends[0][w] : low;
            high = ends[1][w] > high ? ends[1][w] : high;
        }
        if (low == high) break;
        const int bits = 64 - __clzll((long long)(high - low)), shift = bits > kDigitBits ? bits - kDigitBits : 0;
#pragma unroll 4
        for (int i = first + tid; i < last; i += THREADS) {
            const uint64_t k = key_of(i);
            if (k >= low && k <= high) atomicAdd(&bins[(int)((k - low) >> shift)], 1);
        }
        __syncthreads();
        // the bin where the count runs out
        int of[kOwn], own = 0, total;
#pragma unroll
        for (int j = 0; j < kOwn; ++j) own += of[j] = bins[kOwn * tid + j];
        int x = own;
        for (int m = 1; m < 64; m <<= 1) {
            const int y = __shfl_up(x, m);
            x += lane >= m ? y : 0;
        }
        int before = block_before<kWaves>(__shfl(x, 63), scan, total) + x - own;
#pragma unroll
        for (int j = 0; j < kOwn; ++j) {
            if (before < left && left <= before + of[j]) found[0] = kOwn * tid + j, found[1] = before, found[2] = of[j];
            before += of[j];
        }
        __syncthreads();
        low += (uint64_t)(uint32_t)found[0] << shift;
        const uint64_t width = ((uint64_t)1 << shift) - 1;
        if (high - low > width) high = low + width;
        left -= found[1];
        inside = found[2];
        if (left == inside) break;   // all of them go
    }
    int32_t* out_table = p.out_table + s * p.out_table_stride;
    float* out_mass = p.out_mass + s * p.heads * p.max_pages;
    int32_t* evicted = p.evicted + s * p.max_pages;
    // a wave has kOwnPages times 64 pages in a row, so that a part of the walk needs two sums over the waves
    int ties_before = 0, gone_before = 0;
    const uint64_t lower = (1ull << lane) - 1ull;
    for (int base = 0; base < p.max_pages; base += THREADS * kOwnPages) {
        const int at = base + tid / 64 * (64 * kOwnPages) + lane;
        int32_t id[kOwnPages];
        uint64_t below[kOwnPages], tie[kOwnPages];
        int of_wave = 0, total;
#pragma unroll
        for (int j = 0; j < kOwnPages; ++j) {
            const int i = at + j * 64;
            id[j] = i < n ? table[i] : -1;
            const bool may = count > 0 && i >= first && i < last;
            const uint64_t k = may ? key_of(i) : ~0ull;
            below[j] = __ballot(may && k < low);
            tie[j] = __ballot(may && k >= low && k <= high);
            of_wave += __popcll(tie[j]);
        }
        int rank = ties_before + block_before<kWaves>(of_wave, scan, total);
        ties_before += total;
        of_wave = 0;
#pragma unroll
        for (int j = 0; j < kOwnPages; ++j) {
            const bool goes = (tie[j] >> lane & 1) && rank + __popcll(tie[j] & lower) < left;
            rank += __popcll(tie[j]);
            below[j] |= __ballot(goes);   // all that go
            of_wave += __popcll(below[j]);
        }
        rank = gone_before + block_before<kWaves>(of_wave, scan, total);
        gone_before += total;
        int to[kOwnPages];   // where a page that stays moves, or -1 - where the id of one that goes is listed
#pragma unroll
        for (int j = 0; j < kOwnPages; ++j) {
            const int g = rank + __popcll(below[j] & lower);
            to[j] = (below[j] >> lane & 1) ? -1 - g : at + j * 64 - g;
            rank += __popcll(below[j]);
        }
        // every wave has read its share of this part before any of it is written; a barrier alone does not wait for loads
        for (int h = 0; h < p.heads; h += 8) {
            float m[8][kOwnPages];
#pragma unroll
            for (int c = 0; c < 8; ++c)
#pragma unroll
                for (int j = 0; j < kOwnPages; ++j)
                    m[c][j] = h + c < p.heads && at + j * 64 < n ? mass[(int64_t)(h + c) * p.max_pages + at + j * 64] : 0.f;
            __builtin_amdgcn_s_waitcnt(0);
            __syncthreads();
#pragma unroll
            for (int c = 0; c < 8; ++c)
#pragma unroll
                for (int j = 0; j < kOwnPages; ++j)
                    if (h + c < p.heads && at + j * 64 < n && to[j] >= 0)
                        out_mass[(int64_t)(h + c) * p.max_pages + to[j]] = m[c][j];
        }
#pragma unroll
        for (int j = 0; j < kOwnPages; ++j) {
            const int i = at + j * 64;
            if (i >= n) continue;
            if (to[j] >= 0) out_table[to[j]] = id[j];
            else evicted[-1 - to[j]] = id[j];
        }
    }
    __syncthreads();
    for (int i = tid; i < p.max_pages; i += THREADS) {
        if (i >= count) evicted[i] = -1;
        if (i >= n - count) {
            out_table[i] = -1;
            for (int h = 0; h < p.heads; ++h) out_mass[(int64_t)h * p.max_pages + i] = 0.f;
        }
    }
    if (tid == 0) {
        p.out_lens[s] = raw_len - count * p.page_tokens;
        p.n_evicted[s] = count;
    }
}

}  // namespace

extern "C" int ztcp_evict_pages(const float* mass, const int32_t* page_table, int64_t table_stride,
                                const int32_t* kv_lens, int64_t n_seqs, int64_t num_heads, int64_t max_pages,
                                int64_t num_tokens, int64_t budget, int64_t sink, int64_t recent, int32_t* out_table,
                                int64_t out_table_stride, float* out_mass, int32_t* out_lens, int32_t* evicted,
                                int32_t* n_evicted, void* stream) {
    arg_result(ZTCP_OK, "");
    const int64_t most = (int64_t)1 << 31;
    if (n_seqs < 0 || num_heads < 1 || max_pages < 1 || num_tokens < 1 || n_seqs >= most || num_heads >= most ||
        max_pages > most - 4096 || num_tokens >= most || max_pages > (most - 1) / num_tokens)
        return arg_result(ZTCP_EINVAL, "num_heads, max_pages, num_tokens must be positive, max_pages * num_tokens below 2^31, "
                                       "max_pages at most 2^31 - 4096");
    if (budget < 0 || sink < 0 || recent < 1)
        return arg_result(ZTCP_EINVAL, "budget and sink must not be negative, recent at least 1");
    if (n_seqs == 0) return ZTCP_OK;
    if (!mass || !page_table || !kv_lens || !out_table || !out_mass || !out_lens || !evicted || !n_evicted)
        return arg_result(ZTCP_EINVAL, "no array may be NULL");
    if (n_seqs > 1 && (table_stride < max_pages || out_table_stride < max_pages))
        return arg_result(ZTCP_EINVAL, "table strides must cover max_pages");
    struct Rows {
        const void* p;
        int64_t n, bytes, stride;
    };
    const int64_t row = 4 * max_pages, cells = n_seqs * num_heads;
    const Rows in[3] = {{page_table, n_seqs, row, 4 * table_stride}, {mass, cells, row, row}, {kv_lens, n_seqs, 4, 4}};
    const Rows out[5] = {{out_table, n_seqs, row, 4 * out_table_stride}, {out_mass, cells, row, row},
                         {out_lens, n_seqs, 4, 4}, {evicted, n_seqs, row, row}, {n_evicted, n_seqs, 4, 4}};
    auto meet = [](const Rows& a, const Rows& b) {
        return rows_overlap(a.p, a.n, a.bytes, a.stride, b.p, b.n, b.bytes, b.stride);
    };
    for (int o = 0; o < 5; ++o) {
        for (int i = 0; i < 3; ++i)
            if (!(o == i && out[o].p == in[i].p && out[o].stride == in[i].stride) && meet(out[o], in[i]))
                return arg_result(ZTCP_EOVERLAP, "an output may be its own input, and overlap no other");
        for (int i = 0; i < o; ++i)
            if (meet(out[o], out[i])) return arg_result(ZTCP_EOVERLAP, "outputs must not overlap each other");
    }
    EvictParams p{};
    p.mass = mass;
    p.table = page_table;
    p.table_stride = table_stride;
    p.lens = kv_lens;
    p.heads = (int32_t)num_heads;
    p.max_pages = (int32_t)max_pages;
    p.page_tokens = (int32_t)num_tokens;
    p.budget = budget;
    p.sink = sink;
    p.recent = recent;
    p.out_table = out_table;
    p.out_table_stride = out_table_stride;
    p.out_mass = out_mass;
    p.out_lens = out_lens;
    p.evicted = evicted;
    p.n_evicted = n_evicted;
    const size_t lds = max_pages <= kKeysInLds ? (size_t)max_pages * sizeof(uint64_t) : 0;
    auto go = [&](auto kernel, uint32_t threads) {
        // over 64 KiB of dynamic LDS has to be asked for
        if (lds > (size_t)48 * 1024 &&
            hipFuncSetAttribute((const void*)kernel, hipFuncAttributeMaxDynamicSharedMemorySize,
                                kKeysInLds * (int)sizeof(uint64_t)) != hipSuccess)
            return ZTCP_EHIP;
        launch_blocks(kernel, (uint64_t)n_seqs, threads, lds, (hipStream_t)stream, p);
        return hipGetLastError() == hipSuccess ? ZTCP_OK : ZTCP_EHIP;
    };
    if (max_pages <= 1024) return go(evict_kernel<256, true>, 256u);
    return lds ? go(evict_kernel<1024, true>, 1024u) : go(evict_kernel<1024, false>, 1024u);
}
