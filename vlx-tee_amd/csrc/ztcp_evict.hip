// ztcp_evict.hip -- which pages of a sequence go cold: those with the least
// accumulated attention weight.
#include "ztcp_hot.h"

using namespace ztcp;

namespace {

constexpr int kDigitBits = 11;
constexpr int kBins = 1 << kDigitBits;
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

// One workgroup per sequence.  The page that the count-th smallest key belongs
// to is found digit by digit from the highest bit in which the keys differ (11
// bits at a time: a histogram of the keys that share the digits found so far,
// then the bin in which the count runs out); pages below it go, and of the pages
// equal to it the first ones.  Then one walk in page order closes the gaps: a
// page moves down by the number of pages gone before it, so that a chunk that
// has been read whole may be written over itself.
template <int THREADS>
__global__ __launch_bounds__(THREADS) void evict_kernel(EvictParams p) {
    constexpr int kWaves = THREADS / 64, kOwn = kBins / THREADS;
    extern __shared__ uint64_t keys[];
    __shared__ int bins[kBins];
    __shared__ int scan[kWaves];
    __shared__ uint64_t same[2][kWaves];
    __shared__ int found[3];
    const int64_t s = blockIdx.x;
    const int tid = (int)threadIdx.x, lane = tid & 63;
    const float* mass = p.mass + s * p.heads * p.max_pages;
    const int32_t* table = p.table + s * p.table_stride;
    const int32_t raw_len = p.lens[s];
    const int32_t len = raw_len < 0 ? 0 : raw_len;
    const int64_t want = ((int64_t)len + p.page_tokens - 1) / p.page_tokens;
    const int n = (int)(want < p.max_pages ? want : p.max_pages);
    const int first = (int)(p.sink < n ? p.sink : n);
    const int last = (int)(n - p.recent > first ? n - p.recent : first);   // candidates are first .. last - 1
    const int64_t over = (int64_t)n - p.budget;
    const int count = (int)(over < 0 ? 0 : over < last - first ? over : last - first);
    const bool in_lds = p.max_pages <= kKeysInLds;
    auto key_of = [&](int page) { return in_lds ? keys[page] : key_from_accounts(p, mass, page); };

    uint64_t bound = 0;   // the count-th smallest key's digits found so far
    int shift = 64, left = count, ties = 0;
    if (count > 0) {
        uint64_t all = ~0ull, any = 0;
#pragma unroll 4
        for (int i = first + tid; i < last; i += THREADS) {
            const uint64_t k = key_from_accounts(p, mass, i);
            if (in_lds) keys[i] = k;
            all &= k, any |= k;
        }
        for (int m = 1; m < 64; m <<= 1) {
            all &= (uint64_t)__shfl_xor((unsigned long long)all, m);
            any |= (uint64_t)__shfl_xor((unsigned long long)any, m);
        }
        if (lane == 0) same[0][tid / 64] = all, same[1][tid / 64] = any;
        __syncthreads();
        for (int w = 0; w < kWaves; ++w) all &= same[0][w], any |= same[1][w];
        shift = all == any ? 0 : 64 - __clzll((long long)(all ^ any));
        bound = shift < 64 ? all >> shift << shift : 0;
        ties = last - first;   // what is left of the keys if they are all equal
        while (shift > 0) {
            const int bits = shift < kDigitBits ? shift : kDigitBits;
            const int next = shift - bits;
            for (int i = tid; i < kBins; i += THREADS) bins[i] = 0;
            __syncthreads();
            for (int i = first + tid; i < last; i += THREADS) {
                const uint64_t k = key_of(i);
                if (shift == 64 || ((k ^ bound) >> shift) == 0)
                    atomicAdd(&bins[(int)((k >> next) & ((1u << bits) - 1u))], 1);
            }
            __syncthreads();
            // the bin where the count runs out
            int of[kOwn], own = 0;
#pragma unroll
            for (int j = 0; j < kOwn; ++j) own += of[j] = bins[kOwn * tid + j];
            int x = own;
            for (int m = 1; m < 64; m <<= 1) {
                const int y = __shfl_up(x, m);
                x += lane >= m ? y : 0;
            }
            int total;
            int before = block_before<kWaves>(__shfl(x, 63), scan, total) + x - own;
#pragma unroll
            for (int j = 0; j < kOwn; ++j) {
                if (before < left && left <= before + of[j]) found[0] = kOwn * tid + j, found[1] = before, found[2] = of[j];
                before += of[j];
            }
            __syncthreads();
            bound |= (uint64_t)(uint32_t)found[0] << next;
            left -= found[1];
            ties = found[2];
            shift = next;
            __syncthreads();
            if (left == ties) break;   // every key with these digits goes
        }
    }
    int32_t* out_table = p.out_table + s * p.out_table_stride;
    float* out_mass = p.out_mass + s * p.heads * p.max_pages;
    int32_t* evicted = p.evicted + s * p.max_pages;
    // a page goes if its digits are below the bound's, or equal and it is among the first `left` of those
    int ties_before = 0, gone_before = 0;
    for (int base = 0; base < p.max_pages; base += THREADS) {
        const int i = base + tid;
        const bool may = count > 0 && i >= first && i < last;
        const uint64_t k = may ? key_of(i) >> shift : ~0ull;
        const bool below = may && k < (bound >> shift), tie = may && k == (bound >> shift);
        const uint64_t lower = (1ull << lane) - 1ull;
        const uint64_t tm = __ballot(tie);
        int t_total, g_total;
        const int t_at = ties_before + block_before<kWaves>(__popcll(tm), scan, t_total) + __popcll(tm & lower);
        const bool gone = below || (tie && t_at < left);
        const uint64_t gm = __ballot(gone);
        const int g_at = gone_before + block_before<kWaves>(__popcll(gm), scan, g_total) + __popcll(gm & lower);
        const int32_t id = i < n ? table[i] : -1;
        const bool kept = i < n && !gone;
        const int to = i - g_at;
        // every wave has read its part of this chunk before any of it is written; a barrier alone does not wait for loads
        for (int h0 = 0; h0 < p.heads; h0 += 8) {
            float m[8];
#pragma unroll
            for (int h = 0; h < 8; ++h)
                m[h] = kept && h0 + h < p.heads ? mass[(int64_t)(h0 + h) * p.max_pages + i] : 0.f;
            __builtin_amdgcn_s_waitcnt(0);
            __syncthreads();
#pragma unroll
            for (int h = 0; h < 8; ++h)
                if (kept && h0 + h < p.heads) out_mass[(int64_t)(h0 + h) * p.max_pages + to] = m[h];
        }
        if (kept) out_table[to] = id;
        if (gone) evicted[g_at] = id;
        ties_before += t_total;
        gone_before += g_total;
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
        max_pages >= most || num_tokens >= most || max_pages > (most - 1) / num_tokens)
        return arg_result(ZTCP_EINVAL, "num_heads, max_pages, num_tokens must be positive, max_pages * num_tokens below 2^31");
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
        hipLaunchKernelGGL(kernel, dim3((uint32_t)n_seqs), dim3(threads), lds, (hipStream_t)stream, p);
        return hipGetLastError() == hipSuccess ? ZTCP_OK : ZTCP_EHIP;
    };
    return max_pages <= 1024 ? go(evict_kernel<256>, 256u) : go(evict_kernel<1024>, 1024u);
}
