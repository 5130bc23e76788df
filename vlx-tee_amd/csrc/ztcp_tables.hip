// ztcp_tables.hip -- page tables kept on the GPU: pages for a step's new
// tokens, their slots and positions, and pages given back.
#include "ztcp_hot.h"

using namespace ztcp;

namespace {

// ---- pages for new tokens ---------------------------------------------------------
// With L tokens held and q asked for (0 if the table's columns do not hold L + q),
// a sequence needs ceil((L + q) / t) - ceil(L / t) pages of t tokens.  Sums R and P
// of what has been asked for up to a sequence decide alone whether it gets all or
// nothing: R <= max_rows and, if it needs a page, P <= n_free.  No sequence's turn
// depends on another's outcome then, and since both sums only grow, those that get
// pages have all that were asked for before them: the stack is taken from its end
// without gaps, page i of a sequence from place n_free - 1 - (P - needed) - i.
//
// Every new page begins with a new token, whose row writes the table's entry.

struct AllotParams {
    int32_t* table;
    int64_t table_stride;
    const int32_t* lens;
    const int32_t* wanted;
    const int32_t* free_pages;
    const int32_t* n_free;
    const int32_t* counts;           // positions of the sequences' next tokens, or nullptr: their lengths
    int64_t capacity, max_rows;      // of free_pages; of slots and positions
    int32_t n_seqs, max_tokens, page_tokens;
    DivBy page_div;
    int32_t* out_lens;
    int32_t* out_n_free;
    int32_t* out_counts;
    int32_t* starts;
    int64_t* slots;
    int32_t* positions;
    int32_t* granted;
    int32_t* before;                 // [n_seqs] pages taken by the sequences in front
    int32_t* had;                    // free pages there were
    uint32_t first_block;            // of this launch
};

constexpr int kPlanThreads = 1024;
constexpr int kOneLaunchRows = 4096;

struct Sum2 {
    int64_t rows, pages;
};
__device__ __forceinline__ Sum2 up(Sum2 x, int m) {
    return Sum2{(int64_t)__shfl_up((long long)x.rows, m), (int64_t)__shfl_up((long long)x.pages, m)};
}

// Pages that hold so many tokens.
__device__ __forceinline__ int pages_for(const AllotParams& p, int tokens) {
    return tokens > 0 ? div_page(tokens - 1, p.page_div) + 1 : 0;
}

// One new token: its slot and position, and its page's entry if it is the page's first.
__device__ __forceinline__ void fill_row(const AllotParams& p, int64_t row, int s, int start, int len, int before, int count, int had) {
    const int nth = (int)row - start, place = len + nth;
    const int page = div_page(place, p.page_div), in_page = place - page * p.page_tokens;
    const int fresh = page - pages_for(p, len);              // which of the sequence's new pages; below 0: one that it held
    int32_t* cell = p.table + s * p.table_stride + page;
    int32_t id;
    if (fresh >= 0) {
        id = p.free_pages[had - 1 - before - fresh];
        if (in_page == 0) *cell = id;
    } else {
        id = *cell;
    }
    p.slots[row] = id >= 0 ? (int64_t)id * p.page_tokens + in_page : -1;
    p.positions[row] = count + nth;
}

// Sums over the sequences, by one workgroup; ROWS: and the rows too (sequences fit into one turn).
template <bool ROWS>
__global__ __launch_bounds__(kPlanThreads) void plan_kernel(AllotParams p) {
    __shared__ Sum2 waves[kPlanThreads / 64];
    __shared__ int32_t granted_upto[ROWS ? kPlanThreads : kPlanThreads / 64];
    __shared__ int32_t lens[ROWS ? kPlanThreads : 1], before_of[ROWS ? kPlanThreads : 1], counts[ROWS ? kPlanThreads : 1];
    const int tid = (int)threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int had = (int)min((int64_t)max(*p.n_free, 0), p.capacity);
    Sum2 base{0, 0};
    int start = 0, taken = 0;                                // rows and pages granted in the turns before
    for (int first = 0; first < p.n_seqs; first += kPlanThreads) {
        const int s = first + tid;
        const bool is = s < p.n_seqs;
        const int len = is ? min(max(p.lens[s], 0), p.max_tokens) : 0;
        int want = is ? max(p.wanted[s], 0) : 0;
        if (want > p.max_tokens - len) want = 0;
        const int count = is ? (p.counts ? p.counts[s] : len) : 0;
        const int need = pages_for(p, len + want) - pages_for(p, len);
        Sum2 x{want, need};
        for (int m = 1; m < 64; m <<= 1) {
            const Sum2 y = up(x, m);
            if (lane >= m) x.rows += y.rows, x.pages += y.pages;
        }
        __syncthreads();                                     // the last turn's sums have been read
        if (lane == 63) waves[wave] = x;
        __syncthreads();
        x.rows += base.rows, x.pages += base.pages;
#pragma unroll
        for (int w = 0; w < kPlanThreads / 64; ++w) {
            const Sum2 y = waves[w];
            if (w < wave) x.rows += y.rows, x.pages += y.pages;
            base.rows += y.rows, base.pages += y.pages;
        }
        const bool served = x.rows <= p.max_rows && (need == 0 || x.pages <= had);
        const int grant = served ? want : 0, before = (int)min(x.pages - need, (int64_t)had);
        // rows granted: a second sum, of at most max_rows
        int g = grant;
        for (int m = 1; m < 64; m <<= 1) {
            const int y = __shfl_up(g, m);
            if (lane >= m) g += y;
        }
        int most = served && need > 0 ? (int)x.pages : 0;    // pages taken up to the last one served
        for (int m = 1; m < 64; m <<= 1) most = max(most, __shfl_xor(most, m));
        __shared__ int32_t rows_of[kPlanThreads / 64], pages_of[kPlanThreads / 64];
        if (lane == 63) rows_of[wave] = g, pages_of[wave] = most;
        __syncthreads();
        int from = start;
#pragma unroll
        for (int w = 0; w < kPlanThreads / 64; ++w) {
            if (w < wave) from += rows_of[w];
            start += rows_of[w];
            taken = max(taken, pages_of[w]);
        }
        from += g - grant;
        if (is) {
            p.starts[s] = from;
            p.granted[s] = grant;
            p.out_lens[s] = len + grant;
            if (p.out_counts) p.out_counts[s] = count + grant;
            if (!ROWS) p.before[s] = before;
        }
        if constexpr (ROWS) {
            granted_upto[tid] = from + grant;
            lens[tid] = len, before_of[tid] = before, counts[tid] = count;
        }
    }
    if (tid == 0) {
        p.starts[p.n_seqs] = start;
        *p.out_n_free = had - taken;
        if (!ROWS) *p.had = had;
    }
    if constexpr (ROWS) {
        __syncthreads();
        for (int row = tid; row < p.max_rows; row += kPlanThreads) {
            if (row >= start) {
                p.slots[row] = -1;
                p.positions[row] = 0;
                continue;
            }
            int low = 0, high = p.n_seqs - 1;                // the first sequence that ends behind the row
            while (low < high) {
                const int mid = (low + high) >> 1;
                if (granted_upto[mid] > row) high = mid;
                else low = mid + 1;
            }
            fill_row(p, row, low, low ? granted_upto[low - 1] : 0, lens[low], before_of[low], counts[low], had);
        }
    }
}

constexpr int kRowsABlock = 1024;

__global__ __launch_bounds__(256) void rows_kernel(AllotParams p) {
    const int64_t row0 = ((int64_t)p.first_block + blockIdx.x) * kRowsABlock;
    const int total = p.starts[p.n_seqs], had = *p.had;
    int low0 = 0, high0 = 0;
    if (row0 < total) {
        low0 = find_above(p.starts + 1, p.n_seqs, (int)row0);
        high0 = find_above(p.starts + 1, p.n_seqs, (int)min(row0 + kRowsABlock, (int64_t)total) - 1);
    }
#pragma unroll
    for (int i = 0; i < kRowsABlock / 256; ++i) {
        const int64_t row = row0 + i * 256 + (int)threadIdx.x;
        if (row >= p.max_rows) return;
        if (row >= total) {
            p.slots[row] = -1;
            p.positions[row] = 0;
            continue;
        }
        int low = low0, high = high0;
        while (low < high) {
            const int mid = (low + high) >> 1;
            if (p.starts[mid + 1] > row) high = mid;
            else low = mid + 1;
        }
        const int grant = p.granted[low];
        const int len = p.out_lens[low] - grant;             // lengths and counts may have been updated in place
        const int count = p.out_counts ? p.out_counts[low] - grant : len;
        fill_row(p, row, low, p.starts[low], len, p.before[low], count, had);
    }
}

// ---- pages given back -------------------------------------------------------------
// Entries that are pages, in columns that a sequence's tokens do not reach, in the
// order of sequences and columns onto the end of the stack.  The first kernel counts
// them by pieces of rows, the second adds up what lies before its piece.

constexpr int kPiece = 4096;        // columns

struct ReleaseParams {
    const int32_t* table;
    int64_t table_stride;
    const int32_t* lens;
    int32_t* free_pages;
    const int32_t* n_free;
    int64_t capacity;
    int32_t n_seqs, max_pages, page_tokens, pieces;
    int32_t* out_table;
    int64_t out_table_stride;
    int32_t* out_n_free;
    int32_t* released;
    int64_t* counts;                 // [1 + n_seqs * pieces]: free pages there were, entries of each piece
    uint32_t first_block;
};

__device__ __forceinline__ int first_spare(const ReleaseParams& p, int s) {
    const int64_t n = ((int64_t)max(p.lens[s], 0) + p.page_tokens - 1) / p.page_tokens;
    return (int)min(n, (int64_t)p.max_pages);
}

template <class T>
__device__ __forceinline__ T block_sum(T x, T* lds) {        // of 256 threads
    for (int m = 1; m < 64; m <<= 1) x += (T)__shfl_xor((long long)x, m);
    __syncthreads();
    if ((threadIdx.x & 63u) == 0) lds[threadIdx.x / 64] = x;
    __syncthreads();
    return lds[0] + lds[1] + lds[2] + lds[3];
}

__global__ __launch_bounds__(256) void release_count_kernel(ReleaseParams p) {
    __shared__ int64_t lds[4];
    const int64_t unit = (int64_t)p.first_block + blockIdx.x;
    const int s = (int)(unit / p.pieces), piece = (int)(unit % p.pieces);
    const int32_t* row = p.table + s * p.table_stride;
    const int end = (int)min((int64_t)(piece + 1) * kPiece, (int64_t)p.max_pages);
    int64_t n = 0;
    for (int i = max(piece * kPiece, first_spare(p, s)) + (int)threadIdx.x; i < end; i += 256) n += row[i] >= 0;
    n = block_sum(n, lds);
    if (threadIdx.x == 0) {
        p.counts[1 + unit] = n;
        if (unit == 0) p.counts[0] = min((int64_t)max(*p.n_free, 0), p.capacity);
    }
}

__global__ __launch_bounds__(256) void release_kernel(ReleaseParams p) {
    __shared__ int64_t lds[4];
    __shared__ int scan[2][4];
    const int64_t unit = (int64_t)p.first_block + blockIdx.x;
    const int s = (int)(unit / p.pieces), piece = (int)(unit % p.pieces);
    const int tid = (int)threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int32_t* row = p.table + s * p.table_stride;
    int32_t* out = p.out_table + s * p.out_table_stride;
    int64_t at = 0;
    for (int64_t i = tid; i < unit; i += 256) at += p.counts[1 + i];
    const int64_t had = p.counts[0];
    at = had + block_sum(at, lds);
    const int64_t last = (int64_t)p.n_seqs * p.pieces - 1;
    if (piece == 0 && tid == 0) {
        int64_t n = 0;
        for (int i = 0; i < p.pieces; ++i) n += p.counts[1 + unit + i];
        p.released[s] = (int32_t)(min(at + n, p.capacity) - min(at, p.capacity));
    }
    if (unit == last && tid == 0) *p.out_n_free = (int32_t)min(at + p.counts[1 + unit], p.capacity);
    const int begin = piece * kPiece, end = (int)min((int64_t)begin + kPiece, (int64_t)p.max_pages), spare = first_spare(p, s);
    const bool moved = out != row;
    for (int base = moved ? begin : max(begin, spare / 256 * 256), turn = 0; base < end; base += 256, turn ^= 1) {
        const int i = base + tid;
        const int32_t id = i < end ? row[i] : -1;
        const bool goes = i >= spare && id >= 0;
        const uint64_t all = __ballot(goes);
        if (lane == 0) scan[turn][wave] = __popcll(all);
        __syncthreads();
        int64_t to = at + __popcll(all & ((1ull << lane) - 1));
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            const int n = scan[turn][w];
            if (w < wave) to += n;
            at += n;
        }
        const bool fits = goes && to < p.capacity;
        if (fits) p.free_pages[to] = id;
        if (i < end && (moved || fits)) out[i] = fits ? -1 : id;
    }
}

// No sequence: nothing is released.
__global__ void keep_free_kernel(ReleaseParams p) { *p.out_n_free = (int32_t)min((int64_t)max(*p.n_free, 0), p.capacity); }

const char* check_table(const void* table, int64_t stride, int64_t n_seqs, int64_t max_pages, int64_t num_tokens) {
    const int64_t most = (int64_t)1 << 31;
    if (n_seqs < 0 || n_seqs >= (int64_t)1 << 24) return "n_seqs must be 0 .. 2^24 - 1";
    if (num_tokens < 1 || max_pages < 1 || num_tokens >= most || max_pages > (most - 1024) / num_tokens)
        return "num_tokens and max_pages must be positive, their product below 2^31 - 1024";
    if (n_seqs > 0 && !table) return "page_table must not be NULL";
    if (n_seqs > 1 && stride < max_pages) return "table_stride must cover max_pages";
    return nullptr;
}

struct Span {
    const void* p;
    int64_t n, bytes, stride;
};
bool meet(const Span& a, const Span& b) { return rows_overlap(a.p, a.n, a.bytes, a.stride, b.p, b.n, b.bytes, b.stride); }
Span flat(const void* p, int64_t bytes) { return Span{p, 1, bytes, bytes}; }

int64_t release_pieces(int64_t max_pages) { return (max_pages + kPiece - 1) / kPiece; }

}  // namespace

extern "C" size_t ztcp_allot_pages_workspace(int64_t n_seqs) {
    return n_seqs < 0 || n_seqs >= (int64_t)1 << 24 ? (size_t)-1 : (size_t)(n_seqs + 1) * sizeof(int32_t);
}

extern "C" int ztcp_allot_pages(int32_t* page_table, int64_t table_stride, int64_t max_pages, const int32_t* kv_lens,
                                const int32_t* q_lens, int64_t n_seqs, const int32_t* free_pages, int64_t capacity,
                                const int32_t* n_free, const int32_t* next_positions, int64_t num_tokens, int64_t max_rows,
                                int32_t* out_lens, int32_t* out_n_free, int32_t* out_next_positions, int32_t* q_starts,
                                int64_t* slots, int32_t* positions, int32_t* granted, void* workspace, size_t workspace_bytes,
                                void* stream) {
    arg_result(ZTCP_OK, "");
    const int64_t most = (int64_t)1 << 31;
    if (const char* why = check_table(page_table, table_stride, n_seqs, max_pages, num_tokens)) return arg_result(ZTCP_EINVAL, why);
    if (max_rows < 0 || max_rows >= most - 1024 || capacity < 0 || capacity >= most)
        return arg_result(ZTCP_EINVAL, "max_rows must be 0 .. 2^31 - 1025, capacity 0 .. 2^31 - 1");
    if ((next_positions == nullptr) != (out_next_positions == nullptr))
        return arg_result(ZTCP_EINVAL, "next_positions and out_next_positions must both be given or both be NULL");
    if (!n_free || !out_n_free || !q_starts || (capacity > 0 && !free_pages) || (max_rows > 0 && (!slots || !positions)) ||
        (n_seqs > 0 && (!kv_lens || !q_lens || !out_lens || !granted)))
        return arg_result(ZTCP_EINVAL, "no array may be NULL");
    const size_t need = ztcp_allot_pages_workspace(n_seqs);
    if (!workspace || workspace_bytes < need || ((uintptr_t)workspace & 3u) != 0)
        return arg_result(ZTCP_EINVAL, "workspace must hold ztcp_allot_pages_workspace bytes, 4-byte aligned");
    const int64_t seqs = 4 * n_seqs;
    const Span in[5] = {flat(kv_lens, seqs), flat(n_free, 4), flat(next_positions, seqs), flat(q_lens, seqs), flat(free_pages, 4 * capacity)};
    const Span out[9] = {flat(out_lens, seqs), flat(out_n_free, 4), flat(out_next_positions, seqs), flat(q_starts, seqs + 4),
                         flat(granted, seqs), flat(slots, 8 * max_rows), flat(positions, 4 * max_rows),
                         flat(workspace, (int64_t)need), Span{page_table, n_seqs, 4 * max_pages, 4 * table_stride}};
    for (int o = 0; o < 9; ++o) {
        for (int i = 0; i < 5; ++i)
            if (!(o == i && o < 3 && out[o].p == in[i].p) && meet(out[o], in[i]))
                return arg_result(ZTCP_EOVERLAP, "lengths, n_free and next_positions may be updated in place; nothing else may overlap");
        for (int i = 0; i < o; ++i)
            if (meet(out[o], out[i])) return arg_result(ZTCP_EOVERLAP, "outputs must not overlap each other or the workspace");
    }
    AllotParams p{};
    p.table = page_table;
    p.table_stride = table_stride;
    p.lens = kv_lens;
    p.wanted = q_lens;
    p.free_pages = free_pages;
    p.n_free = n_free;
    p.counts = next_positions;
    p.capacity = capacity;
    p.max_rows = max_rows;
    p.n_seqs = (int32_t)n_seqs;
    p.max_tokens = (int32_t)(max_pages * num_tokens);
    p.page_tokens = (int32_t)num_tokens;
    p.page_div = div_by((uint32_t)num_tokens);
    p.out_lens = out_lens;
    p.out_n_free = out_n_free;
    p.out_counts = out_next_positions;
    p.starts = q_starts;
    p.slots = slots;
    p.positions = positions;
    p.granted = granted;
    p.before = (int32_t*)workspace;
    p.had = (int32_t*)workspace + n_seqs;
    if (n_seqs <= kPlanThreads && max_rows <= kOneLaunchRows) {
        hipLaunchKernelGGL((plan_kernel<true>), dim3(1), dim3(kPlanThreads), 0, (hipStream_t)stream, p);
    } else {
        hipLaunchKernelGGL((plan_kernel<false>), dim3(1), dim3(kPlanThreads), 0, (hipStream_t)stream, p);
        launch_blocks(rows_kernel, (uint64_t)((max_rows + kRowsABlock - 1) / kRowsABlock), 256, 0, (hipStream_t)stream, p);
    }
    return hipGetLastError() == hipSuccess ? ZTCP_OK : ZTCP_EHIP;
}

extern "C" size_t ztcp_release_pages_workspace(int64_t n_seqs, int64_t max_pages) {
    if (n_seqs < 0 || n_seqs >= (int64_t)1 << 24 || max_pages < 1 || max_pages >= (int64_t)1 << 31) return (size_t)-1;
    return (size_t)(1 + n_seqs * release_pieces(max_pages)) * sizeof(int64_t);
}

extern "C" int ztcp_release_pages(const int32_t* page_table, int64_t table_stride, int64_t max_pages, const int32_t* kv_lens,
                                  int64_t n_seqs, int64_t num_tokens, int32_t* free_pages, int64_t capacity,
                                  const int32_t* n_free, int32_t* out_table, int64_t out_table_stride, int32_t* out_n_free,
                                  int32_t* n_released, void* workspace, size_t workspace_bytes, void* stream) {
    arg_result(ZTCP_OK, "");
    const int64_t most = (int64_t)1 << 31;
    if (const char* why = check_table(page_table, table_stride, n_seqs, max_pages, num_tokens)) return arg_result(ZTCP_EINVAL, why);
    if (capacity < 0 || capacity >= most) return arg_result(ZTCP_EINVAL, "capacity must be 0 .. 2^31 - 1");
    if (!n_free || !out_n_free || (capacity > 0 && !free_pages) || (n_seqs > 0 && (!kv_lens || !out_table || !n_released)))
        return arg_result(ZTCP_EINVAL, "no array may be NULL");
    if (n_seqs > 1 && out_table_stride < max_pages) return arg_result(ZTCP_EINVAL, "table strides must cover max_pages");
    const size_t need = ztcp_release_pages_workspace(n_seqs, max_pages);
    if (!workspace || workspace_bytes < need || ((uintptr_t)workspace & 7u) != 0)
        return arg_result(ZTCP_EINVAL, "workspace must hold ztcp_release_pages_workspace bytes, 8-byte aligned");
    const int64_t row = 4 * max_pages, seqs = 4 * n_seqs;
    const Span in[3] = {Span{page_table, n_seqs, row, 4 * table_stride}, flat(n_free, 4), flat(kv_lens, seqs)};
    const Span out[5] = {Span{out_table, n_seqs, row, 4 * out_table_stride}, flat(out_n_free, 4), flat(n_released, seqs),
                         flat(free_pages, 4 * capacity), flat(workspace, (int64_t)need)};
    for (int o = 0; o < 5; ++o) {
        for (int i = 0; i < 3; ++i)
            if (!(o == i && o < 2 && out[o].p == in[i].p && (out[o].n <= 1 || out[o].stride == in[i].stride)) && meet(out[o], in[i]))
                return arg_result(ZTCP_EOVERLAP, "the table and n_free may be updated in place; nothing else may overlap");
        for (int i = 0; i < o; ++i)
            if (meet(out[o], out[i])) return arg_result(ZTCP_EOVERLAP, "outputs must not overlap each other or the workspace");
    }
    ReleaseParams p{};
    p.table = page_table;
    p.table_stride = table_stride;
    p.lens = kv_lens;
    p.free_pages = free_pages;
    p.n_free = n_free;
    p.capacity = capacity;
    p.n_seqs = (int32_t)n_seqs;
    p.max_pages = (int32_t)max_pages;
    p.page_tokens = (int32_t)num_tokens;
    p.pieces = (int32_t)release_pieces(max_pages);
    p.out_table = out_table;
    p.out_table_stride = out_table_stride;
    p.out_n_free = out_n_free;
    p.released = n_released;
    p.counts = (int64_t*)workspace;
    if (n_seqs == 0) {
        hipLaunchKernelGGL(keep_free_kernel, dim3(1), dim3(1), 0, (hipStream_t)stream, p);
        return hipGetLastError() == hipSuccess ? ZTCP_OK : ZTCP_EHIP;
    }
    const uint64_t units = (uint64_t)n_seqs * (uint64_t)p.pieces;
    launch_blocks(release_count_kernel, units, 256, 0, (hipStream_t)stream, p);
    launch_blocks(release_kernel, units, 256, 0, (hipStream_t)stream, p);
    return hipGetLastError() == hipSuccess ? ZTCP_OK : ZTCP_EHIP;
}
