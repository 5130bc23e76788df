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
//
// All is latency: one workgroup, a few sequences to a thread, adds up once (sums that pass
// 2^32 stay there, which no limit reaches), and only if some sequence has to wait once
// more, for the rows granted.  Up to 4,096 rows it lays these out as well; more are laid
// out by a second launch, whose workgroups find their sequences by what the first left
// them.  64 decoding sequences: 4.6 us (9.6 a pass with an allocation for each output, 6.0
// with one); 2,048 sequences of 246,000 rows: 8.6 and 6 us (12 and 9 with sums of 64 bits,
// one sequence a thread, and searches in memory).

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
    int32_t* had;                    // for the second launch: free pages there were,
    int32_t* hints;                  // the sequence of each block's first row,
    int4* parts;                     // and of each sequence its first row, length, pages taken in front, count
    uint32_t first_block;            // of this launch
};

constexpr int kOneLaunchSeqs = 1024, kOneLaunchRows = 4096;
constexpr int kRowsABlock = 1024;

// Sums of rows and pages; what passes 2^32 stays at its end.
struct Sums {
    uint32_t rows, pages;
};
__device__ __forceinline__ uint32_t add(uint32_t a, uint32_t b) { return a + b < a ? ~0u : a + b; }
__device__ __forceinline__ Sums add(Sums a, Sums b) { return Sums{add(a.rows, b.rows), add(a.pages, b.pages)}; }

// The sum over the threads in front, and over all.
template <int WAVES>
__device__ __forceinline__ Sums sum_before(Sums x, Sums (&lds)[WAVES], Sums& all) {
    const int lane = (int)threadIdx.x & 63, wave = (int)threadIdx.x >> 6;
    Sums upto = x;
    for (int m = 1; m < 64; m <<= 1) {
        const Sums y{(uint32_t)__shfl_up((int)upto.rows, m), (uint32_t)__shfl_up((int)upto.pages, m)};
        if (lane >= m) upto = add(upto, y);
    }
    const Sums last{(uint32_t)__shfl_up((int)upto.rows, 1), (uint32_t)__shfl_up((int)upto.pages, 1)};
    __syncthreads();                                         // the sums of the turn before have been read
    if (lane == 63) lds[wave] = upto;
    __syncthreads();
    Sums before = lane > 0 ? last : Sums{0, 0};
    all = Sums{0, 0};
#pragma unroll
    for (int w = 0; w < WAVES; ++w) {
        const Sums y = lds[w];
        if (w < wave) before = add(before, y);
        all = add(all, y);
    }
    return before;
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

// The sequence of a row among parts low .. high: the last that starts at it or in front.
__device__ __forceinline__ int part_of(const int4* parts, int low, int high, int row) {
    while (low < high) {
        const int mid = (low + high + 1) >> 1;
        if (parts[mid].x <= row) low = mid;
        else high = mid - 1;
    }
    return low;
}

// ROWS: and the rows too (the sequences fit into one turn).
template <int THREADS, bool ROWS>
__global__ __launch_bounds__(THREADS) void plan_kernel(AllotParams p) {
    constexpr int kOwn = 4, kWaves = THREADS / 64;           // sequences of a thread, side by side
    __shared__ Sums lds[kWaves];
    __shared__ int4 parts[ROWS ? kOneLaunchSeqs : 1];
    const int tid = (int)threadIdx.x;
    const int had = (int)min((int64_t)max(*p.n_free, 0), p.capacity);
    Sums base{0, 0};
    int start = 0, taken = 0;                                // rows and pages granted in the turns before
    for (int first = 0; first < p.n_seqs; first += THREADS * kOwn) {
        const int s0 = first + tid * kOwn;
        int len[kOwn], want[kOwn], count[kOwn], need[kOwn];
#pragma unroll
        for (int i = 0; i < kOwn; ++i) {
            const bool is = s0 + i < p.n_seqs;
            len[i] = is ? p.lens[s0 + i] : 0;
            want[i] = is ? p.wanted[s0 + i] : 0;
            count[i] = is && p.counts ? p.counts[s0 + i] : 0;
        }
        Sums own{0, 0};
#pragma unroll
        for (int i = 0; i < kOwn; ++i) {
            len[i] = min(max(len[i], 0), p.max_tokens);
            want[i] = max(want[i], 0);
            if (want[i] > p.max_tokens - len[i]) want[i] = 0;
            if (!p.counts) count[i] = len[i];
            need[i] = pages_for(p, len[i] + want[i]) - pages_for(p, len[i]);
            own = add(own, Sums{(uint32_t)want[i], (uint32_t)need[i]});
        }
        Sums all;
        const Sums in_front = sum_before(own, lds, all);     // in this turn
        Sums upto = add(base, in_front);
        base = add(base, all);
        int before[kOwn];
        bool every = true;
#pragma unroll
        for (int i = 0; i < kOwn; ++i) {
            before[i] = (int)min(upto.pages, (uint32_t)had);
            upto = add(upto, Sums{(uint32_t)want[i], (uint32_t)need[i]});
            const bool served = upto.rows <= (uint64_t)p.max_rows && (need[i] == 0 || upto.pages <= (uint32_t)had);
            every &= served;
            if (!served) want[i] = need[i] = 0;
        }
        Sums granted = in_front, in_all = all;               // what is granted in front of this thread's, and to all, in this turn
        if (!__syncthreads_and(every)) {
            own = Sums{0, 0};
#pragma unroll
            for (int i = 0; i < kOwn; ++i) own = add(own, Sums{(uint32_t)want[i], (uint32_t)need[i]});
            granted = sum_before(own, lds, in_all);
        }
        int from = start + (int)granted.rows;
#pragma unroll
        for (int i = 0; i < kOwn; ++i) {
            const int s = s0 + i;
            if (s >= p.n_seqs) break;
            p.starts[s] = from;
            p.granted[s] = want[i];
            p.out_lens[s] = len[i] + want[i];
            if (p.out_counts) p.out_counts[s] = count[i] + want[i];
            const int4 part = make_int4(from, len[i], before[i], count[i]);
            if constexpr (ROWS) {
                parts[s] = part;
            } else {
                p.parts[s] = part;
                for (int block = (from + kRowsABlock - 1) / kRowsABlock; block * kRowsABlock < from + want[i]; ++block) p.hints[block] = s;
            }
            from += want[i];
        }
        start += (int)in_all.rows;
        taken += (int)in_all.pages;
    }
    if (tid == 0) {
        p.starts[p.n_seqs] = start;
        *p.out_n_free = had - taken;
        if (!ROWS) *p.had = had;
    }
    if constexpr (ROWS) {
        __syncthreads();
        for (int row = tid; row < p.max_rows; row += THREADS) {
            if (row >= start) {
                p.slots[row] = -1;
                p.positions[row] = 0;
                continue;
            }
            const int s = part_of(parts, 0, p.n_seqs - 1, row);
            const int4 part = parts[s];
            fill_row(p, row, s, part.x, part.y, part.z, part.w, had);
        }
    }
}

__global__ __launch_bounds__(256) void rows_kernel(AllotParams p) {
    __shared__ int4 parts[kRowsABlock];
    const int64_t block = (int64_t)p.first_block + blockIdx.x, row0 = block * kRowsABlock;
    const int total = p.starts[p.n_seqs], had = *p.had;
    int low = 0, high = 0;
    bool staged = false;
    if (row0 < total) {
        low = p.hints[block];
        high = row0 + kRowsABlock < total ? p.hints[block + 1] : p.n_seqs - 1;
        staged = high - low < kRowsABlock;
        if (staged)
            for (int i = (int)threadIdx.x; i <= high - low; i += 256) parts[i] = p.parts[low + i];
        __syncthreads();
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
        int s;
        int4 part;
        if (staged) {
            s = part_of(parts, 0, high - low, (int)row);
            part = parts[s];
            s += low;
        } else {
            s = part_of(p.parts, low, high, (int)row);
            part = p.parts[s];
        }
        fill_row(p, row, s, part.x, part.y, part.z, part.w, had);
    }
}

// ---- pages given back -------------------------------------------------------------
// Entries that are pages, in columns that a sequence's tokens do not reach, in the
// order of sequences and columns onto the end of the stack.  The first kernel counts
// them by pieces of rows, the second adds up what lies before its piece; a thread has
// all its entries of a piece on their way at once.  Of many thousand pieces, where adding up would be
// the work, one workgroup turns the counts into sums in between.  512 sequences of up to 4,098 columns,
// a quarter ended (17 MB): 6.5 and 7.5 us (6 and 14 with 256 columns at a time).

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
    int64_t* counts;                 // [2 + n_seqs * pieces]: free pages there were, entries of each piece
    bool summed;                     // counts[1 + i] are those in front of piece i
    uint32_t first_block;
};
constexpr int64_t kMostCounted = 4096;   // pieces whose counts every workgroup adds up itself

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
    const int spare = first_spare(p, s);
    int32_t id[kPiece / 256];
#pragma unroll
    for (int j = 0; j < kPiece / 256; ++j) {
        const int i = piece * kPiece + j * 256 + (int)threadIdx.x;
        id[j] = i < end && i >= spare ? row[i] : -1;
    }
    int64_t n = 0;
#pragma unroll
    for (int j = 0; j < kPiece / 256; ++j) n += id[j] >= 0;
    n = block_sum(n, lds);
    if (threadIdx.x == 0) {
        p.counts[1 + unit] = n;
        if (unit == 0) p.counts[0] = min((int64_t)max(*p.n_free, 0), p.capacity);
    }
}

// Counts into what lies in front of each, and all behind the last.
__global__ __launch_bounds__(1024) void release_sum_kernel(ReleaseParams p) {
    constexpr int kOwn = 4;
    __shared__ int64_t lds[16];
    const int tid = (int)threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int64_t units = (int64_t)p.n_seqs * p.pieces;
    int64_t before = 0;
    for (int64_t first = 0; first < units; first += 1024 * kOwn) {
        int64_t n[kOwn], own = 0;
#pragma unroll
        for (int j = 0; j < kOwn; ++j) {
            const int64_t i = first + tid * kOwn + j;
            own += n[j] = i < units ? p.counts[1 + i] : 0;
        }
        int64_t upto = own;
        for (int m = 1; m < 64; m <<= 1) {
            const int64_t y = (int64_t)__shfl_up((long long)upto, m);
            upto += lane >= m ? y : 0;
        }
        __syncthreads();                                     // the sums of the turn before have been read
        if (lane == 63) lds[wave] = upto;
        __syncthreads();
        int64_t at = before + upto - own;
#pragma unroll
        for (int w = 0; w < 16; ++w) {
            at += w < wave ? lds[w] : 0;
            before += lds[w];
        }
#pragma unroll
        for (int j = 0; j < kOwn; ++j) {
            const int64_t i = first + tid * kOwn + j;
            if (i < units) p.counts[1 + i] = at;
            at += n[j];
        }
    }
    if (tid == 0) p.counts[1 + units] = before;
}

__global__ __launch_bounds__(256) void release_kernel(ReleaseParams p) {
    __shared__ int64_t lds[4];
    __shared__ int scan[64];
    static_assert(kPiece / 256 * 4 == 64, "a lane for each wave's part");
    const int64_t unit = (int64_t)p.first_block + blockIdx.x;
    const int s = (int)(unit / p.pieces), piece = (int)(unit % p.pieces);
    const int tid = (int)threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int32_t* row = p.table + s * p.table_stride;
    int32_t* out = p.out_table + s * p.out_table_stride;
    int64_t at = 0;
    if (p.summed) {
        at = p.counts[1 + unit];
    } else {
        for (int64_t i = tid; i < unit; i += 256) at += p.counts[1 + i];
        at = block_sum(at, lds);
    }
    at += p.counts[0];
    auto count = [&](int64_t of) { return p.summed ? p.counts[2 + of] - p.counts[1 + of] : p.counts[1 + of]; };
    const int64_t last = (int64_t)p.n_seqs * p.pieces - 1, here = count(unit);
    if (piece == 0 && tid == 0) {
        int64_t n = 0;
        for (int i = 0; i < p.pieces; ++i) n += count(unit + i);
        p.released[s] = (int32_t)(min(at + n, p.capacity) - min(at, p.capacity));
    }
    if (unit == last && tid == 0) *p.out_n_free = (int32_t)min(at + here, p.capacity);
    const int begin = piece * kPiece, end = (int)min((int64_t)begin + kPiece, (int64_t)p.max_pages), spare = first_spare(p, s);
    const bool moved = out != row;
    if (!moved && here == 0) return;
    constexpr int kOwn = kPiece / 256;
    int32_t id[kOwn];
#pragma unroll
    for (int j = 0; j < kOwn; ++j) {
        const int i = begin + j * 256 + tid;
        id[j] = i < end && (moved || i >= spare) ? row[i] : -1;
    }
#pragma unroll
    for (int j = 0; j < kOwn; ++j) {
        const uint64_t all = __ballot(begin + j * 256 + tid >= spare && id[j] >= 0);
        if (lane == 0) scan[4 * j + wave] = __popcll(all);
    }
    __syncthreads();
    int upto = scan[lane];                                    // of 256 columns' four waves' counts, in their order
    const int mine = upto;
    for (int m = 1; m < 64; m <<= 1) {
        const int y = __shfl_up(upto, m);
        upto += lane >= m ? y : 0;
    }
    upto -= mine;
#pragma unroll
    for (int j = 0; j < kOwn; ++j) {
        const int i = begin + j * 256 + tid;
        const bool goes = i >= spare && id[j] >= 0;
        const int64_t to = at + __shfl(upto, 4 * j + wave) + __popcll(__ballot(goes) & ((1ull << lane) - 1));
        const bool fits = goes && to < p.capacity;
        if (fits) p.free_pages[to] = id[j];
        if (i < end && (moved || fits)) out[i] = fits ? -1 : id[j];
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

extern "C" size_t ztcp_allot_pages_workspace(int64_t n_seqs, int64_t max_rows) {
    if (n_seqs < 0 || n_seqs >= (int64_t)1 << 24 || max_rows < 0 || max_rows >= ((int64_t)1 << 31) - 1024) return (size_t)-1;
    if (n_seqs <= kOneLaunchSeqs && max_rows <= kOneLaunchRows) return 0;
    const int64_t blocks = (max_rows + kRowsABlock - 1) / kRowsABlock;
    return (size_t)(n_seqs * (int64_t)sizeof(int4) + 4 * (blocks + 1));
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
    const size_t need = ztcp_allot_pages_workspace(n_seqs, max_rows);
    if (need > 0 && (!workspace || workspace_bytes < need || !hot_aligned(workspace)))
        return arg_result(ZTCP_EINVAL, "workspace must hold ztcp_allot_pages_workspace bytes, 16-byte aligned");
    const int64_t seqs = 4 * n_seqs;
    const Span in[5] = {flat(kv_lens, seqs), flat(n_free, 4), flat(next_positions, seqs), flat(q_lens, seqs), flat(free_pages, 4 * capacity)};
    const Span out[9] = {flat(out_lens, seqs), flat(out_n_free, 4), flat(out_next_positions, seqs), flat(q_starts, seqs + 4),
                         flat(granted, seqs), flat(slots, 8 * max_rows), flat(positions, 4 * max_rows),
                         flat(need ? workspace : nullptr, (int64_t)need), Span{page_table, n_seqs, 4 * max_pages, 4 * table_stride}};
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
    if (need == 0) {
        if (max_rows <= 1024) hipLaunchKernelGGL((plan_kernel<256, true>), dim3(1), dim3(256), 0, (hipStream_t)stream, p);
        else hipLaunchKernelGGL((plan_kernel<1024, true>), dim3(1), dim3(1024), 0, (hipStream_t)stream, p);
    } else {
        p.parts = (int4*)workspace;
        p.had = (int32_t*)(p.parts + n_seqs);
        p.hints = p.had + 1;
        hipLaunchKernelGGL((plan_kernel<1024, false>), dim3(1), dim3(1024), 0, (hipStream_t)stream, p);
        launch_blocks(rows_kernel, (uint64_t)((max_rows + kRowsABlock - 1) / kRowsABlock), 256, 0, (hipStream_t)stream, p);
    }
    return hipGetLastError() == hipSuccess ? ZTCP_OK : ZTCP_EHIP;
}

extern "C" size_t ztcp_release_pages_workspace(int64_t n_seqs, int64_t max_pages) {
    if (n_seqs < 0 || n_seqs >= (int64_t)1 << 24 || max_pages < 1 || max_pages >= (int64_t)1 << 31) return (size_t)-1;
    return (size_t)(2 + n_seqs * release_pieces(max_pages)) * sizeof(int64_t);
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
    p.summed = units > kMostCounted;
    launch_blocks(release_count_kernel, units, 256, 0, (hipStream_t)stream, p);
    if (p.summed) hipLaunchKernelGGL(release_sum_kernel, dim3(1), dim3(1024), 0, (hipStream_t)stream, p);
    launch_blocks(release_kernel, units, 256, 0, (hipStream_t)stream, p);
    return hipGetLastError() == hipSuccess ? ZTCP_OK : ZTCP_EHIP;
}
