// ztcp_select.hip -- which pages of a long context a query attends over: bounds
// of each page's keys, a score made of them, and the pages of the highest scores.
//
// With lo_c and hi_c the least and the greatest number in column c of a page's
// keys, no key k of the page has q . k above
//     score = sum_c max(q_c lo_c, q_c hi_c) = q+ . hi + q- . lo,
// q+ and q- being q's positive and negative numbers with 0 in the others' place:
// two products of 16-bit numbers, which the matrix units make.
#include <type_traits>

#include "ztcp_hot.h"

using namespace ztcp;

namespace {

// ---- bounds -----------------------------------------------------------------------
// The pages that hold new tokens, over all of their tokens.  A wave takes the pages
// that begin, or whose sequence's new tokens begin, in a run of rows, and then another
// run; lanes lie along a token's elements, 8 each, and where these are fewer than 64
// lanes' the lanes' rest takes other tokens.  Bytes are the work: each key is read
// once, 8 loads in flight.

constexpr int kBoundsWaves = 8192;  // at most: 32 for each of 256 compute units

struct BoundsParams {
    PagedView batch;
    const uint8_t* k_pool;
    int64_t k_page;                  // elements between pages
    uint8_t* bounds;
    int64_t bounds_page;
    int32_t row_elements;            // of a token: KV heads times head_dim
    int32_t parts;                   // waves to a row's elements
};

// The pages of `run` rows from run0 on: part `part` of their elements.
template <int DT>
__device__ __forceinline__ void bounds_of(const BoundsParams& p, int64_t run0, int run, int part) {
    const int lane = (int)threadIdx.x & 63;
    const int64_t row_end = run0 + run;
    const int chunks = min(p.row_elements / 8 - 64 * part, 64);   // 16-byte pieces of a row that this wave has
    int width = 1;                                                // lanes along a row
    while (width < chunks) width <<= 1;
    const int chunk = lane % width, turn = lane / width, turns = 64 / width;
    const int64_t column = 8 * (int64_t)(64 * part + chunk);
    int64_t row = run0;
    for (int s = find_above(p.batch.starts + 1, p.batch.n_seqs, (int)run0); s < p.batch.n_seqs && row < row_end; ++s) {
        const Seq seq = uniform(seq_of(p.batch, s));
        row = max(row, (int64_t)seq.row0);
        while (row < min(row_end, (int64_t)seq.row0 + seq.n_new)) {
            const int place = seq.len - seq.n_new + (int)(row - seq.row0);
            if (place < 0) {
                row -= place;
                continue;
            }
            const int at = uniform(div_page(place, p.batch.page_div)), first = at * p.batch.page_tokens;
            const int tokens = min(p.batch.page_tokens, seq.len - first);
            const bool mine = row == seq.row0 || place == first;
            row += p.batch.page_tokens - (place - first);         // the next page's first token
            const int id = seq.table[at];
            if (!mine || id < 0 || id >= p.batch.n_pages) continue;
            const uint8_t* src = p.k_pool + 2 * ((int64_t)id * p.k_page + column);
            float lo[8], hi[8];
            uint32_t nan = 0;
#pragma unroll
            for (int e = 0; e < 8; ++e) lo[e] = INFINITY, hi[e] = -INFINITY;
            auto take = [&](const uint4& x) {
                const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const float y = e & 1 ? hot_hi<DT>(w[e / 2]) : hot_lo<DT>(w[e / 2]);
                    lo[e] = y < lo[e] ? y : lo[e];
                    hi[e] = y > hi[e] ? y : hi[e];
                    nan |= (y != y ? 1u : 0u) << e;
                }
            };
            const int64_t step = 2 * (int64_t)p.row_elements;
            if (chunk < chunks) {
                int t = turn;
                for (; t + 7 * turns < tokens; t += 8 * turns) {
                    uint4 x[8];
#pragma unroll
                    for (int i = 0; i < 8; ++i) x[i] = ldg16_once(src + (t + i * turns) * step);
#pragma unroll
                    for (int i = 0; i < 8; ++i) take(x[i]);
                }
                for (; t < tokens; t += turns) take(ldg16_once(src + t * step));
            }
            for (int m = width; m < 64; m <<= 1) {
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    lo[e] = fminf(lo[e], __shfl_xor(lo[e], m));
                    hi[e] = fmaxf(hi[e], __shfl_xor(hi[e], m));
                }
                nan |= (uint32_t)__shfl_xor((int)nan, m);
            }
            if (chunk >= chunks || turn != 0) continue;
#pragma unroll
            for (int e = 0; e < 8; ++e)
                if (nan >> e & 1) lo[e] = hi[e] = NAN;
            uint8_t* dst = p.bounds + 2 * ((int64_t)id * p.bounds_page + column);
            stg16(dst, 0, make_uint4(pack_hot<DT>(lo[0], lo[1]), pack_hot<DT>(lo[2], lo[3]), pack_hot<DT>(lo[4], lo[5]), pack_hot<DT>(lo[6], lo[7])));
            stg16(dst + step, 0, make_uint4(pack_hot<DT>(hi[0], hi[1]), pack_hot<DT>(hi[2], hi[3]), pack_hot<DT>(hi[4], hi[5]), pack_hot<DT>(hi[6], hi[7])));
        }
    }
}

template <int DT>
__global__ __launch_bounds__(256) void bounds_kernel(BoundsParams p) {
    const int wave = uniform((int)blockIdx.x * 4 + ((int)threadIdx.x >> 6)), waves = (int)gridDim.x * 4;
    const int64_t rows = min(max(p.batch.starts[p.batch.n_seqs], 0), p.batch.n_rows);
    // a page's rows to a run, fewer as long as there are waves enough without
    const int run = (int)min(max(rows * p.parts / kBoundsWaves, (int64_t)1), (int64_t)p.batch.page_tokens);
    for (int64_t unit = wave; unit / p.parts * run < rows; unit += waves) bounds_of<DT>(p, unit / p.parts * run, run, (int)(unit % p.parts));
}
// ---- scores -----------------------------------------------------------------------
// In fp32: pages are the rows of the products, (token, query head) pairs their columns,
// as many heads to a token as leave no column idle.  A wave keeps 16 pages' bounds of one
// KV head in registers and goes over a block of its sequence's new tokens; the greatest
// score of the KV head's query heads is what counts.

constexpr int kTilePages = 64;      // of a workgroup
constexpr int kBlockTokens = 64;

struct SelectParams {
    PagedView batch;
    const uint8_t* q;
    int64_t q_stride;
    const uint8_t* bounds;
    int64_t bounds_page;             // elements between pages
    int32_t kv_heads, group, head_dim;
    int32_t budget, sink, recent;
    int32_t score_stride, tops;      // floats of a row's scores (a multiple of 4), of a sequence's tops for a head
    float* scores;                   // [rows, kv_heads, score_stride]; NaN: no finite number
    float* top;                      // [n_seqs, kv_heads, tops]: the greatest bound of 16 pages, by magnitude
    int32_t* out;
    uint32_t first_block;
};

// Pages that a sequence's first `tokens` new tokens see.
__device__ __forceinline__ int pages_seen(const SelectParams& p, const Seq& q, int tokens) {
    const int limit = q.len - q.n_new + tokens;
    return limit > 0 ? div_page(limit - 1, p.batch.page_div) + 1 : 0;
}

template <int DT, int DP>
__global__ __launch_bounds__(256) void score_kernel(SelectParams p) {
    constexpr int kSteps = DP / 32;
    const int lane = (int)threadIdx.x & 63, wave = uniform((int)threadIdx.x >> 6);
    const int col = lane & 15, quad = lane >> 4;
    const uint32_t unit = p.first_block + blockIdx.x;
    const int head = (int)(unit % (uint32_t)p.kv_heads);
    int tile = (int)(unit / (uint32_t)p.kv_heads);
    auto tiles_of = [&](const Seq& q) { return (pages_seen(p, q, q.n_new) + kTilePages - 1) / kTilePages; };
    auto units_of = [&](const Seq& q) { return q.n_new > 0 ? tiles_of(q) * ((q.n_new - 1) / kBlockTokens + 1) : 0; };
    const int s = uniform(find_tile(p.batch, tile, units_of));
    if (s >= p.batch.n_seqs) return;
    const Seq seq = uniform(seq_of(p.batch, s));
    const int n_tiles = tiles_of(seq);
    if (tile < 0 || tile >= units_of(seq)) return;            // (starts that do not ascend)
    const int block = uniform(tile / n_tiles);
    const int page0 = uniform(tile % n_tiles) * kTilePages + wave * 16;
    const int token0 = block * kBlockTokens, tokens = min(seq.n_new - token0, kBlockTokens);
    if (page0 >= pages_seen(p, seq, token0 + tokens)) return;

    uint4 lo[kSteps], hi[kSteps];
    {
        const int at = page0 + col;
        const int id = at < pages_seen(p, seq, seq.n_new) ? seq.table[at] : -1;
        const bool there = id >= 0 && id < p.batch.n_pages;
        const uint8_t* src = p.bounds + 2 * ((int64_t)(there ? id : 0) * p.bounds_page + (int64_t)head * p.head_dim);
        const int64_t step = 2 * (int64_t)p.kv_heads * p.head_dim;
#pragma unroll
        for (int i = 0; i < kSteps; ++i) {
            const int d = 32 * i + 8 * quad;
            const bool has = there && d < p.head_dim;
            lo[i] = has ? ldg16(src + 2 * d) : make_uint4(0, 0, 0, 0);
            hi[i] = has ? ldg16(src + step + 2 * d) : make_uint4(0, 0, 0, 0);
        }
    }
    if (token0 + tokens == seq.n_new) {   // the block that sees every page
        uint32_t most = 0;
#pragma unroll
        for (int i = 0; i < kSteps; ++i) {
            const uint32_t w[8] = {lo[i].x, lo[i].y, lo[i].z, lo[i].w, hi[i].x, hi[i].y, hi[i].z, hi[i].w};
#pragma unroll
            for (int j = 0; j < 8; ++j) most = max(most, max(w[j] & 0x7FFFu, w[j] >> 16 & 0x7FFFu));
        }
        for (int m = 1; m < 64; m <<= 1) most = max(most, (uint32_t)__shfl_xor((int)most, m));
        if (lane == 0) p.top[((int64_t)s * p.kv_heads + head) * p.tops + page0 / 16] = hot_lo<DT>(most);
    }
    int heads_log = 4;                    // 2^heads_log heads and 2^(4 - heads_log) tokens are the 16 columns
    while (heads_log > 0 && tokens > 16 >> heads_log) --heads_log;
    const int heads = 1 << heads_log, token_step = 16 >> heads_log;
    const int col_token = col >> heads_log, col_head = col & (heads - 1);
    for (int t0 = 0; t0 < tokens; t0 += token_step) {
        const int token = token0 + min(t0 + col_token, tokens - 1);
        const uint8_t* row = p.q + 2 * ((int64_t)(seq.row0 + token) * p.q_stride + (int64_t)head * p.group * p.head_dim);
        float best[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
        for (int h0 = 0; h0 < p.group; h0 += heads) {
            const uint8_t* src = row + 2 * (int64_t)min(h0 + col_head, p.group - 1) * p.head_dim;
            uint4 x[kSteps];
#pragma unroll
            for (int i = 0; i < kSteps; ++i) {
                const int d = 32 * i + 8 * quad;
                x[i] = d < p.head_dim ? ldg16(src + 2 * d) : make_uint4(0, 0, 0, 0);
            }
            f32x4 sc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int i = 0; i < kSteps; ++i) {
                const uint32_t w[4] = {x[i].x, x[i].y, x[i].z, x[i].w};
                uint32_t neg[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) neg[j] = w[j] & ((w[j] >> 15 & 0x00010001u) * 0xFFFFu);
                sc = mfma16<DT>(lo[i], make_uint4(neg[0], neg[1], neg[2], neg[3]), sc);
                sc = mfma16<DT>(hi[i], make_uint4(w[0] ^ neg[0], w[1] ^ neg[1], w[2] ^ neg[2], w[3] ^ neg[3]), sc);
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) best[e] = fmaxf(best[e], fabsf(sc[e]) < INFINITY ? sc[e] : INFINITY);
        }
        for (int m = 1; m < heads; m <<= 1)
#pragma unroll
            for (int e = 0; e < 4; ++e) best[e] = fmaxf(best[e], __shfl_xor(best[e], m));
        const int at = page0 + 4 * quad;
        if (col_head == 0 && t0 + col_token < tokens && at < p.score_stride) {
            float* dst = p.scores + ((int64_t)(seq.row0 + token) * p.kv_heads + head) * p.score_stride + at;
#pragma unroll
            for (int e = 0; e < 4; ++e) best[e] = best[e] < INFINITY ? best[e] : NAN;
            *reinterpret_cast<float4*>(dst) = make_float4(best[0], best[1], best[2], best[3]);
        }
    }
}

// ---- selection --------------------------------------------------------------------
// Which pages have the highest scores must not depend on how fp32 sums were rounded.
// A score of n = 2 head_dim products, each exact in fp32, is off by at most
//     E = n (2^-23 |q|_1 B + 2^-125 (1 + |q|_1 + B)),
// B being the greatest bound (every addition rounds or cuts by 2^-23 of what it holds,
// a number too small for fp32 loses 2^-126 times its partner): if T is the k-th highest
// fp32 score, pages above T + 2 E are among the k highest and those below T - 2 E are
// not.  Those between, hardly ever more than a few, are scored again in fp64 and ranked;
// equal ones by their place.  A score that is no finite number tells nothing: then E is
// infinite.  NaN counts as more than every number.

constexpr int kBins = 2048;
constexpr int kFew = 256;
constexpr uint32_t kChosen = 0xFFFFFFFFu;   // in the place of a page's key: it is taken; 0: it is not

__device__ __forceinline__ uint32_t order_of(float x) {       // of finite numbers: neither 0 nor kChosen; -0 as 0
    const uint32_t b = __float_as_uint(x + 0.f);
    return b >> 31 ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float number_of(uint32_t k) { return __uint_as_float(k >> 31 ? k & 0x7FFFFFFFu : ~k); }
__device__ __forceinline__ uint64_t order_of(double x) {
    if (x != x) return ~0ull;
    const uint64_t b = (uint64_t)__double_as_longlong(x + 0.0);
    return b >> 63 ? ~b : b | 1ull << 63;
}

struct PickShared {
    int bins[kBins];
    uint64_t few[kFew];
    int few_page[kFew];
    uint64_t ends[2][4];
    int scan[4];
    float sums[2][4];
    int found[3], n_few;
    uint64_t kth;
};

__device__ __forceinline__ int block_total(int x, int* lds) {
    for (int m = 1; m < 64; m <<= 1) x += __shfl_xor(x, m);
    __syncthreads();
    if ((threadIdx.x & 63u) == 0) lds[threadIdx.x / 64] = x;
    __syncthreads();
    return lds[0] + lds[1] + lds[2] + lds[3];
}

// Closing in on the `left`-th highest of some keys.  visit(f) calls f(key) for each, all threads taking part.  On
// return keys above `high` are among the highest, and `left` of those from low to high, which are all equal or as
// many as that (then `left` is 0 below: all of them).
template <class Key, class Visit>
__device__ __forceinline__ void close_in(PickShared& sh, Visit&& visit, Key& low, Key& high, int& left) {
    const int tid = (int)threadIdx.x, lane = tid & 63, wave = tid >> 6;
    for (;;) {
        uint64_t least = ~0ull, most = 0;
        visit([&](Key k) {
            if (k >= low && k <= high) least = k < least ? k : least, most = k > most ? k : most;
        });
        for (int m = 1; m < 64; m <<= 1) {
            const uint64_t a = (uint64_t)__shfl_xor((unsigned long long)least, m), b = (uint64_t)__shfl_xor((unsigned long long)most, m);
            least = a < least ? a : least, most = b > most ? b : most;
        }
        __syncthreads();
        if (lane == 0) sh.ends[0][wave] = least, sh.ends[1][wave] = most;
        for (int i = tid; i < kBins; i += 256) sh.bins[i] = 0;
        __syncthreads();
        least = sh.ends[0][0], most = sh.ends[1][0];
#pragma unroll
        for (int w = 1; w < 4; ++w) {
            least = sh.ends[0][w] < least ? sh.ends[0][w] : least;
            most = sh.ends[1][w] > most ? sh.ends[1][w] : most;
        }
        low = (Key)least, high = (Key)most;
        if (low == high) return;
        const uint64_t span = most - least;
        const int bits = 64 - __clzll((long long)span), shift = bits > 11 ? bits - 11 : 0;
        visit([&](Key k) {
            if (k >= low && k <= high) atomicAdd(&sh.bins[(int)((uint64_t)(high - k) >> shift)], 1);   // bin 0: the highest
        });
        __syncthreads();
        int of[kBins / 256], own = 0;
#pragma unroll
        for (int j = 0; j < kBins / 256; ++j) own += of[j] = sh.bins[kBins / 256 * tid + j];
        int x = own;
        for (int m = 1; m < 64; m <<= 1) {
            const int y = __shfl_up(x, m);
            x += lane >= m ? y : 0;
        }
        if (lane == 63) sh.scan[wave] = x;
        __syncthreads();
        int before = x - own;
        for (int w = 0; w < wave; ++w) before += sh.scan[w];
#pragma unroll
        for (int j = 0; j < kBins / 256; ++j) {
            if (before < left && left <= before + of[j]) sh.found[0] = kBins / 256 * tid + j, sh.found[1] = before, sh.found[2] = of[j];
            before += of[j];
        }
        __syncthreads();
        high = (Key)(most - ((uint64_t)sh.found[0] << shift));
        const uint64_t width = ((uint64_t)1 << shift) - 1;
        if ((uint64_t)high - (uint64_t)low > width) low = (Key)((uint64_t)high - width);
        left -= sh.found[1];
    }
}

// A page's score in fp64 as a number's place among all: the wave's lanes lie along the columns, and what is left of
// them along the query heads.
template <int DT>
__device__ __forceinline__ uint64_t exact_key(const SelectParams& p, const uint8_t* q, int id, int head) {
    const int lane = (int)threadIdx.x & 63, chunks = p.head_dim / 8;
    int width = 2;
    while (width < chunks) width <<= 1;
    const int chunk = lane % width;
    const uint8_t* src = p.bounds + 2 * ((int64_t)id * p.bounds_page + (int64_t)head * p.head_dim) + 16 * chunk;
    const bool has = chunk < chunks;
    const uint4 none = make_uint4(0, 0, 0, 0);
    const uint4 lo = has ? ldg16(src) : none, hi = has ? ldg16(src + 2 * (int64_t)p.kv_heads * p.head_dim) : none;
    const uint32_t l[4] = {lo.x, lo.y, lo.z, lo.w}, h[4] = {hi.x, hi.y, hi.z, hi.w};
    uint64_t best = 0;
    for (int g0 = 0; g0 < p.group; g0 += 64 / width) {
        const int g = min(g0 + lane / width, p.group - 1);
        const uint4 x = has ? ldg16(q + 2 * (int64_t)g * p.head_dim + 16 * chunk) : none;
        const uint32_t w[4] = {x.x, x.y, x.z, x.w};
        double sum = 0.0;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const double a = e & 1 ? hot_hi<DT>(w[e / 2]) : hot_lo<DT>(w[e / 2]);
            const double b = e & 1 ? hot_hi<DT>(l[e / 2]) : hot_lo<DT>(l[e / 2]);
            const double c = e & 1 ? hot_hi<DT>(h[e / 2]) : hot_lo<DT>(h[e / 2]);
            sum += (a > 0.0 || a != a ? a : 0.0) * c;
            sum += (a < 0.0 || a != a ? a : 0.0) * b;
        }
        for (int m = 1; m < width; m <<= 1) sum += __shfl_xor(sum, m);
        const uint64_t key = order_of(sum);
        best = key > best ? key : best;
    }
    for (int m = width; m < 64; m <<= 1) {
        const uint64_t y = (uint64_t)__shfl_xor((unsigned long long)best, m);
        best = y > best ? y : best;
    }
    return best;
}

// One workgroup for a row and KV head.  Keys are in LDS, or (IN_LDS false) in the place of the scores.
template <int DT, bool IN_LDS>
__global__ __launch_bounds__(256) void pick_kernel(SelectParams p) {
    extern __shared__ uint32_t lds_keys[];
    __shared__ PickShared sh;
    const int tid = (int)threadIdx.x, lane = tid & 63, wave = uniform(tid >> 6);
    const int64_t unit = (int64_t)p.first_block + blockIdx.x;
    const int row = (int)(unit / p.kv_heads), head = (int)(unit % p.kv_heads);
    int s = find_above(p.batch.starts + 1, p.batch.n_seqs, row);
    if (s >= p.batch.n_seqs) return;
    const Seq seq = uniform(seq_of(p.batch, s));
    if (row < seq.row0 || row >= seq.row0 + seq.n_new) return;
    const int n = pages_seen(p, seq, row - seq.row0 + 1);
    float* scores = p.scores + unit * p.score_stride;
    uint32_t* keys;
    if constexpr (IN_LDS) keys = lds_keys;
    else keys = reinterpret_cast<uint32_t*>(scores);
    const uint8_t* q = p.q + 2 * ((int64_t)row * p.q_stride + (int64_t)head * p.group * p.head_dim);
    int32_t* out = p.out + unit * p.budget;

    int forced = 0, open = 0, unknown = 0;
    for (int i = tid; i < n; i += 256) {
        const float x = scores[i];
        const int id = seq.table[i];
        const bool there = id >= 0 && id < p.batch.n_pages, always = there && (i < p.sink || i >= n - p.recent);
        const bool known = x == x;
        keys[i] = always ? kChosen : there ? (known ? order_of(x) : 1u) : 0u;
        forced += always, open += there && !always, unknown += there && !always && !known;
    }
    forced = block_total(forced, sh.scan);
    open = block_total(open, sh.scan);
    unknown = block_total(unknown, sh.scan);
    const int wanted = p.budget - forced;
    if (open <= wanted) {                                     // all of them
        for (int i = tid; i < n; i += 256)
            if (keys[i] != 0) keys[i] = kChosen;
    } else if (wanted > 0) {
        // the fp32 scores' k-th highest, and how far from it fp32 sums cannot tell
        uint32_t low = 1, high = kChosen - 1;                 // keys of pages that may or may not be taken
        int left = wanted;
        if (unknown == 0) {
            uint32_t least = 1, most = kChosen - 1;
            close_in(sh, [&](auto&& f) { for (int i = tid; i < n; i += 256) f(keys[i]); }, least, most, left);
            float sum = 0.f, top = 0.f;
            for (int h = wave; h < p.group; h += 4) {
                float x = 0.f;
                for (int d = 2 * lane; d < p.head_dim; d += 128) {
                    const uint32_t w = *reinterpret_cast<const uint32_t*>(q + 2 * ((int64_t)h * p.head_dim + d));
                    x += fabsf(hot_lo<DT>(w)) + fabsf(hot_hi<DT>(w));
                }
                x = xor_sum(x, 64);
                sum = x > sum || x != x ? x : sum;
            }
            const float* tops = p.top + ((int64_t)s * p.kv_heads + head) * p.tops;
            for (int i = tid; i < (n + 15) / 16; i += 256) {
                const float x = tops[i];
                top = x > top || x != x ? x : top;
            }
            for (int m = 1; m < 64; m <<= 1) {
                const float x = __shfl_xor(top, m);
                top = x > top || x != x ? x : top;
            }
            __syncthreads();
            if (lane == 0) sh.sums[0][wave] = sum, sh.sums[1][wave] = top;
            __syncthreads();
#pragma unroll
            for (int w = 0; w < 4; ++w) {
                sum = sh.sums[0][w] > sum || sh.sums[0][w] != sh.sums[0][w] ? sh.sums[0][w] : sum;
                top = sh.sums[1][w] > top || sh.sums[1][w] != sh.sums[1][w] ? sh.sums[1][w] : top;
            }
            // (a hundredth more than E for the rounding of the sum, of E itself and of the borders)
            const float err = 2.02f * (float)p.head_dim * (0x1p-23f * sum * top + 0x1p-125f * (1.f + sum + top));
            const float kth = number_of(least), reach = 2.f * err + 0x1p-22f * fabsf(kth);
            if (reach < INFINITY) {
                const float a = kth - reach, b = kth + reach;
                low = a > -INFINITY ? order_of(a) : 1u;
                high = b < INFINITY ? order_of(b) : kChosen - 1;
            }
        }
        int above = 0, near = 0;
        for (int i = tid; i < n; i += 256) {
            const uint32_t k = keys[i];
            above += k > high && k != kChosen;
            near += k >= low && k <= high;
        }
        above = block_total(above, sh.scan);
        near = block_total(near, sh.scan);
        left = wanted - above;
        // above `high`: taken; below `low`: not
        if (near <= left || near > kFew) {
            uint64_t exact_low = 1, exact_high = ~0ull;       // (a score's place is never 0)
            int ties = 0x7FFFFFFF;
            auto chunk = [&](int base) {                      // of 256 pages: the scores of those near the border, 0 for the others
                __syncthreads();
                for (int j = wave; j < 256; j += 4) {
                    const int i = base + j;
                    const uint32_t k = i < n ? keys[i] : 0u;
                    const bool is = k >= low && k <= high;
                    const uint64_t x = is ? exact_key<DT>(p, q, seq.table[i], head) : 0ull;
                    if (lane == 0) sh.few[j] = x;
                }
                __syncthreads();
                return sh.few[tid];
            };
            if (near > left) {
                ties = left;
                close_in(sh, [&](auto&& f) { for (int base = 0; base < n; base += 256) f(chunk(base)); }, exact_low, exact_high, ties);
            } else {
                exact_high = 0;                               // all that are near
            }
            int tied = 0;
            for (int base = 0; base < n; base += 256) {
                const int i = base + tid;
                const uint32_t k = i < n ? keys[i] : 0u;
                const bool is = k >= low && k <= high;
                const uint64_t x = near > left ? chunk(base) : is ? 1ull : 0ull;
                const bool tie = near > left && is && x >= exact_low && x <= exact_high;
                const uint64_t all = __ballot(tie);
                __syncthreads();
                if (lane == 0) sh.scan[wave] = __popcll(all);
                __syncthreads();
                int rank = tied + __popcll(all & ((1ull << lane) - 1));
                for (int w = 0; w < 4; ++w) {
                    rank += w < wave ? sh.scan[w] : 0;
                    tied += sh.scan[w];
                }
                if (i < n && k != kChosen) keys[i] = k > high || (is && x > exact_high) || (tie && rank < ties) ? kChosen : 0u;
            }
        } else {
            if (tid == 0) sh.n_few = 0;
            __syncthreads();
            for (int i = tid; i < n; i += 256) {
                const uint32_t k = keys[i];
                if (k >= low && k <= high) sh.few_page[atomicAdd(&sh.n_few, 1)] = i;
                if (k != kChosen) keys[i] = k > high ? kChosen : 0u;
            }
            __syncthreads();
            for (int j = wave; j < near; j += 4) {
                const uint64_t x = exact_key<DT>(p, q, seq.table[sh.few_page[j]], head);
                if (lane == 0) sh.few[j] = x;
            }
            __syncthreads();
            if (tid < near) {
                const uint64_t mine = sh.few[tid];
                const int page = sh.few_page[tid];
                int rank = 0;
                for (int j = 0; j < near; ++j) rank += sh.few[j] > mine || (sh.few[j] == mine && sh.few_page[j] < page);
                if (rank < left) keys[page] = kChosen;
            }
        }
    } else {
        for (int i = tid; i < n; i += 256)
            if (keys[i] != kChosen) keys[i] = 0u;
    }
    __syncthreads();
    int at = 0;
    for (int base = 0; base < n; base += 256) {
        const int i = base + tid;
        const bool taken = i < n && keys[i] == kChosen;
        const uint64_t all = __ballot(taken);
        __syncthreads();
        if (lane == 0) sh.scan[wave] = __popcll(all);
        __syncthreads();
        int to = at + __popcll(all & ((1ull << lane) - 1));
        for (int w = 0; w < 4; ++w) {
            to += w < wave ? sh.scan[w] : 0;
            at += sh.scan[w];
        }
        if (taken && to < p.budget) out[to] = i;
    }
    for (int i = at + tid; i < p.budget; i += 256) out[i] = -1;
}

constexpr int kKeysInLds = 12288;   // 48 KiB

// What is wrong with bounds [n_pages, 2, num_heads, head_dim], pages `stride` elements apart, or nullptr.
const char* check_bounds(const void* bounds, int64_t stride, const ztcp_geometry* g, int64_t n_pages) {
    if (!bounds || !hot_aligned(bounds) || stride % 8 != 0) return "bounds must not be NULL, and 16-byte aligned";
    if (n_pages > 1 && stride < 2 * g->num_heads * g->head_dim) return "bounds' stride must cover a page's";
    return nullptr;
}

struct SelectPlan {
    int64_t stride, tops, units, floats;
};
SelectPlan plan_select(const ztcp_paged_batch* b, const ztcp_geometry* g) {
    SelectPlan plan;
    plan.stride = (b->max_pages + 3) / 4 * 4;
    plan.tops = (b->max_pages + 15) / 16;
    plan.units = (b->n_rows / kBlockTokens + b->n_seqs) * ((b->max_pages + kTilePages - 1) / kTilePages);
    plan.floats = b->n_rows * g->num_heads * plan.stride + (b->n_seqs * g->num_heads * plan.tops + 3) / 4 * 4;
    return plan;
}

// `bounds` stands for the pool's K: what check_pool asks of one, the bounds have as well.
const char* check_select(const ztcp_paged_batch* batch, const void* bounds, int64_t bounds_stride, int64_t n_pages,
                         const ztcp_geometry* g, int64_t q_heads, PagedView& view) {
    if (!g) return "geometry must not be NULL";
    if (g->num_tokens < 1 || g->num_heads < 1 || g->head_dim < 1) return "num_tokens, num_heads and head_dim must be positive";
    ztcp_page_pool pool{const_cast<void*>(bounds), nullptr, n_pages, 0, 0};
    ztcp_geometry one = *g;
    one.num_tokens = 2;
    pool.k_stride = bounds_stride;
    if (const char* why = check_bounds(bounds, bounds_stride, g, n_pages)) return why;
    if (const char* why = check_pool(&pool, &one, 256)) return why;
    if (g->num_tokens >= (int64_t)1 << 30) return "num_tokens must be below 2^30";
    pool.k_stride = 0;
    if (const char* why = check_batch(batch, &pool, g, q_heads, view)) return why;
    const SelectPlan plan = plan_select(batch, g);
    if (plan.stride >= (int64_t)1 << 31 || plan.units * g->num_heads >= (int64_t)1 << 31 || plan.floats >= (int64_t)1 << 40)
        return "too many rows and pages in one call";
    return nullptr;
}

}  // namespace

extern "C" int ztcp_page_bounds(const ztcp_page_pool* pool, const ztcp_paged_batch* batch, const ztcp_geometry* g, void* bounds,
                                int64_t bounds_stride, void* stream) {
    arg_result(ZTCP_OK, "");
    BoundsParams p{};
    if (const char* why = check_pool(pool, g, 1024)) return arg_result(ZTCP_EINVAL, why);
    if (const char* why = check_batch(batch, pool, g, g->num_heads, p.batch)) return arg_result(ZTCP_EINVAL, why);
    if (const char* why = check_bounds(bounds, bounds_stride, g, pool->n_pages)) return arg_result(ZTCP_EINVAL, why);
    const int64_t row = g->num_heads * g->head_dim;
    if (rows_overlap(bounds, pool->n_pages, 4 * row, 2 * bounds_stride, pool->k, pool->n_pages, 2 * g->num_tokens * row, 2 * pool->k_stride))
        return arg_result(ZTCP_EOVERLAP, "bounds must not overlap the pages");
    if (batch->n_seqs == 0 || batch->n_rows == 0) return ZTCP_OK;
    p.k_pool = (const uint8_t*)pool->k;
    p.k_page = pool->k_stride;
    p.bounds = (uint8_t*)bounds;
    p.bounds_page = bounds_stride;
    p.row_elements = (int32_t)row;
    p.parts = (int32_t)((row / 8 + 63) / 64);
    // how many rows there are, the device knows: waves for as many as there can be, which take several runs if need be
    const int64_t most = batch->max_q_len > 0 && batch->max_q_len < batch->n_rows / batch->n_seqs ? batch->max_q_len * batch->n_seqs
                                                                                                  : batch->n_rows;
    const int64_t waves = most < kBoundsWaves / p.parts ? most * p.parts : kBoundsWaves;
    const dim3 grid((uint32_t)((waves + 3) / 4));
    if (g->hot_dtype == ZTCP_HOT_BF16) hipLaunchKernelGGL(bounds_kernel<kHotBf16>, grid, dim3(256), 0, (hipStream_t)stream, p);
    else hipLaunchKernelGGL(bounds_kernel<kHotFp16>, grid, dim3(256), 0, (hipStream_t)stream, p);
    return hipGetLastError() == hipSuccess ? ZTCP_OK : ZTCP_EHIP;
}

extern "C" size_t ztcp_select_pages_workspace(const ztcp_paged_batch* batch, int64_t n_pages, const ztcp_geometry* g, int64_t q_heads) {
    arg_result(ZTCP_OK, "");
    PagedView view;
    const int64_t stride = g ? 2 * g->num_heads * g->head_dim : 0;
    if (const char* why = check_select(batch, (const void*)16, stride, n_pages, g, q_heads, view)) {
        arg_result(ZTCP_EINVAL, why);
        return (size_t)-1;
    }
    return (size_t)plan_select(batch, g).floats * sizeof(float);
}

extern "C" int ztcp_select_pages(const void* q, int64_t q_stride, int64_t q_heads, const void* bounds, int64_t bounds_stride,
                                 int64_t n_pages, const ztcp_paged_batch* batch, const ztcp_geometry* g, int64_t budget, int64_t sink,
                                 int64_t recent, int32_t* out, void* workspace, size_t workspace_bytes, void* stream) {
    arg_result(ZTCP_OK, "");
    SelectParams p{};
    if (const char* why = check_select(batch, bounds, bounds_stride, n_pages, g, q_heads, p.batch)) return arg_result(ZTCP_EINVAL, why);
    if (sink < 0 || recent < 1 || budget >= (int64_t)1 << 31 || sink > budget || recent > budget - sink)
        return arg_result(ZTCP_EINVAL, "sink must not be negative, recent at least 1, budget at least sink + recent and below 2^31");
    if (batch->n_seqs == 0 || batch->n_rows == 0) return ZTCP_OK;
    if (!q || !out) return arg_result(ZTCP_EINVAL, "q and out must not be NULL");
    if (!hot_aligned(q) || q_stride % 8 != 0 || ((uintptr_t)out & 3u) != 0) return arg_result(ZTCP_EINVAL, "q must be 16-byte aligned, out 4-byte");
    const int64_t d = g->head_dim, row = q_heads * d;
    if (batch->n_rows > 1 && q_stride < row) return arg_result(ZTCP_EINVAL, "q_stride must cover a token's heads");
    const SelectPlan plan = plan_select(batch, g);
    const int64_t need = plan.floats * (int64_t)sizeof(float), out_bytes = 4 * batch->n_rows * g->num_heads * budget;
    if (!workspace || (int64_t)workspace_bytes < need || !hot_aligned(workspace))
        return arg_result(ZTCP_EINVAL, "workspace must hold ztcp_select_pages_workspace bytes, 16-byte aligned");
    const int64_t q_bytes = 2 * ((batch->n_rows - 1) * q_stride + row), bounds_bytes = 2 * ((n_pages - 1) * bounds_stride + 2 * g->num_heads * d);
    if (bytes_overlap(out, out_bytes, q, q_bytes) || bytes_overlap(out, out_bytes, bounds, bounds_bytes) ||
        bytes_overlap(workspace, need, q, q_bytes) || bytes_overlap(workspace, need, bounds, bounds_bytes) ||
        bytes_overlap(workspace, need, out, out_bytes))
        return arg_result(ZTCP_EOVERLAP, "out and workspace must not overlap q, bounds or each other");
    p.q = (const uint8_t*)q;
    p.q_stride = q_stride;
    p.bounds = (const uint8_t*)bounds;
    p.bounds_page = bounds_stride;
    p.kv_heads = (int32_t)g->num_heads;
    p.group = (int32_t)(q_heads / g->num_heads);
    p.head_dim = (int32_t)d;
    p.budget = (int32_t)budget;
    p.sink = (int32_t)sink;
    p.recent = (int32_t)recent;
    p.score_stride = (int32_t)plan.stride;
    p.tops = (int32_t)plan.tops;
    p.top = (float*)workspace;
    p.scores = p.top + (batch->n_seqs * g->num_heads * plan.tops + 3) / 4 * 4;
    p.out = out;
    auto go = [&](auto dt) {
        constexpr int DT = decltype(dt)::value;
        const uint64_t units = (uint64_t)plan.units * (uint64_t)g->num_heads, picks = (uint64_t)batch->n_rows * (uint64_t)g->num_heads;
        launch_blocks(d <= 64 ? score_kernel<DT, 64> : d <= 128 ? score_kernel<DT, 128> : score_kernel<DT, 256>, units, 256, 0,
                      (hipStream_t)stream, p);
        if (batch->max_pages <= kKeysInLds)
            launch_blocks(pick_kernel<DT, true>, picks, 256, (size_t)batch->max_pages * 4, (hipStream_t)stream, p);
        else launch_blocks(pick_kernel<DT, false>, picks, 256, 0, (hipStream_t)stream, p);
    };
    if (g->hot_dtype == ZTCP_HOT_BF16) go(std::integral_constant<int, kHotBf16>{});
    else go(std::integral_constant<int, kHotFp16>{});
    return hipGetLastError() == hipSuccess ? ZTCP_OK : ZTCP_EHIP;
}
