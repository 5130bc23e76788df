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
            const int id = seq.entry(at);
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
// as many heads to a token as leave no column idle.  A unit is 64 pages of a sequence,
// 16 a wave, and a block of its new tokens; units lie sequence behind sequence, and the
// workgroups of a KV head take equal shares of them, with the loads of the next unit's
// bounds, by whole rows through LDS of the wave's own, in flight meanwhile.  The greatest
// score of the KV head's query heads is what counts.
//
// 32 sequences of 512 to 8,192 pages, 4 query heads to each of 8 KV heads of 128 (375 MB
// of bounds): 114 us a workgroup for each unit and bounds as the products want them, 84
// now, of which the loads alone take 74 and all else alone 41.

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
    int32_t row0, row1;              // rows that these launches take
    int32_t score_stride, tops;      // words of a row's scores and keys (a multiple of 4), of a sequence's tops for a head
    float* scores;                   // [row1 - row0, kv_heads, score_stride]; NaN: no finite number
    int32_t score_groups;            // score kernel: workgroups of a KV head
    int32_t few_pages;               // pick kernel: rows of at most so many pages (-1: none) are another kernel's
    float* top;                      // [n_seqs, kv_heads, tops]: the greatest finite bound of 16 pages, by magnitude
    int32_t* out;
    uint32_t first_block;
};

// What a sequence has in rows row0 .. row1: these as its new tokens, of a length that its last one there sees.
__device__ __forceinline__ Seq part_of(const SelectParams& p, Seq q) {
    const int first = max(q.row0, p.row0), behind = q.row0 + q.n_new, end = min(behind, p.row1);
    q.len -= behind - end;
    q.row0 = first;
    q.n_new = max(end - first, 0);
    return q;
}
__device__ __forceinline__ float* scores_of(const SelectParams& p, int row, int head) {
    return p.scores + ((int64_t)(row - p.row0) * p.kv_heads + head) * p.score_stride;
}

// Pages that a sequence's first `tokens` new tokens see.
__device__ __forceinline__ int pages_seen(const SelectParams& p, const Seq& q, int tokens) {
    const int limit = q.len - q.n_new + tokens;
    return limit > 0 ? div_page(limit - 1, p.batch.page_div) + 1 : 0;
}

// The greatest of the 16 lanes of a row, or of as many of them as an aligned 2^log are; a lane's partners by DPP.
template <int CTRL>
__device__ __forceinline__ float partner(float x) {
    return __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(x), CTRL, 0xF, 0xF, true));
}
__device__ __forceinline__ float row_max(float x, int log) {
    if (log > 0) x = fmaxf(x, partner<0xB1>(x));              // lane ^ 1
    if (log > 1) x = fmaxf(x, partner<0x4E>(x));              // lane ^ 2
    if (log > 2) x = fmaxf(x, partner<0x141>(x));             // 7 - lane, within 8
    if (log > 3) x = fmaxf(x, partner<0x140>(x));             // 15 - lane
    return x;
}

typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
typedef int16_t i16x2 __attribute__((ext_vector_type(2)));

// Two numbers, those with the sign bit (NaN too) as they are, 0 for the others.
__device__ __forceinline__ uint32_t negatives(uint32_t w) { return w & __builtin_bit_cast(uint32_t, __builtin_bit_cast(i16x2, w) >> (int16_t)15); }

// The greatest magnitude among a wave's bounds of 16 pages from page0 on, written down; `counts`: the lane's (lane % 16)
// page is there.  Numbers of one sign are ordered as their bits are, infinity and NaN above all others: where there is one,
// the greatest of the others is looked for.  (A page that has one has no finite score.)
template <int DT, int N>
__device__ __forceinline__ void top_of(const SelectParams& p, const uint4 (&lo)[N], const uint4 (&hi)[N], int s, int head, int page0,
                                       bool counts) {
    const int lane = (int)threadIdx.x & 63;
    u16x2 most = {0, 0};
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const uint32_t w[8] = {lo[i].x, lo[i].y, lo[i].z, lo[i].w, hi[i].x, hi[i].y, hi[i].z, hi[i].w};
#pragma unroll
        for (int j = 0; j < 8; ++j) most = __builtin_elementwise_max(most, __builtin_bit_cast(u16x2, w[j] & 0x7FFF7FFFu));
    }
    auto of_all = [&](uint32_t x) {
        const float top = row_max(__int_as_float(counts ? (int)x << 8 : 0), 4);
        return (uint32_t)max(max(__builtin_amdgcn_readlane(__float_as_int(top), 0), __builtin_amdgcn_readlane(__float_as_int(top), 16)),
                             max(__builtin_amdgcn_readlane(__float_as_int(top), 32), __builtin_amdgcn_readlane(__float_as_int(top), 48))) >> 8;
    };
    uint32_t all = of_all(max((uint32_t)most.x, (uint32_t)most.y));
    if (not_finite16<DT>(all)) {
        uint32_t rest = 0;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const uint32_t w[8] = {lo[i].x, lo[i].y, lo[i].z, lo[i].w, hi[i].x, hi[i].y, hi[i].z, hi[i].w};
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                rest = max(rest, not_finite16<DT>(w[j]) ? 0u : w[j] & 0x7FFFu);
                rest = max(rest, not_finite16<DT>(w[j] >> 16) ? 0u : w[j] >> 16 & 0x7FFFu);
            }
        }
        all = of_all(rest);
    }
    if (lane == 0) p.top[((int64_t)s * p.kv_heads + head) * p.tops + page0 / 16] = hot_lo<DT>(all);
}

template <int DT, int DP>
__global__ __launch_bounds__(256) void score_kernel(SelectParams p) {
    constexpr int kSteps = DP / 32, kChunks = DP / 8;         // products of depth 32; 16-byte pieces of a row
    constexpr int kLoadRows = 64 / kChunks, kLoads = 16 / kLoadRows;   // rows of a load; loads of 16 pages' lower, or upper, bounds
    __shared__ __attribute__((aligned(16))) uint8_t lds[4][32 * DP * 2];
    const int lane = (int)threadIdx.x & 63, wave = uniform((int)threadIdx.x >> 6);
    const int col = lane & 15, quad = lane >> 4;
    const int head = (int)(blockIdx.x % (uint32_t)p.kv_heads), group = (int)(blockIdx.x / (uint32_t)p.kv_heads);
    auto tiles_of = [&](const Seq& q) { return (pages_seen(p, q, q.n_new) + kTilePages - 1) / kTilePages; };
    auto blocks_of = [&](const Seq& q) { return q.n_new > 0 ? (q.n_new - 1) / kBlockTokens + 1 : 0; };
    auto units_of = [&](const Seq& whole) {
        const Seq q = part_of(p, whole);
        return tiles_of(q) * blocks_of(q);
    };
    struct Unit {
        int s, tile, block, tiles, pages;
        Seq seq;
    };
    int none;
    const int total = uniform(count_tiles(p.batch, 0, none, units_of));
    const int quota = (total + p.score_groups - 1) / p.score_groups;
    if ((int64_t)group * quota >= total) return;
    int first = group * quota;
    int left = min(quota, total - first);
    auto open = [&](Unit& u) {       // u.s's sequence, or the next one that has units
        for (; u.s < p.batch.n_seqs; ++u.s) {
            u.seq = uniform(part_of(p, seq_of(p.batch, u.s)));
            u.pages = uniform(pages_seen(p, u.seq, u.seq.n_new));
            u.tiles = (u.pages + kTilePages - 1) / kTilePages;
            if (u.seq.n_new > 0 && u.tiles > 0) return;
        }
    };
    auto advance = [&](Unit& u) {
        if (++u.tile < u.tiles) return;
        u.tile = 0;
        if (++u.block < blocks_of(u.seq)) return;
        u.block = 0;
        ++u.s;
        open(u);
    };
    auto ids = [&](const Unit& u) {  // of page lane % 16 of this wave's, as it was read; looked at when it is loaded from
        const int at = u.tile * kTilePages + wave * 16 + col;
        return u.s < p.batch.n_seqs && at < u.pages ? u.seq.entry(at) : -1;
    };
    uint8_t* mine = lds[wave];
    auto swizzle = [](int row, int chunk) { return chunk ^ (row & (kChunks < 16 ? kChunks - 1 : 15)); };
    const int load_row = lane / kChunks, load_chunk = lane % kChunks;
    const int64_t upper = 2 * (int64_t)p.kv_heads * p.head_dim, in_page = 2 * ((int64_t)head * p.head_dim + 8 * load_chunk);
    uint4 raw[2][kLoads];
    uint32_t there = 0;              // of this lane's loads: what they bring counts (a look at it here would wait for them)
    auto load = [&](int id, bool once) {
        const uint8_t* src[kLoads];
        there = 0;
#pragma unroll
        for (int i = 0; i < kLoads; ++i) {
            const int from = __shfl(id, i * kLoadRows + load_row);
            const bool has = (uint32_t)from < (uint32_t)p.batch.n_pages && load_chunk * 8 < p.head_dim;
            src[i] = p.bounds + 2 * ((int64_t)(has ? from : 0) * p.bounds_page) + (has ? in_page : 0);
            there |= has ? 1u << i : 0u;
        }
        if (once) {
#pragma unroll
            for (int i = 0; i < 2 * kLoads; ++i) raw[i % 2][i / 2] = ldg16_once(src[i / 2] + i % 2 * upper);
        } else {
#pragma unroll
            for (int i = 0; i < 2 * kLoads; ++i) raw[i % 2][i / 2] = ldg16(src[i / 2] + i % 2 * upper);
        }
    };
    Unit unit;
    unit.s = uniform(find_tile(p.batch, first, units_of));
    if (unit.s >= p.batch.n_seqs) return;
    open(unit);
    unit.block = uniform(first) / unit.tiles;
    unit.tile = uniform(first) - unit.block * unit.tiles;
    if (first < 0 || unit.s >= p.batch.n_seqs || unit.block >= blocks_of(unit.seq)) return;   // (starts that do not ascend)
    load(ids(unit), unit.seq.n_new <= kBlockTokens);
    Unit next = unit;
    advance(next);
    int next_ids = ids(next);
    uint4 neg[kSteps], pos[kSteps];                           // columns of a product
    int have = -1;                                            // whose: the sequence's, if it has one product only
    for (; left > 0 && unit.s < p.batch.n_seqs; --left) {
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int i = 0; i < kLoads; ++i) {
                const int row = i * kLoadRows + load_row;
                *reinterpret_cast<uint4*>(mine + (16 * u + row) * DP * 2 + swizzle(row, load_chunk) * 16) =
                    there >> i & 1 ? raw[u][i] : make_uint4(0, 0, 0, 0);
            }
        const Seq seq = unit.seq;
        const int s = unit.s, page0 = unit.tile * kTilePages + wave * 16, token0 = unit.block * kBlockTokens;
        const int tokens = min(seq.n_new - token0, kBlockTokens);
        const bool last_block = token0 + tokens == seq.n_new;
        const int pages = last_block ? unit.pages : pages_seen(p, seq, token0 + tokens);
        int heads_log = 4;                    // 2^heads_log heads and 2^(4 - heads_log) tokens are the 16 columns
        while (heads_log > 0 && tokens > 16 >> heads_log) --heads_log;
        const int heads = 1 << heads_log, token_step = 16 >> heads_log;
        const int col_token = col >> heads_log, col_head = col & (heads - 1);
        uint4 x[kSteps];
        auto load_q = [&](int t0, int h0) {
            const int token = token0 + min(t0 + col_token, tokens - 1), h = min(h0 + col_head, p.group - 1);
            const uint8_t* src = p.q + 2 * ((int64_t)(seq.row0 + token) * p.q_stride + ((int64_t)head * p.group + h) * p.head_dim);
#pragma unroll
            for (int i = 0; i < kSteps; ++i) {
                const int d = 32 * i + 8 * quad;
                x[i] = d < p.head_dim ? ldg16(src + 2 * d) : make_uint4(0, 0, 0, 0);
            }
        };
        auto split = [&]() {
#pragma unroll
            for (int i = 0; i < kSteps; ++i) {
                const uint32_t w[4] = {x[i].x, x[i].y, x[i].z, x[i].w};
                uint32_t n[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) n[j] = negatives(w[j]);
                neg[i] = make_uint4(n[0], n[1], n[2], n[3]);
                pos[i] = make_uint4(w[0] ^ n[0], w[1] ^ n[1], w[2] ^ n[2], w[3] ^ n[3]);
            }
        };
        const bool one = tokens <= token_step && p.group <= heads && seq.n_new == tokens;
        const bool keeps = one && have == s;
        if (!keeps) load_q(0, 0);             // ahead of the next unit's bounds, which a wait for it would include
        if (left > 1) load(next_ids, next.seq.n_new <= kBlockTokens);
        unit = next;
        if (left > 1) {
            advance(next);
            next_ids = ids(next);
        }
        if (page0 >= pages) continue;
        uint4 lo[kSteps], hi[kSteps];
#pragma unroll
        for (int i = 0; i < kSteps; ++i) {
            lo[i] = *reinterpret_cast<const uint4*>(mine + col * DP * 2 + swizzle(col, 4 * i + quad) * 16);
            hi[i] = *reinterpret_cast<const uint4*>(mine + (16 + col) * DP * 2 + swizzle(col, 4 * i + quad) * 16);
        }
        if (last_block) top_of<DT>(p, lo, hi, s, head, page0, true);   // it sees every page (what is not there is 0)
        for (int t0 = 0; t0 < tokens; t0 += token_step) {
            float best[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
            for (int h0 = 0; h0 < p.group; h0 += heads) {
                if (!keeps) split();
                have = one ? s : -1;
                const bool same_tokens = h0 + heads < p.group;
                if (same_tokens || t0 + token_step < tokens) load_q(same_tokens ? t0 : t0 + token_step, same_tokens ? h0 + heads : 0);
                f32x4 sc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int i = 0; i < kSteps; ++i) {
                    sc = mfma16<DT>(lo[i], neg[i], sc);
                    sc = mfma16<DT>(hi[i], pos[i], sc);
                }
#pragma unroll
                for (int e = 0; e < 4; ++e) best[e] = fmaxf(best[e], fabsf(sc[e]) < INFINITY ? sc[e] : INFINITY);
            }
            // (columns behind the group's heads repeat its last one)
            const int log = p.group <= 1 ? 0 : min(heads_log, 32 - __clz(p.group - 1));
#pragma unroll
            for (int e = 0; e < 4; ++e) best[e] = row_max(best[e], log);
            const int at = page0 + 4 * quad;
            if (col_head == 0 && t0 + col_token < tokens && at < p.score_stride) {
                const int token = token0 + t0 + col_token;
                float* dst = scores_of(p, seq.row0 + token, head) + at;
#pragma unroll
                for (int e = 0; e < 4; ++e) best[e] = best[e] < INFINITY ? best[e] : NAN;
                *reinterpret_cast<float4*>(dst) = make_float4(best[0], best[1], best[2], best[3]);
            }
        }
    }
}

// Chunks: a workgroup keeps a block of tokens' columns in LDS, up to eight products of 16 tokens and one head each, their
// negative and their positive numbers apart, and goes over up to 1,024 pages with them, 16 a wave and turn, whose bounds
// come as the products want them, from the caches most of the time, a turn ahead.
//
// 2 x 2,000 tokens, 3 query heads to each of 5 KV heads of 96, over 525 pages: 36 us (52 with signs looked at for every
// product, 42 with products as deep as 128; 32 pages a wave and turn, which read the columns half as often, take the
// registers of a third wave a SIMD: 47), 12 of them before the first product; 57 by the kernel above, whose waves wait
// for the columns of each product.
constexpr int kPieceTiles = 16;
// Tokens of a block: as many as make six products (48 KiB at 128 elements, three workgroups a compute unit), or 16 with up
// to eight; half as many for wider vectors; 0: too many heads.
__host__ __device__ inline int chunk_tokens(int group, int width) {
    const int fit = width <= 128 ? 6 : 3, most = width <= 128 ? 8 : 4;
    return group <= fit ? fit / group * 16 : group <= most ? 16 : 0;
}

// STEPS: products of depth 32 that hold head_dim.
template <int DT, int DP, int STEPS>
__global__ __launch_bounds__(256) void score_chunk_kernel(SelectParams p) {
    constexpr int kSteps = STEPS, kChunks = DP / 8, kLoadRows = 64 / kChunks, kRowBytes = DP * 2;
    extern __shared__ __attribute__((aligned(16))) uint8_t columns[];   // [negative, positive][product][16][DP]
    const int lane = (int)threadIdx.x & 63, wave = uniform((int)threadIdx.x >> 6);
    const int col = lane & 15, quad = lane >> 4;
    const uint32_t unit = p.first_block + blockIdx.x;
    const int head = (int)(unit % (uint32_t)p.kv_heads), block_size = chunk_tokens(p.group, DP);
    int at = (int)(unit / (uint32_t)p.kv_heads);
    auto tiles_of = [&](const Seq& q) { return (pages_seen(p, q, q.n_new) + kTilePages - 1) / kTilePages; };
    auto pieces_of = [&](const Seq& q) { return (tiles_of(q) + kPieceTiles - 1) / kPieceTiles; };
    auto units_of = [&](const Seq& whole) {
        const Seq q = part_of(p, whole);
        return q.n_new > 0 ? ((q.n_new - 1) / block_size + 1) * pieces_of(q) : 0;
    };
    const int s = uniform(find_tile(p.batch, at, units_of));
    if (s >= p.batch.n_seqs) return;
    const Seq whole = seq_of(p.batch, s), seq = uniform(part_of(p, whole));
    const int pieces = uniform(pieces_of(seq));
    if (at < 0 || at >= units_of(whole)) return;              // (starts that do not ascend)
    at = uniform(at);
    const int block = at / pieces, piece = at - block * pieces;
    const int token0 = block * block_size, tokens = min(seq.n_new - token0, block_size);
    const bool last_block = token0 + tokens == seq.n_new;
    const int all_pages = pages_seen(p, seq, seq.n_new), pages = min(pages_seen(p, seq, token0 + tokens), (piece + 1) * kPieceTiles * kTilePages);
    const int products = (tokens + 15) / 16 * p.group, block_bytes = block_size * p.group * kRowBytes;
    auto swizzle = [](int row, int chunk) { return chunk ^ (row & (kChunks < 16 ? kChunks - 1 : 15)); };
    int page0 = piece * kPieceTiles * kTilePages + wave * 16;
    // bounds of page lane % 16, at the products' depths
    uint4 bound[2][kSteps];
    int id = -1;
    auto fetch = [&](int page) { return page + col < all_pages ? seq.entry(page + col) : -1; };
    bool there = false;                                       // this lane's page, which is loaded
    auto load = [&](int of) {
        there = (uint32_t)of < (uint32_t)p.batch.n_pages;
        const uint8_t* src = p.bounds + 2 * ((int64_t)(there ? of : 0) * p.bounds_page + (int64_t)head * p.head_dim);
        const int64_t upper = 2 * (int64_t)p.kv_heads * p.head_dim;
#pragma unroll
        for (int i = 0; i < kSteps; ++i) {
            const int d = 32 * i + 8 * quad < p.head_dim ? 32 * i + 8 * quad : 0;   // (columns behind head_dim meet zeros)
#pragma unroll
            for (int u = 0; u < 2; ++u) bound[u][i] = ldg16(src + u * upper + 2 * d);
        }
    };
    load(fetch(page0));
    id = fetch(page0 + kTilePages);
    {
        const int load_row = lane / kChunks, load_chunk = lane % kChunks;
        for (int r0 = wave * kLoadRows; r0 < products * 16; r0 += 4 * kLoadRows) {
            const int r = r0 + load_row, group16 = r / 16 / p.group, h = r / 16 - group16 * p.group;
            const int token = token0 + min(group16 * 16 + (r & 15), tokens - 1);
            const uint8_t* src = p.q + 2 * ((int64_t)(seq.row0 + token) * p.q_stride + ((int64_t)head * p.group + h) * p.head_dim);
            uint4 x = make_uint4(0, 0, 0, 0);
            if (load_chunk * 8 < p.head_dim) x = ldg16(src + 16 * load_chunk);
            const uint4 n = make_uint4(negatives(x.x), negatives(x.y), negatives(x.z), negatives(x.w));
            uint8_t* dst = columns + r * kRowBytes + swizzle(r, load_chunk) * 16;
            *reinterpret_cast<uint4*>(dst) = n;
            *reinterpret_cast<uint4*>(dst + block_bytes) = make_uint4(x.x ^ n.x, x.y ^ n.y, x.z ^ n.z, x.w ^ n.w);
        }
    }
    __syncthreads();
    for (; page0 < pages; page0 += kTilePages) {
        uint4 lo[kSteps], hi[kSteps];
#pragma unroll
        for (int i = 0; i < kSteps; ++i) lo[i] = bound[0][i], hi[i] = bound[1][i];
        if (last_block) top_of<DT>(p, lo, hi, s, head, page0, there);
        if (page0 + kTilePages < pages) {
            load(id);
            id = fetch(page0 + 2 * kTilePages);
        }
        float best[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
        int t0 = 0, h = 0;
        uint4 neg[kSteps], pos[kSteps];
        const uint8_t* mine = columns + col * kRowBytes;
        auto read = [&](int j) {
#pragma unroll
            for (int i = 0; i < kSteps; ++i) {
                const uint8_t* src = mine + 16 * j * kRowBytes + swizzle(col, 4 * i + quad) * 16;
                neg[i] = *reinterpret_cast<const uint4*>(src);
                pos[i] = *reinterpret_cast<const uint4*>(src + block_bytes);
            }
        };
        read(0);
        for (int j = 0; j < products; ++j) {
            f32x4 sum[2] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
#pragma unroll
            for (int i = 0; i < kSteps; ++i) {
                sum[0] = mfma16<DT>(lo[i], neg[i], sum[0]);
                sum[1] = mfma16<DT>(hi[i], pos[i], sum[1]);
            }
            if (j + 1 < products) read(j + 1);
            const f32x4 sc = sum[0] + sum[1];
#pragma unroll
            for (int e = 0; e < 4; ++e) best[e] = fmaxf(best[e], fabsf(sc[e]) < INFINITY ? sc[e] : INFINITY);
            if (++h < p.group) continue;
            const int to = page0 + 4 * quad;
            if (t0 + col < tokens && to < p.score_stride) {
                float* dst = scores_of(p, seq.row0 + token0 + t0 + col, head) + to;
#pragma unroll
                for (int e = 0; e < 4; ++e) best[e] = best[e] < INFINITY ? best[e] : NAN;
                *reinterpret_cast<float4*>(dst) = make_float4(best[0], best[1], best[2], best[3]);
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) best[e] = -INFINITY;
            h = 0;
            t0 += 16;
        }
    }
}

// ---- selection --------------------------------------------------------------------
// Which pages have the highest scores must not depend on how fp32 sums were rounded.
// A score is a sum of head_dim products other than 0 (of a column's two one is), each
// exact in fp32, in two parts at most: it is off by at most
//     E = (head_dim + 2) (2^-23 |q|_1 B + 2^-125 (1 + |q|_1 + B)),
// B being the greatest finite bound (every addition rounds or cuts by 2^-23 of what it
// holds, a number too small for fp32 loses 2^-126 times its partner).  Of k pages that
// are wanted, u have a score that is no finite number, which tells nothing of its rank
// (their sums pass fp32, or infinity or NaN is in them): each may be before or behind
// every other.  If T is the k-th highest of the finite fp32 scores and S the (k - u)-th,
// pages above S + 2 E are among the k highest and those below T - 2 E are not.  Those
// between, hardly ever more than a few, and the u are scored in fp64 and ranked; equal
// ones by their place.  NaN counts as more than every number.

constexpr int kBins = 2048;
constexpr int kFew = 256;
constexpr uint32_t kChosen = 0xFFFFFFFFu;   // in the place of a page's key: it is taken; 0: it is not
constexpr uint32_t kUnknown = 1;            // its score is no finite number

__device__ __forceinline__ uint32_t order_of(float x) {       // of finite numbers: neither 0 nor kChosen; -0 as 0
    const uint32_t b = __float_as_uint(x + 0.f);
    return b >> 31 ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float number_of(uint32_t k) { return __uint_as_float(k >> 31 ? k & 0x7FFFFFFFu : ~k); }
// (Neither word that is upper in the place of a number is 0 or kChosen.)
__device__ __forceinline__ uint64_t order_of(double x) {
    if (x != x) return 0xFFFFFFFE00000000ull;
    const uint64_t b = (uint64_t)__double_as_longlong(x + 0.0);
    return b >> 63 ? ~b : b | 1ull << 63;
}

struct PickSums {
    uint32_t least, most;            // keys of open pages whose scores are finite
    int forced, open, unknown;       // pages
    float sum, top;                  // |q|_1, the greatest bound
};

template <int THREADS>
struct PickShared {
    static constexpr int kThreads = THREADS, kWaves = THREADS / 64;
    int bins[kBins];
    uint64_t few[THREADS];
    int few_page[kFew];
    uint64_t ends[2][kWaves];
    int scan[kWaves];
    PickSums sums[kWaves];
    int found[3], n_few, n_near;
    uint32_t kth;
};

// The bin where a count from bin 0 on reaches `left`: its number, what lies in the bins before it, what is in it.
template <class Shared>
__device__ __forceinline__ void find_bin(Shared& sh, int left) {
    constexpr int kOwn = kBins / Shared::kThreads;
    const int tid = (int)threadIdx.x, lane = tid & 63, wave = tid >> 6;
    int of[kOwn], own = 0;
#pragma unroll
    for (int j = 0; j < kOwn; ++j) own += of[j] = sh.bins[kOwn * tid + j];
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
    for (int j = 0; j < kOwn; ++j) {
        if (before < left && left <= before + of[j]) sh.found[0] = kOwn * tid + j, sh.found[1] = before, sh.found[2] = of[j];
        before += of[j];
    }
    __syncthreads();
}

// The left-th highest of the keys from least to most, which are n keys' range of open pages; bins are 0 and n_few is.
// Two turns at most with a few hundred keys in a bin of the first: these are ranked by counting.
template <class Shared>
__device__ __forceinline__ uint32_t kth_key(Shared& sh, const uint32_t* keys, int n, uint32_t least, uint32_t most, int left) {
    constexpr int kThreads = Shared::kThreads;
    const int tid = (int)threadIdx.x;
    while (least != most) {
        const int bits = 32 - __clz((int)(most - least)), shift = bits > 11 ? bits - 11 : 0;
        for (int i = tid; i < n; i += kThreads) {
            const uint32_t k = keys[i];
            if (k >= least && k <= most) atomicAdd(&sh.bins[(most - k) >> shift], 1);        // bin 0: the highest
        }
        __syncthreads();
        find_bin(sh, left);
        most -= (uint32_t)sh.found[0] << shift;
        least = max(least, most - min(most, (uint32_t)((1ull << shift) - 1)));
        left -= sh.found[1];
        const int inside = sh.found[2];
        if (inside <= kFew) {
            for (int i = tid; i < n; i += kThreads) {
                const uint32_t k = keys[i];
                if (k >= least && k <= most) sh.few[atomicAdd(&sh.n_few, 1)] = k;
            }
            __syncthreads();
            if (tid < inside) {
                const uint64_t mine = sh.few[tid];
                int more = 0, same = 0;
#pragma unroll 8
                for (int j = 0; j < inside; ++j) more += sh.few[j] > mine, same += sh.few[j] == mine;
                if (more < left && left <= more + same) sh.kth = (uint32_t)mine;
            }
            __syncthreads();
            return sh.kth;
        }
        for (int i = tid; i < kBins; i += kThreads) sh.bins[i] = 0;
        __syncthreads();
    }
    return least;
}

// Closing in on the `left`-th highest of some keys.  visit(f) calls f(key) for each, all threads taking part.  On
// return keys above `high` are among the highest, and `left` of those from low to high, which are all equal or as
// many as that (then `left` is 0 below: all of them).
template <class Shared, class Key, class Visit>
__device__ __forceinline__ void close_in(Shared& sh, Visit&& visit, Key& low, Key& high, int& left) {
    constexpr int kThreads = Shared::kThreads;
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
        for (int i = tid; i < kBins; i += kThreads) sh.bins[i] = 0;
        __syncthreads();
        least = sh.ends[0][0], most = sh.ends[1][0];
#pragma unroll
        for (int w = 1; w < Shared::kWaves; ++w) {
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
        find_bin(sh, left);
        high = (Key)(most - ((uint64_t)sh.found[0] << shift));
        const uint64_t width = ((uint64_t)1 << shift) - 1;
        if ((uint64_t)high - (uint64_t)low > width) low = (Key)((uint64_t)high - width);
        left -= sh.found[1];
    }
}

// The keys from low to high are those that fp32 sums cannot tell from the k-th highest.
__device__ __forceinline__ void border(const SelectParams& p, float sum, float top, uint32_t kth_key, uint32_t& low, uint32_t& high) {
    // (a hundredth more than E for the rounding of the sum, of E itself and of the borders)
    const float err = 1.01f * (float)(p.head_dim + 2) * (0x1p-23f * sum * top + 0x1p-125f * (1.f + sum + top));
    const float kth = number_of(kth_key), reach = 2.f * err + 0x1p-22f * fabsf(kth);
    if (!(reach < INFINITY)) return;
    const float a = kth - reach, b = kth + reach;
    low = a > -INFINITY ? order_of(a) : 1u;
    high = b < INFINITY ? order_of(b) : kChosen - 1;
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

// One workgroup for a row and KV head.  Keys are in LDS, or (IN_LDS false) behind the scores.
template <int DT, int THREADS, bool IN_LDS>
__global__ __launch_bounds__(THREADS) void pick_kernel(SelectParams p) {
    extern __shared__ uint32_t lds_keys[];
    constexpr int kWaves = THREADS / 64;
    __shared__ PickShared<THREADS> sh;
    const int tid = (int)threadIdx.x, lane = tid & 63, wave = uniform(tid >> 6);
    const int64_t unit = (int64_t)p.first_block + blockIdx.x;
    const int row = p.row0 + (int)(unit / p.kv_heads), head = (int)(unit % p.kv_heads);
    int s = find_above(p.batch.starts + 1, p.batch.n_seqs, row);
    if (s >= p.batch.n_seqs) return;
    const Seq seq = uniform(seq_of(p.batch, s));
    if (row < seq.row0 || row >= seq.row0 + seq.n_new) return;
    const int n = pages_seen(p, seq, row - seq.row0 + 1);
    if (n <= p.few_pages) return;
    uint32_t* scores = reinterpret_cast<uint32_t*>(scores_of(p, row, head));   // (as words, since keys' lower ones may take their place)
    uint32_t* keys;
    if constexpr (IN_LDS) keys = lds_keys;
    else keys = scores + p.score_stride / 2;
    const uint8_t* q = p.q + 2 * ((int64_t)row * p.q_stride + (int64_t)head * p.group * p.head_dim);
    int32_t* out = p.out + ((int64_t)row * p.kv_heads + head) * p.budget;

    for (int i = tid; i < kBins; i += THREADS) sh.bins[i] = 0;
    if (tid == 0) sh.n_few = sh.n_near = 0;
    PickSums all{kChosen, 0, 0, 0, 0, 0.f, 0.f};
    auto larger = [](float a, float b) { return a > b || a != a ? a : b; };   // NaN above all
    for (int h = wave; h < p.group; h += kWaves) {
        float x = 0.f;
        for (int d = 2 * lane; d < p.head_dim; d += 128) {
            const uint32_t w = *reinterpret_cast<const uint32_t*>(q + 2 * ((int64_t)h * p.head_dim + d));
            x += fabsf(hot_lo<DT>(w)) + fabsf(hot_hi<DT>(w));
        }
        all.sum = larger(xor_sum(x, 64), all.sum);
    }
    const float* tops = p.top + ((int64_t)s * p.kv_heads + head) * p.tops;
    for (int i = tid; i < (n + 15) / 16; i += THREADS) all.top = larger(tops[i], all.top);
    for (int base = 0; base < n; base += 4 * THREADS) {       // four loads in flight
        float x[4];
        int id[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int i = base + j * THREADS + tid;
            x[j] = i < n ? __uint_as_float(scores[i]) : 0.f;
            id[j] = i < n ? seq.entry(i) : -1;
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int i = base + j * THREADS + tid;
            const bool there = id[j] >= 0 && id[j] < p.batch.n_pages, always = there && (i < p.sink || i >= n - p.recent);
            const bool may = there && !always, known = x[j] == x[j];
            const uint32_t k = always ? kChosen : may ? (known ? order_of(x[j]) : kUnknown) : 0u;
            if (i < n) keys[i] = k;
            if (may && known) all.least = min(all.least, k), all.most = max(all.most, k);
            all.forced += __popcll(__ballot(always)), all.open += __popcll(__ballot(may)), all.unknown += __popcll(__ballot(may && !known));
        }
    }
    auto join = [&](int width, bool counts) {
        for (int m = 1; m < width; m <<= 1) {
            all.least = min(all.least, (uint32_t)__shfl_xor((int)all.least, m));
            all.most = max(all.most, (uint32_t)__shfl_xor((int)all.most, m));
            all.top = larger(__shfl_xor(all.top, m), all.top);
            if (!counts) continue;
            all.sum = larger(__shfl_xor(all.sum, m), all.sum);
            all.forced += __shfl_xor(all.forced, m);
            all.open += __shfl_xor(all.open, m);
            all.unknown += __shfl_xor(all.unknown, m);
        }
    };
    join(64, false);
    if (lane == 0) sh.sums[wave] = all;
    __syncthreads();
    all = sh.sums[lane % kWaves];
    join(kWaves, true);
    const int wanted = p.budget - all.forced;
    bool every = all.open <= wanted;                          // what is neither 0 nor kChosen by the end is taken
    if (!every && wanted > 0) {
        // keys of pages that may or may not be taken, beside kUnknown: from what fp32 sums cannot tell from the k-th highest
        // to what they cannot tell from the (k - u)-th
        uint32_t low = kUnknown + 1, high = kChosen - 1;
        for (int nth = wanted;; nth = wanted - all.unknown) {
            if (nth > 0 && nth <= all.open - all.unknown) {
                uint32_t from = low, to = high;
                border(p, all.sum, all.top, kth_key(sh, keys, n, all.least, all.most, nth), from, to);
                if (nth == wanted) low = from;
                if (nth == wanted - all.unknown) high = to;
            }
            if (nth == wanted - all.unknown) break;
            __syncthreads();                                  // the first key has been read
            for (int i = tid; i < kBins; i += THREADS) sh.bins[i] = 0;
            if (tid == 0) sh.n_few = 0;
            __syncthreads();
        }
        int above = 0;
        for (int base = 0; base < n; base += THREADS) {
            const int i = base + tid;
            const uint32_t k = i < n ? keys[i] : 0u;
            const bool over = k > high && k != kChosen;
            above += __popcll(__ballot(over));
            if (over) keys[i] = kChosen;
            if (k == kUnknown || (k >= low && k <= high)) {
                const int at = atomicAdd(&sh.n_near, 1);
                if (at < kFew) sh.few_page[at] = i;
            }
        }
        if (lane == 0) sh.scan[wave] = above;
        __syncthreads();
        above = 0;
#pragma unroll
        for (int w = 0; w < kWaves; ++w) above += sh.scan[w];
        const int left = wanted - above, near = sh.n_near;
        if (near <= left) {                                   // all that are near, and of the others none
            for (int i = tid; i < n; i += THREADS) keys[i] = keys[i] >= low || keys[i] == kUnknown ? kChosen : 0u;
        } else if (near <= kFew) {
            for (int j = wave; j < near; j += kWaves) {
                const uint64_t x = exact_key<DT>(p, q, seq.entry(sh.few_page[j]), head);
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
        } else {
            // each once: their upper words in the place of the keys, the lower ones in that of the scores
            for (int i = wave; i < n; i += kWaves) {
                const uint32_t k = keys[i];
                if (k == kChosen) continue;
                const bool is = k == kUnknown || k >= low;    // (above high they are taken)
                const uint64_t x = is ? exact_key<DT>(p, q, seq.entry(i), head) : 0ull;
                if (lane == 0) keys[i] = (uint32_t)(x >> 32), scores[i] = (uint32_t)x;
            }
            __syncthreads();
            auto exact = [&](int i) {                         // 0: it is taken, or is not near
                const uint32_t k = i < n ? keys[i] : 0u;
                return k == 0 || k == kChosen ? 0ull : (uint64_t)k << 32 | scores[i];
            };
            uint64_t exact_low = 1, exact_high = ~0ull;
            int ties = left;
            close_in(sh, [&](auto&& f) { for (int i = tid; i < n; i += THREADS) f(exact(i)); }, exact_low, exact_high, ties);
            int tied = 0;
            for (int base = 0; base < n; base += THREADS) {
                const int i = base + tid;
                const uint64_t x = exact(i);
                const bool tie = x >= exact_low && x <= exact_high;
                const uint64_t all_ties = __ballot(tie);
                __syncthreads();
                if (lane == 0) sh.scan[wave] = __popcll(all_ties);
                __syncthreads();
                int rank = tied + __popcll(all_ties & ((1ull << lane) - 1));
                for (int w = 0; w < kWaves; ++w) {
                    rank += w < wave ? sh.scan[w] : 0;
                    tied += sh.scan[w];
                }
                if (x != 0) keys[i] = x > exact_high || (tie && rank < ties) ? kChosen : 0u;
            }
        }
    }
    __syncthreads();
    // a wave has a run of pages
    const int run = (n + THREADS - 1) / THREADS * 64, run0 = wave * run, run1 = min(run0 + run, n);
    int mine = 0;
    auto is_taken = [&](int i) { return i < run1 && (keys[i] == kChosen || (every && keys[i] != 0)); };
    for (int base = run0; base < run1; base += 64) mine += __popcll(__ballot(is_taken(base + lane)));
    if (lane == 0) sh.scan[wave] = mine;
    __syncthreads();
    int at = 0, total = 0;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
        at += w < wave ? sh.scan[w] : 0;
        total += sh.scan[w];
    }
    for (int base = run0; base < run1; base += 64) {
        const bool taken = is_taken(base + lane);
        const uint64_t mask = __ballot(taken);
        const int to = at + __popcll(mask & ((1ull << lane) - 1));
        if (taken && to < p.budget) out[to] = base + lane;
        at += __popcll(mask);
    }
    for (int i = total + tid; i < p.budget; i += THREADS) out[i] = -1;
}

// f over a wave's 64 numbers, in every lane, without LDS.
template <class F>
__device__ __forceinline__ uint32_t over_wave(uint32_t x, F&& f, int width = 64) {
    x = f(x, __float_as_uint(partner<0xB1>(__uint_as_float(x))));
    x = f(x, __float_as_uint(partner<0x4E>(__uint_as_float(x))));
    x = f(x, __float_as_uint(partner<0x141>(__uint_as_float(x))));
    x = f(x, __float_as_uint(partner<0x140>(__uint_as_float(x))));
    if (width > 16) {
        const u32x2 r = __builtin_amdgcn_permlane16_swap(x, x, false, false);
        x = f(r.x, r.y);
    }
    if (width > 32) {
        const u32x2 r = __builtin_amdgcn_permlane32_swap(x, x, false, false);
        x = f(r.x, r.y);
    }
    return x;
}
__device__ __forceinline__ float wave_max(float x) {           // NaN if there is one
    const bool nan = __any(x != x);
    x = __uint_as_float(over_wave(__float_as_uint(x), [](uint32_t a, uint32_t b) { return __float_as_uint(fmaxf(__uint_as_float(a), __uint_as_float(b))); }));
    return nan ? NAN : x;
}

// The same for rows of at most 1,024 pages: one wave for a row and KV head, its keys in registers, which pages are taken
// in the bits of a word of each lane, and the k-th highest key found bit by bit.
//
// 4,000 rows of 5 KV heads over 525 pages: 205 us by workgroups, 50 so.
constexpr int kFewPages = 1024;

template <int DT, int OWN>
__global__ __launch_bounds__(256) void pick_few_kernel(SelectParams p) {
    constexpr int kOwn = OWN;                                 // pages of a lane: 64 OWN are enough for every row
    const int lane = (int)threadIdx.x & 63;
    const int64_t unit = ((int64_t)p.first_block + blockIdx.x) * 4 + uniform((int)threadIdx.x >> 6);
    const int64_t wide_row = p.row0 + unit / p.kv_heads;
    if (wide_row >= p.row1) return;
    const int row = (int)wide_row, head = (int)(unit % p.kv_heads);
    const int s = uniform(find_above(p.batch.starts + 1, p.batch.n_seqs, row));
    if (s >= p.batch.n_seqs) return;
    const Seq seq = uniform(seq_of(p.batch, s));
    if (row < seq.row0 || row >= seq.row0 + seq.n_new) return;
    const int n = uniform(pages_seen(p, seq, row - seq.row0 + 1));
    if (n > 64 * OWN) return;                                 // (another kernel's)
    const float* scores = scores_of(p, row, head);
    const uint8_t* q = p.q + 2 * ((int64_t)row * p.q_stride + (int64_t)head * p.group * p.head_dim);
    int32_t* out = p.out + ((int64_t)row * p.kv_heads + head) * p.budget;

    // |q|_1, of four heads at once (two of vectors of more than 128 elements), and the greatest bound
    float sum = 0.f;
    const float top = wave_max(lane < (n + 15) / 16 ? p.top[((int64_t)s * p.kv_heads + head) * p.tops + lane] : 0.f);
    {
        const int width = p.head_dim <= 128 ? 16 : 32, chunk = lane % width;
        for (int h0 = 0; h0 < p.group; h0 += 64 / width) {
            const int h = min(h0 + lane / width, p.group - 1);
            const uint4 x = 8 * chunk < p.head_dim ? ldg16(q + 2 * ((int64_t)h * p.head_dim + 8 * chunk)) : make_uint4(0, 0, 0, 0);
            const uint32_t w[4] = {x.x, x.y, x.z, x.w};
            float part = 0.f;
#pragma unroll
            for (int e = 0; e < 4; ++e) part += fabsf(hot_lo<DT>(w[e])) + fabsf(hot_hi<DT>(w[e]));
            part = __uint_as_float(over_wave(__float_as_uint(part),
                                             [](uint32_t a, uint32_t b) { return __float_as_uint(__uint_as_float(a) + __uint_as_float(b)); }, width));
            part = wave_max(part);
            sum = part > sum || part != part ? part : sum;
        }
    }
    uint32_t key[kOwn], taken = 0, nears = 0;                 // key 0: not open; bit c: of page 64 c + lane
    int forced = 0, open = 0, unknown = 0;
    int id[kOwn];
    {
        float x[kOwn];
#pragma unroll
        for (int c = 0; c < kOwn; ++c) {
            const int i = min(64 * c + lane, n - 1);
            x[c] = 64 * c < n ? scores[i] : 0.f;
            id[c] = 64 * c < n ? seq.entry(i) : -1;
        }
#pragma unroll
        for (int c = 0; c < kOwn; ++c) {
            key[c] = 0;
            if (64 * c >= n) continue;
            const int i = 64 * c + lane;
            const bool there = i < n && (uint32_t)id[c] < (uint32_t)p.batch.n_pages, known = x[c] == x[c];
            if (there) key[c] = known ? order_of(x[c]) : kUnknown;
            if (64 * c < p.sink || 64 * c + 64 > n - p.recent) {   // some that are always taken
                const bool always = there && (i < p.sink || i >= n - p.recent);
                if (always) key[c] = 0, taken |= 1u << c;
                forced += __popcll(__ballot(always));
            }
            open += __popcll(__ballot(key[c] != 0));
            unknown += __popcll(__ballot(key[c] == kUnknown));
        }
    }
    auto count = [&](auto&& is) {
        int total = 0;
#pragma unroll
        for (int c = 0; c < kOwn; ++c) total += __popcll(__ballot(is(c)));
        return total;
    };
    const int wanted = p.budget - forced;
    if (open <= wanted) {
#pragma unroll
        for (int c = 0; c < kOwn; ++c) taken |= key[c] != 0 ? 1u << c : 0u;
    } else if (wanted > 0) {
        uint32_t low = kUnknown + 1, high = kChosen - 1;      // as in pick_kernel
        for (int nth = wanted;; nth = wanted - unknown) {
            if (nth > 0 && nth <= open - unknown) {
                uint32_t least = kChosen, most = 0;           // the nth highest is one of these and those between
#pragma unroll
                for (int c = 0; c < kOwn; ++c) {
                    least = key[c] > kUnknown ? min(least, key[c]) : least;
                    most = max(most, key[c]);
                }
                auto lower = [](uint32_t a, uint32_t b) { return min(a, b); };
                least = (uint32_t)uniform((int)over_wave(least, lower));
                most = (uint32_t)uniform((int)over_wave(most, [](uint32_t a, uint32_t b) { return max(a, b); }));
                while (least < most) {
                    const uint32_t t = least + (most - least + 1) / 2;
                    const int reach = count([&](int c) { return key[c] >= t; });
                    if (reach >= nth) least = t;
                    else most = t - 1;
                    if (reach != nth) continue;
                    most = kChosen;                           // the least of these
#pragma unroll
                    for (int c = 0; c < kOwn; ++c) most = key[c] >= t ? min(most, key[c]) : most;
                    least = most = (uint32_t)uniform((int)over_wave(most, lower));
                }
                uint32_t from = low, to = high;
                border(p, sum, top, least, from, to);
                if (nth == wanted) low = from;
                if (nth == wanted - unknown) high = to;
            }
            if (nth == wanted - unknown) break;
        }
        int above = 0, near = 0;
#pragma unroll
        for (int c = 0; c < kOwn; ++c) {
            if (64 * c >= n) continue;
            const bool over = key[c] > high, is = key[c] == kUnknown || (key[c] >= low && key[c] <= high);
            above += __popcll(__ballot(over));
            near += __popcll(__ballot(is));
            taken |= over ? 1u << c : 0u;
            nears |= is ? 1u << c : 0u;
        }
        const int left = wanted - above;
        if (near <= left) {
            taken |= nears;
        } else {
            uint64_t exact[kOwn];                             // of this lane's near pages; 0 for the others
#pragma unroll
            for (int c = 0; c < kOwn; ++c) {
                exact[c] = 0;
                if (64 * c >= n) continue;
                for (uint64_t todo = __ballot(nears >> c & 1); todo; todo &= todo - 1) {
                    const int from = __ffsll((unsigned long long)todo) - 1;
                    const uint64_t x = exact_key<DT>(p, q, __builtin_amdgcn_readlane(id[c], from), head);
                    if (lane == from) exact[c] = x;
                }
            }
            uint64_t kth_key = 0;
            int reach = near;
            for (int bit = 63; bit >= 0 && reach != left; --bit) {
                const uint64_t t = kth_key | 1ull << bit;
                const int r = count([&](int c) { return exact[c] >= t; });
                if (r >= left) kth_key = t, reach = r;
            }
            // those above are taken, and as many as are left of those equal to it
            int ties = left - (reach == left ? left : count([&](int c) { return exact[c] > kth_key; }));
#pragma unroll
            for (int c = 0; c < kOwn; ++c) {
                if (64 * c >= n) continue;
                const bool tie = reach != left && exact[c] == kth_key;
                const uint64_t all = __ballot(tie);
                const bool in = reach == left ? exact[c] >= kth_key && exact[c] != 0
                                              : exact[c] > kth_key || (tie && __popcll(all & ((1ull << lane) - 1)) < ties);
                taken |= in ? 1u << c : 0u;
                ties -= min(ties, (int)__popcll(all));
            }
        }
    }
    int at = 0;
#pragma unroll
    for (int c = 0; c < kOwn; ++c) {
        if (64 * c >= n) continue;
        const uint64_t all = __ballot(taken >> c & 1);
        const int to = at + __popcll(all & ((1ull << lane) - 1));
        if ((taken >> c & 1) && to < p.budget) out[to] = 64 * c + lane;
        at += __popcll(all);
    }
    for (int i = at + lane; i < p.budget; i += 64) out[i] = -1;
}

// The kernel with as many registers of keys as a table's columns need: every turn of the search compares and counts all of
// them (selections of 2 x 2,000 rows of 5 KV heads over 520 pages: 83 us with 9 registers, 91 with 12; over 600: 90 with 10,
// 93 with 12, 107 with 16).
template <int DT, int OWN>
auto pick_few(int64_t max_pages) -> void (*)(SelectParams) {
    if constexpr (OWN > 1)
        if (max_pages <= 64 * (OWN - 1)) return pick_few<DT, OWN - 1>(max_pages);
    return pick_few_kernel<DT, OWN>;
}

constexpr int kKeysInLds = 12288;   // 48 KiB

// What is wrong with bounds [n_pages, 2, num_heads, head_dim], pages `stride` elements apart, or nullptr.
const char* check_bounds(const void* bounds, int64_t stride, const ztcp_geometry* g, int64_t n_pages) {
    if (!bounds || !hot_aligned(bounds) || stride % 8 != 0) return "bounds must not be NULL, and 16-byte aligned";
    if (n_pages > 1 && stride < 2 * g->num_heads * g->head_dim) return "bounds' stride must cover a page's";
    return nullptr;
}

struct SelectPlan {
    int64_t stride, tops, units;     // words of a row's scores, and of its keys where these are not in LDS; units: 64 pages and a block of tokens each, at most
    int64_t scores, rows, floats;    // scores of the call; rows that are scored and chosen for at a time; the workspace
};
SelectPlan plan_select(const ztcp_paged_batch* b, const ztcp_geometry* g) {
    SelectPlan plan;
    plan.stride = (b->max_pages + 3) / 4 * 4 * (b->max_pages > kKeysInLds ? 2 : 1);
    plan.tops = (b->max_pages + 15) / 16;
    plan.units = (b->n_rows / kBlockTokens + b->n_seqs) * ((b->max_pages + kTilePages - 1) / kTilePages);
    const int64_t row = g->num_heads * plan.stride, most = kMostBetween / (row * (int64_t)sizeof(float));
    plan.scores = b->n_rows * row;
    const int64_t parts = b->n_rows > 0 ? (b->n_rows - 1) / (most > 0 ? most : 1) + 1 : 1;
    plan.rows = (b->n_rows + parts - 1) / parts;             // alike
    plan.floats = plan.rows * row + (b->n_seqs * g->num_heads * plan.tops + 3) / 4 * 4;
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
    if (plan.stride >= (int64_t)1 << 31 || plan.units * g->num_heads >= (int64_t)1 << 31 || plan.scores >= (int64_t)1 << 40)
        return "too many rows and pages in one call";
    return nullptr;
}

}  // namespace

extern "C" int ztcp_page_bounds(const ztcp_page_pool* pool, const ztcp_paged_batch* batch, const ztcp_geometry* g, void* bounds,
                                int64_t bounds_stride, void* stream) {
    arg_result(ZTCP_OK, "");
    BoundsParams p{};
    if (const char* why = check_pool(pool, g, 1024)) return arg_result(ZTCP_EINVAL, why);
    if (!batch) return arg_result(ZTCP_EINVAL, "batch must not be NULL");
    if (batch->n_rows < 0 || batch->n_rows >= (int64_t)1 << 31) return arg_result(ZTCP_EINVAL, "n_rows must be 0 .. 2^31 - 1");
    ztcp_paged_batch rest = *batch;                           // there is no q, whose rows times heads are bounded
    rest.n_rows = 0;
    if (const char* why = check_batch(&rest, pool, g, g->num_heads, p.batch)) return arg_result(ZTCP_EINVAL, why);
    p.batch.n_rows = (int32_t)batch->n_rows;
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
    int cus = 0;
    if (cu_count(cus) != ZTCP_OK) return ZTCP_EHIP;
    // as many as the card holds at once, and no more than units
    const int64_t resident = (int64_t)cus * (d <= 64 ? 5 : d <= 128 ? 3 : 1), each = (resident + g->num_heads - 1) / g->num_heads;
    p.score_groups = (int32_t)(each < plan.units ? each : plan.units);
    // chunks: sequences of more than 16 new tokens on average, as many workgroups as half the compute units at least
    const int64_t block = chunk_tokens(p.group, d <= 128 ? 128 : 256);
    const size_t chunk_lds = (size_t)(block * p.group) * (d <= 64 ? 64 : d <= 128 ? 128 : 256) * 4;
    const int64_t pieces = (batch->max_pages + kPieceTiles * kTilePages - 1) / (kPieceTiles * kTilePages);
    auto go = [&](auto dt) {
        constexpr int DT = decltype(dt)::value;
        const int64_t rows = p.row1 - p.row0;
        int64_t chunk_units = 0;
        if (block > 0 && batch->n_rows > 16 * batch->n_seqs) {
            chunk_units = (rows / block + batch->n_seqs) * pieces * g->num_heads;
            if (rows / block * g->num_heads < cus / 2 || chunk_units >= (int64_t)1 << 31) chunk_units = 0;
        }
        if (chunk_units > 0) {
            auto kernel = d <= 64 ? score_chunk_kernel<DT, 64, 2> : d <= 96 ? score_chunk_kernel<DT, 128, 3> : d <= 128 ? score_chunk_kernel<DT, 128, 4>
                        : d <= 192 ? score_chunk_kernel<DT, 256, 6> : score_chunk_kernel<DT, 256, 8>;
            // over 64 KiB of dynamic LDS has to be asked for
            if (chunk_lds > (size_t)48 * 1024 &&
                hipFuncSetAttribute((const void*)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, 64 * 1024) != hipSuccess)
                return false;
            launch_blocks(kernel, (uint64_t)chunk_units, 256, chunk_lds, (hipStream_t)stream, p);
        } else {
            const dim3 grid((uint32_t)(g->num_heads * p.score_groups));
            hipLaunchKernelGGL((d <= 64 ? score_kernel<DT, 64> : d <= 128 ? score_kernel<DT, 128> : score_kernel<DT, 256>), grid, dim3(256),
                               0, (hipStream_t)stream, p);
        }
        const uint64_t picks = (uint64_t)rows * (uint64_t)g->num_heads;
        const bool many = picks > 2 * (uint64_t)cus;          // rows: a wave each if their pages are few
        if (batch->max_pages <= kFewPages || many)
            launch_blocks(pick_few<DT, kFewPages / 64>(batch->max_pages), (picks + 3) / 4, 256, 0, (hipStream_t)stream, p);
        if (batch->max_pages <= kFewPages) return true;
        p.few_pages = many ? kFewPages : -1;
        const bool in_lds = batch->max_pages <= kKeysInLds;
        const size_t lds = in_lds ? (size_t)batch->max_pages * 4 : 0;
        if (many) launch_blocks(in_lds ? pick_kernel<DT, 256, true> : pick_kernel<DT, 256, false>, picks, 256, lds, (hipStream_t)stream, p);
        else launch_blocks(in_lds ? pick_kernel<DT, 1024, true> : pick_kernel<DT, 1024, false>, picks, 1024, lds, (hipStream_t)stream, p);
        return true;
    };
    // rows of as many scores as the workspace holds, and then those behind them in the same place
    for (int64_t row0 = 0; row0 < batch->n_rows; row0 += plan.rows) {
        p.row0 = (int32_t)row0;
        p.row1 = (int32_t)(batch->n_rows - row0 < plan.rows ? batch->n_rows : row0 + plan.rows);
        if (!(g->hot_dtype == ZTCP_HOT_BF16 ? go(std::integral_constant<int, kHotBf16>{}) : go(std::integral_constant<int, kHotFp16>{})))
            return ZTCP_EHIP;
    }
    return hipGetLastError() == hipSuccess ? ZTCP_OK : ZTCP_EHIP;
}
