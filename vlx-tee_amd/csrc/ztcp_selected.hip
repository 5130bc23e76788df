// ztcp_selected.hip -- attention of new tokens over pages that each of them,
// for each KV head, has picked.
//
// The formula is paged attention's with the sums over the tokens of the listed
// pages that the row sees.
//
// Few rows (decoding): a row and KV head are a unit of their own, whose query heads
// are the columns of the products (16; a group of fewer leaves columns idle, which
// costs nothing where reading K and V is the work), and all of them see the same
// tokens.  Many rows (chunks): a workgroup takes 128 rows of a KV head over the pages
// that any of them lists, and each row's list says which of these it sees.
#include <type_traits>

#include "ztcp_hot.h"

using namespace ztcp;

namespace {

struct SelectedParams {
    PagedView batch;
    const uint8_t* q;
    uint8_t* out;
    float* lse;                      // or nullptr
    int64_t q_stride;                // elements between tokens
    const uint8_t* k_pool;
    const uint8_t* v_pool;
    int64_t k_page, v_page;          // elements between pages
    const int32_t* selected;         // [rows, kv_heads, listed]
    int32_t listed, max_pages;
    int32_t kv_heads, group, head_dim;
    float scale_log2;                // scale * log2(e): exponentials are powers of two
    int32_t splits, piece;           // pieces of a unit's keys, and their keys
    float* partial;                  // results of pieces: sums [head_dim], maximum, total
    int2* lists;                     // blocks: for each workgroup of a launch list_stride columns and pages that its rows list
    uint32_t* masks;                 // and for each of these the tokens that list it
    int64_t list_stride;
    uint32_t first_block;            // of this launch
};

__device__ __forceinline__ float* partial_of(const SelectedParams& p, int row, int q_head, int split) {
    return p.partial + (((int64_t)row * p.kv_heads * p.group + q_head) * p.splits + split) * (p.head_dim + 2);
}

// ---- by rows ----------------------------------------------------------------------
// A workgroup of WAVES waves takes a piece of a unit's keys, 32 a wave and turn, with a wave's loads of the next 32 in
// flight while it works on these: K and V by whole rows through LDS of its own (K of vectors of more than 128 elements
// as the products want it).  Scores are made transposed: a column is a query head.
template <int DT, int DP, int WAVES>
__global__ __launch_bounds__(64 * WAVES) __attribute__((amdgpu_waves_per_eu(DP <= 128 ? 2 : 1)))
void selected_kernel(SelectedParams p) {
    constexpr int kSteps = DP / 32, kChunks = DP / 8;         // products of depth 32; 16-byte pieces of a row
    constexpr int kVLoads = 32 * kChunks / 64, kVRows = 64 / kChunks;
    constexpr int kJoinRow = DP + 4;
    constexpr int kWaveBytes = 32 * DP * 2;
    constexpr bool kKInLds = DP <= 128;
    constexpr int kJoinBytes = WAVES > 1 ? WAVES * 16 * kJoinRow * 4 : 0;
    constexpr int kTileBytes = (kKInLds ? 2 : 1) * WAVES * kWaveBytes;
    __shared__ __attribute__((aligned(16))) uint8_t lds[kTileBytes > kJoinBytes ? kTileBytes : kJoinBytes];
    __shared__ float join_m[WAVES][16], join_l[WAVES][16];
    const int lane = (int)threadIdx.x & 63, wave = uniform((int)threadIdx.x >> 6);
    const int col = lane & 15, quad = lane >> 4;
    const uint32_t unit = p.first_block + blockIdx.x;
    const int head = (int)(unit % (uint32_t)p.kv_heads);
    const uint32_t rest = unit / (uint32_t)p.kv_heads;
    const int split = (int)(rest % (uint32_t)p.splits), row = (int)(rest / (uint32_t)p.splits);
    const int s = uniform(find_above(p.batch.starts + 1, p.batch.n_seqs, row));
    if (s >= p.batch.n_seqs) return;
    const Seq seq = uniform(seq_of(p.batch, s));
    if (row < seq.row0 || row >= seq.row0 + seq.n_new) return;
    const int limit = max(0, seq.len - seq.n_new + (row - seq.row0) + 1);   // tokens that the row sees
    const int32_t* picked = p.selected + ((int64_t)row * p.kv_heads + head) * p.listed;
    // An entry that is not above all (columns of the table) in front of it lists nothing.  Lists ascend: whether this one
    // does is looked at while the first keys are on their way, and only if it does not are the entries in front looked at.
    bool ascends = true;
    const int key0 = split * p.piece, stop = key0 + min(p.listed * p.batch.page_tokens - key0, p.piece);
    uint8_t* vt = lds + wave * kWaveBytes;
    uint8_t* kt = lds + (WAVES + wave) * kWaveBytes;          // (kKInLds)
    // 16-byte pieces are permuted within a row so that the rows of one read lie in different banks
    auto k_swizzle = [](int r, int chunk) { return chunk ^ (r & (kChunks < 16 ? kChunks - 1 : 15)); };
    auto v_swizzle = [](int r, int chunk) {
        if constexpr (DP == 64) return chunk ^ (((r >> 1) & 3) << 1);
        else return chunk ^ ((r & 7) << 1);
    };
    const int v_row = lane / kChunks, v_chunk = lane % kChunks;
    const bool v_has = v_chunk * 8 < p.head_dim;
    auto place = [&](int key) {                               // of the unit's list; page -1: not there, or not seen
        Place at{-1, 0};
        if (key < stop) {
            const int nth = div_page(key, p.batch.page_div);
            at.row = key - nth * p.batch.page_tokens;
            const int page = picked[nth];
            bool counts = page >= 0 && page < p.max_pages && page * p.batch.page_tokens + at.row < limit;
            if (!ascends)
                for (int i = 0; i < nth; ++i) counts &= !(picked[i] >= page && picked[i] < p.max_pages);
            if (counts) {
                const int id = seq.entry(page);
                if (id >= 0 && id < p.batch.n_pages) at.page = id;
            }
        }
        return at;
    };
    for (int h0 = 0; h0 < p.group; h0 += 16) {
        const int q_head = head * p.group + h0 + col;
        const bool is = h0 + col < p.group;
        uint4 qf[kSteps];
        {
            const uint8_t* src = p.q + 2 * ((int64_t)row * p.q_stride + (int64_t)q_head * p.head_dim);
#pragma unroll
            for (int i = 0; i < kSteps; ++i) {
                const int d = 32 * i + 8 * quad;
                qf[i] = is && d < p.head_dim ? ldg16(src + 2 * d) : make_uint4(0, 0, 0, 0);
            }
        }
        float m = -INFINITY, l = 0.f;
        f32x4 o[DP / 16];
#pragma unroll
        for (int i = 0; i < DP / 16; ++i) o[i] = f32x4{0.f, 0.f, 0.f, 0.f};
        uint4 kf[2][kSteps], vf[kVLoads];                     // (K in LDS: loads by whole rows as V's, in order)
        uint32_t valid = 0;                                   // keys of the loaded tile that are there
        // few rows read each page once, and leave no trace of it in the caches (32 sequences' 128 pages of 16 tokens, 269 MB:
        // 56 us with ordinary loads, 49 so); many share pages
        auto get = [](const uint8_t* src) { return WAVES > 1 ? ldg16_once(src) : ldg16(src); };
        auto load = [&](const Place& at) {
            const bool has = at.page >= 0;
            valid = (uint32_t)__ballot(has);
            const int page = has ? at.page : 0, in = has ? at.row : 0;
            if constexpr (!kKInLds) {
#pragma unroll
                for (int t = 0; t < 2; ++t) {
                    const int from = 16 * t + col;
                    const int64_t pg = __shfl(page, from), rw = __shfl(in, from);
                    const uint8_t* src = p.k_pool + 2 * (pg * p.k_page + (rw * p.kv_heads + head) * p.head_dim);
#pragma unroll
                    for (int i = 0; i < kSteps; ++i) {
                        const int d = 32 * i + 8 * quad;
                        kf[t][i] = d < p.head_dim ? ldg16(src + 2 * d) : make_uint4(0, 0, 0, 0);
                    }
                }
            }
#pragma unroll
            for (int i = 0; i < kVLoads; ++i) {
                const int from = i * kVRows + v_row;
                const int64_t pg = __shfl(page, from), rw = __shfl(in, from);
                const int64_t in_page = (rw * p.kv_heads + head) * p.head_dim;
                if constexpr (kKInLds)
                    kf[i / kSteps][i % kSteps] = v_has ? get(p.k_pool + 2 * (pg * p.k_page + in_page) + 16 * v_chunk)
                                                       : make_uint4(0, 0, 0, 0);
                vf[i] = v_has ? get(p.v_pool + 2 * (pg * p.v_page + in_page) + 16 * v_chunk) : make_uint4(0, 0, 0, 0);
            }
        };
        Place at{-1, 0};                                      // of key (lane % 32) of the tile to be loaded
        int kb = key0 + 32 * wave;
        if (kb < stop) {
            load(place(kb + (lane & 31)));
            at = place(kb + 32 * WAVES + (lane & 31));
            if (h0 == 0) {
                int most = -1;                                // of the entries in front
                for (int base = 0; base < p.listed; base += 64) {
                    const int x = base + lane < p.listed ? picked[base + lane] : -1;
                    int upto = x < p.max_pages ? x : -1;
                    const bool column = upto >= 0;
                    for (int k = 1; k < 64; k <<= 1) {
                        const int y = __shfl_up(upto, k);
                        upto = lane >= k ? max(upto, y) : upto;
                    }
                    const int in_front = __shfl_up(upto, 1), before = max(most, lane > 0 ? in_front : -1);
                    if (__any(column && x <= before)) ascends = false;
                    most = max(most, __shfl(upto, 63));
                }
                if (!ascends) {
                    load(place(kb + (lane & 31)));
                    at = place(kb + 32 * WAVES + (lane & 31));
                }
            }
        }
        for (; kb < stop; kb += 32 * WAVES) {
            const uint32_t here = valid;
#pragma unroll
            for (int i = 0; i < kVLoads; ++i) {
                const int r = i * kVRows + v_row;
                if constexpr (kKInLds)
                    *reinterpret_cast<uint4*>(kt + r * DP * 2 + k_swizzle(r, v_chunk) * 16) = kf[i / kSteps][i % kSteps];
                // what is not there or not seen has no weight, but 0 * NaN is NaN
                *reinterpret_cast<uint4*>(vt + r * DP * 2 + v_swizzle(r, v_chunk) * 16) = (here >> r) & 1u ? vf[i] : make_uint4(0, 0, 0, 0);
            }
            auto k_part = [&](int u, int i) {
                if constexpr (kKInLds)
                    return *reinterpret_cast<const uint4*>(kt + (16 * u + col) * DP * 2 + k_swizzle(col, 4 * i + quad) * 16);
                else return kf[u][i];
            };
            f32x4 sc[2];
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                sc[u] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int i = 0; i < kSteps; ++i) sc[u] = mfma16<DT>(k_part(u, i), qf[i], sc[u]);
            }
            if (kb + 32 * WAVES < stop) {
                load(at);
                at = place(kb + 64 * WAVES + (lane & 31));
            }
            float x[8];
#pragma unroll
            for (int u = 0; u < 2; ++u)
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    x[4 * u + i] = (here >> (16 * u + 4 * quad + i)) & 1u ? sc[u][i] * p.scale_log2 : -INFINITY;
            float top = fmaxf(fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])), fmaxf(fmaxf(x[4], x[5]), fmaxf(x[6], x[7])));
            top = fmaxf(top, __shfl_xor(top, 16));
            top = fmaxf(top, __shfl_xor(top, 32));
            const float m_new = fmaxf(m, top);
            const float base = m_new == -INFINITY ? 0.f : m_new;   // no key seen yet: every power is 0
            if (__any(m_new != m)) {
                const float fade = __builtin_amdgcn_exp2f(m - base);
                l *= fade;
#pragma unroll
                for (int i = 0; i < DP / 16; ++i) o[i] *= fade;
            }
            m = m_new;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                x[i] = __builtin_amdgcn_exp2f(x[i] - base);
                l += x[i];
            }
            // probabilities are rounded to the hot dtype for the product with V (their total is not): relative to the
            // result that costs about what its own final rounding does
            const uint4 pf = make_uint4(pack_hot<DT>(x[0], x[1]), pack_hot<DT>(x[2], x[3]), pack_hot<DT>(x[4], x[5]),
                                        pack_hot<DT>(x[6], x[7]));
#pragma unroll
            for (int n = 0; n < DP / 16; ++n) {
                uint2 v[2];
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    const int r = 16 * u + 4 * quad + col / 4, chunk = 2 * n + (col & 3) / 2;
                    v[u] = lds_read_transposed(vt + r * DP * 2 + v_swizzle(r, chunk) * 16 + (col & 1) * 8);
                }
                o[n] = mfma16<DT>(make_uint4(v[0].x, v[0].y, v[1].x, v[1].y), pf, o[n]);
            }
        }
        l += __shfl_xor(l, 16);
        l += __shfl_xor(l, 32);
        const int64_t row_head = (int64_t)row * p.kv_heads * p.group + q_head;
        if constexpr (WAVES == 1) {
            if (!is) continue;
            const float base = m == -INFINITY ? 0.f : m, inv = l > 0.f || l != l ? 1.f / l : 0.f;
            float* part = p.splits > 1 ? partial_of(p, row, q_head, split) : nullptr;
#pragma unroll
            for (int n = 0; n < DP / 16; ++n) {
                const int d = 16 * n + 4 * quad;
                if (d >= p.head_dim) continue;
                if (part) {
                    *reinterpret_cast<float2*>(part + d) = make_float2(o[n][0], o[n][1]);
                    *reinterpret_cast<float2*>(part + d + 2) = make_float2(o[n][2], o[n][3]);
                } else {
                    *reinterpret_cast<uint2*>(p.out + 2 * (row_head * p.head_dim + d)) =
                        make_uint2(pack_hot<DT>(o[n][0] * inv, o[n][1] * inv), pack_hot<DT>(o[n][2] * inv, o[n][3] * inv));
                }
            }
            if (quad == 0) {
                if (part) part[p.head_dim] = m, part[p.head_dim + 1] = l;
                else if (p.lse) p.lse[row_head] = l == 0.f ? -INFINITY : (base + __builtin_amdgcn_logf(l)) * kLn2;
            }
        } else {
            __syncthreads();                                  // the tiles, or the last heads' sums, have been read
            float* join = reinterpret_cast<float*>(lds);
#pragma unroll
            for (int n = 0; n < DP / 16; ++n)
                *reinterpret_cast<f32x4*>(join + (wave * 16 + col) * kJoinRow + 16 * n + 4 * quad) = o[n];
            if (quad == 0) {
                join_m[wave][col] = m;
                join_l[wave][col] = l;
            }
            __syncthreads();
            // a thread has 8 numbers of a query head's result
            for (int i = (int)threadIdx.x; i < 16 * (DP / 8); i += 64 * WAVES) {
                const int h = i / (DP / 8), d = 8 * (i % (DP / 8));
                if (h0 + h >= p.group || d >= p.head_dim) continue;
                float top = -INFINITY, total = 0.f, w[WAVES];
#pragma unroll
                for (int j = 0; j < WAVES; ++j) top = fmaxf(top, join_m[j][h]);
                const float base = top == -INFINITY ? 0.f : top;
#pragma unroll
                for (int j = 0; j < WAVES; ++j) {
                    w[j] = __builtin_amdgcn_exp2f(join_m[j][h] - base);
                    total += w[j] * join_l[j][h];
                }
                const float inv = total > 0.f || total != total ? 1.f / total : 0.f;
                float y[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    y[e] = 0.f;
#pragma unroll
                    for (int j = 0; j < WAVES; ++j) y[e] = __builtin_fmaf(w[j], join[(j * 16 + h) * kJoinRow + d + e], y[e]);
                }
                const int at_head = head * p.group + h0 + h;
                const int64_t at_row = (int64_t)row * p.kv_heads * p.group + at_head;
                if (p.splits > 1) {
                    float* part = partial_of(p, row, at_head, split);
#pragma unroll
                    for (int e = 0; e < 8; e += 2) *reinterpret_cast<float2*>(part + d + e) = make_float2(y[e], y[e + 1]);
                    if (d == 0) part[p.head_dim] = top, part[p.head_dim + 1] = total;
                } else {
                    stg16(p.out + 2 * (at_row * p.head_dim + d), 0,
                          make_uint4(pack_hot<DT>(y[0] * inv, y[1] * inv), pack_hot<DT>(y[2] * inv, y[3] * inv),
                                     pack_hot<DT>(y[4] * inv, y[5] * inv), pack_hot<DT>(y[6] * inv, y[7] * inv)));
                    if (d == 0 && p.lse) p.lse[at_row] = total == 0.f ? -INFINITY : (base + __builtin_amdgcn_logf(total)) * kLn2;
                }
            }
            __syncthreads();                                  // the sums have been read
        }
    }
}

// One wave per row and query head: the pieces' sums under one maximum.
template <int DT>
__global__ __launch_bounds__(256) void join_selected_kernel(SelectedParams p) {
    const int lane = (int)threadIdx.x & 63, q_heads = p.kv_heads * p.group;
    const int64_t row_head = ((int64_t)p.first_block + blockIdx.x) * 4 + ((int)threadIdx.x >> 6);
    const int64_t row = row_head / q_heads;
    if (row >= p.batch.n_rows) return;
    const int s = find_above(p.batch.starts + 1, p.batch.n_seqs, (int)row);
    if (s >= p.batch.n_seqs) return;
    const Seq seq = seq_of(p.batch, s);
    if (row < seq.row0 || row >= seq.row0 + seq.n_new) return;
    const float* src = partial_of(p, (int)row, (int)(row_head % q_heads), 0);
    const int64_t step = p.head_dim + 2;
    const float mine = lane < p.splits ? src[lane * step + p.head_dim] : -INFINITY;
    float top = mine;
    for (int k = 1; k < 64; k <<= 1) top = fmaxf(top, __shfl_xor(top, k));
    const float base = top == -INFINITY ? 0.f : top;
    const float w = __builtin_amdgcn_exp2f(mine - base);
    const float total = xor_sum(lane < p.splits ? w * src[lane * step + p.head_dim + 1] : 0.f, 64);
    const float inv = total > 0.f || total != total ? 1.f / total : 0.f;
    for (int d = 2 * lane; d < (p.head_dim + 127) / 128 * 128; d += 128) {
        float a = 0.f, b = 0.f;
        for (int i = 0; i < p.splits; ++i) {
            const float wi = __shfl(w, i);
            if (d >= p.head_dim) continue;
            const float2 x = *reinterpret_cast<const float2*>(src + i * step + d);
            a = __builtin_fmaf(wi, x.x, a);
            b = __builtin_fmaf(wi, x.y, b);
        }
        if (d < p.head_dim) *reinterpret_cast<uint32_t*>(p.out + 2 * (row_head * p.head_dim + d)) = pack_hot<DT>(a * inv, b * inv);
    }
    if (lane == 0 && p.lse) p.lse[row_head] = total == 0.f ? -INFINITY : (base + __builtin_amdgcn_logf(total)) * kLn2;
}

// ---- by blocks --------------------------------------------------------------------
// 128 rows (new token r / group, query head r % group) by eight waves of 16 rows each.
// Keys are the tokens of the pages that the block's rows list, one behind the other;
// tiles of 64 (32 where vectors have more than 128 elements) are loaded straight into
// LDS, read by all waves whose rows see of them, the next one on its way meanwhile.
// Few rows a wave, so that few waves have work to do for a page that few rows list: all
// wait for those that have.
//
// Two chunks of 1,024 tokens, 16 pages of 64 picked at random for each of 8 KV heads of
// 128, 4 query heads each: 350 us, 1.6 us a tile: the time that a wave with work
// needs for it; 657 by rows, each of which brings its 512 KiB from the caches, 478 by
// four waves of 32 rows.  Rows that pick alike share pages, which random ones hardly do.

constexpr int kBlockWaves = 8, kBlockRows = 16 * kBlockWaves, kBlockThreads = 64 * kBlockWaves;
constexpr int block_tile(int dp) { return dp <= 128 ? 64 : 32; }

// Tokens that a block's rows can belong to, and words of a bit for each.
__host__ __device__ inline int block_tokens(int group) { return kBlockRows % group == 0 ? kBlockRows / group : (kBlockRows - 1) / group + 2; }
__host__ __device__ inline int block_words(int group) { return (block_tokens(group) + 31) / 32; }

// A block's pages: in the order of their columns, each with its entry of the table and a bit for every token of the block
// that lists it.  `bits` is LDS, two words for 32 columns; returns how many.  An entry of a token's list that is no column,
// or not above all columns in front of it, lists nothing.
constexpr int kMostColumns = 1 << 17;
__device__ __forceinline__ int list_pages(const SelectedParams& p, const Seq& seq, int head, int block, uint32_t* bits, int2* list,
                                          uint32_t* masks) {
    __shared__ int32_t scan[kBlockWaves];
    const int tid = (int)threadIdx.x, lane = tid & 63, wave = tid >> 6, t = p.batch.page_tokens;
    const int columns = seq.len > 0 ? div_page(seq.len - 1, p.batch.page_div) + 1 : 0, words = (columns + 31) / 32;
    uint32_t* before = bits + words;                          // pages in the words in front
    for (int i = tid; i < words; i += kBlockThreads) bits[i] = 0;
    __syncthreads();
    const int rows = seq.n_new * p.group, token0 = block * kBlockRows / p.group;
    const int tokens = (min(rows, (block + 1) * kBlockRows) - 1) / p.group + 1 - token0;
    auto each = [&](auto&& f) {                               // f(token of the block, column) for what the tokens list
        for (int token = uniform(wave); token < tokens; token += kBlockWaves) {
            const int limit = seq.len - seq.n_new + token0 + token + 1;
            const int32_t* mine = p.selected + ((int64_t)(seq.row0 + token0 + token) * p.kv_heads + head) * p.listed;
            int most = -1;                                    // of the entries in front
            for (int base = 0; base < p.listed; base += 64) {
                const int column = base + lane < p.listed ? mine[base + lane] : -1;
                int upto = column < p.max_pages ? column : -1;
                const bool is = upto >= 0;
                for (int k = 1; k < 64; k <<= 1) {
                    const int y = __shfl_up(upto, k);
                    upto = lane >= k ? max(upto, y) : upto;
                }
                const int in_front = __shfl_up(upto, 1);
                if (is && column > max(most, lane > 0 ? in_front : -1) && column < columns && column * t < limit) f(token, column);
                most = max(most, __shfl(upto, 63));
            }
        }
    };
    each([&](int, int column) { atomicOr(&bits[column / 32], 1u << (column & 31)); });
    __syncthreads();
    // a thread has a run of words; of pages that are not there the bits go
    const int run = (words + kBlockThreads - 1) / kBlockThreads, word0 = tid * run, word1 = min(word0 + run, words);
    int own = 0;
    for (int i = word0; i < word1; ++i) {
        uint32_t left = bits[i];
        for (uint32_t todo = left; todo; todo &= todo - 1) {
            const int id = seq.entry(32 * i + __ffs((int)todo) - 1);
            if (id < 0 || id >= p.batch.n_pages) left &= ~(todo & (0u - todo));
        }
        bits[i] = left;
        own += __popc(left);
    }
    int upto = own;
    for (int m = 1; m < 64; m <<= 1) {
        const int y = __shfl_up(upto, m);
        upto += lane >= m ? y : 0;
    }
    if (lane == 63) scan[wave] = upto;
    __syncthreads();
    int at = upto - own, total = 0;
    for (int w = 0; w < kBlockWaves; ++w) {
        at += w < wave ? scan[w] : 0;
        total += scan[w];
    }
    const int mask_words = block_words(p.group);
    for (int i = word0; i < word1; ++i) {
        before[i] = (uint32_t)at;
        for (uint32_t todo = bits[i]; todo; todo &= todo - 1) {
            const int column = 32 * i + __ffs((int)todo) - 1;
            list[at++] = make_int2(column, seq.entry(column));
        }
    }
    for (int i = tid; i < total * mask_words; i += kBlockThreads) masks[i] = 0;
    __syncthreads();
    each([&](int token, int column) {
        const uint32_t word = bits[column / 32], bit = 1u << (column & 31);
        if (word & bit) atomicOr(&masks[((int)before[column / 32] + __popc(word & (bit - 1))) * mask_words + token / 32], 1u << (token & 31));
    });
    __syncthreads();                                          // lists and masks are there, and the bits have been read
    return total;
}

// Zeros that the tile loads read in the columns behind head_dim: a row of 256 elements.
__device__ __attribute__((aligned(16))) uint32_t g_no_columns[128];

// EVEN: a wave's share of a tile never crosses a page and rows fill DP, so that the share's address is one scalar;
// otherwise every lane has its own.  WORDS: of a page's tokens at most.
template <int DT, int DP, bool EVEN, int WORDS>
__global__ __launch_bounds__(kBlockThreads) __attribute__((amdgpu_waves_per_eu(DP <= 128 ? 4 : 2)))
void block_kernel(SelectedParams p) {
    constexpr int kTile = block_tile(DP), kShare = kTile / kBlockWaves, kSub = kTile / 16;
    constexpr int kSteps = DP / 32, kChunks = DP / 8, kRowBytes = DP * 2, kTileBytes = kTile * kRowBytes;
    constexpr int kLoadRows = 64 / kChunks, kLoads = kShare / kLoadRows;   // rows of a load; a wave's loads for a tile's K, and V
    __shared__ __attribute__((aligned(16))) uint8_t tiles[2][2][kTileBytes];   // [buffer][K, V]
    const int lane = (int)threadIdx.x & 63, wave = uniform((int)threadIdx.x >> 6);
    const int col = lane & 15, quad = lane >> 4;
    const uint32_t unit = p.first_block + blockIdx.x;
    const int head = (int)(unit % (uint32_t)p.kv_heads);
    int block = (int)(unit / (uint32_t)p.kv_heads);
    const int s = uniform(find_tile(p.batch, block, [&](const Seq& q) { return (q.n_new * p.group + kBlockRows - 1) / kBlockRows; }));
    if (s >= p.batch.n_seqs) return;
    block = uniform(block);
    const Seq seq = uniform(seq_of(p.batch, s));
    const int rows = seq.n_new * p.group;
    const int mask_words = block_words(p.group);
    int2* list = p.lists + (int64_t)blockIdx.x * p.list_stride;
    uint32_t* masks = p.masks + (int64_t)blockIdx.x * p.list_stride * mask_words;
    const int stop = uniform(list_pages(p, seq, head, block, reinterpret_cast<uint32_t*>(&tiles[0][0][0]), list, masks)) * p.batch.page_tokens;
    const int r = block * kBlockRows + wave * 16 + col;
    const int token = r / p.group, q_head = head * p.group + (r - token * p.group);
    const int limit = r < rows ? max(0, seq.len - seq.n_new + token + 1) : 0;
    const int nth_token = r < rows ? token - block * kBlockRows / p.group : 0;           // of the block
    // 16-byte pieces are permuted within a row so that the rows of one read lie in different banks
    auto k_swizzle = [](int row, int chunk) { return chunk ^ (row & (kChunks < 16 ? kChunks - 1 : 15)); };
    auto v_swizzle = [](int row, int chunk) {
        if constexpr (DP == 64) return chunk ^ (((row >> 1) & 3) << 1);
        else return chunk ^ ((row & 7) << 1);
    };
    const int load_row = lane / kChunks, load_chunk = lane % kChunks;

    uint4 qf[kSteps];
    {
        const uint8_t* src = p.q + 2 * ((int64_t)(seq.row0 + token) * p.q_stride + (int64_t)q_head * p.head_dim);
#pragma unroll
        for (int i = 0; i < kSteps; ++i) {
            const int d = 32 * i + 8 * quad;
            qf[i] = r < rows && d < p.head_dim ? ldg16(src + 2 * d) : make_uint4(0, 0, 0, 0);
        }
    }
    // Where a tile's keys are, lane = key: entries of the list as they were read, looked at a tile later.  What is not
    // there is loaded from the page of the list's last entry and taken out of the V tile afterwards.
    struct Entry {
        int2 page;                                            // column, page
        uint32_t mask[WORDS];
    };
    struct Where {
        int page, row;                                        // EVEN: of this wave's share; else of the lane's key
        int column, key_row;                                  // of the lane's key
        uint64_t here;                                        // which keys are there
        uint32_t mask[WORDS];                                 // tokens that list the lane's key's page
    };
    auto fetch = [&](int kb) {
        const int key = kb + (lane & (kTile - 1)), nth = div_page(min(key, stop - 1), p.batch.page_div);
        Entry x;
        x.page = list[nth];
#pragma unroll
        for (int w = 0; w < WORDS; ++w) x.mask[w] = w < mask_words ? masks[nth * mask_words + w] : 0;
        return x;
    };
    auto where = [&](const Entry& entry, int kb) {
        const int key = kb + (lane & (kTile - 1));
        const int row = key - div_page(key, p.batch.page_div) * p.batch.page_tokens;
        Where x;
        x.column = entry.page.x, x.key_row = row;
        x.here = __ballot(key < stop && entry.page.x * p.batch.page_tokens + row < seq.len);
        x.page = entry.page.y, x.row = row;
        if constexpr (EVEN) x.page = __builtin_amdgcn_readlane(x.page, wave * kShare), x.row = __builtin_amdgcn_readlane(x.row, wave * kShare);
#pragma unroll
        for (int w = 0; w < WORDS; ++w) x.mask[w] = entry.mask[w];
        return x;
    };
    // The keys of a tile that this lane's row sees
    auto sees = [&](const Where& at, int keys) {
        uint64_t mask = 0;
        for (int j = 0; j < keys;) {                          // a page after another
            const int column = __builtin_amdgcn_readlane(at.column, j), from = __builtin_amdgcn_readlane(at.key_row, j);
            const int width = min(p.batch.page_tokens - from, kTile - j);
            uint32_t word = (uint32_t)__builtin_amdgcn_readlane((int)at.mask[0], j);
#pragma unroll
            for (int w = 1; w < WORDS; ++w) {
                const uint32_t x = (uint32_t)__builtin_amdgcn_readlane((int)at.mask[w], j);
                word = nth_token / 32 == w ? x : word;
            }
            const int some = word >> (nth_token & 31) & 1u ? min(width, limit - (column * p.batch.page_tokens + from)) : 0;
            if (some > 0) mask |= (some >= 64 ? ~0ull : (1ull << some) - 1) << j;
            j += width;
        }
        return kTile == 32 ? mask | mask << 32 : mask;
    };
    constexpr uint64_t kAll = ~0ull;                          // (tiles of 32 keys: both halves of the lanes)
    const uint32_t lds0 = lds_address(&tiles[0][0][0]);
    const uint32_t row_bytes = 2u * (uint32_t)p.kv_heads * (uint32_t)p.head_dim;         // from a token to the next
    // This wave's share of a tile of K (which = 0) or V (1) into a buffer
    auto load = [&](const Where& at, int buffer, auto which) __attribute__((always_inline)) {
        constexpr bool is_v = decltype(which)::value != 0;
        const uint8_t* pool = is_v ? p.v_pool : p.k_pool;
        const int64_t page_step = is_v ? p.v_page : p.k_page;
        auto swizzle = [&](int row, int chunk) { return is_v ? v_swizzle(row, chunk) : k_swizzle(row, chunk); };
        const uint32_t to = lds0 + (uint32_t)((2 * buffer + (is_v ? 1 : 0)) * kTileBytes + wave * kShare * kRowBytes);
        if constexpr (EVEN) {
            const uint8_t* src = pool + 2 * (at.page * page_step + (int64_t)(at.row * p.kv_heads + head) * DP);
#pragma unroll
            for (int i = 0; i < kLoads; ++i)
                load_lds16(src + (uint64_t)(i * kLoadRows) * row_bytes,
                           load_row * row_bytes + 16 * swizzle(wave * kShare + i * kLoadRows + load_row, load_chunk),
                           to + i * kLoadRows * kRowBytes);
        } else {
            const uint64_t mine = (uint64_t)(pool + 2 * (at.page * page_step + (int64_t)(at.row * p.kv_heads + head) * p.head_dim));
#pragma unroll
            for (int i = 0; i < kLoads; ++i) {
                const int from = wave * kShare + i * kLoadRows + load_row, chunk = swizzle(from, load_chunk);
                const uint8_t* src = (const uint8_t*)__shfl(mine, from) + 16 * chunk;
                if (chunk * 8 >= p.head_dim) src = reinterpret_cast<const uint8_t*>(g_no_columns);
                load_lds16(src, to + i * kLoadRows * kRowBytes);
            }
        }
    };
    using IsK = std::integral_constant<int, 0>;
    using IsV = std::integral_constant<int, 1>;
    float m = -INFINITY, l = 0.f;
    f32x4 o[DP / 16];
#pragma unroll
    for (int n = 0; n < DP / 16; ++n) o[n] = f32x4{0.f, 0.f, 0.f, 0.f};
    bool careful = false, apart = false;                      // V is looked through; V numbers have to be added apart
    // Every tile has keys that some rows see and others do not, and 0 * infinity and 0 * NaN are NaN, which stays: where no
    // row has one, nothing has reached a row that it should not have; where one has, everything is done again with care:
    // numbers of V that are not finite leave the products and are added afterwards to the rows that see them.
    for (;;) {
        Where at{}, next{};
        Entry entry{};
        if (stop > 0) {
            at = where(fetch(0), 0);
            load(at, 0, IsK{});
            load(at, 0, IsV{});
            entry = fetch(kTile);
        }
        for (int kb = 0, buffer = 0; kb < stop; kb += kTile, buffer ^= 1) {
            next = where(entry, kb + kTile);
            __builtin_amdgcn_s_waitcnt(0);                    // this wave's share of this tile
            __syncthreads();                                  // everyone's; and what is loaded over has been read
            entry = fetch(kb + 2 * kTile);
            if (kb + kTile < stop) {
                load(next, buffer ^ 1, IsK{});
                load(next, buffer ^ 1, IsV{});
            }
            const uint64_t listed = sees(at, min(stop - kb, kTile)) & at.here;
            if (at.here != kAll || careful) {
                bool dropped = false;
                for (int i = (int)threadIdx.x; i < kTileBytes / 16; i += kBlockThreads) {
                    uint4* piece = reinterpret_cast<uint4*>(tiles[buffer][1]) + i;
                    uint4 x = *piece;
                    if (!((at.here >> (i / kChunks)) & 1u)) {
                        *piece = make_uint4(0, 0, 0, 0);
                    } else if (careful && drop_not_finite<DT>(x)) {
                        *piece = x;
                        dropped = true;
                    }
                }
                apart |= __syncthreads_or(dropped) != 0;
            }
            at = next;
            if (!__any(listed != 0)) continue;
            // Waves that have work go first, the others' loads and looks at the list wait (352 us where it takes 372 without).
            // LDS reads by fours in front of their products: the compiler, short of registers, would put each read right
            // before its product (442).
            __builtin_amdgcn_s_setprio(1);
            const uint8_t *kt = tiles[buffer][0], *vt = tiles[buffer][1];
            f32x4 sc[kSub];
#pragma unroll
            for (int i = 0; i < kSteps; ++i) {
                uint4 kf[kSub];
#pragma unroll
                for (int u = 0; u < kSub; ++u)
                    kf[u] = *reinterpret_cast<const uint4*>(kt + (16 * u + col) * kRowBytes + k_swizzle(col, 4 * i + quad) * 16);
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int u = 0; u < kSub; ++u) sc[u] = mfma16<DT>(kf[u], qf[i], i == 0 ? f32x4{0.f, 0.f, 0.f, 0.f} : sc[u]);
            }
            const uint64_t mine = listed >> (4 * quad);       // keys 16 u + i of this lane
            float top = -INFINITY;
#pragma unroll
            for (int u = 0; u < kSub; ++u)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const uint32_t bits = u < 2 ? (uint32_t)mine : (uint32_t)(mine >> 32);
                    sc[u][i] = bits >> (16 * (u % 2) + i) & 1u ? sc[u][i] * p.scale_log2 : -INFINITY;
                    top = fmaxf(top, sc[u][i]);
                }
            top = max_halves(top);
            const u32x2 rows_of_16 = __builtin_amdgcn_permlane16_swap(__float_as_uint(top), __float_as_uint(top), false, false);
            top = fmaxf(__uint_as_float(rows_of_16.x), __uint_as_float(rows_of_16.y));   // (the lane's and that 16 further on)
            // the reference of the exponentials follows the maximum only when that has grown by 2^8: weights up to 256 lose
            // nothing in fp32 sums and 16-bit operands
            if (__any(top > m + 8.f)) {
                const float m_new = fmaxf(m, top);
                const float fade = m_new == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - m_new);
                m = m_new;
                l *= fade;
#pragma unroll
                for (int n = 0; n < DP / 16; ++n) o[n] *= fade;
            }
            const float base = m == -INFINITY ? 0.f : m;      // no key seen yet: every power is 0
            uint4 pf[kSub / 2];
#pragma unroll
            for (int h = 0; h < kSub / 2; ++h) {
                float x[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    x[e] = __builtin_amdgcn_exp2f(sc[2 * h + e / 4][e % 4] - base);
                    l += x[e];
                }
                // weights are rounded to the hot dtype for the product with V (their total is not)
                pf[h] = make_uint4(pack_hot<DT>(x[0], x[1]), pack_hot<DT>(x[2], x[3]), pack_hot<DT>(x[4], x[5]), pack_hot<DT>(x[6], x[7]));
            }
#pragma unroll
            for (int h = 0; h < kSub / 2; ++h)
#pragma unroll
                for (int n0 = 0; n0 < DP / 16; n0 += 4) {
                    uint4 vf[4];
#pragma unroll
                    for (int n = 0; n < 4; ++n) {
                        const int row = 4 * quad + col / 4;
                        const uint8_t* src = vt + row * kRowBytes + v_swizzle(row, 2 * (n0 + n) + (col & 3) / 2) * 16 + (col & 1) * 8 + 32 * h * kRowBytes;
                        const uint2 x = lds_read_transposed(src), y = lds_read_transposed(src + 16 * kRowBytes);
                        vf[n] = make_uint4(x.x, x.y, y.x, y.y);
                    }
                    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                    for (int n = 0; n < 4; ++n) o[n0 + n] = mfma16<DT>(vf[n], pf[h], o[n0 + n]);
                }
            __builtin_amdgcn_s_setprio(0);
        }
        bool odd = false;
#pragma unroll
        for (int n = 0; n < DP / 16; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e) odd |= o[n][e] != o[n][e];
        if (careful || __syncthreads_or(odd && r < rows) == 0) break;
        careful = true;
        apart = false;
        m = -INFINITY;
        l = 0.f;
#pragma unroll
        for (int n = 0; n < DP / 16; ++n) o[n] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    if (careful && apart) {
        for (int nth = 0; nth * p.batch.page_tokens < stop; ++nth) {
            const int2 of = list[nth];
            const bool lists = masks[nth * mask_words + nth_token / 32] >> (nth_token & 31) & 1u;
            for (int row = 0; row < p.batch.page_tokens && of.x * p.batch.page_tokens + row < seq.len; ++row) {
                const bool seen = lists && of.x * p.batch.page_tokens + row < limit;
                const uint8_t* src = p.v_pool + 2 * (of.y * p.v_page + ((int64_t)row * p.kv_heads + head) * p.head_dim);
#pragma unroll
                for (int n = 0; n < DP / 16; ++n) {
                    const int d = 16 * n + 4 * quad;
                    if (d >= p.head_dim || !seen) continue;
                    const uint2 w = *reinterpret_cast<const uint2*>(src + 2 * d);
                    const float x[4] = {hot_lo<DT>(w.x), hot_hi<DT>(w.x), hot_lo<DT>(w.y), hot_hi<DT>(w.y)};
#pragma unroll
                    for (int e = 0; e < 4; ++e) o[n][e] += __builtin_fabsf(x[e]) < INFINITY ? 0.f : x[e];
                }
            }
        }
    }
    l += __shfl_xor(l, 16);
    l = sum_halves(l);
    if (r >= rows) return;
    const float base = m == -INFINITY ? 0.f : m, inv = l > 0.f || l != l ? 1.f / l : 0.f;
    const int64_t row_head = (int64_t)(seq.row0 + token) * p.kv_heads * p.group + q_head;
#pragma unroll
    for (int n = 0; n < DP / 16; ++n) {
        const int d = 16 * n + 4 * quad;
        if (d < p.head_dim)
            *reinterpret_cast<uint2*>(p.out + 2 * (row_head * p.head_dim + d)) =
                make_uint2(pack_hot<DT>(o[n][0] * inv, o[n][1] * inv), pack_hot<DT>(o[n][2] * inv, o[n][3] * inv));
    }
    if (quad == 0 && p.lse) p.lse[row_head] = l == 0.f ? -INFINITY : (base + __builtin_amdgcn_logf(l)) * kLn2;
}

// ---- host -------------------------------------------------------------------------

constexpr int64_t kLine = 128;       // bytes

struct SelectedPlan {
    int waves, splits;               // rows: waves of a workgroup, pieces of a unit
    int64_t piece;
    int64_t units, part, list;       // blocks: workgroups (0: by rows), those of a launch, columns of a workgroup's list
    int64_t bytes;                   // of the workspace
};

SelectedPlan plan_selected(const ztcp_paged_batch* b, const ztcp_geometry* g, int64_t q_heads, int64_t listed, int cus) {
    SelectedPlan plan{1, 1, listed * g->num_tokens, 0, 0, 0, 0};
    const int64_t heads = g->num_heads, group = q_heads / heads, rows = b->n_rows * group;
    // by blocks if these keep half of the compute units busy and are not mostly empty: a sequence's last one may be
    if (rows / kBlockRows * heads >= cus / 2 && rows >= 64 * b->n_seqs && b->max_pages <= kMostColumns) {
        const int64_t most = block_tokens((int)group) * listed;
        plan.units = ((rows + kBlockRows - 1) / kBlockRows + b->n_seqs) * heads;
        plan.list = ((most < b->max_pages ? most : b->max_pages) + 31) / 32 * 32;   // whole lines, as the first starts with one: none is two workgroups'
        const int64_t each = plan.list * ((int64_t)sizeof(int2) + 4 * block_words((int)group)), hold = kMostBetween / each;
        const int64_t parts = (plan.units - 1) / hold + 1;
        plan.part = (plan.units + parts - 1) / parts;        // alike
        plan.bytes = plan.part * each + kLine - 16;
        return plan;
    }
    const int64_t units = b->n_rows * heads, keys = listed * g->num_tokens;
    if (units < 4 * (int64_t)cus) {
        plan.waves = g->head_dim <= 128 ? 8 : 4;
        const int64_t turn = 32 * plan.waves, most = (keys + turn - 1) / turn;
        int64_t n = units > 0 ? cus / units : 1;
        n = n < most ? n : most;
        n = n < 64 ? n : 64;
        n = n > 1 ? n : 1;
        plan.piece = ((keys + n - 1) / n + turn - 1) / turn * turn;
        plan.splits = (int)((keys + plan.piece - 1) / plan.piece);
        if (plan.splits > 1) plan.bytes = b->n_rows * q_heads * plan.splits * (g->head_dim + 2) * (int64_t)sizeof(float);
    }
    return plan;
}

const char* check_selected(const ztcp_paged_batch* batch, const ztcp_page_pool* pool, const ztcp_geometry* g, int64_t q_heads,
                           int64_t listed, PagedView& view) {
    if (const char* why = check_pool(pool, g, 256)) return why;
    if (const char* why = check_batch(batch, pool, g, q_heads, view)) return why;
    if (listed < 1 || listed > (((int64_t)1 << 31) - 4096) / g->num_tokens)
        return "listed must be positive, listed * num_tokens at most 2^31 - 4096";
    return nullptr;
}

}  // namespace

extern "C" size_t ztcp_selected_attention_workspace(const ztcp_paged_batch* batch, const ztcp_page_pool* pool, const ztcp_geometry* g,
                                                    int64_t q_heads, int64_t listed) {
    arg_result(ZTCP_OK, "");
    PagedView view;
    if (const char* why = check_selected(batch, pool, g, q_heads, listed, view)) {
        arg_result(ZTCP_EINVAL, why);
        return (size_t)-1;
    }
    int cus = 0;
    if (cu_count(cus) != ZTCP_OK) return (size_t)-1;
    return (size_t)plan_selected(batch, g, q_heads, listed, cus).bytes;
}

extern "C" int ztcp_selected_attention(const void* q, int64_t q_stride, void* out, float* lse, int64_t q_heads,
                                       const ztcp_page_pool* pool, const ztcp_paged_batch* batch, const ztcp_geometry* g,
                                       const int32_t* selected, int64_t listed, float scale, void* workspace,
                                       size_t workspace_bytes, void* stream) {
    arg_result(ZTCP_OK, "");
    SelectedParams p{};
    if (const char* why = check_selected(batch, pool, g, q_heads, listed, p.batch)) return arg_result(ZTCP_EINVAL, why);
    if (!pool->v) return arg_result(ZTCP_EINVAL, "attention needs K and V pages (single-buffer pages have none)");
    if (!(scale > 0.f) || isinf(scale)) return arg_result(ZTCP_EINVAL, "scale must be a positive finite number");
    if (batch->n_seqs == 0 || batch->n_rows == 0) return ZTCP_OK;
    if (!q || !out || !selected) return arg_result(ZTCP_EINVAL, "q, out and selected must not be NULL");
    if (!hot_aligned(q) || !hot_aligned(out) || q_stride % 8 != 0 || ((uintptr_t)selected & 3u) != 0)
        return arg_result(ZTCP_EINVAL, "q and out must be 16-byte aligned, selected 4-byte");
    const int64_t d = g->head_dim, row = q_heads * d, page = 2 * g->num_tokens * g->num_heads * d;
    if (batch->n_rows > 1 && q_stride < row) return arg_result(ZTCP_EINVAL, "q_stride must cover a token's heads");
    const int64_t q_bytes = 2 * ((batch->n_rows - 1) * q_stride + row), list_bytes = 4 * batch->n_rows * g->num_heads * listed;
    auto misses = [&](const void* x, int64_t bytes) {
        return !bytes_overlap(x, bytes, q, q_bytes) && !bytes_overlap(x, bytes, selected, list_bytes) &&
               !rows_overlap(x, 1, bytes, bytes, pool->k, pool->n_pages, page, 2 * pool->k_stride) &&
               !rows_overlap(x, 1, bytes, bytes, pool->v, pool->n_pages, page, 2 * pool->v_stride);
    };
    const int64_t out_bytes = 2 * batch->n_rows * row, lse_bytes = lse ? 4 * batch->n_rows * q_heads : 0;
    constexpr const char* kOverlap = "out, lse and workspace must not overlap q, selected, the pages or each other";
    if (!misses(out, out_bytes) || !misses(lse, lse_bytes) || bytes_overlap(out, out_bytes, lse, lse_bytes))
        return arg_result(ZTCP_EOVERLAP, kOverlap);
    int cus = 0;
    if (cu_count(cus) != ZTCP_OK) return ZTCP_EHIP;
    const SelectedPlan plan = plan_selected(batch, g, q_heads, listed, cus);
    const int64_t need = plan.bytes;
    if (need > 0 && (!workspace || (int64_t)workspace_bytes < need || !hot_aligned(workspace)))
        return arg_result(ZTCP_EINVAL, "workspace must hold ztcp_selected_attention_workspace bytes, 16-byte aligned");
    if (!misses(need ? workspace : nullptr, need) || bytes_overlap(workspace, need, out, out_bytes) ||
        bytes_overlap(workspace, need, lse, lse_bytes))
        return arg_result(ZTCP_EOVERLAP, kOverlap);
    p.q = (const uint8_t*)q;
    p.out = (uint8_t*)out;
    p.lse = lse;
    p.q_stride = q_stride;
    p.k_pool = (const uint8_t*)pool->k;
    p.v_pool = (const uint8_t*)pool->v;
    p.k_page = pool->k_stride;
    p.v_page = pool->v_stride;
    p.selected = selected;
    p.listed = (int32_t)listed;
    p.max_pages = (int32_t)batch->max_pages;
    p.kv_heads = (int32_t)g->num_heads;
    p.group = (int32_t)(q_heads / g->num_heads);
    p.head_dim = (int32_t)d;
    p.scale_log2 = scale * kLog2e;
    p.splits = plan.splits;
    p.piece = (int32_t)plan.piece;
    p.partial = (float*)workspace;
    p.lists = (int2*)(((uintptr_t)workspace + kLine - 1) / kLine * kLine);
    p.masks = (uint32_t*)(p.lists + plan.part * plan.list);
    p.list_stride = plan.list;
    if (plan.units >= (int64_t)1 << 31) return arg_result(ZTCP_EINVAL, "too many rows and heads in one call");
    auto go = [&](auto dt, auto dp) {
        constexpr int DT = decltype(dt)::value, DP = decltype(dp)::value, kMany = DP <= 128 ? 8 : 4;
        if (plan.units > 0) {
            const bool even = g->num_tokens % (block_tile(DP) / kBlockWaves) == 0 && d == DP;
            const bool one = block_words(p.group) == 1;
            auto kernel = one ? even ? block_kernel<DT, DP, true, 1> : block_kernel<DT, DP, false, 1>
                              : even ? block_kernel<DT, DP, true, 4> : block_kernel<DT, DP, false, 4>;
            // launches whose lists lie in the same place, one after the other
            for (int64_t first = 0; first < plan.units; first += plan.part) {
                p.first_block = (uint32_t)first;
                const int64_t n = plan.units - first < plan.part ? plan.units - first : plan.part;
                hipLaunchKernelGGL(kernel, dim3((uint32_t)n), dim3(kBlockThreads), 0, (hipStream_t)stream, p);
            }
            return;
        }
        const uint64_t units = (uint64_t)batch->n_rows * (uint64_t)g->num_heads * (uint64_t)plan.splits;
        if (plan.waves == 1) launch_blocks(selected_kernel<DT, DP, 1>, units, 64, 0, (hipStream_t)stream, p);
        else launch_blocks(selected_kernel<DT, DP, kMany>, units, 64 * kMany, 0, (hipStream_t)stream, p);
        if (plan.splits > 1)
            launch_blocks(join_selected_kernel<DT>, ((uint64_t)batch->n_rows * (uint64_t)q_heads + 3) / 4, 256, 0, (hipStream_t)stream, p);
    };
    auto by_width = [&](auto dt) {
        if (d <= 64) go(dt, std::integral_constant<int, 64>{});
        else if (d <= 128) go(dt, std::integral_constant<int, 128>{});
        else go(dt, std::integral_constant<int, 256>{});
    };
    if (g->hot_dtype == ZTCP_HOT_BF16) by_width(std::integral_constant<int, kHotBf16>{});
    else by_width(std::integral_constant<int, kHotFp16>{});
    return hipGetLastError() == hipSuccess ? ZTCP_OK : ZTCP_EHIP;
}
