// ztcp_attention.hip -- attention of new tokens over hot pages.
//
//   s_ij = scale * q_i . k_j  for the tokens j that row i sees,
//   o_i = sum_j exp(s_ij - m_i) v_j / sum_j exp(s_ij - m_i),  lse_i = m_i + log(sum_j ...)
//
// in one pass over the keys with a running maximum m and sum.  A KV head's
// queries are the rows of its products: row r is new token r / group, query
// head r % group of the KV head's group.  Scores are made transposed (K rows
// times Q columns): a row of the softmax is then one column of the result, one
// lane's registers and its partners', and these registers are, as they stand,
// the operand of the second product (V columns times P columns), whose depth,
// the keys, is in the same order on both sides.
#include <type_traits>

#include "ztcp_hot.h"

using namespace ztcp;

namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

struct AttendParams {
    PagedView batch;
    const uint8_t* q;
    uint8_t* out;
    float* lse;                      // or nullptr
    int64_t q_stride;                // elements between tokens
    const uint8_t* k_pool;
    const uint8_t* v_pool;
    int64_t k_page, v_page;          // elements between pages
    int32_t kv_heads, group, head_dim;
    float scale_log2;                // scale * log2(e): exponentials are powers of two
    int32_t few_rows;                // sequences of at most so many rows are the few kernel's, others the many kernel's
    int32_t few_groups;              // few kernel: workgroups of a KV head
    int32_t splits, resident;        // many kernel: most pieces of a sequence's tokens; workgroups the card holds at once
    float* partial;                  // results of pieces: sums [head_dim], maximum, total
    int32_t* cut;                    // what the many kernel's first workgroup leaves its join: pieces, tokens of a piece
    uint32_t first_block;            // of this launch
};

__device__ __forceinline__ float* many_partial(const AttendParams& p, int row, int q_head, int split) {
    return p.partial + (((int64_t)row * p.kv_heads * p.group + q_head) * p.splits + split) * (p.head_dim + 2);
}

// Pieces of `tokens` that a sequence has (one at least: it answers for a sequence without tokens).
__device__ __forceinline__ int pieces_of(int len, int tokens) { return len > 0 ? (len - 1) / tokens + 1 : 1; }

// What a row does not see must not reach it, but 0 * NaN is NaN: of the keys
// that some rows of a workgroup see and others do not, those from `first_sees`
// on, V numbers that are no finite numbers leave the product (set to 0) and are
// added afterwards to the rows that see them.  An infinity or a NaN needs no
// weight for that.  Keys in front of first_sees every row sees: they stay in
// the product.
template <int DT>
__device__ __forceinline__ bool not_finite16(uint32_t h) {
    constexpr uint32_t e = DT == kHotBf16 ? 0x7F80u : 0x7C00u;
    return (h & e) == e;
}
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
// Four numbers of a V row from column d on: those that are not finite, 0 for the others.
template <int DT>
__device__ __forceinline__ f32x4 only_not_finite(const AttendParams& p, const Place& at, int head, int d) {
    f32x4 y = {0.f, 0.f, 0.f, 0.f};
    if (at.page < 0 || d >= p.head_dim) return y;
    const uint8_t* src = p.v_pool + 2 * ((int64_t)at.page * p.v_page + ((int64_t)at.row * p.kv_heads + head) * p.head_dim + d);
    const uint2 w = *reinterpret_cast<const uint2*>(src);
    const float x[4] = {hot_lo<DT>(w.x), hot_hi<DT>(w.x), hot_lo<DT>(w.y), hot_hi<DT>(w.y)};
#pragma unroll
    for (int i = 0; i < 4; ++i)
        if (!(__builtin_fabsf(x[i]) < INFINITY)) y[i] = x[i];
    return y;
}

// ---- few rows -----------------------------------------------------------------
// Decoding: reading K and V is the work.  The tokens of all sequences of few
// rows lie one behind the other in tiles of 128, and every workgroup of a KV
// head takes an equal number of tiles, so that all end together whatever the
// sequences' lengths are; where it ends inside a sequence it leaves a partial
// result.  Of a tile each of its four waves takes 32 keys, with its loads of
// the next tile in flight while it works on this one: K and V by whole rows,
// through LDS of the wave's own to the products (K of vectors of more than 128
// elements, for which there is no room, as the products want it: lane = key,
// 16 bytes of its row).  Waves join their maxima, totals and sums at the end of a
// sequence.
//
// 64 sequences of 500 to 16,384 tokens, 4 query heads to each of 8 KV heads of
// 128, pages of 16 (1.16 GB): 197 to 203 us, 5.8 TB/s where a kernel that only reads has
// 6.35.  Loads of whole rows that leave no trace in the caches made it that: with
// K in 64-byte parts of rows and ordinary loads it took 237 (V's alone without
// trace: 222; K's parts too: 234, each line fetched twice), and cut by sequence
// instead of in equal shares 281.

constexpr int kFewTile = 128;

__device__ __forceinline__ int few_tiles(const AttendParams& p, const Seq& q, int most_rows) {
    const int64_t rows = (int64_t)q.n_new * p.group;
    if (rows == 0 || rows > p.few_rows) return 0;
    if (rows > most_rows) return 1;                           // more than the caller said: one workgroup does them all
    return max(1, (q.len + kFewTile - 1) / kFewTile);
}

// The partial result of workgroup `group` (of a KV head) for a row of sequence s: the workgroups' pieces in order are
// one further either in the workgroup or in the sequence.
__device__ __forceinline__ float* few_partial(const AttendParams& p, int most_rows, int group, int s, int head, int row) {
    return p.partial + ((((int64_t)group + s) * p.kv_heads + head) * most_rows + row) * (p.head_dim + 2);
}

template <int DT, int DP, int NT>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(DP <= 128 && NT == 1 ? 2 : 1)))
void few_kernel(AttendParams p) {
    constexpr int kSteps = DP / 32, kChunks = DP / 8;         // products of depth 32; 16-byte pieces of a row
    constexpr int kVLoads = 32 * kChunks / 64;                // V loads of a lane for a tile
    constexpr int kVRows = 64 / kChunks;                      // rows a load covers
    constexpr int kJoinRow = DP + 4;
    constexpr int kWaveBytes = 32 * DP * 2;
    constexpr bool kKInLds = DP <= 128;
    constexpr int kVBytes = 4 * kWaveBytes > 4 * 16 * kJoinRow * 4 ? 4 * kWaveBytes : 4 * 16 * kJoinRow * 4;
    constexpr int kBytes = kVBytes + (kKInLds ? 4 * kWaveBytes : 0);
    constexpr int kMostRows = 16 * NT;
    __shared__ __attribute__((aligned(16))) uint8_t lds[kBytes];
    __shared__ float join_m[4][16], join_l[4][16];
    const int lane = (int)threadIdx.x & 63, wave = uniform((int)threadIdx.x >> 6);
    const int col = lane & 15, quad = lane >> 4;
    const int head = (int)(blockIdx.x % (uint32_t)p.kv_heads), group = (int)(blockIdx.x / (uint32_t)p.kv_heads);
    int none;
    auto tiles_of = [&](const Seq& q) { return few_tiles(p, q, kMostRows); };
    const int total = uniform(count_tiles(p.batch, 0, none, tiles_of));
    const int quota = (total + p.few_groups - 1) / p.few_groups;
    if ((int64_t)group * quota >= total) return;
    int tile = group * quota;
    int left = min(quota, total - tile);
    int s = uniform(find_tile(p.batch, tile, tiles_of));
    tile = uniform(tile);
    uint8_t* vt = lds + wave * kWaveBytes;
    uint8_t* kt = lds + kVBytes + wave * kWaveBytes;
    auto k_swizzle = [](int row, int chunk) { return chunk ^ (row & (kChunks < 16 ? kChunks - 1 : 15)); };
    // 16-byte pieces of V rows are permuted within the row so that the rows a
    // transposing read takes lie in different banks
    auto swizzle = [](int row, int chunk) {
        if constexpr (DP == 64) return chunk ^ (((row >> 1) & 3) << 1);
        else return chunk ^ ((row & 7) << 1);
    };
    const int v_row = lane / kChunks, v_chunk = lane % kChunks;
    const bool v_has = v_chunk * 8 < p.head_dim;

    for (; left > 0 && s < p.batch.n_seqs; ++s, tile = 0) {
        const Seq seq = uniform(seq_of(p.batch, s));
        const int rows = seq.n_new * p.group, n_tiles = few_tiles(p, seq, kMostRows);
        const int take = min(n_tiles - tile, left);
        if (n_tiles == 0) continue;
        left -= take;
        const bool whole = take == n_tiles;
        const int key0 = tile * kFewTile, key1 = whole ? seq.len : min(seq.len, key0 + take * kFewTile);
        for (int r0 = 0; r0 < rows; r0 += 16 * NT) {
            int limit[NT];                                        // tokens that the lane's rows see
            uint4 qf[NT][kSteps];
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                const int r = r0 + 16 * t + col;
                const int token = r / p.group, h = r - token * p.group;
                limit[t] = r < rows ? max(0, seq.len - seq.n_new + token + 1) : 0;
                const uint8_t* src = p.q + 2 * ((int64_t)(seq.row0 + token) * p.q_stride + (int64_t)(head * p.group + h) * p.head_dim);
#pragma unroll
                for (int i = 0; i < kSteps; ++i) {
                    const int d = 32 * i + 8 * quad;
                    qf[t][i] = r < rows && d < p.head_dim ? ldg16(src + 2 * d) : make_uint4(0, 0, 0, 0);
                }
            }
            const int last = min(rows, r0 + 16 * NT) - 1;
            const int stop = min(key1, max(0, seq.len - seq.n_new + last / p.group + 1));
            float m[NT], l[NT];
            f32x4 o[NT][DP / 16];
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                m[t] = -INFINITY;
                l[t] = 0.f;
#pragma unroll
                for (int i = 0; i < DP / 16; ++i) o[t][i] = f32x4{0.f, 0.f, 0.f, 0.f};
            }
            uint4 kf[2][kSteps], vf[kVLoads];                     // (K in LDS: loads by whole rows as V's, in order)
            Place at;                                             // of key (lane % 32) of the tile to be loaded
            uint32_t valid = 0, v_valid = 0;                      // keys of the loaded tile that are there; this lane's V rows of them
            auto load = [&](const Place& at) {
                const bool has = at.page >= 0;
                valid = (uint32_t)__ballot(has);
                const int page = has ? at.page : 0, row = has ? at.row : 0;
                v_valid = 0;
                if constexpr (!kKInLds) {
#pragma unroll
                    for (int t = 0; t < 2; ++t) {
                        const int from = 16 * t + col;
                        const int64_t pg = __shfl(page, from), rw = __shfl(row, from);
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
                    const int64_t pg = __shfl(page, from), rw = __shfl(row, from);
                    const int64_t in_page = (rw * p.kv_heads + head) * p.head_dim;
                    if constexpr (kKInLds)
                        kf[i / kSteps][i % kSteps] = v_has ? ldg16_once(p.k_pool + 2 * (pg * p.k_page + in_page) + 16 * v_chunk)
                                                           : make_uint4(0, 0, 0, 0);
                    const uint8_t* src = p.v_pool + 2 * (pg * p.v_page + in_page);
                    vf[i] = v_has ? ldg16_once(src + 16 * v_chunk) : make_uint4(0, 0, 0, 0);
                    v_valid |= ((valid >> from) & 1u) << i;
                }
            };
            const int first_sees = max(0, seq.len - seq.n_new + r0 / p.group + 1);   // the row that sees least
            bool apart = false;                                   // V numbers have to be added apart
            int kb = key0 + 32 * wave;
            if (kb < stop) {
                load(place_of(p.batch, seq, kb + (lane & 31), stop));
                at = place_of(p.batch, seq, kb + 128 + (lane & 31), stop);
            }
            for (; kb < stop; kb += 128) {
                const uint32_t here = valid;
                if constexpr (kKInLds) {
#pragma unroll
                    for (int i = 0; i < kVLoads; ++i) {
                        const int row = i * kVRows + v_row;
                        *reinterpret_cast<uint4*>(kt + row * DP * 2 + k_swizzle(row, v_chunk) * 16) = kf[i / kSteps][i % kSteps];
                    }
                }
                auto k_part = [&](int u, int i) {
                    if constexpr (kKInLds)
                        return *reinterpret_cast<const uint4*>(kt + (16 * u + col) * DP * 2 + k_swizzle(col, 4 * i + quad) * 16);
                    else return kf[u][i];
                };
                f32x4 sc[NT][2];
#pragma unroll
                for (int t = 0; t < NT; ++t)
#pragma unroll
                    for (int u = 0; u < 2; ++u) {
                        sc[t][u] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                        for (int i = 0; i < kSteps; ++i) sc[t][u] = mfma16<DT>(k_part(u, i), qf[t][i], sc[t][u]);
                    }
                if (kb + 32 > first_sees && first_sees < stop) {
#pragma unroll
                    for (int i = 0; i < kVLoads; ++i)
                        if (kb + i * kVRows + v_row >= first_sees) apart |= drop_not_finite<DT>(vf[i]);
                }
#pragma unroll
                for (int i = 0; i < kVLoads; ++i) {
                    const int row = i * kVRows + v_row;
                    const uint4 x = (v_valid >> i) & 1u ? vf[i] : make_uint4(0, 0, 0, 0);
                    *reinterpret_cast<uint4*>(vt + row * DP * 2 + swizzle(row, v_chunk) * 16) = x;
                }
                if (kb + 128 < stop) {
                    load(at);
                    at = place_of(p.batch, seq, kb + 256 + (lane & 31), stop);
                }
                uint4 pf[NT];
#pragma unroll
                for (int t = 0; t < NT; ++t) {
                    float x[8];
#pragma unroll
                    for (int u = 0; u < 2; ++u)
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const int key = 16 * u + 4 * quad + i;
                            const bool seen = ((here >> key) & 1u) && kb + key < limit[t];
                            x[4 * u + i] = seen ? sc[t][u][i] * p.scale_log2 : -INFINITY;
                        }
                    float top = fmaxf(fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])), fmaxf(fmaxf(x[4], x[5]), fmaxf(x[6], x[7])));
                    top = fmaxf(top, __shfl_xor(top, 16));
                    top = fmaxf(top, __shfl_xor(top, 32));
                    const float m_new = fmaxf(m[t], top);
                    const float base = m_new == -INFINITY ? 0.f : m_new;   // no key seen yet: every power is 0
                    if (__any(m_new != m[t])) {
                        const float fade = __builtin_amdgcn_exp2f(m[t] - base);
                        l[t] *= fade;
#pragma unroll
                        for (int i = 0; i < DP / 16; ++i) o[t][i] *= fade;
                    }
                    m[t] = m_new;
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        x[i] = __builtin_amdgcn_exp2f(x[i] - base);
                        l[t] += x[i];
                    }
                    // probabilities are rounded to the hot dtype for the product with V (their total is not):
                    // relative to the result that costs about what its own final rounding does
                    pf[t] = make_uint4(pack_hot<DT>(x[0], x[1]), pack_hot<DT>(x[2], x[3]), pack_hot<DT>(x[4], x[5]),
                                       pack_hot<DT>(x[6], x[7]));
                }
#pragma unroll
                for (int n = 0; n < DP / 16; ++n) {
                    uint2 v[2];
#pragma unroll
                    for (int u = 0; u < 2; ++u) {
                        const int row = 16 * u + 4 * quad + col / 4, chunk = 2 * n + (col & 3) / 2;
                        v[u] = lds_read_transposed(vt + row * DP * 2 + swizzle(row, chunk) * 16 + (col & 1) * 8);
                    }
                    const uint4 a = make_uint4(v[0].x, v[0].y, v[1].x, v[1].y);
#pragma unroll
                    for (int t = 0; t < NT; ++t) o[t][n] = mfma16<DT>(a, pf[t], o[t][n]);
                }
            }
            if (__any(apart))                                     // of this wave's tiles
                for (int key = max(key0, first_sees); key < stop; ++key) {
                    if ((key - key0) / 32 % 4 != wave) continue;
                    const Place where = place_of(p.batch, seq, key, stop);
#pragma unroll
                    for (int n = 0; n < DP / 16; ++n) {
                        const f32x4 x = only_not_finite<DT>(p, where, head, 16 * n + 4 * quad);
#pragma unroll
                        for (int t = 0; t < NT; ++t)
#pragma unroll
                            for (int e = 0; e < 4; ++e) o[t][n][e] += key < limit[t] ? x[e] : 0.f;
                    }
                }
            // join the four waves
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                l[t] += __shfl_xor(l[t], 16);
                l[t] += __shfl_xor(l[t], 32);
                __syncthreads();   // the waves' V rows, or the previous rows' sums, have been read
                float* join = reinterpret_cast<float*>(lds);
#pragma unroll
                for (int n = 0; n < DP / 16; ++n)
                    *reinterpret_cast<f32x4*>(join + (wave * 16 + col) * kJoinRow + 16 * n + 4 * quad) = o[t][n];
                if (quad == 0) {
                    join_m[wave][col] = m[t];
                    join_l[wave][col] = l[t];
                }
                __syncthreads();
                const int row = (int)threadIdx.x / 16, part = (int)threadIdx.x % 16;
                const int r = r0 + 16 * t + row;
                if (r < rows) {
                    float top = -INFINITY, total = 0.f, w[4];
#pragma unroll
                    for (int i = 0; i < 4; ++i) top = fmaxf(top, join_m[i][row]);
                    const float base = top == -INFINITY ? 0.f : top;
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        w[i] = __builtin_amdgcn_exp2f(join_m[i][row] - base);
                        total += w[i] * join_l[i][row];
                    }
                    const int token = r / p.group, q_head = head * p.group + (r - token * p.group);
                    float* part_out = whole ? nullptr : few_partial(p, kMostRows, group, s, head, r);
                    const float inv = total > 0.f || total != total ? 1.f / total : 0.f;
                    uint8_t* dst = p.out + 2 * ((int64_t)(seq.row0 + token) * p.kv_heads * p.group + q_head) * p.head_dim;
                    for (int d = 8 * part; d < p.head_dim; d += 128) {
                        float y[8];
#pragma unroll
                        for (int e = 0; e < 8; ++e) {
                            y[e] = 0.f;
#pragma unroll
                            for (int i = 0; i < 4; ++i) y[e] = __builtin_fmaf(w[i], join[(i * 16 + row) * kJoinRow + d + e], y[e]);
                        }
                        if (part_out) {
#pragma unroll
                            for (int e = 0; e < 8; e += 2) *reinterpret_cast<float2*>(part_out + d + e) = make_float2(y[e], y[e + 1]);
                        } else {
                            stg16(dst + 2 * d, 0, make_uint4(pack_hot<DT>(y[0] * inv, y[1] * inv), pack_hot<DT>(y[2] * inv, y[3] * inv),
                                                             pack_hot<DT>(y[4] * inv, y[5] * inv), pack_hot<DT>(y[6] * inv, y[7] * inv)));
                        }
                    }
                    if (part == 0) {
                        if (part_out) {
                            part_out[p.head_dim] = top;
                            part_out[p.head_dim + 1] = total;
                        } else if (p.lse) {
                            p.lse[(int64_t)(seq.row0 + token) * p.kv_heads * p.group + q_head] =
                                total == 0.f ? -INFINITY : (base + __builtin_amdgcn_logf(total)) * kLn2;
                        }
                    }
                }
            }
            __syncthreads();   // the sums have been read
        }
    }
}

// ---- many rows ----------------------------------------------------------------
// Chunks of prompts: the products are the work.  A workgroup of four waves
// takes 128 rows, 32 a wave, of one KV head; tiles of 64 keys (32 where vectors
// have more than 128 elements) are loaded straight into LDS, read by all four,
// the next one on its way meanwhile.  A tile's exponentials are taken beside the
// products of the previous tile's weights with V, so that the matrix and the
// vector units have work at the same time, with two waves on a SIMD.
//
// Two prompts' second 4,096 tokens over 8,192, 32 + 8 heads of 128, pages of 64
// (825 GFLOP): 840 to 870 us, 980 to 950 TFLOP/s, where the library's largest
// products have 1194.  Through registers, one tile after the other, 2067 us;
// straight to LDS 925.  Matrix units are busy for 46% of the clocks and the vector
// units issue for 43%, which two waves a SIMD overlap in part only; registers
// allow no third.  The spread is the clock's, about 2.0 GHz in such a kernel.

constexpr int kManyRows = 128;
constexpr int many_tile(int dp) { return dp <= 128 ? 64 : 32; }

// The unit-th block of kManyRows rows of the batch's sequences of more than
// p.few_rows rows; false if there are fewer.
__device__ __forceinline__ bool find_unit(const AttendParams& p, int unit, int& s, int& block) {
    auto blocks = [&](const Seq& q) {
        const int rows = q.n_new * p.group;
        return rows > p.few_rows ? (rows + kManyRows - 1) / kManyRows : 0;
    };
    s = find_tile(p.batch, unit, blocks);
    if (s >= p.batch.n_seqs) return false;
    block = blocks(seq_of(p.batch, s)) - 1 - unit;            // the last rows, which see most, first
    return true;
}

// Into how many pieces the tokens of the many kernel's sequences are cut, and how
// long these are: as many as the card holds at once, of 512 tokens at least.  The
// lengths are the device's, so it is decided there, alike by every wave.  Eleven
// decoding sequences beside a chunk of 700 tokens, 5 KV heads: 68 us a call when
// the host cut by the most blocks and tokens that there could be, 56 now.
struct Cut {
    int n, tokens;
};
__device__ __forceinline__ Cut cut_of(const AttendParams& p) {
    if (p.splits == 1) return Cut{1, p.batch.max_tokens};
    const int lane = (int)threadIdx.x & 63;
    int units = 0, longest = 1;
    for (int base = 0; base < p.batch.n_seqs; base += 64) {
        if (base + lane >= p.batch.n_seqs) continue;
        const Seq q = seq_of(p.batch, base + lane);
        const int rows = q.n_new * p.group;
        if (rows <= p.few_rows) continue;
        units += (rows + kManyRows - 1) / kManyRows;
        longest = max(longest, q.len);
    }
    for (int m = 1; m < 64 && m < p.batch.n_seqs; m <<= 1) {  // (lane 0's are used)
        units += __shfl_xor(units, m);
        longest = max(longest, __shfl_xor(longest, m));
    }
    longest = uniform(longest);
    const int n = max(1, min(min(p.splits, (longest + 511) / 512), p.resident / max(1, uniform(units) * p.kv_heads)));
    return Cut{n, ((longest + n - 1) / n + 127) / 128 * 128};
}

// Zeros that the tile loads read in the place of tokens that are not there: a row of 256 elements.
__device__ __attribute__((aligned(16))) uint32_t g_zeros[128];

// EVEN: a wave's quarter of a tile never crosses a page and rows fill DP, so that the quarter's address is
// one scalar; otherwise every lane has its own.
template <int DT, int DP, bool EVEN>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(DP <= 128 ? 2 : 1, DP <= 128 ? 2 : 1)))
void many_kernel(AttendParams p) {
    constexpr int kTile = many_tile(DP);                      // keys of a tile
    constexpr int kShare = kTile / 4;                         // of which a wave loads so many
    constexpr int kSub = kTile / 32;
    constexpr int kSteps = DP / 16, kChunks = DP / 8, kRowBytes = DP * 2, kTileBytes = kTile * kRowBytes;
    constexpr int kLoadRows = 64 / kChunks;                   // rows of a wave's load
    constexpr int kLoads = kShare / kLoadRows;                // loads of a wave for a tile's K, and V
    __shared__ __attribute__((aligned(16))) uint8_t tiles[2][2][kTileBytes];   // [buffer][K, V]
    const int lane = (int)threadIdx.x & 63, wave = uniform((int)threadIdx.x >> 6);
    const int col = lane & 31, half = lane >> 5;
    const uint32_t unit = p.first_block + blockIdx.x;
    const int head = (int)(unit % (uint32_t)p.kv_heads);
    const uint32_t rest = unit / (uint32_t)p.kv_heads;
    const Cut cut = cut_of(p);
    if (unit == 0 && threadIdx.x == 0 && p.splits > 1) p.cut[0] = cut.n, p.cut[1] = cut.tokens;
    const int split = (int)(rest % (uint32_t)cut.n);
    int s, block;
    if (!find_unit(p, (int)(rest / (uint32_t)cut.n), s, block)) return;
    s = uniform(s);
    block = uniform(block);
    const Seq seq = uniform(seq_of(p.batch, s));
    const int rows = seq.n_new * p.group;
    if (split >= pieces_of(seq.len, cut.tokens)) return;
    const int key0 = split * cut.tokens, key1 = key0 + min(seq.len - key0, cut.tokens);
    const int r0 = block * kManyRows + wave * 32, r = r0 + col;
    const int token = r / p.group, q_head = head * p.group + (r - token * p.group);
    const int limit = r < rows ? max(0, seq.len - seq.n_new + token + 1) : 0;
    auto sees = [&](int row) { return max(0, seq.len - seq.n_new + row / p.group + 1); };
    const int stop = min(key1, sees(min(rows, (block + 1) * kManyRows) - 1));            // of the workgroup
    const int wave_stop = r0 < rows ? min(key1, sees(min(rows, r0 + 32) - 1)) : 0;       // of this wave
    const int first_sees = sees(block * kManyRows);                                      // the row that sees least
    const int wave_full = r0 + 32 <= rows ? sees(r0) : 0;                                // keys that all its rows see
    // 16-byte pieces are permuted within a row so that the rows of one read lie in different banks
    auto k_swizzle = [](int row, int chunk) { return chunk ^ (row & (kChunks < 16 ? kChunks - 1 : 15)); };
    auto v_swizzle = [](int row, int chunk) {
        if constexpr (DP == 64) return chunk ^ (((row >> 1) & 1) << 2);
        else return chunk ^ ((row & 3) << 2);
    };
    const int load_row = lane / kChunks, load_chunk = lane % kChunks;

    uint4 qf[kSteps];
    {
        const uint8_t* src = p.q + 2 * ((int64_t)(seq.row0 + token) * p.q_stride + (int64_t)q_head * p.head_dim);
#pragma unroll
        for (int i = 0; i < kSteps; ++i) {
            const int d = 16 * i + 8 * half;
            qf[i] = r < rows && d < p.head_dim ? ldg16(src + 2 * d) : make_uint4(0, 0, 0, 0);
        }
    }
    float m = -INFINITY, l[2] = {0.f, 0.f};
    f32x16 o[DP / 32];
#pragma unroll
    for (int n = 0; n < DP / 32; ++n)
#pragma unroll
        for (int i = 0; i < 16; ++i) o[n][i] = 0.f;

    // Where a tile's keys are, lane = key: table entries as they were read, looked at a tile later.  What is not
    // there is loaded from the pool's page 0 and taken out of the V tile afterwards.
    struct Where {
        int page, row;                                        // EVEN: of this wave's quarter; else of the lane's key
        uint64_t here;                                        // which keys are there
    };
    auto fetch = [&](int kb) {
        const int key = kb + (lane & (kTile - 1));
        return key < stop ? seq.table[div_page(key, p.batch.page_div)] : -1;
    };
    auto where = [&](int entry, int kb) {
        const int key = kb + (lane & (kTile - 1));
        const bool present = (uint32_t)entry < (uint32_t)p.batch.n_pages;
        const int page = present ? entry : 0, row = key - div_page(key, p.batch.page_div) * p.batch.page_tokens;
        const uint64_t here = __ballot(present);
        if constexpr (EVEN)
            return Where{__builtin_amdgcn_readlane(page, wave * kShare), __builtin_amdgcn_readlane(row, wave * kShare), here};
        else return Where{page, row, here};
    };
    constexpr uint64_t kAll = ~0ull;                          // (tiles of 32 keys: both halves of the lanes)
    const uint32_t lds0 = lds_address(&tiles[0][0][0]);
    const uint32_t row_bytes = 2u * (uint32_t)p.kv_heads * (uint32_t)p.head_dim;         // from a token to the next
    // This wave's quarter of a tile of K (which = 0) or V (1) into a buffer
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
                if (chunk * 8 >= p.head_dim) src = reinterpret_cast<const uint8_t*>(g_zeros);   // columns behind head_dim
                load_lds16(src, to + i * kLoadRows * kRowBytes);
            }
        }
    };
    using IsK = std::integral_constant<int, 0>;
    using IsV = std::integral_constant<int, 1>;

    // What a tile's products read of LDS: addresses that differ by constants only
    uint32_t k_at[kSteps], v_at[DP / 32];
#pragma unroll
    for (int i = 0; i < kSteps; ++i) k_at[i] = (uint32_t)(col * kRowBytes + k_swizzle(col, 2 * i + half) * 16);
#pragma unroll
    for (int n = 0; n < DP / 32; ++n) {
        const int row = 4 * half + (lane & 15) / 4;
        v_at[n] = (uint32_t)(row * kRowBytes + v_swizzle(row, 4 * n + 2 * ((lane >> 4) & 1) + (lane & 3) / 2) * 16 + (lane & 1) * 8);
    }
    bool apart = false;                                       // V numbers have to be added apart
    int entry = -1;                                           // of the next tile
    uint64_t before = 0;                                      // keys of the previous tile
    uint32_t pw[8 * kSub];                                    // the previous tile's weights, two a word
    Where at{};                                               // of this tile
    auto weigh = [&](const f32x16 (&sc)[kSub], float base, int w) {
        float x[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            x[e] = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[w / 8][2 * (w % 8) + e], p.scale_log2, -base));
            l[e] += x[e];
        }
        pw[w] = pack_hot<DT>(x[0], x[1]);
        asm volatile("" : "+v"(pw[w]), "+v"(l[0]), "+v"(l[1]));              // here, not where the next tile uses it
    };
    constexpr int kProducts = 2 * kSub * (DP / 32), kAhead = 4;
    // Products with V of the tile whose weights pw are made, and (WEIGH) this tile's weights from its scores sc:
    // a 16-key group's weights take the place of the previous tile's once their products have been issued, so
    // that the wave has products and vector work at the same time.  LDS reads run four products ahead; the
    // barriers keep the compiler from putting each read right before its product.
    auto products = [&](int v_buffer, f32x16 (&sc)[kSub], float base, auto weigh_c) __attribute__((always_inline)) {
        constexpr bool kWeigh = decltype(weigh_c)::value;
        const uint8_t* vt = tiles[v_buffer][1];
        uint4 vf[kAhead + 1];
        auto read_v = [&](int k) {
            const uint8_t* src = vt + v_at[k % (DP / 32)] + 16 * (k / (DP / 32)) * kRowBytes;
            const uint2 x = lds_read_transposed(src), y = lds_read_transposed(src + 8 * kRowBytes);
            vf[k % (kAhead + 1)] = make_uint4(x.x, x.y, y.x, y.y);
        };
#pragma unroll
        for (int k = 0; k < kAhead; ++k) read_v(k);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int k = 0; k < kProducts + DP / 32; ++k) {
            const int u = k / (DP / 32), n = k % (DP / 32);
            if (k + kAhead < kProducts) read_v(k + kAhead);
            __builtin_amdgcn_sched_barrier(0);
            if (k < kProducts)
                o[n] = mfma32<DT>(vf[k % (kAhead + 1)], make_uint4(pw[4 * u], pw[4 * u + 1], pw[4 * u + 2], pw[4 * u + 3]), o[n]);
            if (kWeigh && u > 0)
#pragma unroll
                for (int w = 4 * (u - 1); w < 4 * u; ++w)
                    if ((w - 4 * (u - 1)) * (DP / 32) / 4 == n) weigh(sc, base, w);
            __builtin_amdgcn_sched_barrier(0);
        }
    };
    // Takes out of a V tile what must not reach its products
    auto mend = [&](int kb, int v_buffer, uint64_t there) {
        if (there == kAll && !(kb + kTile > first_sees && first_sees < stop)) return;
        bool dropped = false;
        for (int i = (int)threadIdx.x; i < kTileBytes / 16; i += 256) {
            uint4* piece = reinterpret_cast<uint4*>(tiles[v_buffer][1]) + i;
            uint4 x = *piece;
            if (!((there >> (i / kChunks)) & 1u)) *piece = make_uint4(0, 0, 0, 0);
            else if (kb + i / kChunks >= first_sees && drop_not_finite<DT>(x)) {
                *piece = x;
                dropped = true;
            }
        }
        apart |= __syncthreads_or(dropped) != 0;
    };
    // One tile: its scores, the previous tile's products and its own weights.
    auto step = [&](int kb, auto buffer_c, auto first_c) __attribute__((always_inline)) {
        constexpr int buffer = decltype(buffer_c)::value;
        constexpr bool kFirst = decltype(first_c)::value;
        __builtin_amdgcn_s_waitcnt(0);                        // this wave's share of this tile's K and the last one's V
        __syncthreads();                                      // everyone's; and what is loaded over has been read
        const Where next = where(entry, kb + kTile);
        entry = fetch(kb + 2 * kTile);
        if (kb + kTile < stop) load(next, buffer ^ 1, IsK{});
        load(at, buffer, IsV{});
        if (!kFirst) mend(kb - kTile, buffer ^ 1, before);
        before = at.here;
        at = next;
        f32x16 sc[kSub];
        if (kb >= wave_stop) {
            if (!kFirst && kb - kTile < wave_stop) products(buffer ^ 1, sc, 0.f, std::false_type{});
            return;
        }
        {
            const uint8_t* kt = tiles[buffer][0];
            uint4 kf[3][kSub];
            auto read_k = [&](int i) {
#pragma unroll
                for (int u = 0; u < kSub; ++u) kf[i % 3][u] = *reinterpret_cast<const uint4*>(kt + k_at[i] + 32 * u * kRowBytes);
            };
            read_k(0);
            read_k(1);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int i = 0; i < kSteps; ++i) {
                if (i + 2 < kSteps) read_k(i + 2);
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int u = 0; u < kSub; ++u) {
                    if (i == 0)
#pragma unroll
                        for (int e = 0; e < 16; ++e) sc[u][e] = 0.f;
                    sc[u] = mfma32<DT>(kf[i % 3][u], qf[i], sc[u]);
                }
                __builtin_amdgcn_sched_barrier(0);
            }
        }
        if (kb + kTile > wave_full || before != kAll) {       // (before: this tile's keys by now)
            const int most = limit - kb - 4 * half;           // keys 32 u + 8 (i / 4) + i % 4 of this lane that its row sees
            const uint64_t seen = (before >> (4 * half)) & (most >= 64 ? ~0ull : most > 0 ? (1ull << most) - 1 : 0ull);
            const uint32_t bits[2] = {(uint32_t)seen, (uint32_t)(seen >> 32)};
#pragma unroll
            for (int u = 0; u < kSub; ++u)
#pragma unroll
                for (int i = 0; i < 16; ++i)
                    if (!(bits[u] & (1u << (8 * (i / 4) + i % 4)))) sc[u][i] = -INFINITY;
        }
        float tops[4];                                        // four chains, not one of 16 dependent steps
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            tops[e] = sc[0][e];
#pragma unroll
            for (int i = e; i < 16 * kSub; i += 4) tops[e] = fmaxf(tops[e], sc[i / 16][i % 16]);
        }
        const float top = max_halves(fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3]))) * p.scale_log2;
        // The reference of the exponentials follows the maximum only when that has
        // grown by 2^8: weights up to 256 lose nothing in fp32 sums and 16-bit operands.
        const bool grown = __any(top > m + 8.f);
        float fade = 1.f;
        if (grown) {
            const float m_new = fmaxf(m, top);
            fade = m_new == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - m_new);
            m = m_new;
            l[0] *= fade;
            l[1] *= fade;
        }
        const float base = m == -INFINITY ? 0.f : m;          // no key seen yet: every power is 0
        if constexpr (kFirst) {
#pragma unroll
            for (int w = 0; w < 8 * kSub; ++w) weigh(sc, base, w);
        } else {
            products(buffer ^ 1, sc, base, std::true_type{});
        }
        if (grown)                                            // the sums are relative to the old reference up to here
#pragma unroll
            for (int n = 0; n < DP / 32; ++n) o[n] *= fade;
    };
    if (key0 < stop) {
        at = where(fetch(key0), key0);
        entry = fetch(key0 + kTile);
        load(at, 0, IsK{});
        using B0 = std::integral_constant<int, 0>;
        using B1 = std::integral_constant<int, 1>;
        int kb = key0, last = 0;
        step(kb, B0{}, std::true_type{});
        for (kb += kTile; kb < stop; kb += kTile) {
            step(kb, B1{}, std::false_type{});
            last = 1;
            if ((kb += kTile) >= stop) break;
            step(kb, B0{}, std::false_type{});
            last = 0;
        }
        // the last tile's products
        const int end = key0 + (stop - 1 - key0) / kTile * kTile;
        __builtin_amdgcn_s_waitcnt(0);
        __syncthreads();
        mend(end, last, before);
        f32x16 none[kSub];
        if (end < wave_stop) products(last, none, 0.f, std::false_type{});
    }
    if (apart)
        for (int key = max(key0, first_sees); key < stop; ++key) {
            const Place from = place_of(p.batch, seq, key, stop);
#pragma unroll
            for (int n = 0; n < DP / 32; ++n)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const f32x4 x = only_not_finite<DT>(p, from, head, 32 * n + 8 * i + 4 * half);
#pragma unroll
                    for (int e = 0; e < 4; ++e) o[n][4 * i + e] += key < limit ? x[e] : 0.f;
                }
        }
    const float total = sum_halves(l[0] + l[1]);
    if (r >= rows) return;
    const int64_t row_head = (int64_t)(seq.row0 + token) * p.kv_heads * p.group + q_head;
    const float base = m == -INFINITY ? 0.f : m;
    if (cut.n > 1) {
        float* dst = many_partial(p, seq.row0 + token, q_head, split);
#pragma unroll
        for (int n = 0; n < DP / 32; ++n)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int d = 32 * n + 8 * i + 4 * half;
                if (d < p.head_dim) {
                    *reinterpret_cast<float2*>(dst + d) = make_float2(o[n][4 * i], o[n][4 * i + 1]);
                    *reinterpret_cast<float2*>(dst + d + 2) = make_float2(o[n][4 * i + 2], o[n][4 * i + 3]);
                }
            }
        if (half == 0) {
            dst[p.head_dim] = m;
            dst[p.head_dim + 1] = total;
        }
        return;
    }
    const float inv = total > 0.f || total != total ? 1.f / total : 0.f;
    uint8_t* dst = p.out + 2 * row_head * p.head_dim;
#pragma unroll
    for (int n = 0; n < DP / 32; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int d = 32 * n + 8 * i + 4 * half;
            if (d < p.head_dim)
                *reinterpret_cast<uint2*>(dst + 2 * d) = make_uint2(pack_hot<DT>(o[n][4 * i] * inv, o[n][4 * i + 1] * inv),
                                                                    pack_hot<DT>(o[n][4 * i + 2] * inv, o[n][4 * i + 3] * inv));
        }
    if (half == 0 && p.lse) p.lse[row_head] = total == 0.f ? -INFINITY : (base + __builtin_amdgcn_logf(total)) * kLn2;
}

// ---- pieces joined --------------------------------------------------------------
// One wave per row and query head: the pieces' sums under one maximum.

template <int DT>
__device__ __forceinline__ void join_row(const AttendParams& p, const float* src, int64_t step, int n, int64_t row_head) {
    const int lane = (int)threadIdx.x & 63;
    float top = -INFINITY;
    for (int i = lane; i < n; i += 64) top = fmaxf(top, src[i * step + p.head_dim]);
    for (int k = 1; k < 64; k <<= 1) top = fmaxf(top, __shfl_xor(top, k));
    const float base = top == -INFINITY ? 0.f : top;
    float total = 0.f;
    for (int i = lane; i < n; i += 64)
        total += __builtin_amdgcn_exp2f(src[i * step + p.head_dim] - base) * src[i * step + p.head_dim + 1];
    total = xor_sum(total, 64);
    const float inv = total > 0.f || total != total ? 1.f / total : 0.f;
    for (int d = 2 * lane; d < p.head_dim; d += 128) {
        float a = 0.f, b = 0.f;
#pragma unroll 4
        for (int i = 0; i < n; ++i) {
            const float w = __builtin_amdgcn_exp2f(src[i * step + p.head_dim] - base);
            const float2 x = *reinterpret_cast<const float2*>(src + i * step + d);
            a = __builtin_fmaf(w, x.x, a);
            b = __builtin_fmaf(w, x.y, b);
        }
        *reinterpret_cast<uint32_t*>(p.out + 2 * (row_head * p.head_dim + d)) = pack_hot<DT>(a * inv, b * inv);
    }
    if (lane == 0 && p.lse) p.lse[row_head] = total == 0.f ? -INFINITY : (base + __builtin_amdgcn_logf(total)) * kLn2;
}

template <int DT>
__global__ __launch_bounds__(256) void join_few_kernel(AttendParams p, int most_rows) {
    const int wave = (int)threadIdx.x >> 6;
    const uint32_t unit = p.first_block + blockIdx.x;
    const int head = (int)(unit % (uint32_t)p.kv_heads), s = (int)(unit / (uint32_t)p.kv_heads);
    const Seq seq = seq_of(p.batch, s);
    const int tiles = few_tiles(p, seq, most_rows);
    if (tiles == 0) return;
    int first;
    const int total = count_tiles(p.batch, s, first, [&](const Seq& q) { return few_tiles(p, q, most_rows); });
    const int quota = (total + p.few_groups - 1) / p.few_groups;
    const int group0 = first / quota, group1 = (first + tiles - 1) / quota;
    if (group0 == group1) return;                             // one workgroup had the sequence whole
    const int rows = seq.n_new * p.group;
    const int64_t step = (int64_t)p.kv_heads * most_rows * (p.head_dim + 2);
    for (int r = wave; r < rows; r += 4) {
        const int token = r / p.group, q_head = head * p.group + (r - token * p.group);
        join_row<DT>(p, few_partial(p, most_rows, group0, s, head, r), step, group1 - group0 + 1,
                     (int64_t)(seq.row0 + token) * p.kv_heads * p.group + q_head);
    }
}

// Eight rows of a block a workgroup: a row is a chain of dependent reads, and a block's 128 rows by one workgroup
// took 60 us where their attention had taken 40.
constexpr int kJoinRows = 8;

template <int DT>
__global__ __launch_bounds__(256) void join_many_kernel(AttendParams p) {
    const int wave = (int)threadIdx.x >> 6;
    const uint32_t unit = p.first_block + blockIdx.x;
    const int head = (int)(unit % (uint32_t)p.kv_heads);
    const uint32_t rest = unit / (uint32_t)p.kv_heads;
    const Cut cut{p.cut[0], p.cut[1]};
    int s, block;
    if (cut.n == 1 || !find_unit(p, (int)(rest / (kManyRows / kJoinRows)), s, block)) return;
    const Seq seq = seq_of(p.batch, s);
    const int rows = seq.n_new * p.group, n = pieces_of(seq.len, cut.tokens);
    const int r0 = block * kManyRows + (int)(rest % (kManyRows / kJoinRows)) * kJoinRows;
    for (int r = r0 + wave; r < min(rows, r0 + kJoinRows); r += 4) {
        const int token = r / p.group, q_head = head * p.group + (r - token * p.group);
        join_row<DT>(p, many_partial(p, seq.row0 + token, q_head, 0), p.head_dim + 2, n,
                     (int64_t)(seq.row0 + token) * p.kv_heads * p.group + q_head);
    }
}

// ---- host -------------------------------------------------------------------------

constexpr int64_t kCutFloats = 4;   // in front of the many kernel's pieces

// How a call is cut: what the few and the many kernel take, and into how many pieces.
struct Plan {
    int nt;                         // 16-row tiles of the few kernel, 0: no few kernel
    int few_rows;                   // most rows of its sequences
    int few_groups;                 // its workgroups of a KV head
    bool many;
    int64_t many_units;             // blocks of kManyRows rows at most
    int splits, resident;           // of the many kernel
    int64_t many_groups;            // its workgroups
    int64_t workspace;              // floats
};

Plan plan_call(const ztcp_paged_batch* b, const ztcp_geometry* g, int64_t q_heads, int cus) {
    Plan plan{};
    const int64_t heads = g->num_heads, group = q_heads / heads, piece = g->head_dim + 2;
    const int64_t most_q = b->max_q_len > 0 && b->max_q_len < b->n_rows ? b->max_q_len : b->n_rows;
    const int64_t most_rows = most_q * group, max_tokens = b->max_pages * g->num_tokens;
    const int most_nt = g->head_dim <= 128 ? 2 : 1;
    if (most_rows <= 16 * most_nt) {
        plan.nt = most_rows <= 16 ? 1 : 2;
        plan.few_rows = 0x7FFFFFFF;
    } else {
        plan.nt = b->n_seqs > 1 && group <= 16 * most_nt ? (group <= 16 ? 1 : 2) : 0;
        plan.few_rows = 16 * plan.nt;
        plan.many = true;
        plan.many_units = (b->n_rows * group + kManyRows - 1) / kManyRows + b->n_seqs;
    }
    if (plan.nt) {
        // as many as the card holds at once, and no more than tiles
        const int64_t resident = (int64_t)cus * (g->head_dim <= 64 ? 3 : g->head_dim <= 128 ? 2 : 1);
        const int64_t tiles = b->n_seqs * ((max_tokens + kFewTile - 1) / kFewTile);
        int64_t n = (resident + heads - 1) / heads;
        n = n < tiles ? n : tiles;
        plan.few_groups = (int)(n > 1 ? n : 1);
        if (plan.few_groups > 1) plan.workspace = (plan.few_groups + b->n_seqs) * heads * 16 * plan.nt * piece;
    }
    plan.splits = 1;
    plan.resident = cus * (g->head_dim <= 128 ? 2 : 1);
    if (plan.many) {
        // blocks there are at least if all rows are chunks', and pieces of 512 tokens at least
        const int64_t blocks = (b->n_rows * group + kManyRows - 1) / kManyRows * heads, most = (max_tokens + 511) / 512;
        int64_t n = plan.resident / blocks;
        n = n < most ? n : most;
        n = n < 64 ? n : 64;
        plan.splits = (int)(n > 1 ? n : 1);
        plan.many_groups = plan.many_units * heads;
        const int64_t pieces = (plan.resident + heads - 1) / heads * heads;
        if (plan.splits > 1 && plan.many_groups < pieces) plan.many_groups = pieces;
        const int64_t need = plan.splits > 1 ? b->n_rows * q_heads * plan.splits * piece + kCutFloats : 0;
        plan.workspace = need > plan.workspace ? need : plan.workspace;
    }
    return plan;
}

template <int DT, int DP>
void launch(const AttendParams& base, const Plan& plan, float* workspace, hipStream_t stream) {
    AttendParams p = base;
    p.partial = workspace;
    p.few_rows = plan.few_rows;
    p.few_groups = plan.few_groups;
    p.splits = plan.splits;
    p.resident = plan.resident;
    const uint32_t heads = (uint32_t)p.kv_heads;
    if (plan.nt) {
        const dim3 grid(heads * (uint32_t)plan.few_groups);
        if constexpr (DP <= 128) {
            if (plan.nt == 2) hipLaunchKernelGGL((few_kernel<DT, DP, 2>), grid, dim3(256), 0, stream, p);
        }
        if (plan.nt == 1) hipLaunchKernelGGL((few_kernel<DT, DP, 1>), grid, dim3(256), 0, stream, p);
        if (plan.few_groups > 1)
            launch_blocks(join_few_kernel<DT>, (uint64_t)heads * (uint32_t)p.batch.n_seqs, 256, 0, stream, p, 16 * plan.nt);
    }
    if (plan.many) {
        if (plan.splits > 1) {
            p.cut = (int32_t*)workspace;
            p.partial = workspace + kCutFloats;
        }
        const uint32_t units = (uint32_t)plan.many_units * heads;
        const bool even = p.batch.page_tokens % (many_tile(DP) / 4) == 0 && p.head_dim == DP;
        launch_blocks(even ? many_kernel<DT, DP, true> : many_kernel<DT, DP, false>, (uint64_t)plan.many_groups, 256, 0, stream, p);
        if (p.splits > 1)
            launch_blocks(join_many_kernel<DT>, (uint64_t)units * (kManyRows / kJoinRows), 256, 0, stream, p);
    }
}

const char* check_all(const ztcp_paged_batch* b, const ztcp_page_pool* pool, const ztcp_geometry* g, int64_t q_heads,
                      PagedView& view) {
    if (const char* why = check_pool(pool, g, 256)) return why;
    return check_batch(b, pool, g, q_heads, view);
}

}  // namespace

extern "C" size_t ztcp_paged_attention_workspace(const ztcp_paged_batch* batch, const ztcp_page_pool* pool,
                                                 const ztcp_geometry* g, int64_t q_heads) {
    arg_result(ZTCP_OK, "");
    PagedView view;
    if (const char* why = check_all(batch, pool, g, q_heads, view)) {
        arg_result(ZTCP_EINVAL, why);
        return (size_t)-1;
    }
    int cus = 0;
    if (cu_count(cus) != ZTCP_OK) return (size_t)-1;
    const Plan plan = plan_call(batch, g, q_heads, cus);
    return (size_t)plan.workspace * sizeof(float);
}

extern "C" int ztcp_paged_attention(const void* q, int64_t q_stride, void* out, float* lse, int64_t q_heads,
                                    const ztcp_page_pool* pool, const ztcp_paged_batch* batch, const ztcp_geometry* g,
                                    float scale, void* workspace, size_t workspace_bytes, void* stream) {
    arg_result(ZTCP_OK, "");
    AttendParams p{};
    if (const char* why = check_all(batch, pool, g, q_heads, p.batch)) return arg_result(ZTCP_EINVAL, why);
    if (!pool->v) return arg_result(ZTCP_EINVAL, "attention needs K and V pages (single-buffer pages have none)");
    if (!(scale > 0.f) || isinf(scale)) return arg_result(ZTCP_EINVAL, "scale must be a positive finite number");
    if (batch->n_seqs == 0 || batch->n_rows == 0) return ZTCP_OK;
    if (!q || !out) return arg_result(ZTCP_EINVAL, "q and out must not be NULL");
    if (!hot_aligned(q) || !hot_aligned(out) || q_stride % 8 != 0)
        return arg_result(ZTCP_EINVAL, "q and out must be 16-byte aligned");
    const int64_t d = g->head_dim, row = q_heads * d, page = 2 * g->num_tokens * g->num_heads * d;
    if (batch->n_rows > 1 && q_stride < row) return arg_result(ZTCP_EINVAL, "q_stride must cover a token's heads");
    const int64_t q_bytes = 2 * ((batch->n_rows - 1) * q_stride + row);
    auto misses = [&](const void* x, int64_t bytes) {
        return !bytes_overlap(x, bytes, q, q_bytes) &&
               !rows_overlap(x, 1, bytes, bytes, pool->k, pool->n_pages, page, 2 * pool->k_stride) &&
               !rows_overlap(x, 1, bytes, bytes, pool->v, pool->n_pages, page, 2 * pool->v_stride);
    };
    const int64_t out_bytes = 2 * batch->n_rows * row, lse_bytes = lse ? 4 * batch->n_rows * q_heads : 0;
    int cus = 0;
    if (cu_count(cus) != ZTCP_OK) return ZTCP_EHIP;
    const Plan plan = plan_call(batch, g, q_heads, cus);
    const int64_t need = plan.workspace * (int64_t)sizeof(float);
    if (need > 0 && (!workspace || (int64_t)workspace_bytes < need || !hot_aligned(workspace)))
        return arg_result(ZTCP_EINVAL, "workspace must hold ztcp_paged_attention_workspace bytes, 16-byte aligned");
    if (!misses(out, out_bytes) || !misses(lse, lse_bytes) || !misses(need ? workspace : nullptr, need) ||
        bytes_overlap(out, out_bytes, lse, lse_bytes) || bytes_overlap(workspace, need, out, out_bytes) ||
        bytes_overlap(workspace, need, lse, lse_bytes))
        return arg_result(ZTCP_EOVERLAP, "out, lse and workspace must not overlap q, the pages or each other");
    const int64_t most = (int64_t)1 << 31, tiles = batch->n_seqs * (p.batch.max_tokens / kFewTile + 1);
    if (g->num_heads * plan.many_units * (kManyRows / kJoinRows) >= most ||
        g->num_heads * batch->n_seqs >= most || tiles >= most)
        return arg_result(ZTCP_EINVAL, "too many sequences and heads in one call");
    p.q = (const uint8_t*)q;
    p.out = (uint8_t*)out;
    p.lse = lse;
    p.q_stride = q_stride;
    p.k_pool = (const uint8_t*)pool->k;
    p.v_pool = (const uint8_t*)pool->v;
    p.k_page = pool->k_stride;
    p.v_page = pool->v_stride;
    p.kv_heads = (int32_t)g->num_heads;
    p.group = (int32_t)(q_heads / g->num_heads);
    p.head_dim = (int32_t)d;
    p.scale_log2 = scale * kLog2e;
    auto go = [&](auto dt) {
        constexpr int DT = decltype(dt)::value;
        if (d <= 64) launch<DT, 64>(p, plan, (float*)workspace, (hipStream_t)stream);
        else if (d <= 128) launch<DT, 128>(p, plan, (float*)workspace, (hipStream_t)stream);
        else launch<DT, 256>(p, plan, (float*)workspace, (hipStream_t)stream);
    };
    if (g->hot_dtype == ZTCP_HOT_BF16) go(std::integral_constant<int, kHotBf16>{});
    else go(std::integral_constant<int, kHotFp16>{});
    return hipGetLastError() == hipSuccess ? ZTCP_OK : ZTCP_EHIP;
}
