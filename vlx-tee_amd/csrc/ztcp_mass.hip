// ztcp_mass.hip -- the attention weight that each hot page received.
//
//   mass[s, h, p] = decay * mass[s, h, p] + sum over the rows i of KV head h and
//                   the tokens j of page p that i sees of exp(s_ij - lse_i)
#include <type_traits>

#include "ztcp_hot.h"

using namespace ztcp;

namespace {

constexpr int kFewKeys = 128, kManyKeys = 64;   // keys that a workgroup of either kernel has in registers, 32 a wave

struct MassParams {
    PagedView batch;
    const uint8_t* q;
    const float* lse;
    const float* mass;
    float* out;
    int64_t q_stride;
    const uint8_t* k_pool;
    int64_t k_page;
    int32_t kv_heads, group, head_dim, max_pages;
    int32_t few_rows;                // sequences of at most so many rows are the few kernel's
    int32_t few_groups;              // its workgroups of a KV head
    int32_t group_pages;             // pages of a tile: as many as the kernel's keys hold, one at least
    DivBy group_div;
    float scale_log2, decay;
    uint32_t first_block;            // of this launch
};

// (a page may have so many tokens that a length and a page's tokens together pass 2^31)
__device__ __forceinline__ int mass_tiles(const MassParams& p, const Seq& q) {
    return q.len > 0 ? (q.len - 1) / (p.group_pages * p.batch.page_tokens) + 1 : 0;
}

__device__ __forceinline__ int pages_of(const MassParams& p, const Seq& q) {
    return q.len > 0 ? (q.len - 1) / p.batch.page_tokens + 1 : 0;
}

// A tile of pages is summed key by key into LDS, in blocks of KEYS keys (kb) from its first (key0) on: thread i adds up
// its page's keys, block by block.
template <int KEYS>
__device__ __forceinline__ float page_sum(const MassParams& p, const float* key_sum, int kb, int key0, float sum) {
    const int T = p.batch.page_tokens;
    if ((int)threadIdx.x < p.group_pages) {
        const int from = max(kb, key0 + (int)threadIdx.x * T), to = min(kb + KEYS, key0 + ((int)threadIdx.x + 1) * T);
#pragma unroll 4
        for (int k = from; k < to; ++k) sum += key_sum[k - kb];
    }
    return sum;
}

__device__ __forceinline__ void store_account(const MassParams& p, const Seq& q, int s, int head, int page0, float sum) {
    if ((int)threadIdx.x < p.group_pages && page0 + (int)threadIdx.x < pages_of(p, q)) {
        const int64_t at = ((int64_t)s * p.kv_heads + head) * p.max_pages + page0 + threadIdx.x;
        p.out[at] = __builtin_fmaf(p.decay, p.mass[at], sum);
    }
}

// Accounts of a sequence that receive nothing: of pages behind its tokens, all of them if it has no rows.
__device__ __forceinline__ void rest_of(const MassParams& p, int s, int head) {
    if (p.out == p.mass && p.decay == 1.f) return;
    const Seq seq = seq_of(p.batch, s);
    const int from = seq.n_new > 0 ? pages_of(p, seq) : 0;
    const int64_t at = ((int64_t)s * p.kv_heads + head) * p.max_pages;
    for (int i = from + (int)threadIdx.x; i < p.max_pages; i += 256) p.out[at + i] = p.decay * p.mass[at + i];
}

// ---- few rows -------------------------------------------------------------------
// Decoding: reading K is the work.  The tiles of all sequences lie one behind the
// other and every workgroup of a KV head takes an equal number of them; a wave has
// 32 keys of a block and its loads of the next block in flight while it works on
// this one.  The rows stay in registers for a whole sequence.
//
// 64 sequences of 500 to 16,384 tokens, 8 KV heads of 128, pages of 16 (583 MB):
// 114 to 120 us, 5.0 TB/s where a kernel that only reads has 6.35.  K comes by whole
// rows with loads that leave no trace in the caches, and through LDS of the
// wave's own to the products; taken as the products want it, 64 bytes of a row
// a load, 133, and cut by sequence 198.  Bound by the loads in flight.

// Waves of a SIMD, and so workgroups of a compute unit, that the registers allow without scratch memory.
constexpr int few_waves(int dp, int nt) { return dp <= 128 && nt == 1 ? 3 : dp <= 128 || nt == 1 ? 2 : 1; }

template <int DT, int DP, int NT>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(few_waves(DP, NT))))
void mass_few_kernel(MassParams p) {
    constexpr int kSteps = DP / 32, kChunks = DP / 8, kRowBytes = DP * 2;
    constexpr int kLoads = 2 * kSteps, kLoadRows = 64 / kChunks;   // of a wave for its 32 keys; rows of a load
    __shared__ __attribute__((aligned(16))) uint8_t tiles[4][32 * kRowBytes];
    __shared__ float key_sum[2][kFewKeys];
    const int lane = (int)threadIdx.x & 63, wave = uniform((int)threadIdx.x >> 6);
    const int col = lane & 15, quad = lane >> 4;
    const int head = (int)(blockIdx.x % (uint32_t)p.kv_heads), group = (int)(blockIdx.x / (uint32_t)p.kv_heads);
    auto tiles_of = [&](const Seq& q) {
        const int64_t rows = (int64_t)q.n_new * p.group;
        return rows == 0 || rows > p.few_rows ? 0 : mass_tiles(p, q);
    };
    for (int i = group; i < p.batch.n_seqs; i += p.few_groups) rest_of(p, i, head);
    int none;
    const int total = uniform(count_tiles(p.batch, 0, none, tiles_of)), quota = (total + p.few_groups - 1) / p.few_groups;
    if ((int64_t)group * quota >= total) return;
    int tile = group * quota, left = min(quota, total - tile), flip = 0;
    int s = uniform(find_tile(p.batch, tile, tiles_of));
    tile = uniform(tile);
    const int tile_keys = p.group_pages * p.batch.page_tokens;
    // 16-byte pieces are permuted within a row so that the rows of one read lie in different banks
    uint8_t* kt = tiles[wave];
    const int load_row = lane / kChunks, load_chunk = lane % kChunks;
    auto swizzle = [](int row, int chunk) { return chunk ^ (row & (kChunks < 16 ? kChunks - 1 : 15)); };
    for (; left > 0 && s < p.batch.n_seqs; ++s, tile = 0) {
        const Seq seq = uniform(seq_of(p.batch, s));
        const int rows = seq.n_new * p.group, n_tiles = tiles_of(seq);
        if (n_tiles == 0) continue;
        const int end = tile + min(n_tiles - tile, left);
        left -= end - tile;
        const int key_end = min(seq.len, end * tile_keys);
        int limit[NT];                                        // tokens that the lane's row sees
        float base[NT];
        uint4 qf[NT][kSteps];
        auto load_q = [&](int r0) {
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                const int r = r0 + 16 * t + col, token = r / p.group, q_head = head * p.group + (r - token * p.group);
                const uint8_t* src = p.q + 2 * ((int64_t)(seq.row0 + token) * p.q_stride + (int64_t)q_head * p.head_dim);
#pragma unroll
                for (int i = 0; i < kSteps; ++i) {
                    const int d = 32 * i + 8 * quad;
                    qf[t][i] = r < rows && d < p.head_dim ? ldg16(src + 2 * d) : make_uint4(0, 0, 0, 0);
                }
                const float lse = r < rows ? p.lse[(int64_t)(seq.row0 + token) * p.kv_heads * p.group + q_head] : -INFINITY;
                limit[t] = lse == -INFINITY ? 0 : seq.len - seq.n_new + token + 1;   // -infinity: the row saw nothing
                base[t] = lse == -INFINITY ? 0.f : lse * kLog2e;
            }
        };
        load_q(0);
        uint4 kf[kLoads];
        uint32_t valid = 0;
        int entry = -1;                                       // of key lane % 32 of the wave's share of the block to be loaded
        auto look_up = [&](int kb) {
            const int key = kb + 32 * wave + (lane & 31);
            return key < key_end ? seq.entry(div_page(key, p.batch.page_div)) : -1;
        };
        auto load = [&](int kb) {
            const int key = kb + 32 * wave + (lane & 31);
            const bool has = (uint32_t)entry < (uint32_t)p.batch.n_pages;
            valid = (uint32_t)__ballot(has);
            const int row = key - div_page(key, p.batch.page_div) * p.batch.page_tokens;
            const uint64_t mine =
                (uint64_t)(p.k_pool + (has ? 2 * (entry * p.k_page + (int64_t)(row * p.kv_heads + head) * p.head_dim) : 0));
#pragma unroll
            for (int i = 0; i < kLoads; ++i) {
                const uint8_t* src = (const uint8_t*)__shfl(mine, i * kLoadRows + load_row);
                kf[i] = load_chunk * 8 < p.head_dim ? ldg16_once(src + 16 * load_chunk) : make_uint4(0, 0, 0, 0);
            }
        };
        // blocks of a tile: one, or several of a page of more than kFewKeys tokens
        auto next_block = [&](int kb, int key0) { return kb + kFewKeys < key0 + tile_keys ? kb + kFewKeys : key0 + tile_keys; };
        int key0 = tile * tile_keys, kb = key0;
        entry = look_up(kb);
        load(kb);
        entry = look_up(next_block(kb, key0));
        float sum = 0.f;
        while (kb < key_end) {
            const uint32_t here = valid;
            const int next = next_block(kb, key0), most = min(kb + kFewKeys, min(next, key_end)) - (kb + 32 * wave);
            float x[8] = {};
#pragma unroll
            for (int i = 0; i < kLoads; ++i) {
                const int row = i * kLoadRows + load_row;
                *reinterpret_cast<uint4*>(kt + row * kRowBytes + swizzle(row, load_chunk) * 16) = kf[i];
            }
            if (next < key_end) {
                load(next);
                entry = look_up(next_block(next, next < key0 + tile_keys ? key0 : next));
            }
            auto weigh = [&]() {
#pragma unroll
                for (int t = 0; t < NT; ++t)
#pragma unroll
                    for (int u = 0; u < 2; ++u) {
                        f32x4 sc = {0.f, 0.f, 0.f, 0.f};
                        __builtin_amdgcn_sched_barrier(0);    // no more of K in registers at once
#pragma unroll
                        for (int i = 0; i < kSteps; ++i)
                            sc = mfma16<DT>(*reinterpret_cast<const uint4*>(kt + (16 * u + col) * kRowBytes +
                                                                            swizzle(col, 4 * i + quad) * 16), qf[t][i], sc);
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const float w = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[i], p.scale_log2, -base[t]));
                            x[4 * u + i] += kb + 32 * wave + 16 * u + 4 * quad + i < limit[t] ? w : 0.f;
                        }
                    }
            };
            weigh();
            if (rows > 16 * NT) {                             // more rows than the caller said: they come again for every block
                for (int r0 = 16 * NT; r0 < rows; r0 += 16 * NT) {
                    load_q(r0);
                    weigh();
                }
                load_q(0);
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int key = 16 * (i / 4) + 4 * quad + i % 4;
                const float y = xor_sum(x[i], 16);
                if (col == 0) key_sum[flip][32 * wave + key] = ((here >> key) & 1u) && key < most ? y : 0.f;
            }
            __syncthreads();
            sum = page_sum<kFewKeys>(p, key_sum[flip], kb, key0, sum);
            flip ^= 1;
            kb = next;
            if (next == key0 + tile_keys) {
                store_account(p, seq, s, head, tile * p.group_pages, sum);
                sum = 0.f;
                ++tile;
                key0 = next;
            }
        }
        if (key0 < key_end) store_account(p, seq, s, head, tile * p.group_pages, sum);   // the last page's blocks behind the end
    }
}

// ---- many rows ------------------------------------------------------------------
// Chunks of prompts: the products and exponentials are the work.  A workgroup
// owns a tile of pages of one KV head: K stays in registers, 32 of a block's keys
// a wave, while the rows, 128 (64) at a time, pass through LDS, the next ones on their
// way meanwhile.  Two waves have the same keys and each half of the rows, so that
// tiles are small and many: early ones, which more rows see, start first, and
// the card ends evenly.  Every page's account has one writer and one order of additions.
//
// Two prompts' second 2,048 tokens over 4,096, 32 + 8 heads of 128, pages of 16
// (103 GFLOP): 151 to 153 us, 684 to 675 TFLOP/s; with the rows read from memory
// by every wave and the exponentials after the products 408.  Vector work bounds
// it: the matrix units are busy for 29% of the clocks, the vector units, with
// the time of four instructions for an exponential, for 67%: 43% the 403 million
// exponentials with their scaling and sums, 24% everything else (scores begun at
// zero, masks, the rows' references, addresses).

template <int DT, int DP>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(DP <= 128 ? 2 : 1)))
void mass_many_kernel(MassParams p) {
    constexpr int kSub = DP <= 128 ? 2 : 1;                   // 32-row tiles that a wave works on at a time
    constexpr int kRowTile = 64 * kSub, kScores = 16 * kSub;
    constexpr int kSteps = DP / 16, kChunks = DP / 8, kRowBytes = DP * 2, kTileBytes = kRowTile * kRowBytes;
    constexpr int kLoadRows = 64 / kChunks, kLoads = kRowTile / kLoadRows / 4;
    __shared__ __attribute__((aligned(16))) uint8_t tiles[2][kTileBytes];
    __shared__ float key_sum[2][kManyKeys];
    const int lane = (int)threadIdx.x & 63, wave = uniform((int)threadIdx.x >> 6);
    const int col = lane & 31, half = lane >> 5;
    const int row_half = wave >> 1;
    const uint32_t unit = p.first_block + blockIdx.x;
    const int head = (int)(unit % (uint32_t)p.kv_heads);
    const uint32_t rest = unit / (uint32_t)p.kv_heads;
    const int s = (int)(rest % (uint32_t)p.batch.n_seqs);
    const int tile = (int)(rest / (uint32_t)p.batch.n_seqs);  // early keys, which most rows see, first
    const Seq seq = uniform(seq_of(p.batch, s));
    const int rows = seq.n_new * p.group;
    if (!p.few_groups && tile == 0) rest_of(p, s, head);
    if (rows <= p.few_rows || tile >= mass_tiles(p, seq)) return;
    const int tile_keys = p.group_pages * p.batch.page_tokens, key0 = tile * tile_keys, key_end = min(seq.len, key0 + tile_keys);
    const int before = seq.len - seq.n_new;                   // tokens that every row sees
    const uint32_t lds0 = lds_address(&tiles[0][0]);
    const int load_row = lane / kChunks, load_chunk = lane % kChunks;
    auto swizzle = [](int row, int chunk) { return chunk ^ (row & (kChunks < 16 ? kChunks - 1 : 15)); };
    // This wave's quarter of the rows from r0 on.  Where the group is a power of two that divides the rows, the loads
    // of every step lie alike: a scalar says where the rows begin, eight more how far behind that a load does, and a
    // lane's offset in its load is always the same.  Otherwise, and for the last rows, every lane has its own address
    // (rows behind the last one are the last one's numbers; columns behind head_dim are not written).
    const bool even = p.head_dim == DP && (p.group & (p.group - 1)) == 0 && p.group <= kRowTile &&
                      kRowTile * p.q_stride < ((int64_t)1 << 30);
    const int lane_token = p.group < kLoadRows ? load_row / p.group : 0;
    const uint32_t lane_offset = even ? (uint32_t)(2 * (lane_token * p.q_stride + (load_row - lane_token * p.group) * p.head_dim)) : 0;
    int load_offset[kLoads];
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
        const int first = (wave * kLoads + i) * kLoadRows, token = div_page(first, p.group_div);
        load_offset[i] = even ? (int)(2 * (token * p.q_stride + (first - token * p.group) * DP)) : 0;
    }
    auto load_rows = [&](int r0, int buffer) __attribute__((always_inline)) {
        if (even && r0 + kRowTile <= rows) {
            const uint8_t* base = p.q + 2 * ((int64_t)(seq.row0 + div_page(r0, p.group_div)) * p.q_stride + (int64_t)head * p.group * DP);
#pragma unroll
            for (int i = 0; i < kLoads; ++i) {
                const int first = (wave * kLoads + i) * kLoadRows;
                load_lds16(base + load_offset[i], lane_offset + 16 * swizzle(first + load_row, load_chunk),
                           lds0 + (uint32_t)(buffer * kTileBytes + first * kRowBytes));
            }
        } else {
#pragma unroll
            for (int i = 0; i < kLoads; ++i) {
                const int first = (wave * kLoads + i) * kLoadRows, row = first + load_row, r = min(r0 + row, rows - 1);
                const int token = div_page(r, p.group_div), chunk = swizzle(row, load_chunk);
                const uint8_t* src = p.q + 2 * ((int64_t)(seq.row0 + token) * p.q_stride +
                                                (int64_t)(head * p.group + (r - token * p.group)) * p.head_dim);
                if (chunk * 8 < p.head_dim) load_lds16(src + 16 * chunk, lds0 + (uint32_t)(buffer * kTileBytes + first * kRowBytes));
            }
        }
    };
    if (p.head_dim < DP) {
        for (int i = (int)threadIdx.x; i < 2 * kTileBytes / 16; i += 256)
            reinterpret_cast<uint4*>(&tiles[0][0])[i] = make_uint4(0, 0, 0, 0);
        __syncthreads();
    }
    uint32_t q_at[kSteps];
#pragma unroll
    for (int i = 0; i < kSteps; ++i) q_at[i] = (uint32_t)((32 * kSub * row_half + col) * kRowBytes + swizzle(col, 2 * i + half) * 16);

    float sum = 0.f;
    for (int kb = key0; kb < key_end; kb += kManyKeys) {
        const int wb = kb + 32 * (wave & 1);                        // this wave's first key
        const int most = min(kb + kManyKeys, key_end) - wb;
        uint4 kf[kSteps];
        uint32_t here;
        {
            const Place at = place_of(p.batch, seq, wb + col, min(kb + kManyKeys, key_end));
            here = (uint32_t)__ballot(at.page >= 0);
            const uint8_t* src = p.k_pool + (at.page >= 0 ? 2 * (at.page * p.k_page + (int64_t)(at.row * p.kv_heads + head) * p.head_dim) : 0);
#pragma unroll
            for (int i = 0; i < kSteps; ++i) {
                const int d = 16 * i + 8 * half;
                kf[i] = d < p.head_dim ? ldg16(src + 2 * d) : make_uint4(0, 0, 0, 0);
            }
        }
        // from the first row that sees the block's first key
        const int first_token = max(0, kb - before);
        const int row0 = first_token < seq.n_new ? first_token * p.group / kRowTile * kRowTile : rows;
        float acc[16] = {};
        // a row's lse, and the tokens that it sees, one tile ahead
        float lse[kSub];
        int sees[kSub];
        auto load_lse = [&](int r0) {
#pragma unroll
            for (int u = 0; u < kSub; ++u) {
                const int r = r0 + 32 * kSub * row_half + 32 * u + col, at = min(r, rows - 1), token = div_page(at, p.group_div);
                sees[u] = r < rows ? before + token + 1 : 0;
                lse[u] = p.lse[(int64_t)(seq.row0 + token) * p.kv_heads * p.group + head * p.group + (at - token * p.group)];
            }
        };
        if (row0 < rows) {
            load_lse(row0);
            load_rows(row0, 0);
        }
        // The weights of 64 rows whose scores are made are taken beside the next rows' products, so that the wave has
        // products and vector work at the same time; LDS reads run two steps ahead, and the barriers keep the compiler
        // from putting each right before its product.
        float base[kSub] = {};
        int limit[kSub] = {};
        auto hide = [&](f32x16 (&sc)[kSub]) {                    // what the scores' rows do not see
            if (__all(min(limit[0], limit[kSub - 1]) >= wb + 32)) return;
#pragma unroll
            for (int u = 0; u < kSub; ++u) {
                const int seen = limit[u] - wb - 4 * half;
#pragma unroll
                for (int i = 0; i < 16; ++i)
                    if (8 * (i / 4) + i % 4 >= seen) sc[u][i] = -INFINITY;
                if (base[u] != base[u]) {                        // a NaN goes to the tokens that its row sees
#pragma unroll
                    for (int i = 0; i < 16; ++i)
                        if (8 * (i / 4) + i % 4 < seen) sc[u][i] = base[u];
                    base[u] = 0.f;
                }
            }
        };
        auto weigh = [&](const f32x16 (&sc)[kSub], int w) {
            acc[w % 16] += __builtin_amdgcn_exp2f(__builtin_fmaf(sc[w / 16][w % 16], p.scale_log2, -base[w / 16]));
            asm volatile("" : "+v"(acc[w % 16]));
        };
        auto step = [&](int r0, auto buffer_c, f32x16 (&sc)[kSub], f32x16 (&next)[kSub]) __attribute__((always_inline)) {
            constexpr int buffer = decltype(buffer_c)::value;
            __builtin_amdgcn_s_waitcnt(0);
            __syncthreads();
            float z[kSub];
            int z_sees[kSub];
#pragma unroll
            for (int u = 0; u < kSub; ++u) {
                z[u] = lse[u];
                z_sees[u] = sees[u];
            }
            if (r0 + kRowTile < rows) {
                load_lse(r0 + kRowTile);
                load_rows(r0 + kRowTile, buffer ^ 1);
            }
            hide(sc);
            uint4 qf[3][kSub];
            auto read_q = [&](int i) {
#pragma unroll
                for (int u = 0; u < kSub; ++u)
                    qf[i % 3][u] = *reinterpret_cast<const uint4*>(tiles[buffer] + q_at[i] + 32 * u * kRowBytes);
            };
            read_q(0);
            read_q(1);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int i = 0; i < kSteps; ++i) {
                if (i + 2 < kSteps) read_q(i + 2);
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int u = 0; u < kSub; ++u) {
                    if (i == 0)
#pragma unroll
                        for (int e = 0; e < 16; ++e) next[u][e] = 0.f;
                    next[u] = mfma32<DT>(kf[i], qf[i % 3][u], next[u]);
#pragma unroll
                    for (int w = 0; w < kScores; ++w)
                        if (w * kSub * kSteps / kScores == kSub * i + u) weigh(sc, w);
                    __builtin_amdgcn_sched_barrier(0);
                }
            }
#pragma unroll
            for (int u = 0; u < kSub; ++u) {
                base[u] = z[u] == -INFINITY ? 0.f : z[u] * kLog2e;
                limit[u] = z[u] == -INFINITY ? 0 : z_sees[u];   // -infinity: the row saw nothing
            }
        };
        if (row0 < rows) {
            f32x16 a[kSub], b[kSub];
#pragma unroll
            for (int i = 0; i < kScores; ++i) a[i / 16][i % 16] = -INFINITY;   // no rows yet
            auto finish = [&](f32x16 (&sc)[kSub]) {
                hide(sc);
#pragma unroll
                for (int w = 0; w < kScores; ++w) weigh(sc, w);
            };
            for (int r0 = uniform(row0);;) {
                step(r0, std::integral_constant<int, 0>{}, a, b);
                if ((r0 += kRowTile) >= rows) {
                    finish(b);
                    break;
                }
                step(r0, std::integral_constant<int, 1>{}, b, a);
                if ((r0 += kRowTile) >= rows) {
                    finish(a);
                    break;
                }
            }
        }
        __syncthreads();                                      // the last rows, and the previous block's sums, have been read
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const int key = 8 * (i / 4) + 4 * half + i % 4;
            const float x = xor_sum(acc[i], 32);
            if (col == 0) key_sum[row_half][32 * (wave & 1) + key] = ((here >> key) & 1u) && key < most ? x : 0.f;
        }
        __syncthreads();
        if (threadIdx.x < kManyKeys) key_sum[0][threadIdx.x] += key_sum[1][threadIdx.x];
        __syncthreads();
        sum = page_sum<kManyKeys>(p, key_sum[0], kb, key0, sum);
    }
    store_account(p, seq, s, head, tile * p.group_pages, sum);
}

template <int DT, int DP>
void launch(MassParams p, int64_t most_rows, int cus, hipStream_t stream) {
    const int64_t heads = p.kv_heads;
    auto tiles_of = [&](int keys) {                           // of a table row
        p.group_pages = p.batch.page_tokens >= keys ? 1 : keys / p.batch.page_tokens;
        return (int64_t)(p.max_pages + p.group_pages - 1) / p.group_pages;
    };
    // rows of a decoding sequence fit 16 or 32; where none can have more the few kernel does all
    const int nt = most_rows <= 16 ? 1 : most_rows <= 32 ? 2 : p.group <= 16 ? 1 : p.group <= 32 ? 2 : 0;
    const bool many = most_rows > 32 || nt == 0;
    p.few_rows = many ? 16 * nt : 0x7FFFFFFF;
    if (nt) {
        const int64_t resident = ((int64_t)cus * few_waves(DP, nt) + heads - 1) / heads;
        const int64_t tiles = p.batch.n_seqs * tiles_of(kFewKeys);
        p.few_groups = (int32_t)(resident < tiles ? resident : tiles);
        const dim3 grid((uint32_t)(p.few_groups * heads));
        if (nt == 1) hipLaunchKernelGGL((mass_few_kernel<DT, DP, 1>), grid, dim3(256), 0, stream, p);
        else hipLaunchKernelGGL((mass_few_kernel<DT, DP, 2>), grid, dim3(256), 0, stream, p);
    }
    if (many) {
        const int64_t tiles = p.batch.n_seqs * tiles_of(kManyKeys);
        launch_blocks(mass_many_kernel<DT, DP>, (uint64_t)(tiles * heads), 256, 0, stream, p);
    }
}

}  // namespace

extern "C" int ztcp_attention_mass(const void* q, int64_t q_stride, const float* lse, int64_t q_heads,
                                   const ztcp_page_pool* pool, const ztcp_paged_batch* batch, const ztcp_geometry* g,
                                   float scale, const float* mass, float decay, float* out, void* stream) {
    arg_result(ZTCP_OK, "");
    MassParams p{};
    if (const char* why = check_pool(pool, g, 256)) return arg_result(ZTCP_EINVAL, why);
    if (const char* why = check_batch(batch, pool, g, q_heads, p.batch)) return arg_result(ZTCP_EINVAL, why);
    if (!(scale > 0.f) || isinf(scale)) return arg_result(ZTCP_EINVAL, "scale must be a positive finite number");
    if (!(decay >= 0.f) || isinf(decay)) return arg_result(ZTCP_EINVAL, "decay must be a finite number, not negative");
    if (batch->n_seqs == 0) return ZTCP_OK;
    if (!mass || !out) return arg_result(ZTCP_EINVAL, "mass and out must not be NULL");
    if (batch->n_rows > 0 && (!q || !lse)) return arg_result(ZTCP_EINVAL, "q and lse must not be NULL");
    if (!hot_aligned(q) || q_stride % 8 != 0) return arg_result(ZTCP_EINVAL, "q must be 16-byte aligned");
    const int64_t d = g->head_dim, row = q_heads * d, page = 2 * g->num_tokens * g->num_heads * d;
    if (batch->n_rows > 1 && q_stride < row) return arg_result(ZTCP_EINVAL, "q_stride must cover a token's heads");
    const int64_t cells = 4 * batch->n_seqs * g->num_heads * batch->max_pages;
    if ((mass != out && bytes_overlap(out, cells, mass, cells)) ||
        bytes_overlap(out, cells, q, batch->n_rows ? 2 * ((batch->n_rows - 1) * q_stride + row) : 0) ||
        bytes_overlap(out, cells, lse, 4 * batch->n_rows * q_heads) ||
        rows_overlap(out, 1, cells, cells, pool->k, pool->n_pages, page, 2 * pool->k_stride))
        return arg_result(ZTCP_EOVERLAP, "out may be mass itself, and must not overlap q, lse or the pages");
    p.q = (const uint8_t*)q;
    p.lse = lse;
    p.mass = mass;
    p.out = out;
    p.q_stride = q_stride;
    p.k_pool = (const uint8_t*)pool->k;
    p.k_page = pool->k_stride;
    p.kv_heads = (int32_t)g->num_heads;
    p.group = (int32_t)(q_heads / g->num_heads);
    p.group_div = div_by((uint32_t)p.group);
    p.head_dim = (int32_t)d;
    p.max_pages = (int32_t)batch->max_pages;
    p.scale_log2 = scale * kLog2e;
    p.decay = decay;
    const int64_t most_q = batch->max_q_len > 0 && batch->max_q_len < batch->n_rows ? batch->max_q_len : batch->n_rows;
    const int64_t most_rows = most_q * p.group;
    int cus = 0;
    if (cu_count(cus) != ZTCP_OK) return ZTCP_EHIP;
    if (batch->n_seqs * batch->max_pages * g->num_heads >= (int64_t)1 << 31)
        return arg_result(ZTCP_EINVAL, "too many sequences, pages and heads in one call");
    auto go = [&](auto dt) {
        constexpr int DT = decltype(dt)::value;
        if (d <= 64) launch<DT, 64>(p, most_rows, cus, (hipStream_t)stream);
        else if (d <= 128) launch<DT, 128>(p, most_rows, cus, (hipStream_t)stream);
        else launch<DT, 256>(p, most_rows, cus, (hipStream_t)stream);
    };
    if (g->hot_dtype == ZTCP_HOT_BF16) go(std::integral_constant<int, kHotBf16>{});
    else go(std::integral_constant<int, kHotFp16>{});
    return hipGetLastError() == hipSuccess ? ZTCP_OK : ZTCP_EHIP;
}
