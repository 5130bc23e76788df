// ztcp_selected.hip -- attention of new tokens over pages that each of them,
// for each KV head, has picked.
//
// The formula is paged attention's with the sums over the tokens of the listed
// pages that the row sees.  A row and KV head are a unit of their own: its query
// heads are the columns of the products (16; a group of fewer leaves columns
// idle, which costs nothing where reading K and V is the work), and all of them
// see the same tokens.
#include <type_traits>

#include "ztcp_hot.h"

using namespace ztcp;

namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

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
    uint32_t first_block;            // of this launch
};

__device__ __forceinline__ float* partial_of(const SelectedParams& p, int row, int q_head, int split) {
    return p.partial + (((int64_t)row * p.kv_heads * p.group + q_head) * p.splits + split) * (p.head_dim + 2);
}

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
            if (page >= 0 && page < p.max_pages && page * p.batch.page_tokens + at.row < limit) {
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
                    kf[i / kSteps][i % kSteps] = v_has ? ldg16(p.k_pool + 2 * (pg * p.k_page + in_page) + 16 * v_chunk)
                                                       : make_uint4(0, 0, 0, 0);
                vf[i] = v_has ? ldg16(p.v_pool + 2 * (pg * p.v_page + in_page) + 16 * v_chunk) : make_uint4(0, 0, 0, 0);
            }
        };
        Place at{-1, 0};                                      // of key (lane % 32) of the tile to be loaded
        int kb = key0 + 32 * wave;
        if (kb < stop) {
            load(place(kb + (lane & 31)));
            at = place(kb + 32 * WAVES + (lane & 31));
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
__global__ __launch_bounds__(256) void join_kernel(SelectedParams p) {
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

// ---- host -------------------------------------------------------------------------

struct SelectedPlan {
    int waves, splits;
    int64_t piece, floats;
};

SelectedPlan plan_selected(const ztcp_paged_batch* b, const ztcp_geometry* g, int64_t q_heads, int64_t listed, int cus) {
    SelectedPlan plan{1, 1, listed * g->num_tokens, 0};
    const int64_t units = b->n_rows * g->num_heads, keys = listed * g->num_tokens;
    if (units < 4 * (int64_t)cus) {
        plan.waves = g->head_dim <= 128 ? 8 : 4;
        const int64_t turn = 32 * plan.waves, most = (keys + turn - 1) / turn;
        int64_t n = units > 0 ? cus / units : 1;
        n = n < most ? n : most;
        n = n < 64 ? n : 64;
        n = n > 1 ? n : 1;
        plan.piece = ((keys + n - 1) / n + turn - 1) / turn * turn;
        plan.splits = (int)((keys + plan.piece - 1) / plan.piece);
        if (plan.splits > 1) plan.floats = b->n_rows * q_heads * plan.splits * (g->head_dim + 2);
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
    return (size_t)plan_selected(batch, g, q_heads, listed, cus).floats * sizeof(float);
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
    const int64_t need = plan.floats * (int64_t)sizeof(float);
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
    auto go = [&](auto dt, auto dp) {
        constexpr int DT = decltype(dt)::value, DP = decltype(dp)::value, kMany = DP <= 128 ? 8 : 4;
        const uint64_t units = (uint64_t)batch->n_rows * (uint64_t)g->num_heads * (uint64_t)plan.splits;
        if (plan.waves == 1) launch_blocks(selected_kernel<DT, DP, 1>, units, 64, 0, (hipStream_t)stream, p);
        else launch_blocks(selected_kernel<DT, DP, kMany>, units, 64 * kMany, 0, (hipStream_t)stream, p);
        if (plan.splits > 1)
            launch_blocks(join_kernel<DT>, ((uint64_t)batch->n_rows * (uint64_t)q_heads + 3) / 4, 256, 0, (hipStream_t)stream, p);
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
