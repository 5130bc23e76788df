// ztcp_append.hip -- new tokens into their hot pages: norms of queries and keys
// for each head, position rotation and the write, in one pass.
#include "ztcp_hot.h"

using namespace ztcp;

namespace {

struct AppendParams {
    const uint8_t* q;
    const uint8_t* k;
    const uint8_t* v;
    uint8_t* q_out;
    int64_t q_stride, k_stride, v_stride, q_out_stride;   // elements between tokens
    uint8_t* k_pool;
    uint8_t* v_pool;
    int64_t n_slots, k_page, v_page;                      // slots of the pool; elements between pages
    const int64_t* slots;
    const int32_t* positions;
    const float* rope;
    int32_t max_position;
    const uint8_t* q_weight;
    const uint8_t* k_weight;
    int32_t q_weight_len, k_weight_len;
    uint32_t n_tokens, parts;                             // a token's vectors are shared by `parts` waves,
    int32_t vecs, part_vecs;                              // part_vecs of its vecs each
    int32_t q_heads, kv_heads, head_dim, rope_dim, page_tokens;
    int32_t interleaved;
    float eps;
    uint32_t first_block;                                 // of this launch
};

// Eight elements of a head vector in fp32.
struct Chunk {
    float x[8];
};

template <int DT>
__device__ __forceinline__ Chunk unpack(uint4 w) {
    const uint32_t u[4] = {w.x, w.y, w.z, w.w};
    Chunk c;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        c.x[2 * i] = hot_lo<DT>(u[i]);
        c.x[2 * i + 1] = hot_hi<DT>(u[i]);
    }
    return c;
}

template <int DT>
__device__ __forceinline__ uint4 pack_chunk(const Chunk& c) {
    return make_uint4(pack_hot<DT>(c.x[0], c.x[1]), pack_hot<DT>(c.x[2], c.x[3]), pack_hot<DT>(c.x[4], c.x[5]),
                      pack_hot<DT>(c.x[6], c.x[7]));
}

// A group of LANES lanes (a power of two, eight elements a lane and chunk; CHUNKS > 1 only for vectors of more than
// 512 elements) has a head vector; a wave has a token's vectors, or a part of them, in turns of 64 / LANES.  The pass
// reads and writes every element once and is bound by that: the angles and weights are loaded once for a wave's
// vectors, the next turns' loads are in flight during a turn, the sum of squares is a butterfly over the group, and
// the partner of a rotated pair sits rope_dim / 16 lanes away (or in the same lane when interleaved), so a vector
// never leaves registers.  Prompt of 16,384 tokens of 32 + 8 + 8 vectors of 128 (407 MB): 91 to 92 us, 4.45 TB/s where a
// large copy has 5.0; with loads that leave a trace in the caches 99 us, and a wave for every four vectors, with
// angles and weights of its own, 147 us.
template <int DT, int LANES, int CHUNKS, int AHEAD>
__global__ __launch_bounds__(256) void append_kernel(AppendParams p) {
    constexpr int kTurn = 64 / LANES;                         // vectors of a turn
    constexpr int kAhead = AHEAD;                             // turns in flight
    const int lane = (int)threadIdx.x % LANES, group = ((int)threadIdx.x & 63) / LANES;
    const uint32_t unit = (uint32_t)uniform((int)((p.first_block + blockIdx.x) * 4 + (threadIdx.x >> 6)));
    const uint32_t token = unit / p.parts, part = unit - token * p.parts;
    if (token >= p.n_tokens) return;
    const int first = (int)part * p.part_vecs, end = min(first + p.part_vecs, p.vecs);
    const int n_chunks = p.head_dim / 8;
    const uint8_t* q = p.q + 2 * (int64_t)token * p.q_stride;
    const uint8_t* k = p.k + 2 * (int64_t)token * p.k_stride;
    const uint8_t* v = p.v + 2 * (int64_t)token * p.v_stride;
    uint8_t* q_out = p.q_out + 2 * (int64_t)token * p.q_out_stride;
    const int64_t slot = p.slots[token];
    const int32_t position = p.rope_dim > 0 ? p.positions[token] : 0;

    // where the token's K and V go
    uint8_t* k_out = nullptr;
    uint8_t* v_out = nullptr;
    if (slot >= 0 && slot < p.n_slots) {
        const int64_t page = slot / p.page_tokens, row = slot - page * p.page_tokens;
        const int64_t in_page = row * p.kv_heads * p.head_dim;
        k_out = p.k_pool + 2 * (page * p.k_page + in_page);
        v_out = p.v_pool + 2 * (page * p.v_page + in_page);
    }
    // Cosines and sines of this lane's elements, (1, 0) for those that do not turn; of a pair's second half the sine
    // that its first has, negated, so that both are x cos - partner sin.  All rotated columns are in a lane's chunk 0
    // (rope_dim <= 512).
    const int half = p.rope_dim / 16;                         // chunks of half the rotated columns
    const bool turned = lane < 2 * half;
    float cs[8], sn[8];
    {
        const bool known = position >= 0 && position < p.max_position;
        const float* row = p.rope + (int64_t)(known ? position : 0) * p.rope_dim;
        const int a0 = p.interleaved ? 4 * lane : 8 * (lane < half ? lane : lane - half);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            cs[e] = 1.f;
            sn[e] = 0.f;
            if (turned && (!p.interleaved || e < 4)) {
                cs[e] = known ? row[a0 + e] : __builtin_nanf("");
                sn[e] = known ? row[8 * half + a0 + e] : __builtin_nanf("");
                if (!p.interleaved && lane >= half) sn[e] = -sn[e];
            }
        }
    }
    const int partner = ((int)threadIdx.x & 63) + (!turned ? 0 : lane < half ? half : -half);
    // Weights of this lane's elements
    uint4 wq[CHUNKS], wk[CHUNKS];
    const int q_first = (p.head_dim - p.q_weight_len) / 8, k_first = (p.head_dim - p.k_weight_len) / 8;   // first normed chunk
#pragma unroll
    for (int i = 0; i < CHUNKS; ++i) {
        const int at = lane + i * LANES;
        wq[i] = at >= q_first && at < n_chunks ? ldg16(p.q_weight + 16 * (at - q_first)) : make_uint4(0, 0, 0, 0);
        wk[i] = at >= k_first && at < n_chunks ? ldg16(p.k_weight + 16 * (at - k_first)) : make_uint4(0, 0, 0, 0);
    }

    // (no lambdas: what they choose between by lane they would choose by address, in scratch memory)
    uint4 c[kAhead][CHUNKS];
    for (int h1 = first - kAhead * kTurn; h1 < end; h1 += kAhead * kTurn) {
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
            if (h1 >= first) {
                const int h0 = h1 + i * kTurn, h = h0 + group;
                const bool is_q = h < p.q_heads, is_k = !is_q && h < p.q_heads + p.kv_heads;
                Chunk x[CHUNKS];
#pragma unroll
                for (int j = 0; j < CHUNKS; ++j) x[j] = unpack<DT>(c[i][j]);
                if (h0 < p.q_heads + p.kv_heads) {                    // not V alone
                    const int normed = is_q ? q_first : is_k ? k_first : n_chunks;
                    float ss = 0.f;
#pragma unroll
                    for (int j = 0; j < CHUNKS; ++j)
                        if (lane + j * LANES >= normed)
#pragma unroll
                            for (int e = 0; e < 8; ++e) ss = __builtin_fmaf(x[j].x[e], x[j].x[e], ss);
                    ss = xor_sum(ss, LANES);
                    const int len = p.head_dim - 8 * normed;
                    const float inv = len > 0 ? rsqrtf(ss / (float)len + p.eps) : 1.f;
#pragma unroll
                    for (int j = 0; j < CHUNKS; ++j) {
                        const Chunk w = unpack<DT>(make_uint4(is_q ? wq[j].x : wk[j].x, is_q ? wq[j].y : wk[j].y,
                                                              is_q ? wq[j].z : wk[j].z, is_q ? wq[j].w : wk[j].w));
                        if (lane + j * LANES >= normed)
#pragma unroll
                            for (int e = 0; e < 8; ++e) x[j].x[e] = x[j].x[e] * inv * w.x[e];
                    }
                    if (half > 0) {
                        const bool turns = turned && (is_q || is_k);
                        if (p.interleaved) {
                            if (turns)
#pragma unroll
                                for (int e = 0; e < 4; ++e) {
                                    const float a = x[0].x[2 * e], b = x[0].x[2 * e + 1];
                                    x[0].x[2 * e] = __builtin_fmaf(a, cs[e], -(b * sn[e]));
                                    x[0].x[2 * e + 1] = __builtin_fmaf(b, cs[e], a * sn[e]);
                                }
                        } else {
#pragma unroll
                            for (int e = 0; e < 8; ++e) {
                                const float o = __shfl(x[0].x[e], partner);
                                if (turns) x[0].x[e] = __builtin_fmaf(x[0].x[e], cs[e], -(o * sn[e]));
                            }
                        }
                    }
                }
                uint8_t* dst = is_q ? q_out + 2 * (int64_t)(h * p.head_dim)
                                    : is_k ? k_out + 2 * (int64_t)((h - p.q_heads) * p.head_dim)
                                           : v_out + 2 * (int64_t)((h - p.q_heads - p.kv_heads) * p.head_dim);
                if (h < end && (is_q || k_out))
#pragma unroll
                    for (int j = 0; j < CHUNKS; ++j) {
                        const int at = lane + j * LANES;
                        if (at < n_chunks) stg16(dst, at, pack_chunk<DT>(x[j]));
                    }
            }
            const int h = h1 + (i + kAhead) * kTurn + group;  // the turn after the next ones
            const bool is_q = h < p.q_heads, is_k = !is_q && h < p.q_heads + p.kv_heads;
            const uint8_t* src = is_q ? q + 2 * (int64_t)(h * p.head_dim)
                                      : is_k ? k + 2 * (int64_t)((h - p.q_heads) * p.head_dim)
                                             : v + 2 * (int64_t)((h - p.q_heads - p.kv_heads) * p.head_dim);
#pragma unroll
            for (int j = 0; j < CHUNKS; ++j) {
                const int at = lane + j * LANES;
                c[i][j] = h < end && at < n_chunks ? ldg16_once(src + 16 * at) : make_uint4(0, 0, 0, 0);
            }
        }
    }
}

template <int DT>
void launch(AppendParams p, int cus, hipStream_t stream) {
    const int chunks = p.head_dim / 8;
    auto go = [&](auto kernel1, auto kernel4, int lanes) {
        // A wave has all of a token's vectors where that leaves 16 waves to a SIMD's queue, fewer where tokens are
        // few: a decoding step's 32 tokens of 48 vectors are 384 waves of one turn, 4.6 us (7.3 with four in flight).
        const int turn = 64 / lanes, turns = (p.vecs + turn - 1) / turn;
        int64_t parts = ((int64_t)cus * 64 + p.n_tokens - 1) / p.n_tokens;
        parts = parts < turns ? parts : turns;
        const int per_part = (int)((turns + parts - 1) / parts);
        p.part_vecs = per_part * turn;
        p.parts = (uint32_t)((turns + per_part - 1) / per_part);
        const uint64_t units = (uint64_t)p.n_tokens * p.parts;
        launch_blocks(per_part < 4 ? kernel1 : kernel4, (units + 3) / 4, 256, 0, stream, p);
    };
#define ZT_GO(lanes, chunks) go(append_kernel<DT, lanes, chunks, 1>, append_kernel<DT, lanes, chunks, 4>, lanes)
    if (chunks <= 2) ZT_GO(2, 1);
    else if (chunks <= 4) ZT_GO(4, 1);
    else if (chunks <= 8) ZT_GO(8, 1);
    else if (chunks <= 16) ZT_GO(16, 1);
    else if (chunks <= 32) ZT_GO(32, 1);
    else if (chunks <= 64) ZT_GO(64, 1);
    else ZT_GO(64, 2);
#undef ZT_GO
}

}  // namespace

extern "C" int ztcp_append_tokens(const void* q, int64_t q_stride, void* q_out, int64_t q_out_stride, const void* k,
                                  int64_t k_stride, const void* v, int64_t v_stride, int64_t n_tokens,
                                  int64_t q_heads, const ztcp_page_pool* pool, const ztcp_geometry* g,
                                  const int64_t* slots, const int32_t* positions, const float* rope,
                                  int64_t max_position, const void* q_weight, int64_t q_weight_len,
                                  const void* k_weight, int64_t k_weight_len, float eps, int32_t interleaved,
                                  void* stream) {
    arg_result(ZTCP_OK, "");
    if (const char* why = check_pool(pool, g, 1024)) return arg_result(ZTCP_EINVAL, why);
    if (n_tokens < 0 || q_heads < 0) return arg_result(ZTCP_EINVAL, "n_tokens and q_heads must not be negative");
    if (n_tokens == 0) return ZTCP_OK;
    const int64_t d = g->head_dim, r = g->rope_dim, per_token = q_heads + g->num_heads * (pool->v ? 2 : 1);
    if (per_token > (int64_t)1 << 20 || n_tokens > ((int64_t)1 << 31) / per_token - 1)
        return arg_result(ZTCP_EINVAL, "too many head vectors in one call (n_tokens * heads must be below 2^31)");
    if (r > 512) return arg_result(ZTCP_EINVAL, "rope_dim must be at most 512");
    if (!k || (q_heads > 0 && (!q || !q_out)) || !slots || (r > 0 && (!positions || !rope)))
        return arg_result(ZTCP_EINVAL, "q, k, slots, positions and rope must not be NULL");
    if ((v != nullptr) != (pool->v != nullptr))
        return arg_result(ZTCP_EINVAL, "v and the pool's v must both be given or both be NULL");
    if (r > 0 && (max_position < 1 || max_position > (int64_t)0x7FFFFFFF))
        return arg_result(ZTCP_EINVAL, "max_position must be 1 .. 2^31 - 1");
    for (int64_t len : {q_weight_len, k_weight_len})
        if (len != 0 && len != d && !(len == d - r && len > 0))
            return arg_result(ZTCP_EINVAL, "a norm weight must have head_dim or head_dim - rope_dim entries");
    if ((q_weight_len > 0) != (q_weight != nullptr) || (k_weight_len > 0) != (k_weight != nullptr))
        return arg_result(ZTCP_EINVAL, "a norm weight and its length must agree");
    if (!(eps >= 0.f) || isinf(eps)) return arg_result(ZTCP_EINVAL, "eps must be a finite number, not negative");
    if (!hot_aligned(q) || !hot_aligned(q_out) || !hot_aligned(k) || !hot_aligned(v) || !hot_aligned(q_weight) ||
        !hot_aligned(k_weight) || (q_stride | q_out_stride | k_stride | v_stride) % 8 != 0)
        return arg_result(ZTCP_EINVAL, "token rows and weights must be 16-byte aligned");
    const int64_t qw = q_heads * d, kw = g->num_heads * d;
    if (n_tokens > 1 && (q_stride < qw || q_out_stride < qw || k_stride < kw || (v && v_stride < kw)))
        return arg_result(ZTCP_EINVAL, "token strides must cover a token's heads");
    // q_out may be q; no output may be another input, and the pool none at all
    const bool in_place = q == q_out && q_stride == q_out_stride;
    struct Rows {
        const void* p;
        int64_t n, bytes, stride;
    };
    const int64_t page = g->num_tokens * kw;
    const Rows in[3] = {{q, n_tokens, 2 * qw, 2 * q_stride}, {k, n_tokens, 2 * kw, 2 * k_stride},
                        {v, n_tokens, 2 * kw, 2 * v_stride}};
    const Rows out[3] = {{qw ? q_out : nullptr, n_tokens, 2 * qw, 2 * q_out_stride},
                         {pool->k, pool->n_pages, 2 * page, 2 * pool->k_stride},
                         {pool->v, pool->n_pages, 2 * page, 2 * pool->v_stride}};
    for (int o = 0; o < 3; ++o)
        for (int i = 0; i < 3; ++i)
            if (!(o == 0 && i == 0 && in_place) && rows_overlap(out[o].p, out[o].n, out[o].bytes, out[o].stride, in[i].p,
                                                               in[i].n, in[i].bytes, in[i].stride))
                return arg_result(ZTCP_EOVERLAP, "q_out and the pages must not overlap q, k or v");
    for (int o = 0; o < 3; ++o)
        for (int i = 0; i < o; ++i)
            if (rows_overlap(out[o].p, out[o].n, out[o].bytes, out[o].stride, out[i].p, out[i].n, out[i].bytes,
                             out[i].stride))
                return arg_result(ZTCP_EOVERLAP, "q_out and the pages must not overlap each other");

    AppendParams p{};
    p.q = (const uint8_t*)q;
    p.k = (const uint8_t*)k;
    p.v = (const uint8_t*)v;
    p.q_out = (uint8_t*)q_out;
    p.q_stride = q_stride;
    p.k_stride = k_stride;
    p.v_stride = v_stride;
    p.q_out_stride = q_out_stride;
    p.k_pool = (uint8_t*)pool->k;
    p.v_pool = (uint8_t*)pool->v;
    p.n_slots = pool->n_pages * g->num_tokens;
    p.k_page = pool->k_stride;
    p.v_page = pool->v_stride;
    p.slots = slots;
    p.positions = positions;
    p.rope = rope;
    p.max_position = (int32_t)max_position;
    p.q_weight = (const uint8_t*)q_weight;
    p.k_weight = (const uint8_t*)k_weight;
    p.q_weight_len = (int32_t)q_weight_len;
    p.k_weight_len = (int32_t)k_weight_len;
    p.n_tokens = (uint32_t)n_tokens;
    p.vecs = (int32_t)per_token;
    p.q_heads = (int32_t)q_heads;
    p.kv_heads = (int32_t)g->num_heads;
    p.head_dim = (int32_t)d;
    p.rope_dim = (int32_t)r;
    p.page_tokens = (int32_t)g->num_tokens;
    p.interleaved = interleaved;
    p.eps = eps;
    int cus = 0;
    if (cu_count(cus) != ZTCP_OK) return ZTCP_EHIP;
    if (g->hot_dtype == ZTCP_HOT_BF16) launch<kHotBf16>(p, cus, (hipStream_t)stream);
    else launch<kHotFp16>(p, cus, (hipStream_t)stream);
    return hipGetLastError() == hipSuccess ? ZTCP_OK : ZTCP_EHIP;
}
