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
    uint32_t vecs, vecs_per_token;                        // head vectors of the call, of a token
    int32_t q_heads, kv_heads, head_dim, rope_dim, page_tokens;
    int32_t interleaved;
    float eps;
};

// Eight elements of a head vector in fp32.
struct Chunk {
    float x[8];
};

template <int DT>
__device__ __forceinline__ Chunk load_chunk(const uint8_t* p) {
    const uint4 w = ldg16(p);
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

// One head vector per group of LANES lanes (a power of two, eight elements a
// lane and chunk; CHUNKS > 1 only for the vectors of more than 512 elements).
// The pass reads and writes every element once and is bound by that; the sum
// of squares is a butterfly over the group, and the partner of a rotated pair
// sits rope_dim / 16 lanes away (or in the same lane when interleaved), so a
// vector never leaves registers.
template <int DT, int LANES, int CHUNKS>
__global__ __launch_bounds__(256) void append_kernel(AppendParams p) {
    const int lane = (int)threadIdx.x % LANES;
    const uint32_t vec = blockIdx.x * (256u / LANES) + threadIdx.x / LANES;
    const bool live = vec < p.vecs;
    const uint32_t token = live ? vec / p.vecs_per_token : 0u;
    const int h = live ? (int)(vec - token * p.vecs_per_token) : 0;
    const bool is_q = h < p.q_heads, is_k = !is_q && h < p.q_heads + p.kv_heads;
    const int head = is_q ? h : is_k ? h - p.q_heads : h - p.q_heads - p.kv_heads;
    const int64_t stride = is_q ? p.q_stride : is_k ? p.k_stride : p.v_stride;
    const uint8_t* src = (is_q ? p.q : is_k ? p.k : p.v) + 2 * ((int64_t)token * stride + (int64_t)head * p.head_dim);
    const int n_chunks = live ? p.head_dim / 8 : 0;
    Chunk c[CHUNKS];
#pragma unroll
    for (int i = 0; i < CHUNKS; ++i) {
        const int at = lane + i * LANES;
        if (at < n_chunks) c[i] = load_chunk<DT>(src + 16 * at);
        else
#pragma unroll
            for (int e = 0; e < 8; ++e) c[i].x[e] = 0.f;
    }
    // where the vector goes
    uint8_t* dst = nullptr;
    if (live) {
        if (is_q) {
            dst = p.q_out + 2 * ((int64_t)token * p.q_out_stride + (int64_t)head * p.head_dim);
        } else {
            const int64_t slot = p.slots[token];
            if (slot >= 0 && slot < p.n_slots) {
                const int64_t page = slot / p.page_tokens, row = slot - page * p.page_tokens;
                dst = (is_k ? p.k_pool + 2 * page * p.k_page : p.v_pool + 2 * page * p.v_page) +
                      2 * (row * p.kv_heads + head) * p.head_dim;
            }
        }
    }
    // norm of the last weight_len columns
    const int weight_len = is_q ? p.q_weight_len : is_k ? p.k_weight_len : 0;
    const int first = (p.head_dim - weight_len) / 8;   // first normed chunk
    float ss = 0.f;
#pragma unroll
    for (int i = 0; i < CHUNKS; ++i)
        if (lane + i * LANES >= first)
#pragma unroll
            for (int e = 0; e < 8; ++e) ss = __builtin_fmaf(c[i].x[e], c[i].x[e], ss);
    ss = xor_sum(ss, LANES);
    if (weight_len > 0) {
        const float inv = rsqrtf(ss / (float)weight_len + p.eps);
        const uint8_t* weight = is_q ? p.q_weight : p.k_weight;
#pragma unroll
        for (int i = 0; i < CHUNKS; ++i) {
            const int at = lane + i * LANES;
            if (at >= first && at < n_chunks) {
                const Chunk w = load_chunk<DT>(weight + 16 * (at - first));
#pragma unroll
                for (int e = 0; e < 8; ++e) c[i].x[e] = c[i].x[e] * inv * w.x[e];
            }
        }
    }
    // rotation; all rotated columns are in chunk 0 of a lane (rope_dim <= 512)
    const int half = p.rope_dim / 16;   // chunks of half the rotated columns
    if (half > 0) {
        const bool turned = lane < 2 * half && live && (is_q || is_k);
        const int32_t pos = turned ? p.positions[token] : 0;
        const bool known = pos >= 0 && pos < p.max_position;
        const float* row = p.rope + (int64_t)(known ? pos : 0) * p.rope_dim;
        float cs[8], sn[8];
        const int a0 = p.interleaved ? 4 * lane : 8 * (lane < half ? lane : lane - half);
        const int n = p.interleaved ? 4 : 8;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const bool has = turned && e < n;
            cs[e] = has ? (known ? row[a0 + e] : __builtin_nanf("")) : 1.f;
            sn[e] = has ? (known ? row[8 * half + a0 + e] : __builtin_nanf("")) : 0.f;
        }
        if (p.interleaved) {
            if (turned)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float a = c[0].x[2 * e], b = c[0].x[2 * e + 1];
                    c[0].x[2 * e] = __builtin_fmaf(a, cs[e], -(b * sn[e]));
                    c[0].x[2 * e + 1] = __builtin_fmaf(b, cs[e], a * sn[e]);
                }
        } else {
            const int partner = (int)(threadIdx.x & 63u) + (lane < half ? half : -half);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const float o = __shfl(c[0].x[e], partner & 63);
                if (turned)
                    c[0].x[e] = lane < half ? __builtin_fmaf(c[0].x[e], cs[e], -(o * sn[e]))
                                            : __builtin_fmaf(c[0].x[e], cs[e], o * sn[e]);
            }
        }
    }
    if (dst)
#pragma unroll
        for (int i = 0; i < CHUNKS; ++i) {
            const int at = lane + i * LANES;
            if (at < n_chunks) stg16(dst, at, pack_chunk<DT>(c[i]));
        }
}

template <int DT>
void launch(const AppendParams& p, hipStream_t stream) {
    const int chunks = p.head_dim / 8;
    auto go = [&](auto kernel, uint32_t lanes) {
        const uint32_t per_block = 256 / lanes;
        hipLaunchKernelGGL(kernel, dim3((p.vecs + per_block - 1) / per_block), dim3(256), 0, stream, p);
    };
    if (chunks <= 2) go(append_kernel<DT, 2, 1>, 2);
    else if (chunks <= 4) go(append_kernel<DT, 4, 1>, 4);
    else if (chunks <= 8) go(append_kernel<DT, 8, 1>, 8);
    else if (chunks <= 16) go(append_kernel<DT, 16, 1>, 16);
    else if (chunks <= 32) go(append_kernel<DT, 32, 1>, 32);
    else if (chunks <= 64) go(append_kernel<DT, 64, 1>, 64);
    else go(append_kernel<DT, 64, 2>, 64);
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
    p.vecs = (uint32_t)(n_tokens * per_token);
    p.vecs_per_token = (uint32_t)per_token;
    p.q_heads = (int32_t)q_heads;
    p.kv_heads = (int32_t)g->num_heads;
    p.head_dim = (int32_t)d;
    p.rope_dim = (int32_t)r;
    p.page_tokens = (int32_t)g->num_tokens;
    p.interleaved = interleaved;
    p.eps = eps;
    if (g->hot_dtype == ZTCP_HOT_BF16) launch<kHotBf16>(p, (hipStream_t)stream);
    else launch<kHotFp16>(p, (hipStream_t)stream);
    return hipGetLastError() == hipSuccess ? ZTCP_OK : ZTCP_EHIP;
}
