// ztcp_mass.hip -- the attention weight that each hot page received.
//
//   mass[s, h, p] = decay * mass[s, h, p] + sum over the rows i of KV head h and
//                   the tokens j of page p that i sees of exp(s_ij - lse_i)
#include <type_traits>

#include "ztcp_hot.h"

using namespace ztcp;

namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr int kBlockKeys = 256;

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
    int32_t group_pages;             // pages of a workgroup
    float scale_log2, decay;
};

// A workgroup owns whole pages of one KV head, 64 of up to 256 keys a wave: K
// stays in registers while the rows pass by, each key's sum over the rows in
// fp32 registers, so every page's account has one writer and one order of
// additions.
template <int DT, int DP>
__global__ __launch_bounds__(256) void mass_kernel(MassParams p) {
    constexpr int kSteps = DP / 32;
    __shared__ float key_sum[kBlockKeys];
    const int lane = (int)threadIdx.x & 63, wave = (int)threadIdx.x >> 6;
    const int col = lane & 15, quad = lane >> 4;
    const int head = (int)(blockIdx.x % (uint32_t)p.kv_heads);
    const uint32_t rest = blockIdx.x / (uint32_t)p.kv_heads;
    const int groups = (p.max_pages + p.group_pages - 1) / p.group_pages;
    const int page0 = (int)(rest % (uint32_t)groups) * p.group_pages, s = (int)(rest / (uint32_t)groups);
    const Seq seq = seq_of(p.batch, s);
    const int rows = seq.n_new * p.group;
    const int pages = min(p.group_pages, p.max_pages - page0);
    const int T = p.batch.page_tokens;
    const int key0 = page0 * T, key1 = min(seq.len, key0 + pages * T);
    const float* account = p.mass + ((int64_t)s * p.kv_heads + head) * p.max_pages + page0;
    float* out = p.out + ((int64_t)s * p.kv_heads + head) * p.max_pages + page0;
    float sum = 0.f;                                          // thread i: of page page0 + i
    for (int kb = key0; kb < key1 && rows > 0; kb += kBlockKeys) {
        const int wb = kb + 64 * wave;
        uint64_t here = 0;
        float acc[4][4] = {};
        if (wb < key1) {
            const Place at = place_of(p.batch, seq, wb + lane, key1);
            here = __ballot(at.page >= 0);
            const int page = max(at.page, 0), row = at.page >= 0 ? at.row : 0;
            uint4 kf[4][kSteps];
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                const int64_t pg = __shfl(page, 16 * u + col), rw = __shfl(row, 16 * u + col);
                const uint8_t* src = p.k_pool + 2 * (pg * p.k_page + (rw * p.kv_heads + head) * p.head_dim);
#pragma unroll
                for (int i = 0; i < kSteps; ++i) {
                    const int d = 32 * i + 8 * quad;
                    kf[u][i] = d < p.head_dim ? ldg16(src + 2 * d) : make_uint4(0, 0, 0, 0);
                }
            }
            // rows that see the wave's first key
            const int t0 = max(0, wb - (seq.len - seq.n_new));
            for (int r0 = t0 < seq.n_new ? t0 * p.group / 16 * 16 : rows; r0 < rows; r0 += 16) {
                const int r = r0 + col;
                const int token = r / p.group, q_head = head * p.group + (r - token * p.group);
                int limit = r < rows ? seq.len - seq.n_new + token + 1 : 0;
                const uint8_t* src = p.q + 2 * ((int64_t)(seq.row0 + token) * p.q_stride + (int64_t)q_head * p.head_dim);
                uint4 qf[kSteps];
#pragma unroll
                for (int i = 0; i < kSteps; ++i) {
                    const int d = 32 * i + 8 * quad;
                    qf[i] = r < rows && d < p.head_dim ? ldg16(src + 2 * d) : make_uint4(0, 0, 0, 0);
                }
                const float lse = r < rows ? p.lse[(int64_t)(seq.row0 + token) * p.kv_heads * p.group + q_head] : 0.f;
                if (lse == -INFINITY) limit = 0;             // the row saw nothing
                const float base = lse == -INFINITY ? 0.f : lse * kLog2e;
#pragma unroll
                for (int u = 0; u < 4; ++u) {
                    f32x4 sc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int i = 0; i < kSteps; ++i) sc = mfma16<DT>(kf[u][i], qf[i], sc);
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const float w = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[i], p.scale_log2, -base));
                        acc[u][i] += wb + 16 * u + 4 * quad + i < limit ? w : 0.f;
                    }
                }
            }
        }
#pragma unroll
        for (int u = 0; u < 4; ++u)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int key = 16 * u + 4 * quad + i;
                const float x = xor_sum(acc[u][i], 16);
                if (col == 0) key_sum[64 * wave + key] = (here >> key) & 1u ? x : 0.f;
            }
        __syncthreads();
        if ((int)threadIdx.x < pages) {
            const int from = max(kb, key0 + (int)threadIdx.x * T), to = min(kb + kBlockKeys, key0 + ((int)threadIdx.x + 1) * T);
            for (int k = from; k < to; ++k) sum += key_sum[k - kb];
        }
        __syncthreads();
    }
    if ((int)threadIdx.x < pages) out[threadIdx.x] = __builtin_fmaf(p.decay, account[threadIdx.x], sum);
}

template <int DT, int DP>
void launch(const MassParams& p, hipStream_t stream) {
    const int64_t groups = (p.max_pages + p.group_pages - 1) / p.group_pages;
    hipLaunchKernelGGL((mass_kernel<DT, DP>), dim3((uint32_t)(p.batch.n_seqs * groups * p.kv_heads)), dim3(256), 0, stream, p);
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
    p.head_dim = (int32_t)d;
    p.max_pages = (int32_t)batch->max_pages;
    p.group_pages = (int32_t)(g->num_tokens >= kBlockKeys ? 1 : kBlockKeys / g->num_tokens);
    p.scale_log2 = scale * kLog2e;
    p.decay = decay;
    const int64_t groups = (p.max_pages + p.group_pages - 1) / p.group_pages;
    if (batch->n_seqs * groups * g->num_heads >= (int64_t)1 << 31)
        return arg_result(ZTCP_EINVAL, "too many sequences, pages and heads in one call");
    auto go = [&](auto dt) {
        constexpr int DT = decltype(dt)::value;
        if (d <= 64) launch<DT, 64>(p, (hipStream_t)stream);
        else if (d <= 128) launch<DT, 128>(p, (hipStream_t)stream);
        else launch<DT, 256>(p, (hipStream_t)stream);
    };
    if (g->hot_dtype == ZTCP_HOT_BF16) go(std::integral_constant<int, kHotBf16>{});
    else go(std::integral_constant<int, kHotFp16>{});
    return hipGetLastError() == hipSuccess ? ZTCP_OK : ZTCP_EHIP;
}
