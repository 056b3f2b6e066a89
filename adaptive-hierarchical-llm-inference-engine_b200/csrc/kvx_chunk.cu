// kvx_chunk.cu -- attention of several new tokens per sequence over int8
// pages (kvx_attend_chunk).
//
// With x = zp + (c + 128) s for every block of 16 tokens x 128 dims and
// mid = zp + 128 s,
//     q . k = s (q . c) + mid sum(q)
//     sum_t p_t v_t = sum_t (p_t s_t) c_t + sum_t p_t mid_t.
#include <math_constants.h>

#include <algorithm>

#include "kvx_common.cuh"

namespace kvx {
namespace {

struct ChunkParams {
    const uint8_t *pool;
    const float *stats;
    const int32_t *block_table, *q_start, *positions;
    const void *q;
    void *out;
    int32_t *error_flag;
    int batch, total, hq, hkv, group, max_pages, num_pages, causal;
    float scale_log2;
};

// One CTA per (token, kv-head), a warp per q-head of the group, lane: 4 dims.
template <typename T>
__global__ void __launch_bounds__(128) attend_rows_kernel(const __grid_constant__ ChunkParams p) {
    __shared__ int slot;
    const int t = blockIdx.x, kvh = blockIdx.y, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (threadIdx.x == 0) slot = -1;
    __syncthreads();
    for (int i = threadIdx.x; i < p.batch; i += blockDim.x)
        if (p.q_start[i] <= t && t < p.q_start[i + 1]) slot = i;
    __syncthreads();
    const int s = slot;
    if (s < 0) return;
    const int pos = p.positions[s], a = p.q_start[s], b = min(p.q_start[s + 1], p.total);
    long long keys = pos < 0 ? 0 : (p.causal ? (long long)pos + t - a + 1 : (long long)pos + b - a);
    if (pos < 0 && p.error_flag) atomicOr(p.error_flag, 2);
    if (keys > (long long)p.max_pages * kPageTokens) {
        keys = (long long)p.max_pages * kPageTokens;
        if (p.error_flag) atomicOr(p.error_flag, 4);
    }
    const int T_ = (int)keys;
    for (int g = warp; g < p.group; g += 4) {
        const T *qr = static_cast<const T *>(p.q) + ((size_t)t * p.hq + kvh * p.group + g) * kHeadDim + 4 * lane;
        float q[4], acc[4] = {0.f, 0.f, 0.f, 0.f}, qs = 0.f;
        for (int k = 0; k < 4; ++k) {
            q[k] = io_traits<T>::load(qr + k) * p.scale_log2;
            qs += q[k];
        }
        for (int o = 16; o; o >>= 1) qs += __shfl_xor_sync(0xffffffffu, qs, o);
        float m = -CUDART_INF_F, l = 0.f;
        for (int k0 = 0; k0 < T_; k0 += kPageTokens) {
            const int phys = p.block_table[(size_t)s * p.max_pages + k0 / kPageTokens];
            if (phys < 0 || phys >= p.num_pages) {
                if (p.error_flag) atomicOr(p.error_flag, 2);
                continue;
            }
            const size_t kb = ((size_t)phys * 2) * p.hkv + kvh, vb = kb + p.hkv;
            const float4 ks = reinterpret_cast<const float4 *>(p.stats)[kb], vs = reinterpret_cast<const float4 *>(p.stats)[vb];
            const float kmid = fmaf(128.f, ks.z, ks.w), vmid = fmaf(128.f, vs.z, vs.w);
            for (int j = 0; j < min(kPageTokens, T_ - k0); ++j) {
                const char4 kc = reinterpret_cast<const char4 *>(p.pool + (kb * kPageTokens + j) * kHeadDim)[lane];
                const char4 vc = reinterpret_cast<const char4 *>(p.pool + (vb * kPageTokens + j) * kHeadDim)[lane];
                float dot = q[0] * kc.x + q[1] * kc.y + q[2] * kc.z + q[3] * kc.w;
                for (int o = 16; o; o >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, o);
                const float sc = fmaf(ks.z, dot, kmid * qs);
                const float mn = fmaxf(m, sc), al = exp2f(m - mn), pr = exp2f(sc - mn);
                m = mn;
                l = l * al + pr;
                const float ps = pr * vs.z, pm = pr * vmid;
                acc[0] = fmaf(acc[0], al, fmaf(ps, (float)vc.x, pm));
                acc[1] = fmaf(acc[1], al, fmaf(ps, (float)vc.y, pm));
                acc[2] = fmaf(acc[2], al, fmaf(ps, (float)vc.z, pm));
                acc[3] = fmaf(acc[3], al, fmaf(ps, (float)vc.w, pm));
            }
        }
        T *o = static_cast<T *>(p.out) + ((size_t)t * p.hq + kvh * p.group + g) * kHeadDim + 4 * lane;
        for (int k = 0; k < 4; ++k) io_traits<T>::store(o + k, l == 0.f ? 0.f : acc[k] / l);
    }
}

}  // namespace
}  // namespace kvx

using namespace kvx;

extern "C" KVX_API size_t kvx_attend_chunk_workspace_bytes(int32_t batch, int32_t total_tokens, int32_t num_q_heads,
                                                           int32_t num_kv_heads, int32_t max_pages) {
    if (batch <= 0 || total_tokens <= 0 || num_q_heads <= 0 || num_kv_heads <= 0 || num_q_heads % num_kv_heads ||
        max_pages <= 0)
        return 0;
    return 16;
}

extern "C" KVX_API int kvx_attend_chunk(const kvx_paged *kv, const int32_t *block_table, int32_t max_pages,
                                        const int32_t *q_start, const int32_t *positions, int32_t batch,
                                        int32_t total_tokens, int32_t num_q_heads, const void *q, void *out,
                                        int32_t io_dtype, float sm_scale, int32_t causal, void *workspace,
                                        size_t workspace_bytes, int32_t *error_flag, void *stream) {
    if (!kv || !kv->pool || !block_table || !q_start || !positions) return KVX_EINVAL;
    if (batch < 0 || total_tokens < 0 || max_pages <= 0 || kv->num_kv_heads <= 0 || num_q_heads <= 0 || kv->num_pages <= 0)
        return KVX_EINVAL;
    if (num_q_heads % kv->num_kv_heads != 0 || (causal != 0 && causal != 1)) return KVX_EINVAL;
    if (io_dtype != KVX_F16 && io_dtype != KVX_F32) return KVX_EINVAL;
    if (kv->dtype != KVX_I8 || kv->head_dim != kHeadDim || kv->page_tokens != kPageTokens) return KVX_EUNSUPPORTED;
    if (kv->num_kv_heads > 65535 || num_q_heads > 65535) return KVX_EUNSUPPORTED;
    if (!kv->stats) return KVX_EINVAL;
    if (batch == 0 || total_tokens == 0) return KVX_OK;
    if (!q || !out) return KVX_EINVAL;
    if ((reinterpret_cast<uintptr_t>(kv->pool) | reinterpret_cast<uintptr_t>(kv->stats) | reinterpret_cast<uintptr_t>(q) |
         reinterpret_cast<uintptr_t>(out)) & 15)
        return KVX_EINVAL;
    if (!workspace || workspace_bytes < kvx_attend_chunk_workspace_bytes(batch, total_tokens, num_q_heads,
                                                                         kv->num_kv_heads, max_pages))
        return KVX_ENOSPC;
    if (reinterpret_cast<uintptr_t>(workspace) & 15) return KVX_EINVAL;
    ChunkParams p{};
    p.pool = static_cast<const uint8_t *>(kv->pool);
    p.stats = kv->stats;
    p.block_table = block_table, p.q_start = q_start, p.positions = positions;
    p.q = q, p.out = out, p.error_flag = error_flag;
    p.batch = batch, p.total = total_tokens, p.hq = num_q_heads, p.hkv = kv->num_kv_heads;
    p.group = num_q_heads / kv->num_kv_heads, p.max_pages = max_pages, p.num_pages = kv->num_pages, p.causal = causal;
    p.scale_log2 = (sm_scale > 0.f ? sm_scale : 1.0f / sqrtf((float)kHeadDim)) * 1.4426950408889634f;
    const dim3 grid((unsigned)total_tokens, (unsigned)kv->num_kv_heads);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (io_dtype == KVX_F16)
        attend_rows_kernel<__half><<<grid, 128, 0, st>>>(p);
    else
        attend_rows_kernel<float><<<grid, 128, 0, st>>>(p);
    return launch_status();
}
