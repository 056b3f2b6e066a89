// kvx_rope.cu -- rotary positions (kvx_rope) and the ragged, rotated append
// into fp16 / fp32 / int8 pages (kvx_rope_append).
//
// Both are bound by the bytes of their rows.  One CTA per token: its
// (cos, sin) pairs are worked out once into shared memory (rotary/2 sincospi
// for heads * rotary/2 pairs), each thread keeps one item of a row -- a
// 16-byte vector, or the two that pair up in the half layout -- with its
// cosines in registers and walks the token's rows, the first of which are
// asked for before the cosines are worked out (afterwards: 98 against 93 us).
// Backward of 8191 tokens x 72 heads of 128 (64 rotated, interleaved, fp32,
// strided): 93 us, 6.5 TB/s, the measured copy rate; 64 tokens of 32 heads:
// 2.3 us, a launch.
#include <math.h>

#include <algorithm>
#include <cmath>

#include "kvx_common.cuh"
#include "kvx_decode_params.cuh"  // grid_dependents_launch, grid_dependency_wait
#include "kvx_rope.cuh"

namespace kvx {
namespace {

constexpr int kMaxRopeDim = 1024;
constexpr int kRopeThreads = 256;
constexpr int kRowsInFlight = 4;  // rows whose loads a thread issues together
constexpr int kRowsBeside = 2;    // the same, of rope_append_q_kernel (59 us at the size below; 4 and 2 CTAs an SM: 84; 1 and 5: 65)

struct RopeTensor {
    const void *in;
    void *out;
    int heads;
    int64_t in_token, in_head, out_token, out_head;
};

struct RopeParams {
    const uint64_t *turns;
    const int32_t *positions;
    RopeTensor x[2];
    int rotary, items;
    float amplitude, sine_sign;
};

// The token's (cos, sin) pairs into shared memory.
__device__ __forceinline__ void fill_cs(float2 *cs, const uint64_t *turns, int pairs, int64_t pos, float amplitude,
                                        float sine_sign) {
    for (int i = threadIdx.x; i < pairs; i += blockDim.x) {
        float2 v = rope_turn(turns[i], pos, amplitude);
        v.y *= sine_sign;
        cs[i] = v;
    }
}

// Rows row0, row0 + step, ... < rows of the tensors, this thread's item of
// each.  ready() runs once (in every thread, rows or not) when the first rows
// have been asked for: the cosines are worked out while they are on their way.
template <int kRows, typename Item, typename T, typename Address, typename Ready>
__device__ __forceinline__ void rope_rows(const Item &item, int row0, int step, int rows, Address at, Ready ready) {
    bool asked = false;
    for (int r = row0; r < rows || !asked; r += kRows * step) {
        typename Item::Data d[kRows];
        const T *src[kRows];
        T *dst[kRows];
        bool turn[kRows];
#pragma unroll
        for (int u = 0; u < kRows; ++u) {
            dst[u] = nullptr;
            if (r + u * step < rows) {
                at(r + u * step, src[u], dst[u], turn[u]);
                if (dst[u]) item.load(src[u], d[u]);
            }
        }
        if (!asked) ready();
        asked = true;
#pragma unroll
        for (int u = 0; u < kRows; ++u)
            if (dst[u]) {
                if (turn[u]) item.turn(d[u]);
                item.store(dst[u], d[u]);
            }
    }
}

template <typename T, bool kHalf, bool kVec>
__global__ void __launch_bounds__(kVec ? kRopeThreads : kMaxRopeDim) rope_kernel(const __grid_constant__ RopeParams p) {
    __shared__ float2 cs[kMaxRopeDim / 2];
    const int64_t t = blockIdx.x;
    const int step = blockDim.x / p.items, row0 = threadIdx.x / p.items;
    RopeItem<T, kHalf, kVec> item(threadIdx.x % p.items, p.rotary);
    rope_rows<kRowsInFlight, RopeItem<T, kHalf, kVec>, T>(
        item, row0, step, row0 < step ? p.x[0].heads + p.x[1].heads : 0,  // threads left over by whole rows: none
        [&](int r, const T *&src, T *&dst, bool &turn) {
            const int which = r >= p.x[0].heads;
            const RopeTensor &x = p.x[which];
            const int64_t h = which ? r - p.x[0].heads : r;
            src = static_cast<const T *>(x.in) + t * x.in_token + h * x.in_head;
            dst = static_cast<T *>(x.out) + t * x.out_token + h * x.out_head;
            turn = true;
        },
        [&] {
            fill_cs(cs, p.turns, p.rotary / 2, p.positions[t], p.amplitude, p.sine_sign);
            __syncthreads();
            item.cosines(cs);
        });
}

// ---------------------------------------------------------------------------
// kvx_rope_append

struct RopeAppendParams {
    uint8_t *pool;
    float *stats;
    const int32_t *block_table, *q_start, *positions;
    int32_t *error_flag;
    const uint64_t *turns;  // null: no rotation
    const void *q, *k, *v;
    void *q_out;
    int64_t q_stride, k_stride, v_stride;
    int batch, total, hq, hkv, max_pages, num_pages, rotary, items;
    float amplitude;
    int kv_blocks, tokens_per_block;  // int8: CTAs that write pages, and the tokens each looks at
    bool apart;                       // int8: q is rotated by a launch of its own
};

// The sequence that owns packed row t, or -1: all threads look at the
// boundaries at once (one round trip for up to blockDim sequences).
__device__ __forceinline__ int find_sequence(const int32_t *q_start, int batch, int t, int *slot) {
    if (threadIdx.x == 0) *slot = -1;
    __syncthreads();
    for (int i = threadIdx.x; i < batch; i += blockDim.x)
        if (q_start[i] <= t && t < q_start[i + 1]) *slot = i;
    __syncthreads();
    return *slot;
}

// Token blockIdx: rotate q, and (fp16 / fp32 pools) rotate k and store k, v.
template <int kRows, typename T, bool kHalf, bool kVec>
__device__ __forceinline__ void rope_append_rows(const RopeAppendParams &p, int t, bool with_kv, float2 *cs, int *slot) {
    const int s = find_sequence(p.q_start, p.batch, t, slot);
    if (s < 0) return;
    const int off = t - p.q_start[s];
    const long long pos = (long long)p.positions[s] + off;
    T *page_row = nullptr;  // K row of head 0 at the token's slot
    if (with_kv) {
        const long long lp = pos >> 4;
        const int phys = p.positions[s] >= 0 && lp < p.max_pages ? p.block_table[(size_t)s * p.max_pages + lp] : -1;
        if (phys >= 0 && phys < p.num_pages)
            page_row = reinterpret_cast<T *>(p.pool) + ((size_t)phys * 2 * p.hkv * kPageTokens + (pos & 15)) * kHeadDim;
        else if (p.error_flag && threadIdx.x == 0)
            atomicOr(p.error_flag, 2);
    }
    const int step = blockDim.x / p.items, row0 = threadIdx.x / p.items;
    RopeItem<T, kHalf, kVec> item(threadIdx.x % p.items, p.rotary);
    const bool turning = p.turns != nullptr;
    rope_rows<kRows, RopeItem<T, kHalf, kVec>, T>(
        item, row0, step, row0 < step ? p.hq + (page_row ? 2 * p.hkv : 0) : 0, [&](int r, const T *&src, T *&dst, bool &turn) {
            turn = turning;
            if (r < p.hq) {
                src = static_cast<const T *>(p.q) + (int64_t)t * p.q_stride + r * kHeadDim;
                dst = static_cast<T *>(p.q_out) + ((int64_t)t * p.hq + r) * kHeadDim;
                return;
            }
            r -= p.hq;
            dst = page_row + (size_t)r * kPageTokens * kHeadDim;  // K heads, then V heads of the page
            if (r < p.hkv) {
                src = static_cast<const T *>(p.k) + (int64_t)t * p.k_stride + r * kHeadDim;
            } else {
                src = static_cast<const T *>(p.v) + (int64_t)t * p.v_stride + (r - p.hkv) * kHeadDim;
                turn = false;
            }
        },
        [&] {
            if (!turning) return;
            fill_cs(cs, p.turns, p.rotary / 2, pos, p.amplitude, 1.f);
            __syncthreads();
            item.cosines(cs);
        });
}

// Without a table the item geometry is that of rotary_dim 2 * kRopeVec in the
// interleaved layout (any that covers a row would do) and nothing turns.
template <typename T, bool kHalf, bool kVec>
__global__ void __launch_bounds__(kRopeThreads) rope_append_kernel(const __grid_constant__ RopeAppendParams p) {
    __shared__ float2 cs[kHeadDim / 2];
    __shared__ int slot;
    rope_append_rows<kRowsInFlight, T, kHalf, kVec>(p, blockIdx.x, true, cs, &slot);
}

// ---- int8 pages

constexpr float kTieLimit = 0.5f - 4.0e-5f;  // as in kvx_quant.cu: nearer to a half-integer, divide exactly
constexpr float kTwo23 = 8388608.0f;

// code + 128 of x: clamp(round((x - mn) / scale), 0, 255), NaN -> 0.
__device__ __noinline__ uint32_t level_exact(float x, float mn, float scale) {
    const float r = roundf(__fdiv_rn(__fsub_rn(x, mn), scale));
    return r >= 255.f && r < 2147483648.f ? 255u : (r > 0.f && r < 255.f ? (uint32_t)r : 0u);
}

// Four codes.  The product with the reciprocal decides; next to a
// half-integer, and where anything is not finite (a NaN wins the maximum),
// the division does.
__device__ __forceinline__ uint32_t code4(const float *x, float mn, float scale, float rcp) {
    uint32_t u[4];
    float worst = 0.f;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const float t = __fmul_rn(__fsub_rn(x[k], mn), rcp), s = __fadd_rn(t, kTwo23);
        const float off = fabsf(__fsub_rn(t, __fsub_rn(s, kTwo23)));
        asm("max.NaN.f32 %0, %0, %1;" : "+f"(worst) : "f"(off));
        u[k] = __float_as_uint(s);
    }
    if (!(worst <= kTieLimit)) {
#pragma unroll 1
        for (int k = 0; k < 4; ++k) {
            const uint32_t exact = level_exact(k < 2 ? (k ? x[1] : x[0]) : (k == 2 ? x[2] : x[3]), mn, scale);
            if (k == 0) u[0] = exact;
            if (k == 1) u[1] = exact;
            if (k == 2) u[2] = exact;
            if (k == 3) u[3] = exact;
        }
    }
    return __byte_perm(__byte_perm(u[0], u[1], 0x0040), __byte_perm(u[2], u[3], 0x0040), 0x5410) ^ 0x80808080u;
}

// Four elements as they lie in memory.
template <typename T> struct Raw4;
template <> struct Raw4<float> {
    float4 v;
    __device__ __forceinline__ void load(const float *p) { v = *reinterpret_cast<const float4 *>(p); }
    __device__ __forceinline__ void unpack(float *f) const { f[0] = v.x, f[1] = v.y, f[2] = v.z, f[3] = v.w; }
};
template <> struct Raw4<__half> {
    uint2 v;
    __device__ __forceinline__ void load(const __half *p) { v = *reinterpret_cast<const uint2 *>(p); }
    __device__ __forceinline__ void unpack(float *f) const {
        const float2 a = h2_to_f2(v.x), b = h2_to_f2(v.y);
        f[0] = a.x, f[1] = a.y, f[2] = b.x, f[3] = b.y;
    }
};

// One warp: the new rows (n from slot `slot0`) of one (page, K|V, head)
// block.  Lane: elements 4 lane .. 4 lane + 3 of every row, in registers from
// the range to the codes (read, unpacked and turned twice instead, the kernel
// issued 2.5 times the instructions and took 55 us, not 43).  cs: (cos,
// sin) of row i's pairs at cs + i * rotary/2, null for V and without a table.
// kVec: partners in the half layout lie a multiple of 4 away.
template <typename T, bool kHalf, bool kVec>
__device__ __forceinline__ void append_block_i8(const T *src, int64_t stride, uint8_t *codes, float *stats, int slot0,
                                                int n, const float2 *cs, int rotary) {
    const int lane = threadIdx.x & 31, d = 4 * lane, half = rotary / 2;
    const float4 old = *reinterpret_cast<const float4 *>(stats);
    float x[kPageTokens][4];
#pragma unroll
    for (int i = 0; i < kPageTokens; ++i)
        if (i < n) {
            Raw4<T> raw;
            raw.load(src + i * stride + d);
            raw.unpack(x[i]);
        }
    if (cs && d < rotary) {
        if constexpr (!kHalf) {
#pragma unroll
            for (int i = 0; i < kPageTokens; ++i)
                if (i < n) {
                    const float2 *c = cs + i * half + d / 2;
                    rope_pair(x[i][0], x[i][1], c[0]);
                    if (d + 2 < rotary) rope_pair(x[i][2], x[i][3], c[1]);
                }
        } else if constexpr (kVec) {  // rope_pair's half of the pair: a where d < half, else b
            const int far = d < half ? half : -half, at = d < half ? d : d - half;
            const float sign = d < half ? -1.f : 1.f;
#pragma unroll
            for (int i = 0; i < kPageTokens; ++i)
                if (i < n) {
                    Raw4<T> raw;
                    float y[4];
                    raw.load(src + i * stride + d + far);
                    raw.unpack(y);
                    const float4 c0 = *reinterpret_cast<const float4 *>(cs + i * half + at),
                                 c1 = *reinterpret_cast<const float4 *>(cs + i * half + at + 2);
                    x[i][0] = fmaf(x[i][0], c0.x, __fmul_rn(y[0], sign * c0.y));
                    x[i][1] = fmaf(x[i][1], c0.z, __fmul_rn(y[1], sign * c0.w));
                    x[i][2] = fmaf(x[i][2], c1.x, __fmul_rn(y[2], sign * c1.y));
                    x[i][3] = fmaf(x[i][3], c1.z, __fmul_rn(y[3], sign * c1.w));
                }
        } else {
#pragma unroll
            for (int i = 0; i < kPageTokens; ++i)
                if (i < n) {
                    const T *row = src + i * stride;
#pragma unroll
                    for (int k = 0; k < 4; ++k)
                        if (d + k < rotary) {
                            const bool first = d + k < half;
                            const float y = io_traits<T>::load(row + (first ? d + k + half : d + k - half));
                            const float2 c = cs[i * half + (first ? d + k : d + k - half)];
                            x[i][k] = fmaf(x[i][k], c.x, __fmul_rn(y, first ? -c.y : c.y));
                        }
                }
        }
    }
    float mn = INFINITY, mx = -INFINITY;
#pragma unroll
    for (int i = 0; i < kPageTokens; ++i)
        if (i < n)
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                mn = fminf(mn, x[i][k]);
                mx = fmaxf(mx, x[i][k]);
            }
#pragma unroll
    for (int o = 16; o; o >>= 1) {
        mn = fminf(mn, __shfl_xor_sync(0xffffffffu, mn, o));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
    }
    if (slot0 > 0) {
        mn = fminf(mn, old.x);
        mx = fmaxf(mx, old.y);
    }
    if (!(mn <= mx)) mn = mx = NAN;  // nothing but NaN
    float scale = __fdiv_rn(__fsub_rn(mx, mn), 255.f);
    if (scale == 0.f) scale = 1.f;
    const float rcp = __frcp_rn(scale);
    uint32_t *rows = reinterpret_cast<uint32_t *>(codes) + lane;
    if (slot0 > 0 && !(mn == old.x && mx == old.y)) {  // earlier rows in the wider range
#pragma unroll 4
        for (int r = 0; r < slot0; ++r) {
            const uint32_t u = rows[r * 32] ^ 0x80808080u;
            float v[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) v[k] = __fadd_rn(old.w, __fmul_rn((float)((u >> (8 * k)) & 0xffu), old.z));
            rows[r * 32] = code4(v, mn, scale, rcp);
        }
    }
#pragma unroll
    for (int i = 0; i < kPageTokens; ++i)
        if (i < n) rows[(slot0 + i) * 32] = code4(x[i], mn, scale, rcp);
    if (lane == 0) *reinterpret_cast<float4 *>(stats) = make_float4(mn, mx, scale, mn);
}

// CTAs 0 .. kv_blocks-1 write pages (even ones K, odd ones V blocks), the
// others rotate the q rows of one token each.  A page is written by whoever
// holds its first new token (the sequence's first, or one at a page start)
// among its tokens_per_block packed rows: one token a CTA while tokens are few
// (a decode step, where every token leads), 16 when they fill the GPU anyway.
// 32 sequences x 1 token (24 q-heads on 8): 4.2 us, three dependent reads and
// a launch.  6 chunks of up to 2731 tokens (64 q-heads on 8, fp16): 102 us for
// 410 MB, 43 of them the pages and 59 the q rows.  The pages are 65 MB, 10 us at
// the copy rate: with a block's rows in registers 16 warps fit on an SM, 42 % of
// the issue slots are used, and the rest is latency (fixed waits, scoreboards and
// barriers, 4.6 cycles an instruction) that so few warps do not hide.
//
// A warp with more than kDirectRows rows brings them to shared memory first,
// a bulk copy (TMA) a row, all in flight together; fewer are read in place,
// which is one round trip sooner.
constexpr int kDirectRows = 2;
template <typename T> constexpr int kStageBytes = kRopeThreads / 32 * kPageTokens * kHeadDim * (int)sizeof(T);

template <typename T, bool kHalf, bool kVec>
__global__ void __launch_bounds__(kRopeThreads, 2) rope_append_i8_kernel(const __grid_constant__ RopeAppendParams p) {
    extern __shared__ __align__(128) uint8_t stage[];
    __shared__ __align__(16) float2 cs[kPageTokens * kHeadDim / 2];
    __shared__ uint64_t bars[kRopeThreads / 32];
    __shared__ int slot, found;
    __shared__ int2 lead[kPageTokens];  // (sequence, packed row)
    // rope_append_q_kernel beside this one reads nothing that it writes; any
    // other launch may (kvx_decode reads pages before it waits)
    if (p.apart) grid_dependents_launch();
    if (blockIdx.x >= p.kv_blocks) {
        rope_append_rows<kRowsInFlight, T, kHalf, kVec>(p, blockIdx.x - p.kv_blocks, false, cs, &slot);
        return;
    }
    const bool is_v = blockIdx.x & 1;
    const int r0 = (blockIdx.x >> 1) * p.tokens_per_block, r1 = min(r0 + p.tokens_per_block, p.total);
    if (threadIdx.x == 0) found = 0;
    if (threadIdx.x < kRopeThreads / 32) mbar_init(&bars[threadIdx.x], 1);
    fence_barrier_init();
    __syncthreads();
    for (int s = threadIdx.x; s < p.batch; s += blockDim.x) {
        const int a = p.q_start[s], b = min(p.q_start[s + 1], p.total);
        const int lo = max(a, r0), hi = min(b, r1);
        if (a < 0 || lo >= hi) continue;
        const int pos = p.positions[s];
        if (pos < 0) {
            if (p.error_flag) atomicOr(p.error_flag, 2);
            continue;
        }
        for (int t = lo; t < hi;) {
            const int in_page = (int)(((long long)pos + t - a) & 15);
            if (t == a || in_page == 0) {
                const int i = atomicAdd(&found, 1);
                if (i < kPageTokens) lead[i] = make_int2(s, t);
            }
            t += 16 - in_page;
        }
    }
    __syncthreads();
    const int n_lead = min(found, kPageTokens), warp = threadIdx.x >> 5, lane = threadIdx.x & 31, half = p.rotary / 2;
    T *rows = reinterpret_cast<T *>(stage) + warp * kPageTokens * kHeadDim;
    uint32_t phase = 0;
    for (int i = 0; i < n_lead; ++i) {
        const int s = lead[i].x, t = lead[i].y;
        const int a = p.q_start[s], b = min(p.q_start[s + 1], p.total);
        const long long pos = (long long)p.positions[s] + t - a, lp = pos >> 4;
        const int slot0 = (int)(pos & 15), n = min(kPageTokens - slot0, b - t);
        const int phys = lp < p.max_pages ? p.block_table[(size_t)s * p.max_pages + lp] : -1;
        if (phys < 0 || phys >= p.num_pages) {
            if (p.error_flag && threadIdx.x == 0) atomicOr(p.error_flag, 2);
            continue;
        }
        const int64_t stride = is_v ? p.v_stride : p.k_stride;
        const T *row0 = static_cast<const T *>(is_v ? p.v : p.k) + t * stride;
        const bool staged = n > kDirectRows;
        auto fetch = [&](int h) {  // head h's rows, a lane each
            if (lane == 0) mbar_arrive_expect_tx(&bars[warp], n * kHeadDim * (int)sizeof(T));
            __syncwarp();
            if (lane < n)
                bulk_g2s(rows + lane * kHeadDim, row0 + lane * stride + h * kHeadDim, kHeadDim * (int)sizeof(T), &bars[warp]);
        };
        if (staged && warp < p.hkv) fetch(warp);  // under the work on the cosines
        if (p.turns && !is_v) {
            __syncthreads();  // the previous page's rows are rotated
            for (int j = threadIdx.x; j < n * half; j += blockDim.x)
                cs[j] = rope_turn(p.turns[j % half], pos + j / half, p.amplitude);
            __syncthreads();
        }
        for (int h = warp; h < p.hkv; h += kRopeThreads / 32) {
            const size_t block = (size_t)phys * 2 * p.hkv + (is_v ? p.hkv : 0) + h;
            uint8_t *codes = p.pool + block * kPageTokens * kHeadDim;
            float *stats = p.stats + block * 4;
            const float2 *turn = !is_v && p.turns ? cs : nullptr;
            if (staged) {
                if (!mbar_wait_bounded(&bars[warp], phase, p.error_flag)) {
                    (void)mbar_wait_bounded(&bars[warp], phase, nullptr);
                    return;
                }
                phase ^= 1;
                append_block_i8<T, kHalf, kVec>(rows, kHeadDim, codes, stats, slot0, n, turn, p.rotary);
                fence_proxy_async_smem();  // these reads before the next copies
                __syncwarp();
                if (h + kRopeThreads / 32 < p.hkv) fetch(h + kRopeThreads / 32);
            } else {
                append_block_i8<T, kHalf, kVec>(row0 + h * kHeadDim, stride, codes, stats, slot0, n, turn, p.rotary);
            }
        }
    }
}

// The q rows of many tokens, beside the CTAs that write their pages: placed
// while those run (nothing here depends on them), done when they are done.
template <typename T, bool kHalf, bool kVec>
__global__ void __launch_bounds__(kRopeThreads, 4) rope_append_q_kernel(const __grid_constant__ RopeAppendParams p) {
    __shared__ float2 cs[kHeadDim / 2];
    __shared__ int slot;
    rope_append_rows<kRowsBeside, T, kHalf, kVec>(p, blockIdx.x, false, cs, &slot);
    grid_dependency_wait();
}

template <typename T>
int launch_rope(const RopeParams &p, int tokens, int threads, bool half, bool vec, cudaStream_t st) {
    auto kern = half ? (vec ? rope_kernel<T, true, true> : rope_kernel<T, true, false>)
                     : (vec ? rope_kernel<T, false, true> : rope_kernel<T, false, false>);
    kern<<<(unsigned)tokens, threads, 0, st>>>(p);
    return launch_status();
}

template <typename T>
int launch_rope_append(const RopeAppendParams &p, bool i8, bool half, bool vec, cudaStream_t st) {
    if (i8) {
        auto kern = half ? (vec ? rope_append_i8_kernel<T, true, true> : rope_append_i8_kernel<T, true, false>)
                         : (vec ? rope_append_i8_kernel<T, false, true> : rope_append_i8_kernel<T, false, false>);
        // rows to stage: only where a page gets more than kDirectRows of them
        const int smem = p.total > kDirectRows ? kStageBytes<T> : 0;
        static std::atomic<bool> attr_done[4][kMaxDevices];
        if (smem && ensure_smem_attr(attr_done[2 * half + vec], kern, smem) != KVX_OK) return KVX_ECUDA;
        // Many tokens: the CTAs that rotate q get a launch of their own, whose
        // 64 registers let 4 of them on an SM (with the other role's 128 it is
        // 2, too few to keep the memory busy).
        kern<<<(unsigned)p.kv_blocks + (p.hq && !p.apart ? (unsigned)p.total : 0u), kRopeThreads, smem, st>>>(p);
        const int rc = launch_status();  // clears the error: asked once
        if (!p.apart || rc != KVX_OK) return rc;
        auto q_kern = half ? (vec ? rope_append_q_kernel<T, true, true> : rope_append_q_kernel<T, true, false>)
                           : (vec ? rope_append_q_kernel<T, false, true> : rope_append_q_kernel<T, false, false>);
        cudaLaunchConfig_t cfg{};
        cfg.gridDim = dim3((unsigned)p.total);
        cfg.blockDim = dim3(kRopeThreads);
        cfg.stream = st;
        cudaLaunchAttribute attr[1];
        attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[0].val.programmaticStreamSerializationAllowed = 1;
        cfg.attrs = attr;
        cfg.numAttrs = 1;
        if (cudaLaunchKernelEx(&cfg, q_kern, p) != cudaSuccess) {
            cudaGetLastError();
            return KVX_ECUDA;
        }
    } else {
        auto kern = half ? (vec ? rope_append_kernel<T, true, true> : rope_append_kernel<T, true, false>)
                         : (vec ? rope_append_kernel<T, false, true> : rope_append_kernel<T, false, false>);
        kern<<<(unsigned)p.total, kRopeThreads, 0, st>>>(p);
    }
    return launch_status();
}

bool table_ok(const kvx_rope_table *t, int head_dim) {
    return t->turns && !(reinterpret_cast<uintptr_t>(t->turns) & 7) && t->rotary_dim >= 2 && t->rotary_dim % 2 == 0 &&
           t->rotary_dim <= head_dim && (t->layout == KVX_ROPE_HALF || t->layout == KVX_ROPE_INTERLEAVED);
}

}  // namespace
}  // namespace kvx

using namespace kvx;

extern "C" KVX_API int kvx_rope_frequencies(const kvx_rope_config *cfg, uint64_t *turns, float *amplitude) {
    if (!cfg || !turns || !amplitude) return KVX_EINVAL;
    const int d = cfg->rotary_dim, kind = cfg->scaling;
    if (d < 2 || d % 2 || d > kMaxRopeDim || kind < KVX_ROPE_NONE || kind > KVX_ROPE_YARN) return KVX_EINVAL;
    if (!(cfg->base > 0) || !std::isfinite(cfg->base)) return KVX_EINVAL;
    const double factor = kind == KVX_ROPE_NONE ? 1.0 : cfg->factor;
    if (!(factor >= 1) || !std::isfinite(factor)) return KVX_EINVAL;
    const bool bands = kind == KVX_ROPE_LLAMA3 || kind == KVX_ROPE_YARN;
    if (bands && (!(cfg->low > 0) || !(cfg->high > cfg->low) || !std::isfinite(cfg->high) ||
                  !(cfg->original_context > 0) || !std::isfinite(cfg->original_context)))
        return KVX_EINVAL;
    if (kind == KVX_ROPE_YARN && !(cfg->base > 1)) return KVX_EINVAL;
    constexpr double two_pi = 6.283185307179586476925286766559;
    double base = cfg->base;
    if (kind == KVX_ROPE_NTK && d > 2) base *= std::pow(factor, (double)d / (d - 2));
    double first = 0, last = 0;  // YaRN: pairs the ramp runs between
    if (kind == KVX_ROPE_YARN) {
        auto pair_of = [&](double n) { return d * std::log(cfg->original_context / (n * two_pi)) / (2 * std::log(base)); };
        first = std::max(std::floor(pair_of(cfg->high)), 0.0);
        last = std::min(std::ceil(pair_of(cfg->low)), (double)(d - 1));
    }
    for (int i = 0; i < d / 2; ++i) {
        double f = std::pow(base, -2.0 * i / d);
        if (kind == KVX_ROPE_LINEAR) f /= factor;
        if (kind == KVX_ROPE_LLAMA3) {
            const double mix = (cfg->original_context * f / two_pi - cfg->low) / (cfg->high - cfg->low);
            const double m = std::min(std::max(mix, 0.0), 1.0);
            f = (1 - m) * f / factor + m * f;
        }
        if (kind == KVX_ROPE_YARN) {
            const double r = std::min(std::max((i - first) / std::max(last - first, 0.001), 0.0), 1.0);
            f = f * (1 - r) + f / factor * r;
        }
        // fraction of a turn in units of 2^-64 (whole turns drop out at every
        // integer position)
        const long double turn = (long double)f / 6.283185307179586476925286766559L;
        const long double frac = turn - std::floor(turn);
        const long double units = std::floor(frac * 18446744073709551616.0L + 0.5L);
        turns[i] = units >= 18446744073709551616.0L ? 0 : (uint64_t)units;
    }
    *amplitude = kind == KVX_ROPE_YARN ? (float)(0.1 * std::log(factor) + 1.0) : 1.0f;
    return KVX_OK;
}

extern "C" KVX_API int kvx_rope(const kvx_rope_table *table, const int32_t *positions, int32_t tokens,
                                int32_t head_dim, int32_t dtype, const kvx_rope_rows *rows, int32_t num_rows,
                                int32_t inverse, void *stream) {
    if (!table || !rows || num_rows < 1 || num_rows > 2 || tokens < 0 || head_dim <= 0) return KVX_EINVAL;
    if (inverse != 0 && inverse != 1) return KVX_EINVAL;
    if (dtype != KVX_F16 && dtype != KVX_F32) return KVX_EUNSUPPORTED;
    if (head_dim > kMaxRopeDim) return KVX_EUNSUPPORTED;
    if (!table_ok(table, head_dim)) return KVX_EINVAL;
    const int size = dtype == KVX_F16 ? 2 : 4;
    const bool half = table->layout == KVX_ROPE_HALF;
    RopeParams p{};
    int64_t total = 0;
    bool vec = rope_vector_sizes(head_dim, table->rotary_dim, half, 16 / size);
    for (int i = 0; i < num_rows; ++i) {
        const kvx_rope_rows &r = rows[i];
        if (r.heads < 0 || r.heads > (1 << 20)) return KVX_EINVAL;
        if (r.heads == 0 || tokens == 0) continue;
        if (!r.in || !r.out) return KVX_EINVAL;
        if (r.in == r.out && (r.in_token_stride != r.out_token_stride || r.in_head_stride != r.out_head_stride))
            return KVX_EINVAL;
        const uintptr_t at = reinterpret_cast<uintptr_t>(r.in) | reinterpret_cast<uintptr_t>(r.out);
        const int64_t strides = r.in_token_stride | r.in_head_stride | r.out_token_stride | r.out_head_stride;
        if (at & (size - 1)) return KVX_EINVAL;
        if ((at & 15) || ((strides * size) & 15)) vec = false;
        p.x[i] = {r.in, r.out, r.heads, r.in_token_stride, r.in_head_stride, r.out_token_stride, r.out_head_stride};
        total += r.heads;
    }
    if (total == 0 || tokens == 0) return KVX_OK;
    if (!positions) return KVX_EINVAL;
    p.turns = table->turns;
    p.positions = positions;
    p.rotary = table->rotary_dim;
    p.items = rope_items(head_dim, table->rotary_dim, half, vec ? 16 / size : 1);
    p.amplitude = table->amplitude;
    p.sine_sign = inverse ? -1.f : 1.f;
    // as many threads as one token's rows have items, 256 at most (beyond
    // that a row has to fit: scalar rows of up to 1024 items)
    const int64_t want = std::max<int64_t>(p.items, std::min<int64_t>(total * p.items, kRopeThreads));
    const int threads = (int)((want + 31) / 32 * 32);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    return dtype == KVX_F16 ? launch_rope<__half>(p, tokens, threads, half, vec, st)
                            : launch_rope<float>(p, tokens, threads, half, vec, st);
}

extern "C" KVX_API int kvx_rope_append(const kvx_paged *kv, const int32_t *block_table, int32_t max_pages,
                                       const int32_t *q_start, const int32_t *positions, int32_t batch,
                                       int32_t total_tokens, const kvx_rope_table *table, int32_t io_dtype,
                                       const void *q, int64_t q_stride, void *q_out, int32_t num_q_heads,
                                       const void *k, int64_t k_stride, const void *v, int64_t v_stride,
                                       int32_t *error_flag, void *stream) {
    if (!kv || !kv->pool || !block_table || !q_start || !positions) return KVX_EINVAL;
    if (batch < 0 || total_tokens < 0 || max_pages <= 0 || kv->num_kv_heads <= 0 || kv->num_pages <= 0 ||
        num_q_heads < 0)
        return KVX_EINVAL;
    if (kv->dtype != KVX_F32 && kv->dtype != KVX_F16 && kv->dtype != KVX_I8) return KVX_EINVAL;
    if (kv->page_tokens != kPageTokens || kv->head_dim != kHeadDim) return KVX_EUNSUPPORTED;
    if (io_dtype != KVX_F16 && io_dtype != KVX_F32) return KVX_EINVAL;
    const bool i8 = kv->dtype == KVX_I8;
    if (!i8 && io_dtype != kv->dtype) return KVX_EUNSUPPORTED;
    if (i8 && !kv->stats) return KVX_EINVAL;
    if (kv->num_kv_heads > (1 << 16) || num_q_heads > (1 << 16)) return KVX_EUNSUPPORTED;
    if (table && !table_ok(table, kHeadDim)) return KVX_EINVAL;
    if (batch == 0 || total_tokens == 0) return KVX_OK;
    if (!k || !v || (num_q_heads > 0 && (!q || !q_out))) return KVX_EINVAL;
    const int size = io_dtype == KVX_F16 ? 2 : 4;
    if (k_stride < (int64_t)kv->num_kv_heads * kHeadDim || v_stride < (int64_t)kv->num_kv_heads * kHeadDim ||
        (num_q_heads > 0 && q_stride < (int64_t)num_q_heads * kHeadDim))
        return KVX_EINVAL;
    if (num_q_heads > 0 && q == q_out && q_stride != (int64_t)num_q_heads * kHeadDim) return KVX_EINVAL;
    const int64_t strides = k_stride | v_stride | (num_q_heads > 0 ? q_stride : 0);
    if (((reinterpret_cast<uintptr_t>(kv->pool) | reinterpret_cast<uintptr_t>(kv->stats) | reinterpret_cast<uintptr_t>(k) |
          reinterpret_cast<uintptr_t>(v) | (num_q_heads > 0 ? reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(q_out) : 0)) &
         15) ||
        ((strides * size) & 15))
        return KVX_EINVAL;
    RopeAppendParams p{};
    p.pool = static_cast<uint8_t *>(kv->pool);
    p.stats = const_cast<float *>(kv->stats);
    p.block_table = block_table;
    p.q_start = q_start;
    p.positions = positions;
    p.error_flag = error_flag;
    p.turns = table ? table->turns : nullptr;
    p.q = q, p.k = k, p.v = v, p.q_out = q_out;
    p.q_stride = q_stride, p.k_stride = k_stride, p.v_stride = v_stride;
    p.batch = batch, p.total = total_tokens, p.hq = num_q_heads, p.hkv = kv->num_kv_heads;
    p.max_pages = max_pages, p.num_pages = kv->num_pages;
    const int e = 16 / size;
    p.rotary = table ? table->rotary_dim : 2 * e;
    const bool half = table && table->layout == KVX_ROPE_HALF;
    const bool vec = rope_vector_sizes(kHeadDim, p.rotary, half, e);
    p.items = rope_items(kHeadDim, p.rotary, half, vec ? e : 1);
    p.amplitude = table ? table->amplitude : 1.f;
    // 16 tokens a CTA once their pages alone fill the SMs
    p.tokens_per_block = total_tokens >= kPageTokens * sm_count() ? kPageTokens : 1;
    p.kv_blocks = (total_tokens + p.tokens_per_block - 1) / p.tokens_per_block * 2;
    p.apart = p.hq > 0 && p.tokens_per_block > 1;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    return io_dtype == KVX_F16 ? launch_rope_append<__half>(p, i8, half, vec, st)
                               : launch_rope_append<float>(p, i8, half, vec, st);
}
