// kvx_pages.cu -- who holds which page: reserve, fork, free, compact, copy.
//
// The decisions (which free pages, in which order) come from one CTA of
// 1024 threads that scans the reference counts 16,384 at a time, so they are
// the same on every run; what has many bytes or many entries (block-table
// rows, page contents in every layer) is done by a second launch of the whole
// GPU that reads the first one's lists (a programmatic dependent: its CTAs
// are placed while the plan runs).  Compaction of 6000 pages, 2000 of them
// held, 4 fp16 layers: 127 us for 699 MB (5.5 TB/s, 0.85 of the measured copy
// rate).  A fork of 4 rows, a reserve and a free, 28 int8 layers: 16 us, a chain
// of launches and of dependent reads in one CTA.
#include <algorithm>

#include "kvx_common.cuh"
#include "kvx_decode_params.cuh"  // grid_dependents_launch, grid_dependency_wait

namespace kvx {
namespace {

constexpr int kPlanThreads = 1024;
constexpr int kScanPer = 16;  // pages a thread looks at per step of a scan
constexpr int kMostEntries = 0x7fffffff - 2 * kPlanThreads * kScanPer;
constexpr int kErrRange = 2, kErrLong = 4, kErrPages = 8, kErrRows = 16;

// Workspace: header, then the lists.
struct PlanHeader {
    int32_t count;  // pairs in (src, dst): pages to copy
    int32_t ok;     // the call was accepted
};
struct PlanSpace {
    PlanHeader *head;
    int32_t *src, *dst;  // [num_pages]: copies; reserve and fork: src doubles as the list of pages taken
    int32_t *map;        // [num_pages]: compact: new id of a page; fork: pages taken
    int32_t *rows_a, *rows_b;  // [num_rows]
};
constexpr size_t kHeadBytes = 64;

size_t space_bytes(int num_pages, int num_rows) {
    return kHeadBytes + ((size_t)num_pages * 3 + (size_t)num_rows * 2) * sizeof(int32_t);
}
PlanSpace plan_space(void *w, int num_pages, int num_rows) {
    PlanSpace s;
    s.head = static_cast<PlanHeader *>(w);
    s.src = reinterpret_cast<int32_t *>(static_cast<uint8_t *>(w) + kHeadBytes);
    s.dst = s.src + num_pages;
    s.map = s.dst + num_pages;
    s.rows_a = s.map + num_pages;
    s.rows_b = s.rows_a + num_rows;
    return s;
}

// Pages of len tokens (len >= 0, up to the largest int).
__device__ __forceinline__ int pages_of(int len) { return len / kPageTokens + (len % kPageTokens != 0); }

// Exclusive prefix sum over the CTA's threads in thread order; *total gets
// the sum.  red: 33 ints of shared memory.
__device__ __forceinline__ int cta_prefix(int v, int *red, int *total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int x = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, x, o);
        if (lane >= o) x += y;
    }
    __syncthreads();  // red is free
    if (lane == 31) red[warp] = x;
    __syncthreads();
    if (warp == 0) {
        int s = lane < (int)(blockDim.x >> 5) ? red[lane] : 0;
        const int mine = s;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int y = __shfl_up_sync(0xffffffffu, s, o);
            if (lane >= o) s += y;
        }
        red[lane] = s - mine;
        if (lane == 31) red[32] = s;
    }
    __syncthreads();
    *total = red[32];
    return red[warp] + x - v;
}

// Bit i: page base + i is free (the thread's kScanPer pages).
__device__ __forceinline__ uint32_t free_bits(const int32_t *refs, int base, int num_pages) {
    uint32_t bits = 0;
    if (base + kScanPer <= num_pages && !(reinterpret_cast<uintptr_t>(refs) & 15)) {
        int4 v[kScanPer / 4];
#pragma unroll
        for (int j = 0; j < kScanPer / 4; ++j) v[j] = reinterpret_cast<const int4 *>(refs + base)[j];
#pragma unroll
        for (int j = 0; j < kScanPer / 4; ++j)
            bits |= ((v[j].x <= 0 ? 1u : 0u) | (v[j].y <= 0 ? 2u : 0u) | (v[j].z <= 0 ? 4u : 0u) | (v[j].w <= 0 ? 8u : 0u)) << (4 * j);
    } else {
        for (int j = 0; j < kScanPer; ++j)
            if (base + j < num_pages && refs[base + j] <= 0) bits |= 1u << j;
    }
    return bits;
}

// The lowest `need` free pages, ascending, into list; returns how many there
// are (< need: all of them).  Stops once it has enough.
__device__ int take_free(const int32_t *refs, int num_pages, int need, int32_t *list, int *red) {
    int have = 0;
    for (int at = 0; at < num_pages && have < need; at += kPlanThreads * kScanPer) {
        const int base = at + threadIdx.x * kScanPer;
        uint32_t bits = base < num_pages ? free_bits(refs, base, num_pages) : 0;
        int total, rank = have + cta_prefix(__popc(bits), red, &total);
        for (; bits && rank < need; bits &= bits - 1) list[rank++] = base + __ffs(bits) - 1;
        have += total;
    }
    return min(have, need);
}

__global__ void __launch_bounds__(kPlanThreads)
reserve_kernel(const kvx_pages t, const int32_t *new_tokens, PlanSpace w, int32_t *error_flag) {
    __shared__ int red[33], s_bad;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    if (threadIdx.x == 0) s_bad = 0;
    __syncthreads();
    // a warp per row: how many entries it lacks
    int bad = 0;
    for (int r = warp; r < t.num_rows; r += kPlanThreads / 32) {
        const int len = t.seq_lens[r], grow = new_tokens[r];
        int lack = 0;
        if (len < 0 || grow < 0) {
            bad = kErrRange;
        } else {
            const long long want = ((long long)len + grow + kPageTokens - 1) / kPageTokens;
            if (want > t.max_pages) {
                bad = kErrLong;
            } else {
                const int32_t *row = t.block_table + (size_t)r * t.max_pages;
                for (int lp = pages_of(len) + lane; lp < want; lp += 32) lack += row[lp] < 0;
            }
        }
        lack = __reduce_add_sync(0xffffffffu, lack);
        if (lane == 0) w.rows_a[r] = lack;
    }
    if (bad && lane == 0) atomicOr(&s_bad, bad);
    __syncthreads();
    // where each row's pages begin in the list of pages taken
    int need = 0;
    for (int at = 0; at < t.num_rows; at += kPlanThreads) {
        const int r = at + threadIdx.x;
        const int lack = r < t.num_rows ? w.rows_a[r] : 0;
        int total;
        const int before = cta_prefix(lack, red, &total);
        if (r < t.num_rows) w.rows_b[r] = need + before;
        need = (int)min((long long)need + total, 0x7fffffffll);
    }
    if (!s_bad && need > t.num_pages) {
        if (threadIdx.x == 0) s_bad = kErrPages;
    }
    __syncthreads();
    if (!s_bad && need > 0 && take_free(t.refcounts, t.num_pages, need, w.src, red) < need) {
        __syncthreads();
        if (threadIdx.x == 0) s_bad = kErrPages;
    }
    __syncthreads();
    if (s_bad) {
        if (error_flag && threadIdx.x == 0) atomicOr(error_flag, s_bad);
        return;
    }
    for (int r = warp; r < t.num_rows; r += kPlanThreads / 32) {
        const int len = t.seq_lens[r];
        const int want = (int)(((long long)len + new_tokens[r] + kPageTokens - 1) / kPageTokens);
        int32_t *row = t.block_table + (size_t)r * t.max_pages;
        int next = w.rows_b[r];
        for (int lp0 = pages_of(len); lp0 < want; lp0 += 32) {
            const int lp = lp0 + lane;
            const bool lacks = lp < want && row[lp] < 0;
            const uint32_t mask = __ballot_sync(0xffffffffu, lacks);
            if (lacks) {
                const int page = w.src[next + __popc(mask & ((1u << lane) - 1))];
                row[lp] = page;
                t.refcounts[page] = 1;
            }
            next += __popc(mask);
        }
    }
}

// Check a fork, choose the children's own last pages and list the copies:
// pair i of (src, dst) is the last page of fork rows_a[i].
__global__ void __launch_bounds__(kPlanThreads)
fork_plan_kernel(const kvx_pages t, const int32_t *parents, const int32_t *children, int n, PlanSpace w,
                 int32_t *error_flag) {
    __shared__ int red[33], s_bad;
    grid_dependents_launch();
    if (threadIdx.x == 0) s_bad = 0;
    for (int r = threadIdx.x; r < t.num_rows; r += kPlanThreads) w.rows_b[r] = 0;  // 1: somebody's child
    __syncthreads();
    int bad = 0;
    for (int i = threadIdx.x; i < n; i += kPlanThreads) {
        const int a = parents[i], b = children[i];
        if (a < 0 || a >= t.num_rows || b < 0 || b >= t.num_rows) {
            bad |= kErrRange;
            continue;
        }
        if (atomicExch(&w.rows_b[b], 1) || t.seq_lens[b] != 0 || t.block_table[(size_t)b * t.max_pages] >= 0)
            bad |= kErrRows;
    }
    __syncthreads();
    int need = 0;
    for (int at = 0; at < n; at += kPlanThreads) {
        const int i = at + threadIdx.x;
        int tail = 0;
        if (i < n) {
            const int a = parents[i];
            if (a >= 0 && a < t.num_rows) {
                const int len = t.seq_lens[a];
                if (__ldcg(&w.rows_b[a])) bad |= kErrRows;  // a child of this call as a parent
                if (len < 0) {
                    bad |= kErrRange;
                } else if (pages_of(len) > t.max_pages) {
                    bad |= kErrLong;
                } else if (len % kPageTokens) {
                    const int page = t.block_table[(size_t)a * t.max_pages + len / kPageTokens];
                    if (page < 0 || page >= t.num_pages)
                        bad |= kErrRange;
                    else
                        tail = 1;
                }
            }
        }
        int total;
        const int rank = need + cta_prefix(tail, red, &total);
        if (tail && rank < t.num_pages) {
            const int a = parents[i], len = t.seq_lens[a];
            w.src[rank] = t.block_table[(size_t)a * t.max_pages + len / kPageTokens];
            w.map[rank] = i;
        }
        need += total;
    }
    if (bad) atomicOr(&s_bad, bad);
    __syncthreads();
    if (!s_bad && need > 0 && (need > t.num_pages || take_free(t.refcounts, t.num_pages, need, w.dst, red) < need)) {
        __syncthreads();
        if (threadIdx.x == 0) s_bad = kErrPages;
    }
    __syncthreads();
    if (threadIdx.x == 0) {
        if (s_bad && error_flag) atomicOr(error_flag, s_bad);
        w.head->count = s_bad ? 0 : need;
        w.head->ok = !s_bad;
    }
}

// ---- page contents

constexpr int kCopyThreads = 256;
constexpr int kCopyVecs = 8;                              // 16-byte vectors a thread moves per unit
constexpr int kUnitBytes = kCopyThreads * kCopyVecs * 16;  // 32 KB
constexpr int kMaxLayers = 128;                           // pointers a launch carries

struct CopyLayers {
    uint8_t *pool[kMaxLayers];
    uint8_t *stats[kMaxLayers];  // int8 pools
    int num_layers, page_bytes, stats_bytes, units, num_pages;  // units: of kUnitBytes (the last partial) a page
};

__device__ __forceinline__ void copy_span(uint8_t *dst, const uint8_t *src, int bytes) {
    const int vecs = bytes / 16;
    uint4 v[kCopyVecs];
#pragma unroll
    for (int j = 0; j < kCopyVecs; ++j) {
        const int i = j * kCopyThreads + threadIdx.x;
        if (i < vecs) v[j] = __ldcs(reinterpret_cast<const uint4 *>(src) + i);
    }
#pragma unroll
    for (int j = 0; j < kCopyVecs; ++j) {
        const int i = j * kCopyThreads + threadIdx.x;
        if (i < vecs) __stcs(reinterpret_cast<uint4 *>(dst) + i, v[j]);
    }
}

// CTA `cta` of `ctas`: its share of count x layers x units, layer-major, so
// that the CTAs at work together stay within a layer or two.
__device__ __forceinline__ void copy_pages(const CopyLayers &c, const int32_t *src, const int32_t *dst, int count, int cta,
                                           int ctas, int32_t *error_flag) {
    const long long total = (long long)count * c.num_layers * c.units;
    for (long long u = cta; u < total; u += ctas) {
        const int unit = (int)(u % c.units);
        const long long pl = u / c.units;
        const int pair = (int)(pl % count), layer = (int)(pl / count);
        const int a = src[pair], b = dst[pair];
        if (a < 0 || a >= c.num_pages || b < 0 || b >= c.num_pages) {
            if (error_flag && threadIdx.x == 0 && unit == 0 && layer == 0) atomicOr(error_flag, kErrRange);
            continue;
        }
        if (a == b) continue;
        const size_t off = (size_t)unit * kUnitBytes;
        const int bytes = min(kUnitBytes, c.page_bytes - unit * kUnitBytes);
        copy_span(c.pool[layer] + (size_t)b * c.page_bytes + off, c.pool[layer] + (size_t)a * c.page_bytes + off, bytes);
        if (c.stats_bytes && unit == 0) {
            const uint4 *s = reinterpret_cast<const uint4 *>(c.stats[layer] + (size_t)a * c.stats_bytes);
            uint4 *d = reinterpret_cast<uint4 *>(c.stats[layer] + (size_t)b * c.stats_bytes);
            for (int i = threadIdx.x; i < c.stats_bytes / 16; i += kCopyThreads) d[i] = s[i];
        }
    }
}

__global__ void __launch_bounds__(kCopyThreads)
copy_kernel(const __grid_constant__ CopyLayers c, const int32_t *src, const int32_t *dst, int count, int32_t *error_flag) {
    copy_pages(c, src, dst, count, blockIdx.x, gridDim.x, error_flag);
}

// Table rows and counts (the first CTAs), then the page copies.
__global__ void __launch_bounds__(kCopyThreads)
fork_apply_kernel(const kvx_pages t, const int32_t *parents, const int32_t *children, int n, PlanSpace w,
                  const __grid_constant__ CopyLayers c, int first_layers, int32_t *error_flag) {
    grid_dependency_wait();
    if (!w.head->ok) return;
    const int count = w.head->count;
    if (first_layers) {
        // shared pages; the child's own last page comes from the loop below
        for (int i = blockIdx.x; i < n; i += gridDim.x) {
            const int a = parents[i], b = children[i], len = t.seq_lens[a], full = len / kPageTokens;
            const int32_t *from = t.block_table + (size_t)a * t.max_pages;
            int32_t *to = t.block_table + (size_t)b * t.max_pages;
            for (int lp = threadIdx.x; lp < full; lp += kCopyThreads) {
                const int page = from[lp];
                const bool known = page >= 0 && page < t.num_pages;
                to[lp] = known ? page : -1;
                if (known)
                    atomicAdd(&t.refcounts[page], 1);
                else if (error_flag)
                    atomicOr(error_flag, kErrRange);
            }
            if (threadIdx.x == 0) t.seq_lens[b] = len;
        }
        for (int i = blockIdx.x * kCopyThreads + threadIdx.x; i < count; i += gridDim.x * kCopyThreads) {
            const int f = w.map[i], page = w.dst[i];
            t.block_table[(size_t)children[f] * t.max_pages + t.seq_lens[parents[f]] / kPageTokens] = page;
            t.refcounts[page] = 1;
        }
    }
    copy_pages(c, w.src, w.dst, count, blockIdx.x, gridDim.x, nullptr);
}

__global__ void __launch_bounds__(256) free_kernel(const kvx_pages t, const int32_t *rows, int n, int32_t *error_flag) {
    for (int i = blockIdx.x; i < n; i += gridDim.x) {
        const int r = rows[i];
        if (r < 0 || r >= t.num_rows) {
            if (error_flag && threadIdx.x == 0) atomicOr(error_flag, kErrRange);
            continue;
        }
        int32_t *row = t.block_table + (size_t)r * t.max_pages;
        for (int lp = threadIdx.x; lp < t.max_pages; lp += blockDim.x) {
            if (row[lp] < 0) continue;
            const int page = atomicExch(&row[lp], -1);  // one of the CTAs that were given this row gets it
            if (page < 0) continue;
            if (page >= t.num_pages || atomicSub(&t.refcounts[page], 1) <= 0) {
                if (page < t.num_pages) atomicAdd(&t.refcounts[page], 1);
                if (error_flag) atomicOr(error_flag, kErrRange);
            }
        }
        if (threadIdx.x == 0) t.seq_lens[r] = 0;
    }
}

__global__ void __launch_bounds__(kPlanThreads) compact_plan_kernel(const kvx_pages t, PlanSpace w, int32_t *num_live) {
    __shared__ int red[33];
    grid_dependents_launch();
    int live = 0;
    for (int at = 0; at < t.num_pages; at += kPlanThreads * kScanPer) {
        const int base = at + threadIdx.x * kScanPer;
        int total;
        const int inside = base < t.num_pages ? min(kScanPer, t.num_pages - base) : 0;
        cta_prefix(inside ? inside - __popc(free_bits(t.refcounts, base, t.num_pages)) : 0, red, &total);
        live += total;
    }
    int holes = 0, moving = 0;
    for (int at = 0; at < t.num_pages; at += kPlanThreads * kScanPer) {
        const int base = at + threadIdx.x * kScanPer;
        const int inside = base < t.num_pages ? min(kScanPer, t.num_pages - base) : 0;
        const uint32_t valid = (1u << inside) - 1u;
        const uint32_t low = base >= live ? 0u : (live - base >= 32 ? ~0u : (1u << (live - base)) - 1u);  // ids below live
        const uint32_t empty = inside ? free_bits(t.refcounts, base, t.num_pages) : 0;
        uint32_t hole = empty & low & valid, move = ~empty & ~low & valid;
        int total;
        int rank = holes + cta_prefix(__popc(hole), red, &total);
        holes += total;
        for (; hole; hole &= hole - 1) w.dst[rank++] = base + __ffs(hole) - 1;
        rank = moving + cta_prefix(__popc(move), red, &total);
        moving += total;
        for (; move; move &= move - 1) w.src[rank++] = base + __ffs(move) - 1;
        for (int j = 0; j < inside; ++j) w.map[base + j] = empty >> j & 1 ? -1 : base + j;
    }
    __syncthreads();
    for (int i = threadIdx.x; i < moving; i += kPlanThreads) {  // as many holes as pages behind them
        const int a = w.src[i], b = w.dst[i];
        w.map[a] = b;
        t.refcounts[b] = t.refcounts[a];
        t.refcounts[a] = 0;
    }
    if (threadIdx.x == 0) {
        w.head->count = moving;
        w.head->ok = 1;
        if (num_live) *num_live = live;
    }
}

__global__ void __launch_bounds__(kCopyThreads)
compact_apply_kernel(const kvx_pages t, PlanSpace w, const __grid_constant__ CopyLayers c, int first_layers,
                     int32_t *error_flag) {
    grid_dependency_wait();
    if (first_layers) {
        const size_t entries = (size_t)t.num_rows * t.max_pages;
        for (size_t e = blockIdx.x * (size_t)kCopyThreads + threadIdx.x; e < entries; e += (size_t)gridDim.x * kCopyThreads) {
            const int page = t.block_table[e];
            if (page < 0) continue;
            const int to = page < t.num_pages ? w.map[page] : -1;
            if (to < 0) {
                if (error_flag) atomicOr(error_flag, kErrRange);
            } else if (to != page) {
                t.block_table[e] = to;
            }
        }
    }
    copy_pages(c, w.src, w.dst, w.head->count, blockIdx.x, gridDim.x, nullptr);
}

// ---- host

int pages_status(const kvx_pages *t) {
    if (!t || !t->refcounts || !t->block_table || !t->seq_lens) return KVX_EINVAL;
    if (t->num_pages <= 0 || t->num_rows <= 0 || t->max_pages <= 0) return KVX_EINVAL;
    // sums of entries, and the steps of the loops over pages and entries, fit an int
    if ((long long)t->num_rows * t->max_pages > kMostEntries || t->num_pages > kMostEntries) return KVX_EUNSUPPORTED;
    if ((reinterpret_cast<uintptr_t>(t->refcounts) | reinterpret_cast<uintptr_t>(t->block_table) |
         reinterpret_cast<uintptr_t>(t->seq_lens)) & 3)
        return KVX_EINVAL;
    return KVX_OK;
}

int space_status(const kvx_pages *t, const void *w, size_t bytes) {
    if (!w || bytes < space_bytes(t->num_pages, t->num_rows)) return KVX_ENOSPC;
    return reinterpret_cast<uintptr_t>(w) & 15 ? KVX_EINVAL : KVX_OK;
}

int element_bytes(int dtype) { return dtype == KVX_F32 ? 4 : (dtype == KVX_F16 ? 2 : 1); }

int layers_status(const kvx_paged *layers, int num_layers) {
    if (!layers || num_layers <= 0) return KVX_EINVAL;
    const kvx_paged &a = layers[0];
    if (a.dtype != KVX_F32 && a.dtype != KVX_F16 && a.dtype != KVX_I8) return KVX_EINVAL;
    if (a.num_pages <= 0 || a.num_kv_heads <= 0 || a.page_tokens <= 0 || a.head_dim <= 0) return KVX_EINVAL;
    const long long page = 2LL * a.num_kv_heads * a.page_tokens * a.head_dim * element_bytes(a.dtype);
    if (page % 16 || page > (1LL << 30)) return KVX_EUNSUPPORTED;
    for (int l = 0; l < num_layers; ++l) {
        const kvx_paged &b = layers[l];
        if (!b.pool || (reinterpret_cast<uintptr_t>(b.pool) & 15)) return KVX_EINVAL;
        if (b.dtype != a.dtype || b.num_pages != a.num_pages || b.num_kv_heads != a.num_kv_heads ||
            b.page_tokens != a.page_tokens || b.head_dim != a.head_dim)
            return KVX_EINVAL;
        if (a.dtype == KVX_I8 && (!b.stats || (reinterpret_cast<uintptr_t>(b.stats) & 15))) return KVX_EINVAL;
    }
    return KVX_OK;
}

CopyLayers copy_layers(const kvx_paged *layers, int from, int num_layers) {
    CopyLayers c{};
    const kvx_paged &a = layers[0];
    c.num_layers = std::min(kMaxLayers, num_layers - from);
    c.page_bytes = 2 * a.num_kv_heads * a.page_tokens * a.head_dim * element_bytes(a.dtype);
    c.stats_bytes = a.dtype == KVX_I8 ? 2 * a.num_kv_heads * 16 : 0;
    c.units = (c.page_bytes + kUnitBytes - 1) / kUnitBytes;
    c.num_pages = a.num_pages;
    for (int l = 0; l < c.num_layers; ++l) {
        c.pool[l] = static_cast<uint8_t *>(layers[from + l].pool);
        c.stats[l] = reinterpret_cast<uint8_t *>(const_cast<float *>(layers[from + l].stats));
    }
    return c;
}

// CTAs for a copy whose length only the device knows: `most` units at most,
// and no more than are resident together.
unsigned copy_grid(long long most) { return (unsigned)std::max<long long>(1, std::min<long long>(most, (long long)sm_count() * 6)); }

template <typename... P, typename... A>
int launch_dependent(void (*kern)(P...), unsigned grid, int threads, cudaStream_t st, A... args) {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(grid);
    cfg.blockDim = dim3(threads);
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    if (cudaLaunchKernelEx(&cfg, kern, args...) != cudaSuccess) {
        cudaGetLastError();
        return KVX_ECUDA;
    }
    return launch_status();
}

}  // namespace
}  // namespace kvx

using namespace kvx;

extern "C" KVX_API size_t kvx_pages_workspace_bytes(int32_t num_pages, int32_t num_rows) {
    if (num_pages <= 0 || num_rows <= 0) return 0;
    return (space_bytes(num_pages, num_rows) + 15) / 16 * 16;
}

extern "C" KVX_API int kvx_pages_reserve(const kvx_pages *pages, const int32_t *new_tokens, void *workspace,
                                         size_t workspace_bytes, int32_t *error_flag, void *stream) {
    int rc = pages_status(pages);
    if (rc != KVX_OK) return rc;
    if (!new_tokens) return KVX_EINVAL;
    if ((rc = space_status(pages, workspace, workspace_bytes)) != KVX_OK) return rc;
    reserve_kernel<<<1, kPlanThreads, 0, static_cast<cudaStream_t>(stream)>>>(
        *pages, new_tokens, plan_space(workspace, pages->num_pages, pages->num_rows), error_flag);
    return launch_status();
}

extern "C" KVX_API int kvx_pages_fork(const kvx_pages *pages, const kvx_paged *layers, int32_t num_layers,
                                      const int32_t *parents, const int32_t *children, int32_t n, void *workspace,
                                      size_t workspace_bytes, int32_t *error_flag, void *stream) {
    int rc = pages_status(pages);
    if (rc != KVX_OK) return rc;
    if ((rc = layers_status(layers, num_layers)) != KVX_OK) return rc;
    if (n < 0 || n > pages->num_rows || layers[0].num_pages != pages->num_pages) return KVX_EINVAL;
    if (layers[0].page_tokens != kPageTokens) return KVX_EUNSUPPORTED;
    if (n == 0) return KVX_OK;
    if (!parents || !children) return KVX_EINVAL;
    if ((rc = space_status(pages, workspace, workspace_bytes)) != KVX_OK) return rc;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    const PlanSpace w = plan_space(workspace, pages->num_pages, pages->num_rows);
    fork_plan_kernel<<<1, kPlanThreads, 0, st>>>(*pages, parents, children, n, w, error_flag);
    rc = launch_status();
    for (int from = 0; from < num_layers && rc == KVX_OK; from += kMaxLayers) {
        const CopyLayers c = copy_layers(layers, from, num_layers);
        rc = launch_dependent(fork_apply_kernel, copy_grid((long long)n * c.num_layers * c.units), kCopyThreads, st, *pages,
                              parents, children, n, w, c, from == 0 ? 1 : 0, error_flag);
    }
    return rc;
}

extern "C" KVX_API int kvx_pages_free(const kvx_pages *pages, const int32_t *rows, int32_t n, int32_t *error_flag,
                                      void *stream) {
    const int rc = pages_status(pages);
    if (rc != KVX_OK) return rc;
    if (n < 0) return KVX_EINVAL;
    if (n > kMostEntries) return KVX_EUNSUPPORTED;
    if (n == 0) return KVX_OK;
    if (!rows) return KVX_EINVAL;
    free_kernel<<<(unsigned)std::min<long long>(n, (long long)sm_count() * 8), 256, 0, static_cast<cudaStream_t>(stream)>>>(
        *pages, rows, n, error_flag);
    return launch_status();
}

extern "C" KVX_API int kvx_pages_compact(const kvx_pages *pages, const kvx_paged *layers, int32_t num_layers,
                                         void *workspace, size_t workspace_bytes, int32_t *num_live, int32_t *error_flag,
                                         void *stream) {
    int rc = pages_status(pages);
    if (rc != KVX_OK) return rc;
    if ((rc = layers_status(layers, num_layers)) != KVX_OK) return rc;
    if (layers[0].num_pages != pages->num_pages) return KVX_EINVAL;
    if ((rc = space_status(pages, workspace, workspace_bytes)) != KVX_OK) return rc;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    const PlanSpace w = plan_space(workspace, pages->num_pages, pages->num_rows);
    compact_plan_kernel<<<1, kPlanThreads, 0, st>>>(*pages, w, num_live);
    rc = launch_status();
    for (int from = 0; from < num_layers && rc == KVX_OK; from += kMaxLayers) {
        const CopyLayers c = copy_layers(layers, from, num_layers);
        rc = launch_dependent(compact_apply_kernel, copy_grid((long long)pages->num_pages * c.num_layers * c.units),
                              kCopyThreads, st, *pages, w, c, from == 0 ? 1 : 0, error_flag);
    }
    return rc;
}

extern "C" KVX_API int kvx_pages_copy(const kvx_paged *layers, int32_t num_layers, const int32_t *src,
                                      const int32_t *dst, int32_t n, int32_t *error_flag, void *stream) {
    int rc = layers_status(layers, num_layers);
    if (rc != KVX_OK) return rc;
    if (n < 0) return KVX_EINVAL;
    if (n == 0) return KVX_OK;
    if (!src || !dst) return KVX_EINVAL;
    for (int from = 0; from < num_layers && rc == KVX_OK; from += kMaxLayers) {
        const CopyLayers c = copy_layers(layers, from, num_layers);
        copy_kernel<<<copy_grid((long long)n * c.num_layers * c.units), kCopyThreads, 0, static_cast<cudaStream_t>(stream)>>>(
            c, src, dst, n, from == 0 ? error_flag : nullptr);
        rc = launch_status();
    }
    return rc;
}
