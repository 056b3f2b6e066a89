// kvx_chunk.cu -- attention of several new tokens per sequence over int8
// pages (kvx_attend_chunk), on the 5th-generation tensor cores.
//
// With x = zp + (c + 128) s for every block of 16 tokens x 128 dims and
// mid = zp + 128 s, the codes c enter the products as they are (exact in
// fp16) and the block's statistics are applied around them:
//     q . k = s (q . c) + mid sum(q)
//     sum_t p_t v_t = sum_t (p_t s_t) c_t + sum_t p_t mid_t
// so a score costs one multiply-add on the accumulator, and the second sum is
// one scalar per row.
//
// Rows: the new tokens of a sequence times the q-heads of a kv-head, token
// major.  A CTA owns a tile of rows and a range of 128-key tiles (8 pages):
//  * loader warp: a bulk copy (TMA) per page and K|V, 2 KB of codes each, into
//    staging slots;
//  * 8 convert warps (4 for K, 4 for V): codes -> fp16 into the 128-byte-swizzled K and V tiles
//    (K: the K-major B operand of Q K^T; V: the MN-major B operand of P V,
//    the same bytes), two stages each;
//  * MMA warp: one thread issues S = Q K^T (M 128, N 128, 8 steps of K 16)
//    and O += P V with P read from tensor memory;
//  * 2 softmax warpgroups, a thread per row: running maximum and sum in
//    registers, P (fp16) written over the columns of S it came from; O stays in
//    tensor memory and is rescaled only when a row's maximum has grown by
//    more than 2^8 (p <= 2^8 until then).
// The two warpgroups have an S and an O each (512 tensor-memory columns in
// all), so one's MMAs run under the other's exponentials.  With more than 128
// rows they own 128 rows each and share every key tile; up to 128 rows they
// take turns at the key tiles of the same rows and are merged at the end.
//
// fp16 calls: P' = p s 2^(7 - E) with 2^E above the largest V scale so far: at
// most 2^15 and normal in fp16 down to p s = 2^-21 of that scale, so a block
// of small scale keeps its precision.  fp32 calls: q (scaled to 2^13) and P'
// enter as fp16 high + low parts (22 bits), two MMAs for each product.
#include <math_constants.h>

#include <algorithm>

#include "kvx_common.cuh"
#include "kvx_decode_params.cuh"  // grid_dependents_launch, grid_dependency_wait

namespace kvx {
namespace {

constexpr int kTileKeys = 128, kTilePages = kTileKeys / kPageTokens;
constexpr int kBlockBytes = kPageTokens * kHeadDim;  // codes of one (page, K|V, head)
constexpr int kConvertWarp = 8, kMmaWarp = 16, kLoadWarp = 17, kStatWarp = 18, kChunkThreads = 20 * 32;
// registers a thread, by warpgroup (setmaxnreg): 2 x 128 x 128 + 2 x 128 x 72
// + 128 x 80 = the 640 x 96 of the launch
constexpr int kSoftmaxRegs = 128, kConvertRegs = 72, kIssueRegs = 80;
static_assert(2 * kSoftmaxRegs + 2 * kConvertRegs + kIssueRegs == 5 * 96, "the launch's registers, dealt out");
constexpr int kTileBytes = 128 * kHeadDim * 2;  // an fp16 tile of Q, K or V: two halves of 64 dims
constexpr int kHalfBytes = kTileBytes / 2, kSlotBytes = kTileKeys * kHeadDim;
// What the softmax needs of a key tile's statistics.
constexpr int kStatSlots = 4;
struct TileStats {
    float4 page[kTilePages];  // K: scale, mid (times the softmax scale, log2); V: scale 2^(7 - exponent), mid
    int exponent;             // 2^exponent is above every V scale up to this tile
    uint32_t known;           // bit i: page i is there
    uint32_t pad[2];
};
// shared memory: Q0, Q1 (staging slots 2, 3 when unused), K x 2, V x 2, staging x 2, the rest
constexpr int kAtK = 2 * kTileBytes, kAtV = kAtK + 2 * kTileBytes, kAtStage = kAtV + 2 * kTileBytes,
              kAtMisc = kAtStage + 2 * kSlotBytes, kChunkSmem = 1024 + kAtMisc + 512 + kStatSlots * (int)sizeof(TileStats);
static_assert(kChunkSmem <= 227 * 1024, "chunk attention exceeds the shared memory of a CTA");
constexpr float kLazy = 8.f;  // log2 of the growth of a row's maximum that is let pass

struct ChunkParams {
    const uint8_t *pool;
    const float *stats;
    const int32_t *block_table, *q_start, *positions;
    const void *q;
    void *out;
    float *part_o;     // [split][total * hq][128]
    float2 *part_ml;   // [split][total * hq]
    int32_t *error_flag;
    int batch, total, hq, hkv, group, max_pages, num_pages, causal, chunk;  // chunk: key tiles of a split
    float scale_log2;
};

struct ChunkBars {
    uint64_t ld_full[4], ld_empty[4], stat_full[kStatSlots], stat_empty[kStatSlots], k_full[2], k_empty[2], v_full[2], v_empty[2], s_full[2], p_full[2], q_full, done;
    uint32_t tmem, gave_up;
    uint32_t known[4];  // staging slot: bit i, page i was loaded
    int seq, tile;
};
static_assert(sizeof(ChunkBars) <= 512, "");

// Rows of one (sequence, row tile): what the kernel and the combine agree on.
struct RowTile {
    int begin, n;      // packed rows of the sequence
    int pos, rows;     // rows in the tile
    int keys, tiles;   // keys the tile's last row sees, in 128-key tiles
    int splits;
};

__device__ __forceinline__ int sequence_tokens(const ChunkParams &p, int s) {
    const int a = p.q_start[s], b = min(p.q_start[s + 1], p.total);
    return a >= 0 && b > a ? b - a : 0;
}

__device__ __forceinline__ int row_keys(const ChunkParams &p, const RowTile &t, int row) {
    if (t.pos < 0) return 0;
    const long long k = (long long)t.pos + (p.causal ? row / p.group + 1 : t.n);
    return (int)min(k, (long long)p.max_pages * kPageTokens);
}

__device__ __forceinline__ RowTile row_tile(const ChunkParams &p, int s, int tile, int tile_rows) {
    RowTile t;
    t.begin = p.q_start[s];
    t.n = sequence_tokens(p, s);
    t.pos = p.positions[s];
    const int all = t.n * p.group;
    t.rows = min(tile_rows, all - tile * tile_rows);
    t.keys = row_keys(p, t, tile * tile_rows + t.rows - 1);
    t.tiles = (t.keys + kTileKeys - 1) / kTileKeys;
    t.splits = max(1, (t.tiles + p.chunk - 1) / p.chunk);
    return t;
}

// ---- tcgen05

// Shared-memory descriptor of a 128-byte-swizzled operand whose 8-row groups
// lie 1024 bytes apart: the low word holds the address and the leading
// offset (both count 16 bytes), the high word is the same for all.
__device__ __forceinline__ uint32_t umma_desc_low(uint32_t addr, uint32_t leading) { return (addr >> 4) | (leading >> 4) << 16; }
constexpr uint32_t kDescHigh = (1024u >> 4) | 1u << 14 /* sm100 descriptor */ | 2u << 29 /* 128-byte swizzle */;
// D fp32, A and B fp16, M = N = 128, A K-major
constexpr uint32_t kIdescQK = (1u << 4) | ((128u >> 3) << 17) | ((128u >> 4) << 24);
constexpr uint32_t kIdescPV = kIdescQK | (1u << 16);  // B MN-major

// Issued by the lane whose `issues` is set, under a predicate and not a
// branch: the operands stay in uniform registers.
__device__ __forceinline__ void umma_f16_ss(uint32_t issues, uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, uint32_t acc) {
    asm volatile(
        "{\n\t.reg .pred p, q;\n\t.reg .b64 x, y;\n\tsetp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 q, %5, 0;\n\t"
        "mov.b64 x, {%1, %6};\n\tmov.b64 y, {%2, %6};\n\t"
        "@q tcgen05.mma.cta_group::1.kind::f16 [%0], x, y, %3, p;\n\t}" ::"r"(d), "r"(a), "r"(b), "r"(idesc), "r"(acc), "r"(issues), "n"(kDescHigh)
        : "memory");
}
__device__ __forceinline__ void umma_f16_ts(uint32_t issues, uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, uint32_t acc) {
    asm volatile(
        "{\n\t.reg .pred p, q;\n\t.reg .b64 y;\n\tsetp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 q, %5, 0;\n\t"
        "mov.b64 y, {%2, %6};\n\t"
        "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], y, %3, p;\n\t}" ::"r"(d), "r"(a), "r"(b), "r"(idesc), "r"(acc), "r"(issues), "n"(kDescHigh)
        : "memory");
}
__device__ __forceinline__ uint32_t elect_one() {
    uint32_t r;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(r));
    return r;
}
__device__ __forceinline__ void umma_commit(uint32_t issues, uint64_t *bar) {
    asm volatile(
        "{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %1, 0;\n\t"
        "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(smem_addr(bar)), "r"(issues)
        : "memory");
}
// The same value in every lane, known to be so.
__device__ __forceinline__ uint32_t uniform(uint32_t x) { return __reduce_max_sync(0xffffffffu, x); }
__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
// ... and nothing that uses these registers moves above it
__device__ __forceinline__ void tmem_wait_ld(uint32_t (&a)[16]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;" : "+r"(a[0]), "+r"(a[1]), "+r"(a[2]), "+r"(a[3]), "+r"(a[4]), "+r"(a[5]), "+r"(a[6]), "+r"(a[7]), "+r"(a[8]), "+r"(a[9]), "+r"(a[10]), "+r"(a[11]), "+r"(a[12]), "+r"(a[13]), "+r"(a[14]), "+r"(a[15]) : : "memory");
}
__device__ __forceinline__ void tmem_wait_ld(uint32_t (&a)[32]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;" : "+r"(a[0]), "+r"(a[1]), "+r"(a[2]), "+r"(a[3]), "+r"(a[4]), "+r"(a[5]), "+r"(a[6]), "+r"(a[7]), "+r"(a[8]), "+r"(a[9]), "+r"(a[10]), "+r"(a[11]), "+r"(a[12]), "+r"(a[13]), "+r"(a[14]), "+r"(a[15]), "+r"(a[16]), "+r"(a[17]), "+r"(a[18]), "+r"(a[19]), "+r"(a[20]), "+r"(a[21]), "+r"(a[22]), "+r"(a[23]), "+r"(a[24]), "+r"(a[25]), "+r"(a[26]), "+r"(a[27]), "+r"(a[28]), "+r"(a[29]), "+r"(a[30]), "+r"(a[31]) : : "memory");
}
__device__ __forceinline__ void tmem_wait_ld(uint32_t (&a)[32], uint32_t (&b)[32]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;" : "+r"(a[0]), "+r"(a[1]), "+r"(a[2]), "+r"(a[3]), "+r"(a[4]), "+r"(a[5]), "+r"(a[6]), "+r"(a[7]), "+r"(a[8]), "+r"(a[9]), "+r"(a[10]), "+r"(a[11]), "+r"(a[12]), "+r"(a[13]), "+r"(a[14]), "+r"(a[15]), "+r"(a[16]), "+r"(a[17]), "+r"(a[18]), "+r"(a[19]), "+r"(a[20]), "+r"(a[21]), "+r"(a[22]), "+r"(a[23]), "+r"(a[24]), "+r"(a[25]), "+r"(a[26]), "+r"(a[27]), "+r"(a[28]), "+r"(a[29]), "+r"(a[30]), "+r"(a[31]), "+r"(b[0]), "+r"(b[1]), "+r"(b[2]), "+r"(b[3]), "+r"(b[4]), "+r"(b[5]), "+r"(b[6]), "+r"(b[7]), "+r"(b[8]), "+r"(b[9]), "+r"(b[10]), "+r"(b[11]), "+r"(b[12]), "+r"(b[13]), "+r"(b[14]), "+r"(b[15]), "+r"(b[16]), "+r"(b[17]), "+r"(b[18]), "+r"(b[19]), "+r"(b[20]), "+r"(b[21]), "+r"(b[22]), "+r"(b[23]), "+r"(b[24]), "+r"(b[25]), "+r"(b[26]), "+r"(b[27]), "+r"(b[28]), "+r"(b[29]), "+r"(b[30]), "+r"(b[31]) : : "memory");
}
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

__device__ __forceinline__ void tmem_ld16(uint32_t at, uint32_t (&r)[16]) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
                 : "r"(at));
}
__device__ __forceinline__ void tmem_ld32(uint32_t at, uint32_t (&r)[32]) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
                 : "r"(at));
}
__device__ __forceinline__ void tmem_st8(uint32_t at, const uint32_t (&r)[8]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%8], {%0, %1, %2, %3, %4, %5, %6, %7};" ::"r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(at) : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t at, const uint32_t (&r)[16]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15};" ::"r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(at) : "memory");
}

// 2^x on the special-function unit (2^-inf = +0)
__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// Two floats side by side: the packed fp32 operations of sm_100.
__device__ __forceinline__ uint64_t pack2(float a, float b) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ float2 unpack2(uint64_t v) {
    float2 r;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
    return r;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}

template <int kRegs> __device__ __forceinline__ void more_registers() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRegs)); }
template <int kRegs> __device__ __forceinline__ void fewer_registers() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegs)); }

__device__ __forceinline__ float pow2i(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }  // -126 <= e <= 127

// Smallest e with |x| < 2^e, kept in [-100, 128]; x finite.
__device__ __forceinline__ int exponent_above(float x) {
    return max((int)((__float_as_uint(x) >> 23) & 0xff) - 126, -100);
}

// Bounded wait.  Once one has run out, every later wait of the CTA returns at
// once: the CTA finishes (with wrong results and bit 0 of the error flag)
// instead of waiting again and again.
__device__ __forceinline__ void wait_or_give_up(uint64_t *bar, uint32_t parity, ChunkBars *b, int32_t *error_flag) {
#pragma unroll 1
    for (uint32_t i = 0; i < kWaitPolls; ++i) {
        if (mbar_try_wait(bar, parity)) return;
        if ((i & 255) == 255 && *reinterpret_cast<volatile uint32_t *>(&b->gave_up)) return;
    }
    *reinterpret_cast<volatile uint32_t *>(&b->gave_up) = 1;
    if (error_flag) atomicOr(error_flag, 1);
}

__device__ __forceinline__ void st_shared16(uint32_t at, uint32_t x, uint32_t y, uint32_t z, uint32_t w) {
    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(x), "r"(y), "r"(z), "r"(w) : "memory");
}

// Byte offset of 16-byte chunk c (0..15: 8 dims each) of row r in a tile.
__device__ __forceinline__ uint32_t tile_chunk(int r, int c) {
    return (uint32_t)((c >> 3) * kHalfBytes + r * 128 + (((c & 7) ^ (r & 7)) << 4));
}

// Four int8 codes -> four fp16, exact: the byte c + 128 becomes the low
// mantissa bits of 1024 + c + 128, from which 1152 is taken.
__device__ __forceinline__ uint2 codes_to_half(uint32_t w) {
    const uint32_t u = w ^ 0x80808080u;
    uint2 r;
    const __half2 off = __half2half2(__ushort_as_half((unsigned short)0x6480));  // 1152
    uint32_t lo = __byte_perm(u, 0x64646464u, 0x4140), hi = __byte_perm(u, 0x64646464u, 0x4342);
    const __half2 a = __hsub2(*reinterpret_cast<__half2 *>(&lo), off), b = __hsub2(*reinterpret_cast<__half2 *>(&hi), off);
    r.x = *reinterpret_cast<const uint32_t *>(&a);
    r.y = *reinterpret_cast<const uint32_t *>(&b);
    return r;
}

__device__ __forceinline__ uint32_t pack_half(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t *>(&h);
}

// The row's 16-byte chunk of 8 dims: as fp16, or fp16 high and low parts.
template <typename T> __device__ __forceinline__ void load_q8(const T *row, int c, float *f);
template <> __device__ __forceinline__ void load_q8<__half>(const __half *row, int c, float *f) {
    const uint4 w = reinterpret_cast<const uint4 *>(row)[c];
    const float2 a = h2_to_f2(w.x), b = h2_to_f2(w.y), d = h2_to_f2(w.z), e = h2_to_f2(w.w);
    f[0] = a.x, f[1] = a.y, f[2] = b.x, f[3] = b.y, f[4] = d.x, f[5] = d.y, f[6] = e.x, f[7] = e.y;
}
template <> __device__ __forceinline__ void load_q8<float>(const float *row, int c, float *f) {
    const float4 a = reinterpret_cast<const float4 *>(row)[2 * c], b = reinterpret_cast<const float4 *>(row)[2 * c + 1];
    f[0] = a.x, f[1] = a.y, f[2] = a.z, f[3] = a.w, f[4] = b.x, f[5] = b.y, f[6] = b.z, f[7] = b.w;
}

template <typename T> __device__ __forceinline__ void store_out4(T *o, float a, float b, float c, float d);
template <> __device__ __forceinline__ void store_out4<float>(float *o, float a, float b, float c, float d) {
    *reinterpret_cast<float4 *>(o) = make_float4(a, b, c, d);
}
template <> __device__ __forceinline__ void store_out4<__half>(__half *o, float a, float b, float c, float d) {
    *reinterpret_cast<uint2 *>(o) = make_uint2(pack_half(a, b), pack_half(c, d));
}

// kSplit (fp32 calls): q and P' as high + low parts.
template <typename T, bool kSplit>
__global__ void __launch_bounds__(kChunkThreads, 1) attend_chunk_kernel(const __grid_constant__ ChunkParams p) {
    constexpr int kTileRows = kSplit ? 128 : 256;
    extern __shared__ __align__(1024) uint8_t chunk_smem[];
    uint8_t *sm = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(chunk_smem) + 1023) & ~uintptr_t(1023));
    const uint32_t base = smem_addr(sm);
    ChunkBars *bars = reinterpret_cast<ChunkBars *>(sm + kAtMisc);
    TileStats *tile_stats = reinterpret_cast<TileStats *>(sm + kAtMisc + 512);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int kvh = blockIdx.y, split = blockIdx.z;

    grid_dependents_launch();  // the combine may place its CTAs; it waits for this grid
    // ---- which rows: the last tiles first (causal: they have the most keys)
    if (warp == 0) {
        const int want = gridDim.x - 1 - blockIdx.x;
        int before = 0, seq = -1, tile = 0;
        for (int s0 = 0; s0 < p.batch && seq < 0; s0 += 32) {
            const int s = s0 + lane;
            const int mine = s < p.batch ? (sequence_tokens(p, s) * p.group + kTileRows - 1) / kTileRows : 0;
            int x = mine;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int y = __shfl_up_sync(0xffffffffu, x, o);
                if (lane >= o) x += y;
            }
            const uint32_t hit = __ballot_sync(0xffffffffu, want < before + x);
            if (hit) {
                const int l = __ffs(hit) - 1;
                seq = s0 + l;
                tile = want - before - __shfl_sync(0xffffffffu, x - mine, l);
            }
            before += __shfl_sync(0xffffffffu, x, 31);
        }
        if (lane == 0) {
            bars->seq = seq;
            bars->tile = tile;
            bars->gave_up = 0;
        }
    }
    __syncthreads();
    const int seq = bars->seq, tile = bars->tile;
    if (seq < 0) return;  // the grid is an upper bound
    const RowTile rt = row_tile(p, seq, tile, kTileRows);
    if (split >= rt.splits) return;
    const int row0 = tile * kTileRows;
    if (threadIdx.x == 0 && split == 0 && p.error_flag) {
        if (rt.pos < 0) atomicOr(p.error_flag, 2);
        if ((long long)rt.pos + rt.n > (long long)p.max_pages * kPageTokens) atomicOr(p.error_flag, 4);
    }
    auto row_index = [&](int r) {  // row of q / out: (token, q-head)
        const int row = row0 + r;
        return (size_t)(rt.begin + row / p.group) * p.hq + kvh * p.group + row % p.group;
    };
    if (rt.tiles == 0) {  // nothing to see
        for (int i = threadIdx.x; i < rt.rows * (kHeadDim / 4); i += kChunkThreads)
            store_out4<T>(static_cast<T *>(p.out) + row_index(i / (kHeadDim / 4)) * kHeadDim + 4 * (i % (kHeadDim / 4)), 0.f, 0.f,
                          0.f, 0.f);
        return;
    }
    const int t0 = split * p.chunk, tiles = min(p.chunk, rt.tiles - t0);  // this CTA's key tiles
    const bool turns = kSplit || rt.rows <= 128;  // the warpgroups take turns at the key tiles
    const int items = turns ? tiles : 2 * tiles;  // item w: warpgroup w % 2, key tile w or w / 2
    const int slot_bits = turns && !kSplit ? 2 : 1, slot_mask = (1 << slot_bits) - 1;  // 4 or 2 staging slots
    const int32_t *table = p.block_table + (size_t)seq * p.max_pages;
    if (threadIdx.x == 32) {
        for (int i = 0; i < 4; ++i) {
            mbar_init(&bars->ld_full[i], 1);
            mbar_init(&bars->ld_empty[i], 4);
        }
        for (int i = 0; i < kStatSlots; ++i) {
            mbar_init(&bars->stat_full[i], 1);
            mbar_init(&bars->stat_empty[i], turns ? 4 : 8);  // the softmax warps that look at a tile
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(&bars->k_full[i], 4);
            mbar_init(&bars->k_empty[i], 1);
            mbar_init(&bars->v_full[i], 4);
            mbar_init(&bars->v_empty[i], 1);
            mbar_init(&bars->s_full[i], 1);
            mbar_init(&bars->p_full[i], 128);
        }
        mbar_init(&bars->q_full, 256);
        mbar_init(&bars->done, 1);
        fence_barrier_init();
    }
    if (warp == kMmaWarp) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_addr(&bars->tmem)) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    // S0, S1, O0, O1: 128 columns each.  All 512 columns were asked for, so
    // they begin at 0 (were they to begin elsewhere, nothing is done).
    constexpr uint32_t tmem = 0;
    if (bars->tmem != 0) {
        if (threadIdx.x == 0 && p.error_flag) atomicOr(p.error_flag, 1);
        if (warp == kMmaWarp)
            asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(bars->tmem) : "memory");
        return;
    }
    auto slot_at = [&](int s) { return s < 2 ? kAtStage + s * kSlotBytes : kTileBytes + (s - 2) * kSlotBytes; };

    if (warp >= kMmaWarp) {
        fewer_registers<kIssueRegs>();
        if (warp == kLoadWarp) {
            // ---- loader: lane i < 8 copies page i of the tile's K, then V codes
            auto wanted = [&](int i) { return lane < 8 && i < tiles && ((t0 + i) * kTilePages + lane) * kPageTokens < rt.keys; };
            int next = wanted(0) ? table[t0 * kTilePages + lane] : -1;
            for (int i = 0; i < tiles; ++i) {
                const bool want = wanted(i);
                const int phys = next;
                if (wanted(i + 1)) next = table[(t0 + i + 1) * kTilePages + lane];
                const bool have = want && phys >= 0 && phys < p.num_pages;
                if (want && !have && p.error_flag) atomicOr(p.error_flag, 2);
                const uint32_t known = __ballot_sync(0xffffffffu, have);
                for (int kv = 0; kv < 2; ++kv) {
                    const int u = 2 * i + kv, s = u & slot_mask;
                    wait_or_give_up(&bars->ld_empty[s], (u >> slot_bits & 1) ^ 1, bars, p.error_flag);
                    if (lane == 0) {
                        bars->known[s] = known;
                        mbar_arrive_expect_tx(&bars->ld_full[s], __popc(known) * kBlockBytes);
                    }
                    __syncwarp();
                    if (have)
                        bulk_g2s(sm + slot_at(s) + lane * kBlockBytes,
                                 p.pool + (((size_t)phys * 2 + kv) * p.hkv + kvh) * kBlockBytes, kBlockBytes, &bars->ld_full[s]);
                }
            }
            // no copy is in flight when the CTA ends, however it ends
            for (int u = max(0, 2 * tiles - slot_mask - 1); u < 2 * tiles; ++u)
                (void)mbar_wait_bounded(&bars->ld_full[u & slot_mask], u >> slot_bits & 1, nullptr);
        } else if (warp == kStatWarp) {
            // ---- statistics: lane i < 8 takes page i's of K, lane 8 + i of V;
            // page ids two tiles ahead, statistics one
            auto page_of = [&](int i) {
                const int lp = (t0 + i) * kTilePages + (lane & 7);
                return lane < 16 && i < tiles && lp * kPageTokens < rt.keys ? table[lp] : -1;
            };
            auto stat_of = [&](int phys) {
                return phys >= 0 && phys < p.num_pages
                           ? __ldg(reinterpret_cast<const float4 *>(p.stats) + ((size_t)phys * 2 + (lane >> 3)) * p.hkv + kvh)
                           : make_float4(0.f, 0.f, 0.f, 0.f);
            };
            int id = page_of(0), id_next = page_of(1), E = -100;
            float4 stat = stat_of(id);
            for (int i = 0; i < tiles; ++i) {
                const uint32_t known = __ballot_sync(0xffffffffu, id >= 0 && id < p.num_pages) & 0xffu;
                const float4 cur = stat;
                id = id_next;
                stat = stat_of(id);
                id_next = page_of(i + 2);
                // scales that are no numbers do not count
                const int e = lane >= 8 && lane < 16 && fabsf(cur.z) < CUDART_INF_F ? exponent_above(cur.z) : -100;
                E = max(E, __reduce_max_sync(0xffffffffu, e));
                const float mid = fmaf(128.f, cur.z, cur.w), f = lane < 8 ? p.scale_log2 : pow2i(7 - E);
                TileStats &t = tile_stats[i & (kStatSlots - 1)];
                wait_or_give_up(&bars->stat_empty[i & (kStatSlots - 1)], (i / kStatSlots & 1) ^ 1, bars, p.error_flag);
                if (lane < 16)
                    reinterpret_cast<float2 *>(&t.page[lane & 7])[lane >> 3] = make_float2(cur.z * f, lane < 8 ? mid * f : mid);
                if (lane == 0) {
                    t.exponent = E;
                    t.known = known;
                }
                __syncwarp();
                if (lane == 0) mbar_arrive(&bars->stat_full[i & (kStatSlots - 1)]);
            }
        } else if (warp == kMmaWarp) {
            // The whole warp walks the items and one lane issues, from uniform
            // registers: an MMA is 64 cycles, so its issue has to be a few
            // instructions.  The 512 tensor-memory columns begin at 0.
            const uint32_t issues = elect_one(), at = uniform(base);
            const bool u_turns = uniform(turns);
            const int u_items = (int)uniform(items);
            wait_or_give_up(&bars->q_full, 0, bars, p.error_flag);
#pragma unroll 1
            for (int w = -2; w < u_items; ++w) {  // P V of item w, then the scores of item w + 2
                const int j = w & 1;
                if (w >= 0) {
                    const int i = u_turns ? w : w >> 1, st = i & 1;
                    wait_or_give_up(&bars->v_full[st], (i >> 1) & 1, bars, p.error_flag);
                    wait_or_give_up(&bars->p_full[j], (w >> 1) & 1, bars, p.error_flag);
                    tc_fence_after();
                    const uint32_t v = umma_desc_low(at + kAtV + st * kTileBytes, kHalfBytes);
#pragma unroll
                    for (int part = 0; part < (kSplit ? 2 : 1); ++part)
#pragma unroll
                        for (int ks = 0; ks < 8; ++ks)  // a page: its P over its columns of S
                            umma_f16_ts(issues, tmem + 256 + j * 128, tmem + j * 128 + ks * 16 + part * 8, v + (ks * 2048 >> 4),
                                        kIdescPV, (w > 1) | part | ks);
                    if (u_turns || j) umma_commit(issues, &bars->v_empty[st]);
                }
                if (w + 2 < u_items) {
                    const int i = u_turns ? w + 2 : (w + 2) >> 1, st = i & 1;
                    wait_or_give_up(&bars->k_full[st], (i >> 1) & 1, bars, p.error_flag);
                    tc_fence_after();
                    const uint32_t q = umma_desc_low(at + (u_turns ? 0 : j * kTileBytes), 16),
                                   k = umma_desc_low(at + kAtK + st * kTileBytes, 16);
#pragma unroll
                    for (int part = 0; part < (kSplit ? 2 : 1); ++part)
#pragma unroll
                        for (int ks = 0; ks < 8; ++ks) {
                            const uint32_t off = ((ks >> 2) * kHalfBytes + (ks & 3) * 32) >> 4;
                            umma_f16_ss(issues, tmem + j * 128, q + ((part * kTileBytes >> 4) + off), k + off, kIdescQK, part | ks);
                        }
                    umma_commit(issues, &bars->s_full[j]);
                    if (u_turns || j) umma_commit(issues, &bars->k_empty[st]);
                }
            }
            umma_commit(issues, &bars->done);
            __syncwarp();
        }
    } else if (warp >= kConvertWarp) {
        fewer_registers<kConvertRegs>();
        // ---- convert: a warpgroup for K, one for V.  8 lanes take row r (even)
        // chunks 0-3 and row r + 1 chunks 4-7: reads of 128 contiguous bytes,
        // writes to 8 different 16-byte banks.  The slot is free as soon as its
        // codes are in registers: its next copy runs under the conversion.
        const int kv = warp >> 2 & 1, g = (warp & 3) * 4 + (lane >> 3), j = lane & 7;  // groups 0..15 of 8 lanes
        auto row_of = [&](int k) { return 2 * (g + 16 * (k >> 1)) + ((j >> 2) ^ (k & 1)); };
        for (int i = 0; i < tiles; ++i) {
            const int u = 2 * i + kv, s = u & slot_mask, st = i & 1;
            wait_or_give_up(&bars->ld_full[s], u >> slot_bits & 1, bars, p.error_flag);
            const uint32_t known = bars->known[s];
            const uint8_t *src = sm + slot_at(s);
            uint4 w[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) w[k] = *reinterpret_cast<const uint4 *>(src + row_of(k) * 128 + j * 16);
            if (known != 0xffu) {
#pragma unroll
                for (int k = 0; k < 8; ++k)
                    if (!(known >> (row_of(k) >> 4) & 1)) w[k] = make_uint4(0, 0, 0, 0);
            }
            fence_proxy_async_smem();  // these reads before the slot's next copy
            __syncwarp();
            if (lane == 0) mbar_arrive(&bars->ld_empty[s]);
            wait_or_give_up(kv ? &bars->v_empty[st] : &bars->k_empty[st], ((i >> 1) & 1) ^ 1, bars, p.error_flag);
            const uint32_t dst = base + (kv ? kAtV : kAtK) + st * kTileBytes;
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                const int r = row_of(k);
                const uint2 a = codes_to_half(w[k].x), b = codes_to_half(w[k].y), d = codes_to_half(w[k].z), e = codes_to_half(w[k].w);
                st_shared16(dst + tile_chunk(r, 2 * j), a.x, a.y, b.x, b.y);
                st_shared16(dst + tile_chunk(r, 2 * j + 1), d.x, d.y, e.x, e.y);
            }
            fence_proxy_async_smem();  // before the tensor core's reads
            __syncwarp();
            if (lane == 0) mbar_arrive(kv ? &bars->v_full[st] : &bars->k_full[st]);
        }
    } else {
        more_registers<kSoftmaxRegs>();
        // ---- softmax: thread = row
        const int j = warp >> 2, r = threadIdx.x & 127;
        const uint32_t lanes = (uint32_t)(32 * (warp & 3)) << 16;
        const uint32_t t_s = tmem + j * 128 + lanes, t_o = tmem + 256 + j * 128 + lanes;
        const int my_row = turns ? r : j * 128 + r;
        const bool valid = my_row < rt.rows;
        float q_sum = 0.f, unscale = 1.f;
        {
            const T *row = static_cast<const T *>(p.q) + (valid ? row_index(my_row) : 0) * kHeadDim;
            const bool writes = !turns || j == 0;
            const uint32_t dst = base + (turns ? 0 : j * kTileBytes);
            float up = 1.f;
            if constexpr (kSplit) {
                float big = 0.f;
#pragma unroll 4
                for (int c = 0; c < 16; ++c) {
                    float f[8];
                    if (valid) {
                        load_q8<T>(row, c, f);
#pragma unroll
                        for (int k = 0; k < 8; ++k) big = fmaxf(big, fabsf(f[k]));
                    }
                }
                if (big > 0.f && big < CUDART_INF_F) {
                    const int e = exponent_above(big);
                    up = pow2i(13 - e);
                    unscale = pow2i(e - 13);
                }
            }
#pragma unroll 4
            for (int c = 0; c < 16; ++c) {
                float f[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
                if (valid) load_q8<T>(row, c, f);
#pragma unroll
                for (int k = 0; k < 8; ++k) q_sum += f[k];
                if (writes) {
                    uint32_t hi[4], lo[4];
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        const float a = f[2 * k] * up, b = f[2 * k + 1] * up;
                        hi[k] = pack_half(a, b);
                        const float2 h = h2_to_f2(hi[k]);
                        lo[k] = pack_half(a - h.x, b - h.y);
                    }
                    st_shared16(dst + tile_chunk(r, c), hi[0], hi[1], hi[2], hi[3]);
                    if (kSplit) st_shared16(dst + kTileBytes + tile_chunk(r, c), lo[0], lo[1], lo[2], lo[3]);
                }
            }
            fence_proxy_async_smem();
            mbar_arrive(&bars->q_full);
        }
        const int limit = valid ? row_keys(p, rt, row0 + my_row) : 0x7fffffff;  // a row that is none needs no mask
        const int step = turns ? 2 : 1;
        // O by f (rare, so in little code)
        auto scale_o = [&](float f) {
#pragma unroll 1
            for (int c = 0; c < 8; ++c) {
                uint32_t o[16];
                tmem_ld16(t_o + 16 * c, o);
                tmem_wait_ld(o);
#pragma unroll
                for (int k = 0; k < 16; ++k) o[k] = __float_as_uint(__uint_as_float(o[k]) * f);
                tmem_st16(t_o + 16 * c, o);
            }
        };
        float m = -CUDART_INF_F, l = 0.f, z = 0.f;  // maximum (log2), sum, sum of p mid
        int E = -100;
        int i = turns ? j : 0;
        for (int w = j; w < items; w += 2, i += step) {
            const TileStats &ts = tile_stats[i & (kStatSlots - 1)];
            wait_or_give_up(&bars->stat_full[i & (kStatSlots - 1)], i / kStatSlots & 1, bars, p.error_flag);
            const uint32_t known = ts.known;
            const int e = ts.exponent, seen = limit - (t0 + i) * kTileKeys;  // the tile's keys that the row sees
            const bool masked = __any_sync(0xffffffffu, seen < kTileKeys) || known != 0xffu;
            // a page this row sees nothing of: scores of -inf, whatever its statistics
            auto hidden = [&](int page) { return seen <= page * kPageTokens || !(known >> page & 1); };
            wait_or_give_up(&bars->s_full[j], (w >> 1) & 1, bars, p.error_flag);
            __syncwarp();
            tc_fence_after();
            if (masked) {  // few tiles: their scores are masked where they are
#pragma unroll 1
                for (int page = 0; page < kTilePages; ++page) {
                    uint32_t v[16];
                    tmem_ld16(t_s + 16 * page, v);
                    tmem_wait_ld(v);
                    const int n = known >> page & 1 ? seen - page * kPageTokens : 0;
#pragma unroll
                    for (int k = 0; k < 16; ++k)
                        if (k >= n) v[k] = 0xff800000u;  // -inf
                    tmem_st16(t_s + 16 * page, v);
                }
                tmem_wait_st();
            }
            // Two loops of two chunks of 32 keys each: the code of all warps
            // together has to stay in the instruction cache.
            float top = -CUDART_INF_F;
#pragma unroll 1
            for (int c = 0; c < 4; c += 2) {
                uint32_t x[2][32];
                tmem_ld32(t_s + 32 * c, x[0]);
                tmem_ld32(t_s + 32 * c + 32, x[1]);
                tmem_wait_ld(x[0], x[1]);
#pragma unroll
                for (int h = 0; h < 4; ++h) {
                    const int page = 2 * c + h;
                    uint32_t(&v)[32] = x[h >> 1];
                    float2 ks = *reinterpret_cast<const float2 *>(&ts.page[page]);
                    ks.x *= unscale, ks.y *= q_sum;
                    if (masked && hidden(page)) ks = make_float2(1.f, 0.f);
                    float a = __uint_as_float(v[16 * (h & 1)]), b = __uint_as_float(v[16 * (h & 1) + 1]);
#pragma unroll
                    for (int k = 2; k < 14; k += 4) {  // three-input maxima
                        a = fmaxf(fmaxf(a, __uint_as_float(v[16 * (h & 1) + k])), __uint_as_float(v[16 * (h & 1) + k + 1]));
                        b = fmaxf(fmaxf(b, __uint_as_float(v[16 * (h & 1) + k + 2])), __uint_as_float(v[16 * (h & 1) + k + 3]));
                    }
                    a = fmaxf(fmaxf(a, __uint_as_float(v[16 * (h & 1) + 14])), __uint_as_float(v[16 * (h & 1) + 15]));
                    top = fmaxf(top, fmaf(ks.x, fmaxf(a, b), ks.y));
                }
            }
            // the maximum in use may lag by kLazy; O follows where it catches
            // up, and where a larger V scale came
            const bool lags = __any_sync(0xffffffffu, top > m + kLazy);
            if (lags || e > E) {
                float f = 1.f;
                if (lags) {
                    const float mn = fmaxf(m, top);
                    if (mn != -CUDART_INF_F) f = ex2(m - mn);
                    m = mn;
                    l *= f;
                    z *= f;
                }
                if (w >= 2) scale_o(E - e < -126 ? 0.f : f * pow2i(E - e));
                E = e;
            }
            const float m_use = m == -CUDART_INF_F ? 0.f : m;
#pragma unroll 1
            for (int c = 0; c < 4; c += 2) {
                uint32_t x[2][32];
                tmem_ld32(t_s + 32 * c, x[0]);
                tmem_ld32(t_s + 32 * c + 32, x[1]);
                tmem_wait_ld(x[0], x[1]);
#pragma unroll
                for (int h = 0; h < 4; ++h) {
                    const int page = 2 * c + h;
                    uint32_t(&v)[32] = x[h >> 1];
                    float4 st = ts.page[page];
                    st.x *= unscale;
                    st.y = fmaf(st.y, q_sum, -m_use);
                    if (masked && hidden(page)) st = make_float4(1.f, 0.f, 0.f, 0.f);
                    const uint64_t aa = pack2(st.x, st.x), bb = pack2(st.y, st.y), ss = pack2(st.z, st.z);
                    uint64_t sum = 0;
                    uint32_t hi[8], lo[8];
#pragma unroll
                    for (int k = 0; k < 16; k += 2) {
                        const float2 t = unpack2(fma2(aa, pack2(__uint_as_float(v[16 * (h & 1) + k]), __uint_as_float(v[16 * (h & 1) + k + 1])), bb));
                        const uint64_t e2 = pack2(ex2(t.x), ex2(t.y));
                        sum = add2(sum, e2);
                        const float2 f = unpack2(mul2(e2, ss));
                        hi[k / 2] = pack_half(f.x, f.y);
                        if constexpr (kSplit) {
                            const float2 g = h2_to_f2(hi[k / 2]);
                            lo[k / 2] = pack_half(f.x - g.x, f.y - g.y);
                        }
                    }
                    const float2 both = unpack2(sum);
                    l += both.x + both.y;
                    z = fmaf(both.x + both.y, st.w, z);
                    tmem_st8(t_s + 16 * page, hi);  // over the page's own scores
                    if constexpr (kSplit) tmem_st8(t_s + 16 * page + 8, lo);
                }
            }
            tmem_wait_st();
            tc_fence_before();
            mbar_arrive(&bars->p_full[j]);
            __syncwarp();
            if (lane == 0) mbar_arrive(&bars->stat_empty[i & (kStatSlots - 1)]);
        }

        // ---- O
        wait_or_give_up(&bars->done, 0, bars, p.error_flag);
        __syncwarp();
        tc_fence_after();
        const float back = pow2i(E - 7);
        const bool worked = j < items;  // this warpgroup had a tile
        float *shared_o = reinterpret_cast<float *>(sm + kAtK);  // [dim][row] over K, V, now free
        float *shared_ml = reinterpret_cast<float *>(sm);        // over Q
        float mine = 1.f, other = 0.f;
        if (turns) {
            if (j == 1) {
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    if (!worked) break;
                    uint32_t x[32];
                    tmem_ld32(t_o + 32 * c, x);
                    tmem_wait_ld(x);
#pragma unroll
                    for (int k = 0; k < 32; ++k)
                        shared_o[(32 * c + k) * 128 + r] = fmaf(__uint_as_float(x[k]), back, z);
                }
                shared_ml[r] = m;
                shared_ml[128 + r] = l;
            }
            asm volatile("bar.sync 1, 256;" ::: "memory");
            if (j == 0 && items > 1) {
                const float m1 = shared_ml[r], l1 = shared_ml[128 + r], mn = fmaxf(m, m1);
                if (mn != -CUDART_INF_F) {
                    mine = ex2(m - mn);
                    other = ex2(m1 - mn);
                }
                l = l * mine + l1 * other;
                m = mn;
            }
        }
        if (!turns || j == 0) {
            const size_t at = valid ? row_index(my_row) : 0;
            const bool direct = rt.splits == 1, merge = turns && items > 1;
            const float inv = direct ? (l == 0.f ? 0.f : 1.f / l) : 1.f;
            T *out = static_cast<T *>(p.out) + at * kHeadDim;
            const size_t part = (size_t)split * p.total * p.hq + at;
            if (!direct && valid) p.part_ml[part] = make_float2(m, l);
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                uint32_t x[32];
                tmem_ld32(t_o + 32 * c, x);  // by whole warps: rows that are none are loaded, not stored
                tmem_wait_ld(x);
#pragma unroll
                for (int k = 0; k < 32; k += 4) {
                    float f[4];
#pragma unroll
                    for (int d = 0; d < 4; ++d) {
                        f[d] = fmaf(__uint_as_float(x[k + d]), back, z);
                        if (merge) f[d] = f[d] * mine + shared_o[(32 * c + k + d) * 128 + r] * other;
                        f[d] *= inv;
                    }
                    if (valid) {
                        if (direct)
                            store_out4<T>(out + 32 * c + k, f[0], f[1], f[2], f[3]);
                        else
                            *reinterpret_cast<float4 *>(p.part_o + part * kHeadDim + 32 * c + k) =
                                make_float4(f[0], f[1], f[2], f[3]);
                    }
                }
                __syncwarp();
            }
        }
        tc_fence_before();
    }
    __syncthreads();
    if (warp == kMmaWarp) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
    }
}

// out[row] of the rows whose keys were split: one warp per row, 4 dims a lane.
template <typename T>
__global__ void __launch_bounds__(256) attend_combine_kernel(const __grid_constant__ ChunkParams p, int tile_rows) {
    grid_dependency_wait();
    const size_t row = (size_t)blockIdx.x * 8 + (threadIdx.x >> 5);
    const int lane = threadIdx.x & 31, t = (int)(row / p.hq), h = (int)(row % p.hq);
    if (t >= p.total) return;
    int s = -1;
    for (int s0 = 0; s0 < p.batch && s < 0; s0 += 32) {
        const int i = s0 + lane;
        const uint32_t hit = __ballot_sync(0xffffffffu, i < p.batch && p.q_start[i] >= 0 && p.q_start[i] <= t && t < p.q_start[i + 1]);
        if (hit) s = s0 + __ffs(hit) - 1;
    }
    if (s < 0) return;
    const int tile = ((t - p.q_start[s]) * p.group + h % p.group) / tile_rows;
    const int splits = row_tile(p, s, tile, tile_rows).splits;
    if (splits == 1) return;
    const size_t step = (size_t)p.total * p.hq;
    float M = -CUDART_INF_F;
    for (int c = lane; c < splits; c += 32) M = fmaxf(M, p.part_ml[c * step + row].x);
#pragma unroll
    for (int o = 16; o; o >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, o));
    float L = 0.f;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
    for (int c = 0; c < splits; ++c) {
        const float2 ml = p.part_ml[c * step + row];
        const float4 v = reinterpret_cast<const float4 *>(p.part_o + (c * step + row) * kHeadDim)[lane];
        const float w = ml.x == -CUDART_INF_F ? 0.f : ex2(ml.x - M);
        L += w * ml.y;
        acc.x += w * v.x, acc.y += w * v.y, acc.z += w * v.z, acc.w += w * v.w;
    }
    const float inv = L == 0.f ? 0.f : 1.f / L;
    store_out4<T>(static_cast<T *>(p.out) + row * kHeadDim + 4 * lane, acc.x * inv, acc.y * inv, acc.z * inv, acc.w * inv);
}

constexpr int kMinChunk = 4;  // key tiles: below, a CTA's start and end outweigh its work

int key_tiles(int max_pages) { return (max_pages + kTilePages - 1) / kTilePages; }

// Key tiles of a split: one split while the row tiles (an upper bound of them)
// fill the SMs, else as many as give every SM about two CTAs.
long long most_splits(int batch, long long rows, int hkv, int max_pages, int tile_rows) {
    const long long ctas = (rows / tile_rows + batch) * hkv;
    return std::min<long long>(std::max<long long>(1, 2LL * sm_count() / ctas), std::max(1, key_tiles(max_pages) / kMinChunk));
}

template <typename T, bool kSplit>
int launch_attend(ChunkParams &p, void *workspace, cudaStream_t st) {
    constexpr int tile_rows = kSplit ? 128 : 256;
    auto kern = attend_chunk_kernel<T, kSplit>;
    static std::atomic<bool> attr_done[kMaxDevices];
    if (ensure_smem_attr(attr_done, kern, kChunkSmem) != KVX_OK) return KVX_ECUDA;
    const long long rows = (long long)p.total * p.group;
    const int tiles = key_tiles(p.max_pages);
    const long long most = most_splits(p.batch, rows, p.hkv, p.max_pages, tile_rows);
    p.chunk = (int)((tiles + most - 1) / most);
    const int splits = (tiles + p.chunk - 1) / p.chunk;
    const size_t all = (size_t)p.total * p.hq;
    p.part_o = static_cast<float *>(workspace);
    p.part_ml = reinterpret_cast<float2 *>(p.part_o + (size_t)splits * all * kHeadDim);
    const dim3 grid((unsigned)(rows / tile_rows + p.batch), (unsigned)p.hkv, (unsigned)splits);
    kern<<<grid, kChunkThreads, kChunkSmem, st>>>(p);
    int rc = launch_status();
    if (rc != KVX_OK || splits == 1) return rc;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)((all + 7) / 8));
    cfg.blockDim = dim3(256);
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    if (cudaLaunchKernelEx(&cfg, attend_combine_kernel<T>, p, tile_rows) != cudaSuccess) {
        cudaGetLastError();
        return KVX_ECUDA;
    }
    return launch_status();
}

}  // namespace
}  // namespace kvx

using namespace kvx;

// For every call of at most this many sequences, tokens and pages: with
// ctas >= hkv * (rows / tile_rows + 1), splits * rows * hkv < 2 SMs * tile_rows.
extern "C" KVX_API size_t kvx_attend_chunk_workspace_bytes(int32_t batch, int32_t total_tokens, int32_t num_q_heads,
                                                           int32_t num_kv_heads, int32_t max_pages) {
    if (batch <= 0 || total_tokens <= 0 || num_q_heads <= 0 || num_kv_heads <= 0 || num_q_heads % num_kv_heads ||
        max_pages <= 0)
        return 0;
    const long long splits = most_splits(1, 1, num_kv_heads, max_pages, 128);
    if (splits == 1) return 16;
    const long long rows = std::min(splits * total_tokens * num_q_heads, 2LL * sm_count() * 256);
    return (size_t)std::max(rows, 1LL) * (kHeadDim + 2) * sizeof(float) / 16 * 16 + 16;
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
    if (kv->num_kv_heads > 65535 || max_pages > (0x7fffffff - kTileKeys) / kPageTokens ||
        (long long)total_tokens * num_q_heads > 0x3fffffff)
        return KVX_EUNSUPPORTED;  // grid, key and row counts fit an int
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
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    return io_dtype == KVX_F16 ? launch_attend<__half, false>(p, workspace, st) : launch_attend<float, true>(p, workspace, st);
}
