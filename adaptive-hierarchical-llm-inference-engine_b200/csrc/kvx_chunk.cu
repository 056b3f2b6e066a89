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
// A block of one value is stored as scale 1, codes -128, zero point = the value:
// its mid is 128 off what it holds, and a sum of rounded weights times -128
// would not take that back.  block_values() gives such a block scale 0 instead.
//
// Rows: the new tokens of a sequence times the q-heads of a kv-head, token
// major.  A CTA owns a tile of 128 or 256 rows and a range of 128-key tiles
// (8 pages); 5 warpgroups, registers dealt out with setmaxnreg:
//  * loader warp: a bulk copy (TMA) per page and K|V, 2 KB of codes each, into
//    staging slots;
//  * statistics warp: scales and middles of the next tiles, as the softmax
//    takes them;
//  * 2 convert warpgroups (K, V): codes -> fp16 into the 128-byte-swizzled
//    tiles (K: the K-major B operand of Q K^T; V: the MN-major B operand of
//    P V, the same bytes), two stages each;
//  * MMA warp: one lane issues S = Q K^T (M 128, N 128, 8 steps of K 16) and
//    O += P V with P read from tensor memory;
//  * 2 softmax warpgroups, a thread per row: running maximum and sum in
//    registers, P (fp16 high and low parts) written over the columns of S it
//    came from; O stays in
//    tensor memory and is rescaled only when a row's maximum has grown by
//    more than 2^8 (p <= 2^8 until then).
// The two warpgroups have an S and an O each (512 tensor-memory columns in
// all), so one's MMAs run under the other's exponentials.  With 256 rows they
// own 128 each and share every key tile; with 128 they take turns at the key
// tiles of the same rows and are merged at the end.
//
// What bounds it (4096 new tokens behind 28672, 24 q-heads on 8: 2.15 to 2.37
// ms by box and clock, 650 to 720 TFLOP/s of Q K^T and P V counted once, 39 to
// 43 % of the measured bf16 rate): a step of 256 rows x 128 keys takes about
// 6000 cycles.  In it the tensor cores work 3070 (two thirds of it P V's
// two parts), the exponential units 2050, shared memory about 3100 (Q and K
// read by Q K^T, V twice by P V, codes copied in, read and written back as
// fp16), and a warpgroup's own chain is maximum, exponentials, P V, the next
// Q K^T.  Tried before the weights had a low part: 64-key steps with two score
// buffers, which take the MMAs out of that chain (2.19 against 1.80 ms: both
// warpgroups then want the exponentials at once), and P handed over by halves
// (1.85).  Splitting the row tiles of the last, partly filled turn of the SMs
// gave 1.80 -> 1.63 then (384 on 148 SMs).
//
// Sequences of at most 16 rows (a decode step, a few drafted tokens) would use
// an eighth of those tiles: attend_rows_kernel takes them, on mma.sync (8
// sequences of 5 new tokens behind up to 8192 keys, 90 MB of codes: 43 us; as
// of one part a weight 37 us, against 75 us in the tiles above).
//
// P' = p s 2^(7 - E) with 2^E above the largest V scale that the row has seen (not
// that of pages behind its last key, whose range is none of its): at most 2^15
// and normal in fp16 down to p s = 2^-21 of that scale, so a block of small
// scale keeps its precision.  It enters P V as fp16 high + low parts, as in
// kvx_decode: the weights multiply a block's whole range, and one rounding of
// them costs up to 2^-12 of it, which in a block with outliers is far more than
// the output's own rounding (1 % of V a hundred times the rest, 2 to 33 keys:
// off by up to 0.09).  fp16 calls add both parts to the same sums.  The second
// MMA costs 1.62 -> 2.02 ms (4096 new tokens behind 28672), 28.0 -> 30.2 us (a
// prompt of 1001), 38.8 -> 41.2 us (8 x 5 tokens).
//
// Sums: the tensor core cuts the sum that an MMA adds to, always towards zero,
// so a sum of one sign loses a part that grows with its length: 2.9e-4 of it
// over 30,000 keys, 7.2e-4 over 60,000 with both parts in one sum (measured, V
// with an element at the top of its range in every token).  So O is moved out
// of tensor memory every 32 key tiles of a warpgroup (fp32: 8; settle()), and
// loses up to 1.2e-4 of it, less than an fp16 rounding (fp32: 3e-6 measured).
// That costs 2.02 -> 2.15 ms and 217 -> 254 us at the sizes named here; every 16
// and 4 tiles: 2.28 ms, 276 us, 64: 2.08 ms.  attend_rows_kernel adds each
// page's part in fp32 registers (41.2 -> 43.3 us).
//
// fp32 calls: q (scaled to 2^13) enters as high + low parts too, 22 bits or
// more, two MMAs for each product.  The high parts of q are on a grid (multiples
// of 8), so their sums of products with the codes stay below 2^24 grid steps and
// are exact although the tensor core cuts; the low parts of both products have
// sums of their own.  So a row tile is 128 rows, O takes 256 columns (high,
// low), S as many, and the two warpgroups take 64 keys each of every tile, with
// one running maximum.  4 ragged sequences of up to 300 new tokens behind 4096,
// 64 q-heads on 8: 265 us and an error of 5.0e-7 (fp32 products and sums of the
// plain form: 5850 us, 6.2e-7).
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
// fp32 calls: the low part of P' (at most 2^3, half a step of 2^15) enters times
// 2^11, so that it stays normal in fp16 down to a P' of 2^-14 and below.
constexpr float kLowUp = 2048.f;
// What the softmax needs of a key tile's statistics.
constexpr int kStatSlots = 4;
struct TileStats {
    float4 page[kTilePages];  // K: scale, mid (times the softmax scale, log2); V: scale, mid
    int exponent;             // 2^exponent is above every V scale up to this tile
    uint32_t known;           // bit i: page i is there
    uint32_t pad[2];
};
constexpr int kBarBytes = 320;
// shared memory: Q0, Q1 (staging slots 2, 3 when unused), K x 2, V x 2, staging x 2, the rest
constexpr int kAtK = 2 * kTileBytes, kAtV = kAtK + 2 * kTileBytes, kAtStage = kAtV + 2 * kTileBytes,
              kAtMisc = kAtStage + 2 * kSlotBytes, kChunkSmem = 1024 + kAtMisc + kBarBytes + kStatSlots * (int)sizeof(TileStats) + 256 * 4;
static_assert(kChunkSmem <= 227 * 1024, "chunk attention exceeds the shared memory of a CTA");
// Key tiles of a warpgroup after which O is taken out of tensor memory.
template <bool kSplit> constexpr int kSettle = kSplit ? 8 : 32;
constexpr float kLazy = 8.f;  // log2 of the growth of a row's maximum that is let pass

struct ChunkParams {
    const uint8_t *pool;
    const float *stats;
    const int32_t *block_table, *q_start, *positions;
    const void *q;
    void *out;
    float *part_o;     // attend_chunk_kernel, split row tiles: [piece][tile_rows][128]
    float2 *part_ml;   // [piece][tile_rows]
    float *few_o;      // attend_rows_kernel: [CTA][2][16][128]
    float2 *few_ml;    // [CTA][2][16]
    int32_t *error_flag;
    int batch, total, hq, hkv, group, max_pages, num_pages, causal;
    int followed;  // attend_chunk_kernel is not the call's last launch
    int sms, max_tiles, max_pieces, max_splits;  // attend_chunk_kernel: row tiles, pieces of split ones, of one of them
    int tile_rows, tile_shift;  // attend_chunk_kernel: rows of a CTA (and log2 of it)
    int few_ctas, few_keys;  // attend_rows_kernel: CTAs; log2 of a unit's keys
    int few_rows;          // sequences of at most so many rows are attend_rows_kernel's (0: none)
    float scale_log2;
};

// Rows of one (sequence, row tile): what the kernel and the combine agree on.
struct RowTile {
    int begin, n;      // packed rows of the sequence
    int pos, rows;     // rows in the tile
    int keys, tiles;   // keys the tile's last row sees, in 128-key tiles
    int splits, chunk; // pieces, key tiles of a piece
};

struct ChunkBars {
    uint64_t ld_full[4], ld_empty[4], stat_full[kStatSlots], stat_empty[kStatSlots], k_full[2], k_empty[2], v_full[2], v_empty[2], s_full[2], p_full[2], q_full, done;
    uint32_t tmem, gave_up;
    uint32_t known[4];  // staging slot: bit i, page i was loaded
    int seq, tile, kvh, split, part;
    RowTile rt;
};
static_assert(sizeof(ChunkBars) <= kBarBytes);


// {scale, zero point} of a block's statistics {min, max, scale, zero point};
// scale 0 for a block of one value (stored with scale 1).
__device__ __forceinline__ float2 block_values(const float4 &st) {
    return make_float2(st.x == st.y && st.z == 1.f && st.w == st.x ? 0.f : st.z, st.w);
}

__device__ __forceinline__ int sequence_tokens(const ChunkParams &p, int s) {
    const int a = p.q_start[s], b = min(p.q_start[s + 1], p.total);
    return a >= 0 && b > a ? b - a : 0;
}

__device__ __forceinline__ int row_keys(const ChunkParams &p, const RowTile &t, int row) {
    if (t.pos < 0) return 0;
    const long long k = (long long)t.pos + (p.causal ? row / p.group + 1 : t.n);
    return (int)min(k, (long long)p.max_pages * kPageTokens);
}

// A CTA's start and end, in key tiles.
__host__ __device__ constexpr int piece_start(int tile_rows) { return tile_rows == 256 ? 6 : 8; }
constexpr int kMinChunk = 4;  // key tiles of a piece: below, a CTA's start and end outweigh its work

__device__ __forceinline__ RowTile row_tile(const ChunkParams &p, int s, int tile, int tile_rows, int pieces) {
    RowTile t;
    t.begin = p.q_start[s];
    t.n = sequence_tokens(p, s);
    t.pos = p.positions[s];
    const int all = t.n * p.group;
    t.rows = min(tile_rows, all - tile * tile_rows);
    t.keys = row_keys(p, t, tile * tile_rows + t.rows - 1);
    t.tiles = (t.keys + kTileKeys - 1) / kTileKeys;
    t.splits = max(1, min(pieces, t.tiles / kMinChunk));
    t.chunk = max(1, (t.tiles + t.splits - 1) / t.splits);
    t.splits = max(1, (t.tiles + t.chunk - 1) / t.chunk);
    return t;
}

// The (row tile, kv-head) pairs by rank: kv-heads next to one another, the
// last row tiles first (causal: they have the most keys).  A CTA, of which an
// SM holds one, takes a pair, but those of the last, partly filled turn of
// the SMs are split by keys so that the turn is filled: one pair in `pieces`.
struct ChunkWork {
    int tiles;   // row tiles of all sequences
    int pairs;   // tiles * hkv
    int whole;   // ranks below are not split
    int pieces;  // of each of the others (at most: of at least kMinChunk key tiles each)
};
__device__ __forceinline__ int chunk_tiles(const ChunkParams &p, int s) {
    const int rows = sequence_tokens(p, s) * p.group;
    return rows > p.few_rows ? (rows + p.tile_rows - 1) >> p.tile_shift : 0;
}
// By a whole warp.  mine: the row tiles of sequence `lane`.
__device__ __forceinline__ ChunkWork chunk_work(const ChunkParams &p, int *mine) {
    const int lane = threadIdx.x & 31;
    int tiles = 0;
    unsigned longest = 0;  // key tiles
    *mine = 0;
    for (int s = lane; s < p.batch; s += 32) {
        const int pos = p.positions[s], n = sequence_tokens(p, s), t = n * p.group > p.few_rows ? (n * p.group + p.tile_rows - 1) >> p.tile_shift : 0;
        tiles += t;
        if (s == lane) *mine = t;
        if (t && pos >= 0)
            longest = max(longest, ((unsigned)min((long long)pos + n, (long long)p.max_pages * kPageTokens) + kTileKeys - 1) / kTileKeys);
    }
    ChunkWork w;
    // a q_start that does not ascend may claim more rows than there are
    w.tiles = min(__reduce_add_sync(0xffffffffu, tiles), p.max_tiles);
    w.pairs = w.tiles * p.hkv;
    const int rest = w.pairs % p.sms;
    w.whole = w.pairs - rest;
    w.pieces = 1;
    longest = __reduce_max_sync(0xffffffffu, longest);
    if (rest && longest >= 2 * kMinChunk) {
        // Least of turns x (key tiles + a CTA's start and end, 10 us), and for
        // partial results their writing and reading (64 pieces: a key tile's
        // time) and the combine, in 64ths of a key tile.  Against 3 key tiles
        // for a CTA and nothing for the rest: 2600 tokens behind 2000 (24 q-heads
        // on 8) 183 and 224 us, 1001 behind 3000 (64 on 8) 199 and 235, 3500
        // behind 30000 (24 on 8) 2057 and 2045 to 2075.
        const unsigned start = piece_start(p.tile_rows);
        const int most = min(min(p.max_splits, (int)longest / kMinChunk), p.max_pieces / rest);
        unsigned best = 0xffffffffu, at = 1;
        for (int n = 1 + lane; n <= most; n += 32) {
            const unsigned cost =
                64u * ((rest * n + p.sms - 1) / p.sms) * ((longest + n - 1) / n + start) + (n > 1 ? rest * n + 128 : 0);
            if (cost < best) best = cost, at = n;
        }
        w.pieces = (int)__reduce_min_sync(0xffffffffu, best == __reduce_min_sync(0xffffffffu, best) ? at : 0xffffffffu);
    }
    return w;
}
// By a whole warp: the sequence of row tile x, *x becomes its tile there (-1:
// none).  mine as of chunk_work.
__device__ __forceinline__ int chunk_sequence(const ChunkParams &p, int mine, int *x) {
    const int lane = threadIdx.x & 31;
    int before = 0;
    for (int s0 = 0; s0 < p.batch; s0 += 32) {
        if (s0) mine = s0 + lane < p.batch ? chunk_tiles(p, s0 + lane) : 0;
        int sum = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int y = __shfl_up_sync(0xffffffffu, sum, o);
            if (lane >= o) sum += y;
        }
        const uint32_t hit = __ballot_sync(0xffffffffu, *x < before + sum);
        if (hit) {
            const int l = __ffs(hit) - 1;
            *x -= before + __shfl_sync(0xffffffffu, sum - mine, l);
            return s0 + l;
        }
        before += __shfl_sync(0xffffffffu, sum, 31);
    }
    return -1;
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

template <typename T> __device__ __forceinline__ void load_q4(const T *p, float *f);
template <> __device__ __forceinline__ void load_q4<__half>(const __half *p, float *f) {
    const uint2 w = *reinterpret_cast<const uint2 *>(p);
    const float2 a = h2_to_f2(w.x), b = h2_to_f2(w.y);
    f[0] = a.x, f[1] = a.y, f[2] = b.x, f[3] = b.y;
}
template <> __device__ __forceinline__ void load_q4<float>(const float *p, float *f) {
    const float4 v = *reinterpret_cast<const float4 *>(p);
    f[0] = v.x, f[1] = v.y, f[2] = v.z, f[3] = v.w;
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
    const int tile_rows = p.tile_rows;
    extern __shared__ __align__(1024) uint8_t chunk_smem[];
    uint8_t *sm = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(chunk_smem) + 1023) & ~uintptr_t(1023));
    const uint32_t base = smem_addr(sm);
    ChunkBars *bars = reinterpret_cast<ChunkBars *>(sm + kAtMisc);
    TileStats *tile_stats = reinterpret_cast<TileStats *>(sm + kAtMisc + kBarBytes);
    float *row_sum = reinterpret_cast<float *>(tile_stats + kStatSlots), *row_unscale = row_sum + 128;  // [256]; fp32 calls: [128] each
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

    // A launch of this call may place its CTAs; it waits for this grid.  The
    // call's last launch lets nothing start: kvx_decode reads its queries and
    // pages before it waits.
    if (p.followed) grid_dependents_launch();
    // ---- which rows, which keys
    if (warp == 0) {
        int mine;
        const ChunkWork work_of = chunk_work(p, &mine);
        const int b = (int)blockIdx.x - work_of.whole;
        const int rank = b < 0 ? (int)blockIdx.x : work_of.whole + b / work_of.pieces;
        int tile = work_of.tiles - 1 - rank / p.hkv;
        const int seq = rank < work_of.pairs ? chunk_sequence(p, mine, &tile) : -1;
        if (lane == 0) {
            if (seq >= 0) bars->rt = row_tile(p, seq, tile, tile_rows, b < 0 ? 1 : work_of.pieces);
            bars->seq = seq;
            bars->tile = tile;
            bars->kvh = rank % p.hkv;
            bars->split = b < 0 ? 0 : b % work_of.pieces;
            bars->part = b;
            bars->gave_up = 0;
        }
    }
    // ---- meanwhile barriers and tensor memory
    if (threadIdx.x == 32) {
        for (int i = 0; i < 4; ++i) {
            mbar_init(&bars->ld_full[i], 1);
            mbar_init(&bars->ld_empty[i], 4);
        }
        for (int i = 0; i < kStatSlots; ++i) {
            mbar_init(&bars->stat_full[i], 1);
            mbar_init(&bars->stat_empty[i], 8);  // the softmax warps that look at a tile (alternate: 4, twice each)
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(&bars->k_full[i], 4);
            mbar_init(&bars->k_empty[i], 1);
            mbar_init(&bars->v_full[i], 4);
            mbar_init(&bars->v_empty[i], 1);
            mbar_init(&bars->s_full[i], kSplit && i == 1 ? 256 : 1);  // fp32: [1] says that the scores are read
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
    auto release = [&] {
        if (warp == kMmaWarp)
            asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(bars->tmem) : "memory");
    };
    const int seq = bars->seq, tile = bars->tile, kvh = bars->kvh, split = bars->split;
    const RowTile rt = bars->rt;
    if (seq < 0 || split >= rt.splits) {  // the grid is an upper bound
        release();
        return;
    }
    const int row0 = tile * tile_rows;
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
        release();
        return;
    }
    const int t0 = split * rt.chunk, tiles = min(rt.chunk, rt.tiles - t0);  // this CTA's key tiles
    // the warpgroups take the same rows: whole key tiles in turn, or (fp32) both
    // halves of each
    const bool turns = kSplit || rt.rows <= 128, alternate = turns && !kSplit;
    const int items = turns ? tiles : 2 * tiles;  // item w: warpgroup w % 2 (fp32: both), key tile w or w / 2
    // 4 or 2 staging slots (two are Q1's place, which settle() takes in long runs)
    const int slot_bits = alternate && tiles <= 2 * kSettle<kSplit> ? 2 : 1, slot_mask = (1 << slot_bits) - 1;
    const int32_t *table = p.block_table + (size_t)seq * p.max_pages;
    // S0, S1, O0, O1: 128 columns each.  All 512 columns were asked for, so
    // they begin at 0 (were they to begin elsewhere, nothing is done).
    constexpr uint32_t tmem = 0;
    if (bars->tmem != 0) {
        if (threadIdx.x == 0 && p.error_flag) atomicOr(p.error_flag, 1);
        release();
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
                const float2 cur = block_values(stat);
                id = id_next;
                stat = stat_of(id);
                id_next = page_of(i + 2);
                // scales that are no numbers do not count
                const int e = lane >= 8 && lane < 16 && fabsf(cur.x) < CUDART_INF_F ? exponent_above(cur.x) : -100;
                E = max(E, __reduce_max_sync(0xffffffffu, e));
                const float mid = fmaf(128.f, cur.x, cur.y), f = lane < 8 ? p.scale_log2 : 1.f;
                TileStats &t = tile_stats[i & (kStatSlots - 1)];
                wait_or_give_up(&bars->stat_empty[i & (kStatSlots - 1)], (i / kStatSlots & 1) ^ 1, bars, p.error_flag);
                // a K scale below 2^-70 becomes that: the -inf of a masked key stays
                // one also times an fp32 row's 2^-50 (row_unscale), and products
                // below 2^30 of the others stay nothing
                if (lane < 16)
                    reinterpret_cast<float2 *>(&t.page[lane & 7])[lane >> 3] =
                        make_float2(lane < 8 && cur.x * f < 0x1p-70f ? 0x1p-70f : cur.x * f, mid * f);
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
            if constexpr (kSplit) {
                // P V of a key tile and the scores of the next; high and low parts
                // have sums of their own.  The low scores' columns are free as
                // soon as they are read: the next ones come under the exponentials.
                const uint32_t q = umma_desc_low(at, 16);
#pragma unroll 1
                for (int i = -1; i < u_items; ++i) {
                    const int st = (i + 1) & 1;
                    const uint32_t k = umma_desc_low(at + kAtK + st * kTileBytes, 16);
                    auto scores = [&](int part) {
#pragma unroll
                        for (int ks = 0; ks < 8; ++ks) {
                            const uint32_t off = ((ks >> 2) * kHalfBytes + (ks & 3) * 32) >> 4;
                            umma_f16_ss(issues, tmem + part * 128, q + ((part * kTileBytes >> 4) + off), k + off, kIdescQK, ks);
                        }
                    };
                    if (i + 1 < u_items) {
                        wait_or_give_up(&bars->k_full[st], ((i + 1) >> 1) & 1, bars, p.error_flag);
                        if (i >= 0) wait_or_give_up(&bars->s_full[1], i & 1, bars, p.error_flag);
                        tc_fence_after();
                        scores(1);
                    }
                    if (i >= 0) {
                        wait_or_give_up(&bars->v_full[i & 1], (i >> 1) & 1, bars, p.error_flag);
                        wait_or_give_up(&bars->p_full[0], i & 1, bars, p.error_flag);
                        wait_or_give_up(&bars->p_full[1], i & 1, bars, p.error_flag);
                        tc_fence_after();
                        const uint32_t v = umma_desc_low(at + kAtV + (i & 1) * kTileBytes, kHalfBytes);
#pragma unroll
                        for (int part = 0; part < 2; ++part)
#pragma unroll
                            for (int ks = 0; ks < 8; ++ks)
                                umma_f16_ts(issues, tmem + 256 + part * 128, tmem + ks * 16 + part * 8, v + (ks * 2048 >> 4), kIdescPV, i | ks);
                        umma_commit(issues, &bars->v_empty[i & 1]);
                    }
                    if (i + 1 < u_items) {
                        scores(0);
                        umma_commit(issues, &bars->s_full[0]);
                        umma_commit(issues, &bars->k_empty[st]);
                    }
                }
            } else {
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
                    for (int ks = 0; ks < 16; ++ks)  // a page: its P, high and low, over its columns of S
                        umma_f16_ts(issues, tmem + 256 + j * 128, tmem + j * 128 + ks * 8, v + ((ks >> 1) * 2048 >> 4), kIdescPV, (w > 1) | ks);
                    if (u_turns || j) umma_commit(issues, &bars->v_empty[st]);
                }
                if (w + 2 < u_items) {
                    const int i = u_turns ? w + 2 : (w + 2) >> 1, st = i & 1;
                    wait_or_give_up(&bars->k_full[st], (i >> 1) & 1, bars, p.error_flag);
                    tc_fence_after();
                    const uint32_t q = umma_desc_low(at + (u_turns ? 0 : j * kTileBytes), 16),
                                   k = umma_desc_low(at + kAtK + st * kTileBytes, 16);
#pragma unroll
                    for (int ks = 0; ks < 8; ++ks) {
                        const uint32_t off = ((ks >> 2) * kHalfBytes + (ks & 3) * 32) >> 4;
                        umma_f16_ss(issues, tmem + j * 128, q + off, k + off, kIdescQK, ks);
                    }
                    umma_commit(issues, &bars->s_full[j]);
                    if (u_turns || j) umma_commit(issues, &bars->k_empty[st]);
                }
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
        // fp32: this warpgroup's half of the keys, high parts (the low ones 128 columns on)
        const uint32_t t_s = tmem + j * (kSplit ? 64 : 128) + lanes, t_o = tmem + 256 + j * 128 + lanes;
        const int my_row = turns ? r : j * 128 + r;
        const bool valid = my_row < rt.rows;
        // Q: 16 loads of 512 contiguous bytes a warp, all in flight at once
        // (fp16: 2 rows each, fp32: 1); rows that are none are zero
        {
            const int rows_all = turns ? 128 : 256;
            constexpr int kUnits = 16, kPerUnit = kSplit ? 1 : 2;
            uint4 x[kUnits];
            const int first = warp * kUnits * kPerUnit, mine = first + (lane & (kUnits * kPerUnit - 1));
            const int at = mine < rt.rows ? (int)row_index(mine) : 0;  // total * hq fits an int
#pragma unroll
            for (int u = 0; u < kUnits; ++u) {
                const int i = u * kPerUnit + (kSplit ? 0 : lane >> 4), row_at = __shfl_sync(0xffffffffu, at, i);
                x[u] = make_uint4(0, 0, 0, 0);
                if (first + i < rt.rows)
                    x[u] = *reinterpret_cast<const uint4 *>(static_cast<const T *>(p.q) + (size_t)row_at * kHeadDim +
                                                            (kSplit ? 4 * lane : 8 * (lane & 15)));
            }
#pragma unroll
            for (int u = 0; u < kUnits; ++u) {
                const int row = (warp * kUnits + u) * kPerUnit + (kSplit ? 0 : lane >> 4);
                const uint32_t dst = base + (row >> 7) * kTileBytes;
                if constexpr (!kSplit) {
                    if (row < rows_all) st_shared16(dst + tile_chunk(row & 127, lane & 15), x[u].x, x[u].y, x[u].z, x[u].w);
                } else {
                    // Scaled to 2^13.  The high part is a multiple of 8, so its
                    // product with the codes is below 2^24 eights: exact, however
                    // the tensor core rounds.  The low part is the rest (to 2^-9).
                    const float f[4] = {__uint_as_float(x[u].x), __uint_as_float(x[u].y), __uint_as_float(x[u].z), __uint_as_float(x[u].w)};
                    uint32_t big = 0, hi[2], lo[2];
#pragma unroll
                    for (int k = 0; k < 4; ++k) big = max(big, __float_as_uint(fabsf(f[k])));
                    big = __reduce_max_sync(0xffffffffu, big);
                    const int e = big > 0 && big < 0x7f800000u ? max(exponent_above(__uint_as_float(big)), -37) : 13;
                    const float up = pow2i(13 - e);
#pragma unroll
                    for (int k = 0; k < 2; ++k) {
                        const float a = f[2 * k] * up, b = f[2 * k + 1] * up;
                        hi[k] = pack_half(rintf(a * 0.125f) * 8.f, rintf(b * 0.125f) * 8.f);
                        const float2 h = h2_to_f2(hi[k]);
                        lo[k] = pack_half(a - h.x, b - h.y);
                    }
                    const uint32_t at = dst + tile_chunk(row, lane >> 1) + 8 * (lane & 1);
                    asm volatile("st.shared.v2.b32 [%0], {%1, %2};" ::"r"(at), "r"(hi[0]), "r"(hi[1]) : "memory");
                    asm volatile("st.shared.v2.b32 [%0], {%1, %2};" ::"r"(at + kTileBytes), "r"(lo[0]), "r"(lo[1]) : "memory");
                    if (lane == 0) row_unscale[row] = pow2i(e - 13);
                }
            }
            fence_proxy_async_smem();
            mbar_arrive(&bars->q_full);
            // the rows' sums: the 16 lanes (fp32: 32) of each of the 16 units, so
            // that lane u ends with unit u's
            float sum[kUnits];
#pragma unroll
            for (int u = 0; u < kUnits; ++u) {
                if constexpr (kSplit) {
                    sum[u] = (__uint_as_float(x[u].x) + __uint_as_float(x[u].y)) + (__uint_as_float(x[u].z) + __uint_as_float(x[u].w));
                } else {
                    const float2 a = h2_to_f2(x[u].x), b = h2_to_f2(x[u].y), c = h2_to_f2(x[u].z), d = h2_to_f2(x[u].w);
                    sum[u] = ((a.x + a.y) + (b.x + b.y)) + ((c.x + c.y) + (d.x + d.y));
                }
            }
#pragma unroll
            for (int n = kUnits / 2; n; n >>= 1) {
                const bool upper = lane & n;
#pragma unroll
                for (int u = 0; u < n; ++u) {
                    const float keep = upper ? sum[u + n] : sum[u], give = upper ? sum[u] : sum[u + n];
                    sum[u] = keep + __shfl_xor_sync(0xffffffffu, give, n);
                }
            }
            if constexpr (kSplit) sum[0] += __shfl_xor_sync(0xffffffffu, sum[0], 16);
            if (!kSplit || lane < 16) row_sum[first + (lane & 15) * kPerUnit + (kSplit ? 0 : lane >> 4)] = sum[0];
            asm volatile("bar.sync 1, 256;" ::: "memory");
        }
        const float q_sum = row_sum[my_row], unscale = kSplit ? row_unscale[r] : 1.f;
        if (kSplit) asm volatile("bar.sync 1, 256;" ::: "memory");  // row_sum, row_unscale are free
        const int limit = valid ? row_keys(p, rt, row0 + my_row) : 0x7fffffff;  // a row that is none needs no mask
        const int step = alternate ? 2 : 1;
        // the columns of O that this thread looks after, 16 at a time: its own O's
        // (fp32: its half of the dims, high parts, then low parts)
        auto o_at = [&](int c) { return kSplit ? tmem + 256 + lanes + (c >> 2) * 128 + 64 * j + 16 * (c & 3) : t_o + 16 * c; };
        // O by f (rare, so in little code)
        auto scale_o = [&](float f) {
#pragma unroll 1
            for (int c = 0; c < 8; ++c) {
                uint32_t o[16];
                tmem_ld16(o_at(c), o);
                tmem_wait_ld(o);
#pragma unroll
                for (int k = 0; k < 16; ++k) o[k] = __float_as_uint(__uint_as_float(o[k]) * f);
                tmem_st16(o_at(c), o);
            }
        };
        // The tensor core cuts every sum it adds to (about 2^-22 of it an MMA, and
        // always towards zero), so every kSettle key tiles O moves on to the row's
        // place in the output or in the partial results, times 1 / settled.  fp16
        // rows there hold the nearest fp16 (of at most 2^15: |O| <= 2^14 l) and the
        // rest, exact, stays in O; the second of two warpgroups with the same rows
        // has Q1's place in shared memory.
        float settled = 0.f;  // 0: nothing there yet
        auto home = [&] {
            return rt.splits == 1 ? static_cast<uint8_t *>(p.out) + row_index(my_row) * (kHeadDim * sizeof(T))
                                  : reinterpret_cast<uint8_t *>(p.part_o + ((size_t)bars->part * tile_rows + my_row) * kHeadDim);
        };
        auto home_vec = [&](uint8_t *at, int k) {  // its 16-byte vector k
            return reinterpret_cast<uint4 *>(alternate && j ? sm + kTileBytes + tile_chunk(r, k) : at + 16 * k);
        };
        constexpr int kVec = 16 / (int)sizeof(T);
        auto vec_dims = [&](const uint4 &w, float *h) {
            if constexpr (kSplit) {
                h[0] = __uint_as_float(w.x), h[1] = __uint_as_float(w.y), h[2] = __uint_as_float(w.z), h[3] = __uint_as_float(w.w);
            } else {
                const float2 a = h2_to_f2(w.x), b = h2_to_f2(w.y), d = h2_to_f2(w.z), e = h2_to_f2(w.w);
                h[0] = a.x, h[1] = a.y, h[2] = b.x, h[3] = b.y, h[4] = d.x, h[5] = d.y, h[6] = e.x, h[7] = e.y;
            }
        };
        auto settle = [&](float l) {  // rows that are none have no home
            uint8_t *at = home();
            if constexpr (kSplit) {  // added in memory: nothing to wait for
                const bool add = settled > 0x1p-60f;
                const float times = add ? 1.f / settled : 1.f;
#pragma unroll 1
                for (int c = 0; c < 4; ++c) {
                    uint32_t o[16], low[16];
                    tmem_ld16(o_at(c), o);
                    tmem_ld16(o_at(c + 4), low);
                    tmem_wait_ld(o);
                    tmem_wait_ld(low);
                    if (valid) {
#pragma unroll
                        for (int k = 0; k < 4; ++k) {
                            float4 *to = reinterpret_cast<float4 *>(at) + 16 * j + 4 * c + k;
                            float f[4];
#pragma unroll
                            for (int d = 0; d < 4; ++d) f[d] = fmaf(__uint_as_float(low[4 * k + d]), 1.f / kLowUp, __uint_as_float(o[4 * k + d])) * times;
                            if (add) {
                                asm volatile("red.global.add.v4.f32 [%0], {%1, %2, %3, %4};" ::"l"(to), "f"(f[0]), "f"(f[1]), "f"(f[2]), "f"(f[3]) : "memory");
                            } else {
                                const float4 old = settled != 0.f ? __ldcg(to) : make_float4(0.f, 0.f, 0.f, 0.f);
                                *to = make_float4(fmaf(old.x, settled, f[0]), fmaf(old.y, settled, f[1]), fmaf(old.z, settled, f[2]), fmaf(old.w, settled, f[3]));
                            }
                        }
                    }
#pragma unroll
                    for (int k = 0; k < 16; ++k) o[k] = 0;
                    tmem_st16(o_at(c), o);
                    tmem_st16(o_at(c + 4), o);
                }
                if (!add) settled = 1.f;
            } else {
                const int e = min(exponent_above(l), 100);
                const float down = pow2i(e - 1), up = pow2i(1 - e);
#pragma unroll 1
                for (int b = 0; b < 16; b += 8) {
                    uint4 w[8];  // asked for together
#pragma unroll
                    for (int k = 0; k < 8; ++k) w[k] = settled != 0.f && valid ? *home_vec(at, b + k) : make_uint4(0, 0, 0, 0);
#pragma unroll
                    for (int c = 0; c < 4; ++c) {
                        uint32_t o[16], u[8];
                        tmem_ld16(o_at(b / 2 + c), o);
                        tmem_wait_ld(o);
                        float h[16];
                        vec_dims(w[2 * c], h);
                        vec_dims(w[2 * c + 1], h + 8);
#pragma unroll
                        for (int k = 0; k < 16; ++k) h[k] = fmaf(h[k], settled, __uint_as_float(o[k]));
#pragma unroll
                        for (int k = 0; k < 8; ++k) {
                            u[k] = pack_half(h[2 * k] * up, h[2 * k + 1] * up);
                            const float2 g = h2_to_f2(u[k]);
                            o[2 * k] = __float_as_uint(fmaf(g.x, -down, h[2 * k]));
                            o[2 * k + 1] = __float_as_uint(fmaf(g.y, -down, h[2 * k + 1]));
                        }
                        if (valid) {
                            *home_vec(at, b + 2 * c) = make_uint4(u[0], u[1], u[2], u[3]);
                            *home_vec(at, b + 2 * c + 1) = make_uint4(u[4], u[5], u[6], u[7]);
                        }
                        tmem_st16(o_at(b / 2 + c), o);
                    }
                }
                settled = down;
            }
            tmem_wait_st();
        };
        // the 64 scores of pages c .. c + kStep - 1
        auto load_scores = [&](int c, uint32_t(&x)[2][32]) {
            if constexpr (kSplit) {
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    uint32_t low[32];
                    tmem_ld32(t_s + 32 * h, x[h]);
                    tmem_ld32(t_s + 32 * h + 128, low);
                    tmem_wait_ld(x[h], low);
#pragma unroll
                    for (int k = 0; k < 32; ++k) x[h][k] = __float_as_uint(__uint_as_float(x[h][k]) + __uint_as_float(low[k]));
                }
            } else {
                tmem_ld32(t_s + 16 * c, x[0]);
                tmem_ld32(t_s + 16 * c + 32, x[1]);
                tmem_wait_ld(x[0], x[1]);
            }
        };
        float m = -CUDART_INF_F, l = 0.f, z = 0.f;  // maximum (log2), sum, sum of p mid
        int E = -100;
        constexpr int kPages = kSplit ? 4 : 8, kStep = 4;  // of an item; of those, at once
        const int page0 = kSplit ? 4 * j : 0;
        int i = alternate ? j : 0;
        for (int w = kSplit ? 0 : j; w < items; w += kSplit ? 1 : 2, i += step) {
            const TileStats &ts = tile_stats[i & (kStatSlots - 1)];
            wait_or_give_up(&bars->stat_full[i & (kStatSlots - 1)], i / kStatSlots & 1, bars, p.error_flag);
            const uint32_t known = kSplit ? ts.known >> page0 & 0xfu : ts.known;
            const auto *stats = ts.page + page0;
            const int seen = limit - (t0 + i) * kTileKeys - page0 * kPageTokens;  // the item's keys that the row sees
            const bool masked = __any_sync(0xffffffffu, seen < kPages * kPageTokens) || known != (1u << kPages) - 1;
            // a page this row sees nothing of: scores of -inf, whatever its statistics
            auto hidden = [&](int page) { return seen <= page * kPageTokens || !(known >> page & 1); };
            const int past = kSplit ? w : w >> 1;  // items in O, or moved on from it
            wait_or_give_up(&bars->s_full[kSplit ? 0 : j], (kSplit ? w : w >> 1) & 1, bars, p.error_flag);
            __syncwarp();
            tc_fence_after();
            if (past && !(past & (kSettle<kSplit> - 1))) settle(l);
            if (masked) {  // few tiles: their scores are masked where they are
#pragma unroll 1
                for (int page = 0; page < kPages; ++page) {
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
            // together has to stay in the instruction cache.  fp32: one chunk, held.
            float top = -CUDART_INF_F;
            uint32_t held[2][32];
#pragma unroll 1
            for (int c = 0; c < kPages; c += kStep) {
                uint32_t fresh[2][32], (&x)[2][32] = kSplit ? held : fresh;
                load_scores(c, x);
                if constexpr (kSplit) {
                    tc_fence_before();
                    mbar_arrive(&bars->s_full[1]);
                }
#pragma unroll
                for (int h = 0; h < kStep; ++h) {
                    const int page = c + h;
                    uint32_t(&v)[32] = x[h >> 1];
                    float2 ks = *reinterpret_cast<const float2 *>(&stats[page]);
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
            if constexpr (kSplit) {  // of both halves of the keys (read before the next scores are asked for)
                row_sum[128 * j + r] = top;
                asm volatile("bar.sync 1, 256;" ::: "memory");
                top = fmaxf(top, row_sum[128 * (j ^ 1) + r]);
            }
            // the largest V scale of the pages that the row has seen (both warpgroups
            // of fp32 calls: of the whole tile); those behind its last key do not count
            int e = ts.exponent;
            const int in_tile = limit - (t0 + i) * kTileKeys;
            if (kSplit ? __any_sync(0xffffffffu, in_tile < kTileKeys) || ts.known != 0xffu : masked) {
                e = E;
#pragma unroll 1
                for (int page = 0; page < kTilePages; ++page) {
                    const float v = ts.page[page].z;
                    if (in_tile > page * kPageTokens && (ts.known >> page & 1) && fabsf(v) < CUDART_INF_F) e = max(e, exponent_above(v));
                }
            }
            // the maximum in use may lag by kLazy; O follows where it catches
            // up, and where a larger V scale came
            const bool lags = __any_sync(0xffffffffu, top > m + kLazy);
            if (lags || __any_sync(0xffffffffu, e > E)) {
                float f = 1.f;
                if (lags) {
                    const float mn = fmaxf(m, top);
                    if (mn != -CUDART_INF_F) f = ex2(m - mn);
                    m = mn;
                    l *= f;
                    z *= f;
                }
                f = E - e < -126 ? 0.f : f * pow2i(E - e);
                if (w >= (kSplit ? 1 : 2)) scale_o(f);
                settled *= f;
                E = e;
            }
            const float m_use = m == -CUDART_INF_F ? 0.f : m, v_up = pow2i(7 - E);
#pragma unroll 1
            for (int c = 0; c < kPages; c += kStep) {
                uint32_t fresh[2][32], (&x)[2][32] = kSplit ? held : fresh;
                if constexpr (!kSplit) load_scores(c, x);
#pragma unroll
                for (int h = 0; h < kStep; ++h) {
                    const int page = c + h;
                    uint32_t(&v)[32] = x[h >> 1];
                    float4 st = stats[page];
                    st.x *= unscale;
                    st.y = fmaf(st.y, q_sum, -m_use);
                    st.z *= v_up;
                    if (masked && hidden(page)) st = make_float4(1.f, 0.f, 0.f, 0.f);
                    const uint64_t aa = pack2(st.x, st.x), bb = pack2(st.y, st.y), ss = pack2(st.z, st.z);
                    uint64_t sum = 0;
                    uint32_t hi[8], lo[8];
#pragma unroll
                    for (int k = 0; k < 16; k += 2) {
                        const float2 t = unpack2(fma2(aa, pack2(__uint_as_float(v[16 * (h & 1) + k]), __uint_as_float(v[16 * (h & 1) + k + 1])), bb));
                        const uint64_t e2 = pack2(ex2(t.x), ex2(t.y));
                        sum = add2(sum, e2);
                        const uint64_t p2 = mul2(e2, ss);
                        const float2 f = unpack2(p2);
                        if constexpr (kSplit) {
                            hi[k / 2] = pack_half(f.x, f.y);
                            const float2 g = h2_to_f2(hi[k / 2]);
                            lo[k / 2] = pack_half((f.x - g.x) * kLowUp, (f.y - g.y) * kLowUp);
                        } else {
                            // high part cut to 11 bits, so that the rest is exact
                            const float a = __uint_as_float(__float_as_uint(f.x) & 0xffffe000u), b = __uint_as_float(__float_as_uint(f.y) & 0xffffe000u);
                            hi[k / 2] = pack_half(a, b);
                            const float2 g = unpack2(fma2(pack2(a, b), pack2(-1.f, -1.f), p2));
                            lo[k / 2] = pack_half(g.x, g.y);
                        }
                    }
                    const float2 both = unpack2(sum);
                    l += both.x + both.y;
                    z = fmaf(both.x + both.y, st.w, z);
                    tmem_st8(t_s + 16 * page, hi);  // over the page's own scores
                    tmem_st8(t_s + 16 * page + 8, lo);
                }
            }
            tmem_wait_st();
            tc_fence_before();
            mbar_arrive(&bars->p_full[j]);
            __syncwarp();
            if (lane == 0) {
                mbar_arrive(&bars->stat_empty[i & (kStatSlots - 1)]);
                if (alternate) mbar_arrive(&bars->stat_empty[i & (kStatSlots - 1)]);
            }
        }

        // ---- O
        wait_or_give_up(&bars->done, 0, bars, p.error_flag);
        __syncwarp();
        tc_fence_after();
        const float back = pow2i(E - 7);
        const bool direct = rt.splits == 1, merge = alternate && items > 1;
        float mine = 1.f, other = 0.f;
        // turns: warpgroup j ends with dims 64 j .. + 63 of all rows, the other
        // half of its sums goes to the other one by shared memory, [dim][row]
        // over K, now free
        float *shared_o = reinterpret_cast<float *>(sm + kAtK);
        // dims 32 c .. + 31 of the row's sums
        auto sums = [&](int c, uint32_t(&x)[32]) {
            if constexpr (kSplit) {
                uint32_t low[32];
                tmem_ld32(tmem + 256 + lanes + 32 * c, x);
                tmem_ld32(tmem + 384 + lanes + 32 * c, low);
                tmem_wait_ld(x, low);
#pragma unroll
                for (int k = 0; k < 32; ++k) x[k] = __float_as_uint(fmaf(__uint_as_float(low[k]), 1.f / kLowUp, __uint_as_float(x[k])));
            } else {
                tmem_ld32(t_o + 32 * c, x);
                tmem_wait_ld(x);
            }
            if (settled != 0.f && valid) {
                uint8_t *at = home();
#pragma unroll
                for (int n = 0; n < 32 / kVec; ++n) {
                    float h[kVec];
                    uint4 *from = home_vec(at, c * (32 / kVec) + n);
                    vec_dims(kSplit ? __ldcg(from) : *from, h);
#pragma unroll
                    for (int k = 0; k < kVec; ++k)
                        x[kVec * n + k] = __float_as_uint(fmaf(h[k], settled, __uint_as_float(x[kVec * n + k])));
                }
            }
        };
        if (merge) {
            float *shared_ml = reinterpret_cast<float *>(sm);  // over Q
#pragma unroll 1
            for (int c = 2 - 2 * j; c < 4 - 2 * j; ++c) {
                uint32_t x[32];
                sums(c, x);
#pragma unroll
                for (int k = 0; k < 32; ++k) shared_o[(32 * c + k) * 128 + r] = fmaf(__uint_as_float(x[k]), back, z);
            }
            shared_ml[256 * j + r] = m;
            shared_ml[256 * j + 128 + r] = l;
            asm volatile("bar.sync 1, 256;" ::: "memory");
            const float m1 = shared_ml[256 * (j ^ 1) + r], l1 = shared_ml[256 * (j ^ 1) + 128 + r], mn = fmaxf(m, m1);
            if (mn != -CUDART_INF_F) {
                mine = ex2(m - mn);
                other = ex2(m1 - mn);
            }
            l = l * mine + l1 * other;
            m = mn;
        }
        if constexpr (kSplit) {
            float *shared_lz = reinterpret_cast<float *>(sm);  // over Q
            shared_lz[256 * j + r] = l;
            shared_lz[256 * j + 128 + r] = z;
            asm volatile("bar.sync 1, 256;" ::: "memory");
            l += shared_lz[256 * (j ^ 1) + r];
            z += shared_lz[256 * (j ^ 1) + 128 + r];
        }
        // alternate without merge: a single tile, which was warpgroup 0's
        const int c0 = merge || kSplit ? 2 * j : 0, chunks = merge || kSplit ? 2 : !turns || j == 0 ? 4 : 0;
        const size_t at = valid ? row_index(my_row) : 0, part = (size_t)bars->part * tile_rows + my_row;
        const float inv = direct ? (l == 0.f ? 0.f : 1.f / l) : 1.f;
        if (!direct && valid && (!turns || j == 0)) p.part_ml[part] = make_float2(m, l);
        // through shared memory (rows 16 bytes longer: no two of 8 lanes in a
        // bank)
        const int size = direct ? (int)sizeof(T) : 4;
        uint8_t *row = sm + (turns ? kAtV : kAtK) + my_row * (kHeadDim * size + 16);
#pragma unroll 1
        for (int c = c0; c < c0 + chunks; ++c) {
            uint32_t x[32];
            sums(c, x);  // by whole warps: rows that are none are loaded, not stored
#pragma unroll
            for (int k = 0; k < 32; k += 8) {
                float f[8];
#pragma unroll
                for (int d = 0; d < 8; ++d) {
                    f[d] = fmaf(__uint_as_float(x[k + d]), back, z);
                    if (merge) f[d] = f[d] * mine + shared_o[(32 * c + k + d) * 128 + r] * other;
                    f[d] *= inv;
                }
                if (sizeof(T) == 2 && direct) {
                    *reinterpret_cast<uint4 *>(row + 2 * (32 * c + k)) =
                        make_uint4(pack_half(f[0], f[1]), pack_half(f[2], f[3]), pack_half(f[4], f[5]), pack_half(f[6], f[7]));
                } else {
                    *reinterpret_cast<float4 *>(row + 4 * (32 * c + k)) = make_float4(f[0], f[1], f[2], f[3]);
                    *reinterpret_cast<float4 *>(row + 4 * (32 * c + k) + 16) = make_float4(f[4], f[5], f[6], f[7]);
                }
            }
        }
        __syncwarp();
        // 16 bytes a lane, whole stretches of rows together (a bulk copy a row
        // took 1.2 us to issue, for all rows of the CTA)
        const int shift = 31 - __clz(max(1, 32 * chunks * size / 16)), some = direct ? (int)at : (int)part;
        const uint32_t rows_there = __ballot_sync(0xffffffffu, valid);
        uint8_t *to = direct ? static_cast<uint8_t *>(p.out) : reinterpret_cast<uint8_t *>(p.part_o);
        const uint8_t *from = row - lane * (kHeadDim * size + 16) + 32 * c0 * size;
        if (chunks)
#pragma unroll 4
            for (int i = lane; i < 32 << shift; i += 32) {
                const int of = i >> shift, byte = 16 * (i & ((1 << shift) - 1));
                const int its = __shfl_sync(0xffffffffu, some, of);
                if (rows_there >> of & 1)
                    *reinterpret_cast<uint4 *>(to + (size_t)its * (kHeadDim * size) + 32 * c0 * size + byte) =
                        *reinterpret_cast<const uint4 *>(from + of * (kHeadDim * size + 16) + byte);
            }
        tc_fence_before();
    }
    __syncthreads();
    if (warp == kMmaWarp) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
    }
}

// ---- at most 16 rows

constexpr int kFewRows = 16;
// Warps of a CTA and CTAs on an SM: as many warps as the registers hold.
template <bool kSplit> constexpr int kFewWarps = kSplit ? 4 : 8;
template <bool kSplit> constexpr int kFewCtas = kSplit ? 3 : 2;
// P' = p s 2^(kFewUp - v_exp) is at most 2^15: p may reach 2^kFewLazy before the
// maximum in use follows.  fp32: little leeway, so that the weights of distant
// keys are normal fp16 numbers (p of 2^-24: 2^-10, high and low part 2^-14 of it).
template <bool kSplit> constexpr int kFewLazy = kSplit ? 1 : 8;
template <bool kSplit> constexpr int kFewUp = 15 - kFewLazy<kSplit>;

__device__ __forceinline__ void mma_f16(float (&c)[4], const uint4 &a, uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a.x), "r"(a.y), "r"(a.z), "r"(a.w), "r"(b0), "r"(b1));
}

// The product alone (a zero accumulator).
__device__ __forceinline__ void mma_f16_zero(float (&c)[4], const uint4 &a, uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %10, %10, %10};"
        : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
        : "r"(a.x), "r"(a.y), "r"(a.z), "r"(a.w), "r"(b0), "r"(b1), "f"(0.f));
}

// 16 bytes, memory to shared memory, in this thread's next group
__device__ __forceinline__ void copy16(uint32_t to, const void *from) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to), "l"(from) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int kLeft> __device__ __forceinline__ void copy_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(kLeft) : "memory"); }

// One page of one head: 16 rows of K, 16 of V, their statistics.  16-byte
// chunk c of row r lies at few_chunk(r, c), so that neither reader (K: the
// same chunk of rows r and r + 1; V: rows r, r + 4, r + 8, r + 12) meets
// itself in a bank.
constexpr int kFewStages = 2;
struct FewPage {
    uint8_t k[kBlockBytes], v[kBlockBytes];
    float4 ks, vs;
};
__device__ __forceinline__ int few_chunk(int row, int chunk) {
    return row * kHeadDim + 16 * (chunk ^ (((row >> 2) << 1) ^ ((row & 1) << 2)));
}
template <bool kSplit> struct FewShared {
    union {
        FewPage page[kFewStages];
        float o[kFewRows][kHeadDim + 4];  // once the warp has no more pages
    } of[kFewWarps<kSplit>];
    uint4 q_frag[kSplit ? 2 : 1][8][32];
    int row_at[kFewRows], row_limit[kFewRows];
    float row_sum[kFewRows], row_unscale[kFewRows], m[kFewWarps<kSplit>][kFewRows], l[kFewWarps<kSplit>][kFewRows];
};

// The work of the sequences of at most 16 rows, one (sequence, kv-head) pair
// after the other, is dealt out to the CTAs in equal ranges, whatever the
// lengths (which the host does not know).  It is counted in units of a page
// for each warp of a CTA (p.few_keys keys).  A pair is kFewStart empty units, then its
// own: what the start and end of a pair cost a CTA, so that one whose range
// holds two ends has less to read (8 x 5 tokens: 43.2 us, with 2 units 42.8; as of
// one part a weight 35.4 and 37.2).
constexpr int kFewStart = 4;
struct FewWork {
    int units;  // of all
    int ctas;   // that have a range (longer than kFewStart, where there are so many)
};

__device__ __forceinline__ int few_units(const ChunkParams &p, int keys) {  // one even where nothing is seen
    return max(1, (keys + (1 << p.few_keys) - 1) >> p.few_keys);
}
__device__ __forceinline__ int few_pair(const ChunkParams &p, int s) {  // units of a pair of the sequence, empty ones included
    const int rows = sequence_tokens(p, s) * p.group;
    return rows > 0 && rows <= p.few_rows ? kFewStart + few_units(p, row_tile(p, s, 0, kFewRows, 1).keys) : 0;
}
__device__ __forceinline__ int few_used(const ChunkParams &p, int units) { return max(1, min(p.few_ctas, units / (kFewStart + 1))); }
// By a whole warp: the work, and the units before sequence `seq`.
__device__ __forceinline__ FewWork few_work(const ChunkParams &p, int seq, int *before) {
    int all = 0, first = 0;
    for (int s = threadIdx.x & 31; s < p.batch; s += 32) {
        const int t = few_pair(p, s) * p.hkv;
        all += t;
        if (s < seq) first += t;
    }
    *before = __reduce_add_sync(0xffffffffu, first);
    FewWork w;
    w.units = __reduce_add_sync(0xffffffffu, all);
    w.ctas = few_used(p, w.units);
    return w;
}
// Ranges of units / ctas units, the first units % ctas of them one longer.
__device__ __forceinline__ int few_begin(const FewWork &w, int cta) {
    return cta * (w.units / w.ctas) + min(cta, w.units % w.ctas);
}
__device__ __forceinline__ int few_owner(const FewWork &w, int unit) {
    const int each = w.units / w.ctas, longer = w.units % w.ctas;
    return unit < longer * (each + 1) ? unit / (each + 1) : (unit - longer) / each;
}

// Sequences of at most 16 rows.  The warps of a CTA take the pages of its
// range in turn; pages come by cp.async into the warp's own stages (no barrier
// in the loop), two ahead (three: 43.9 against 43.2 us at the size below).  The
// codes become the operands of mma.sync (m16n8k16) in registers: the order of
// the dims within Q K^T, and of the keys and dims within P V, is free as long as
// both operands agree, so with g = lane / 4, q = lane % 4
//  * K: a lane reads dims 16 q .. + 15 and 64 + 16 q .. + 15 of key
//    4 (g / 2) + g % 2 (+ 2 for the second n-tile); word s of those 32 bytes
//    is its B fragment of k-step s.  Its scores are then keys 4 q .. 4 q + 3;
//  * V: a lane reads dims 16 g .. + 15 of keys 4 q .. 4 q + 3, transposes them
//    4 x 4 bytes at a time, and has its B fragments of the 16 n-tiles: n-tile
//    t holds dims 16 n + t, so the lane ends with dims 32 q .. 32 q + 31 of O.
// A page is one k-step of P V and has one V scale, which P takes.  Where a
// range ends inside a (sequence, kv-head) pair the rows' partial results go to
// the workspace; a CTA has two such ends at most.
//
// 8 sequences of 5 new tokens behind up to 8192 keys, 24 q-heads on 8: 90 MB
// of codes, 14 us at the copy rate; 34 us here (2.7 TB/s), and 9 us for the
// launch of the empty tiles beside it and the combine.  Issue slots are 54 %
// full (about 800 instructions a page in all, 4 warps a scheduler), the
// start (lengths, page ids, first pages: three dependent reads) is a fifth.
// 8 warps x 2 CTAs an SM against 4 x 4: 40.3 and 42.6 us at the time, for
// fewer starts, ends and partial results.
template <typename T, bool kSplit>
__global__ void __launch_bounds__(kFewWarps<kSplit> * 32, kFewCtas<kSplit>) attend_rows_kernel(const __grid_constant__ ChunkParams p) {
    constexpr int kWarps = kFewWarps<kSplit>;
    extern __shared__ __align__(16) uint8_t few_smem[];
    FewShared<kSplit> &sh = *reinterpret_cast<FewShared<kSplit> *>(few_smem);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, q4 = lane & 3, cta = blockIdx.x;
    grid_dependents_launch();
    // this CTA's units, and the sequence that the first belongs to
    int w0 = 0, w1 = 0, seq = 0, before = 0;  // before: units of earlier sequences
    {
        const int t = lane < p.batch ? few_pair(p, lane) * p.hkv : 0;  // the first 32 sequences, looked at once
        int all = t;
        for (int i = 32 + lane; i < p.batch; i += 32) all += few_pair(p, i) * p.hkv;
        FewWork work_of;
        work_of.units = __reduce_add_sync(0xffffffffu, all);
        work_of.ctas = few_used(p, work_of.units);
        if (cta < work_of.ctas) {
            w0 = few_begin(work_of, cta);
            w1 = few_begin(work_of, cta + 1);
            for (int s0 = 0;; s0 += 32) {
                const int mine = s0 == 0 ? t : (s0 + lane < p.batch ? few_pair(p, s0 + lane) * p.hkv : 0);
                int x = mine;
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) {
                    const int y = __shfl_up_sync(0xffffffffu, x, o);
                    if (lane >= o) x += y;
                }
                const uint32_t hit = __ballot_sync(0xffffffffu, w0 < before + x);
                if (hit || s0 + 32 >= p.batch) {
                    const int at = hit ? __ffs(hit) - 1 : 0;
                    seq = s0 + at;
                    before += __shfl_sync(0xffffffffu, x - mine, at);
                    break;
                }
                before += __shfl_sync(0xffffffffu, x, 31);
            }
        }
    }
    bool later = false;  // not this CTA's first pair
#pragma unroll 1
    for (int w = w0; w < w1;) {
        RowTile rt = row_tile(p, seq, 0, kFewRows, 1);
        const int n_rows = rt.n * p.group, units = n_rows > 0 && n_rows <= p.few_rows ? few_units(p, rt.keys) : 0;
        const int pair = units ? kFewStart + units : 0;
        if (w >= before + pair * p.hkv) {
            before += pair * p.hkv;
            ++seq;
            continue;
        }
        const int kvh = (w - before) / pair, at = (w - before) % pair, unit0 = max(at - kFewStart, 0);
        const int piece = min(pair - at, w1 - w) - max(kFewStart - at, 0);  // units of its own in this range
        w += min(pair - at, w1 - w);
        if (piece <= 0) continue;  // the range ends before them
        const bool whole = piece == units, second = later;
        later = true;
        if (threadIdx.x == 0 && unit0 == 0 && p.error_flag) {
            if (rt.pos < 0) atomicOr(p.error_flag, 2);
            if ((long long)rt.pos + rt.n > (long long)p.max_pages * kPageTokens) atomicOr(p.error_flag, 4);
        }
        const int page0 = unit0 * kWarps, page1 = min(page0 + piece * kWarps, (rt.keys + kPageTokens - 1) / kPageTokens);
        const int32_t *table = p.block_table + (size_t)seq * p.max_pages;
        auto page_of = [&](int lp) { return lp < page1 ? table[lp] : -1; };
        const int key_a = 4 * (g >> 1) + (g & 1);  // key of this lane's column of Q K^T (+ 2 for the second n-tile)
        // this warp's pages page0 + warp, + kWarps, ...: contents kFewStages ahead, ids of 32 at once
        const int first = page0 + warp, count = first < page1 ? (page1 - first + kWarps - 1) / kWarps : 0;
        FewPage *page = sh.of[warp].page;
        int ids = page_of(first + lane * kWarps);
        uint32_t here = 0;  // bit i % 32: page i has an id that is one
        // q is asked for before the pages, and used once they are under way
        auto row_at = [&](int row) { return (rt.begin + row / p.group) * p.hq + kvh * p.group + row % p.group; };
        float q_raw[kFewRows / kWarps][4] = {};
#pragma unroll
        for (int j = 0; j < kFewRows / kWarps; ++j) {
            const int row = warp + kWarps * j;
            if (row < n_rows) load_q4<T>(static_cast<const T *>(p.q) + (size_t)row_at(row) * kHeadDim + 4 * lane, q_raw[j]);
        }
        auto fetch = [&](int i, int stage) {
            if (i < count) {
                if (i && !(i & 31)) ids = page_of(first + (i + lane) * kWarps);
                const int phys = __shfl_sync(0xffffffffu, ids, i & 31);
                const bool known = phys >= 0 && phys < p.num_pages;
                here = (here & ~(1u << (i & 31))) | (uint32_t)known << (i & 31);
                if (known) {
                    const size_t kb = (size_t)phys * 2 * p.hkv + kvh;
                    const int row = lane >> 3, chunk = lane & 7;
                    const uint8_t *k = p.pool + kb * kBlockBytes + 16 * lane, *v = k + (size_t)p.hkv * kBlockBytes;
                    const uint32_t to = smem_addr(&page[stage]);
#pragma unroll
                    for (int j = 0; j < 4; ++j) copy16(to + few_chunk(row + 4 * j, chunk), k + 512 * j);
#pragma unroll
                    for (int j = 0; j < 4; ++j) copy16(to + kBlockBytes + few_chunk(row + 4 * j, chunk), v + 512 * j);
                    if (lane < 2) copy16(to + 2 * kBlockBytes + 16 * lane, reinterpret_cast<const float4 *>(p.stats) + kb + lane * p.hkv);
                }
            }
            copy_commit();
        };
#pragma unroll
        for (int i = 0; i < kFewStages; ++i) fetch(i, i);

        // q: a warp's rows, 4 dims a lane, to the A fragments: the dims of a lane
        // are those of one lane of one k-step
#pragma unroll
        for (int j = 0; j < kFewRows / kWarps; ++j) {
            const int row = warp + kWarps * j;
            float up = 1.f, *f = q_raw[j];
            if (row < n_rows) {
                float sum = f[0] + f[1] + f[2] + f[3];
#pragma unroll
                for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
                float unscale = 1.f;
                if constexpr (kSplit) {
                    float big = fmaxf(fmaxf(fabsf(f[0]), fabsf(f[1])), fmaxf(fabsf(f[2]), fabsf(f[3])));
#pragma unroll
                    for (int o = 16; o; o >>= 1) big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, o));
                    if (big > 0.f && big < CUDART_INF_F) unscale = pow2i(exponent_above(big) - 13);
                    up = 1.f / unscale;  // a power of two
                }
                if (lane == 0) {
                    sh.row_sum[row] = sum;
                    sh.row_unscale[row] = unscale;
                }
            }
            if (lane == 0) {
                const int r = min(row, n_rows - 1);  // rows that are none see what the last one sees
                sh.row_at[row] = row_at(r);
                sh.row_limit[row] = row_keys(p, rt, r);
            }
            const int step = (lane >> 4) * 4 + (lane & 3), to = (row & 7) * 4 + ((lane >> 2) & 3), half = row >> 3;
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                const float x = f[2 * k] * up, y = f[2 * k + 1] * up;
                const uint32_t hi = pack_half(x, y);
                reinterpret_cast<uint32_t *>(&sh.q_frag[0][step][to])[2 * k + half] = hi;
                if constexpr (kSplit) {
                    const float2 h = h2_to_f2(hi);
                    reinterpret_cast<uint32_t *>(&sh.q_frag[1][step][to])[2 * k + half] = pack_half(x - h.x, y - h.y);
                }
            }
        }
        __syncthreads();

        float o[16][4];  // n-tile t: two dims of row g, of row g + 8; times 2^(kFewUp - v_exp)
#pragma unroll
        for (int t = 0; t < 16; ++t)
#pragma unroll
            for (int k = 0; k < 4; ++k) o[t][k] = 0.f;
        int v_exp = -100, v_top = -100;
        // rows g and g + 8
        int limit[2];
        float m[2], l[2], z[2], q_sum[2], unscale[2];
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            const int row = g + 8 * r;
            limit[r] = sh.row_limit[row];
            m[r] = -CUDART_INF_F;
            l[r] = z[r] = 0.f;
            q_sum[r] = row < n_rows ? sh.row_sum[row] : 0.f;
            unscale[r] = row < n_rows ? sh.row_unscale[row] : 1.f;
        }
        const int least = sh.row_limit[0];  // the first row sees the fewest keys

        int stage = 0;
#pragma unroll 1
        for (int i = 0; i < count; ++i) {
            copy_wait<kFewStages - 1>();
            __syncwarp();
            const FewPage &f = page[stage];
            if (!(here >> (i & 31) & 1)) {
                if (p.error_flag && lane == 0) atomicOr(p.error_flag, 2);
                fetch(i + kFewStages, stage);
                stage = stage == kFewStages - 1 ? 0 : stage + 1;
                continue;
            }
            const float2 ks = block_values(f.ks), vs = block_values(f.vs);
            uint4 kw[2][2];
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
                for (int h = 0; h < 2; ++h) kw[j][h] = *reinterpret_cast<const uint4 *>(f.k + few_chunk(key_a + 2 * j, q4 + 4 * h));
            float c[2][4], c2[2][4];  // even and odd steps: two chains each
#pragma unroll
            for (int s = 0; s < 8; ++s) {
                const uint4 a = sh.q_frag[0][s][lane];
                uint4 al;
                if constexpr (kSplit) al = sh.q_frag[1][s][lane];
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    const uint4 &w = kw[j][s >> 2];
                    const uint2 b = codes_to_half((s & 3) == 0 ? w.x : (s & 3) == 1 ? w.y : (s & 3) == 2 ? w.z : w.w);
                    float(&d)[4] = s & 1 ? c2[j] : c[j];
                    if (s < 2)
                        mma_f16_zero(d, a, b.x, b.y);
                    else
                        mma_f16(d, a, b.x, b.y);
                    if constexpr (kSplit) mma_f16(d, al, b.x, b.y);
                }
            }
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) c[j][e] += c2[j][e];
            // scores (log2): keys key0 + 4 q + 2 j + e of rows g (c[j][e]) and g + 8 (c[j][2 + e])
            const int key0 = (first + i * kWarps) * kPageTokens;
            const bool masked = least < key0 + kPageTokens;
            const float k_mid = fmaf(128.f, ks.x, ks.y) * p.scale_log2, v_mid = fmaf(128.f, vs.x, vs.y);
            float top[2];
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                const float a = ks.x * p.scale_log2 * unscale[r], b = k_mid * q_sum[r];
                top[r] = -CUDART_INF_F;
#pragma unroll
                for (int j = 0; j < 2; ++j)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        float &x = c[j][2 * r + e];
                        x = fmaf(a, x, b);
                        if (masked && key0 + 4 * q4 + 2 * j + e >= limit[r]) x = -CUDART_INF_F;
                        top[r] = fmaxf(top[r], x);
                    }
            }
            // P V takes p times the page's scale times 2^(kFewUp - v_exp), as fp16
            // high and low parts that keep 22 bits while the scale is near 2^v_exp.
            // v_exp goes down no further than
            // 60 below the largest so far, so that the sums stay finite.
            const float v_abs = fabsf(vs.x);
            const int e_v = v_abs > 0.f && v_abs < CUDART_INF_F ? max(min(exponent_above(v_abs), 126), v_top - 60) : v_exp;
            const bool far = e_v > v_exp || e_v < v_exp - 4;
            if (__any_sync(0xffffffffu, far || top[0] > m[0] + kFewLazy<kSplit> || top[1] > m[1] + kFewLazy<kSplit>)) {
                const float to = v_exp - e_v < -126 ? 0.f : far ? pow2i(v_exp - e_v) : 1.f;
                if (far) v_exp = e_v;
                v_top = max(v_top, v_exp);
#pragma unroll
                for (int r = 0; r < 2; ++r) {
                    top[r] = fmaxf(top[r], __shfl_xor_sync(0xffffffffu, top[r], 1));
                    top[r] = fmaxf(top[r], __shfl_xor_sync(0xffffffffu, top[r], 2));
                    const float mn = fmaxf(m[r], top[r]), f_ = mn == -CUDART_INF_F ? 1.f : ex2(m[r] - mn);
                    m[r] = mn;
                    l[r] *= f_;
                    z[r] *= f_;
                    const float f_o = f_ * to;
#pragma unroll
                    for (int t = 0; t < 16; ++t) {
                        o[t][2 * r] *= f_o;
                        o[t][2 * r + 1] *= f_o;
                    }
                }
            }
            const float v_scale = vs.x * pow2i(kFewUp<kSplit> - v_exp);
            uint4 ph, pl;
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                const float m_use = m[r] == -CUDART_INF_F ? 0.f : m[r];
                float e4[4], sum = 0.f;
#pragma unroll
                for (int k = 0; k < 4; ++k) {  // keys 4 q + k
                    e4[k] = ex2(c[k >> 1][2 * r + (k & 1)] - m_use);
                    sum += e4[k];
                }
                l[r] += sum;
                // a row that sees nothing of the page takes nothing from it, whatever its statistics
                const bool sees = !masked || limit[r] > key0;
                if (sees) z[r] = fmaf(sum, v_mid, z[r]);
#pragma unroll
                for (int k = 0; k < 4; ++k) e4[k] = sees ? e4[k] * v_scale : 0.f;
                const uint32_t a = pack_half(e4[0], e4[1]), b = pack_half(e4[2], e4[3]);
                (r ? ph.y : ph.x) = a;
                (r ? ph.w : ph.z) = b;
                const float2 x = h2_to_f2(a), y = h2_to_f2(b);
                (r ? pl.y : pl.x) = pack_half(e4[0] - x.x, e4[1] - x.y);
                (r ? pl.w : pl.z) = pack_half(e4[2] - y.x, e4[3] - y.y);
            }
            uint4 vw[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) vw[j] = *reinterpret_cast<const uint4 *>(f.v + few_chunk(4 * q4 + j, g));
            __syncwarp();  // the warp is done with the stage
            fetch(i + kFewStages, stage);
            stage = stage == kFewStages - 1 ? 0 : stage + 1;
#pragma unroll
            for (int w = 0; w < 4; ++w) {
                uint32_t r4[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) r4[j] = w == 0 ? vw[j].x : w == 1 ? vw[j].y : w == 2 ? vw[j].z : vw[j].w;
                const uint32_t a = __byte_perm(r4[0], r4[1], 0x5140), b = __byte_perm(r4[2], r4[3], 0x5140);
                const uint32_t d = __byte_perm(r4[0], r4[1], 0x7362), e = __byte_perm(r4[2], r4[3], 0x7362);
                const uint32_t col[4] = {__byte_perm(a, b, 0x5410), __byte_perm(a, b, 0x7632), __byte_perm(d, e, 0x5410),
                                         __byte_perm(d, e, 0x7632)};
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const uint2 v = codes_to_half(col[i]);
                    // the page's part alone, then added: the tensor core cuts the
                    // sum it adds to, always towards zero
                    float d[4];
                    mma_f16_zero(d, pl, v.x, v.y);
                    mma_f16(d, ph, v.x, v.y);
#pragma unroll
                    for (int e = 0; e < 4; ++e) o[4 * w + i][e] += d[e];
                }
            }
        }
        copy_wait<0>();
        __syncwarp();

        // ---- the quad's sums, then the warps
        const float v_unit = pow2i(v_exp - kFewUp<kSplit>);
#pragma unroll
        for (int r = 0; r < 2; ++r) {
#pragma unroll
            for (int off = 1; off < 4; off <<= 1) {
                l[r] += __shfl_xor_sync(0xffffffffu, l[r], off);
                z[r] += __shfl_xor_sync(0xffffffffu, z[r], off);
            }
            const int row = g + 8 * r;
            if (q4 == 0) {
                sh.m[warp][row] = m[r];
                sh.l[warp][row] = l[r];
            }
#pragma unroll
            for (int t = 0; t < 16; t += 4) {
                float *to = &sh.of[warp].o[row][32 * q4 + t];
#pragma unroll
                for (int h = 0; h < 2; ++h)
                    *reinterpret_cast<float4 *>(to + 16 * h) =
                        make_float4(fmaf(o[t][2 * r + h], v_unit, z[r]), fmaf(o[t + 1][2 * r + h], v_unit, z[r]),
                                    fmaf(o[t + 2][2 * r + h], v_unit, z[r]), fmaf(o[t + 3][2 * r + h], v_unit, z[r]));
            }
        }
        __syncthreads();
        for (int i = threadIdx.x; i < n_rows * (kHeadDim / 4); i += kWarps * 32) {
            const int row = i / (kHeadDim / 4), d = 4 * (i % (kHeadDim / 4));
            float M = sh.m[0][row];
#pragma unroll
            for (int w = 1; w < kWarps; ++w) M = fmaxf(M, sh.m[w][row]);
            float L = 0.f;
            float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int w = 0; w < kWarps; ++w) {
                const float f = sh.m[w][row] == -CUDART_INF_F && sh.l[w][row] == 0.f ? 0.f : ex2(sh.m[w][row] - M);
                const float4 v = *reinterpret_cast<const float4 *>(&sh.of[w].o[row][d]);
                L = fmaf(f, sh.l[w][row], L);
                acc.x = fmaf(f, v.x, acc.x), acc.y = fmaf(f, v.y, acc.y), acc.z = fmaf(f, v.z, acc.z), acc.w = fmaf(f, v.w, acc.w);
            }
            if (whole) {
                const float inv = L == 0.f ? 0.f : 1.f / L;
                store_out4<T>(static_cast<T *>(p.out) + (size_t)sh.row_at[row] * kHeadDim + d, acc.x * inv, acc.y * inv, acc.z * inv,
                               acc.w * inv);
            } else {
                const size_t at = ((size_t)2 * cta + second) * kFewRows + row;
                *reinterpret_cast<float4 *>(p.few_o + at * kHeadDim + d) = acc;
                if (d == 0) p.few_ml[at] = make_float2(M, L);
            }
        }
        __syncthreads();  // shared memory is free for the next piece
    }
    grid_dependency_wait();  // the other kernel's rows are done when this grid is
}

// out[row] of one row whose keys were split: by a warp, 4 dims a lane.
// part(c): the row of part_ml, part_o that holds piece c.
template <typename T, typename Part>
__device__ __forceinline__ void combine_row(T *out, const float *part_o, const float2 *part_ml, int splits, Part part) {
    const int lane = threadIdx.x & 31;
    float M = -CUDART_INF_F;
    for (int c = lane; c < splits; c += 32) M = fmaxf(M, part_ml[part(c)].x);
#pragma unroll
    for (int o = 16; o; o >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, o));
    float L = 0.f;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 8
    for (int c = 0; c < splits; ++c) {
        const float2 ml = part_ml[part(c)];
        const float4 v = reinterpret_cast<const float4 *>(part_o + part(c) * kHeadDim)[lane];
        const float w = ml.x == -CUDART_INF_F && ml.y == 0.f ? 0.f : ex2(ml.x - M);
        L = fmaf(w, ml.y, L);
        acc.x = fmaf(w, v.x, acc.x), acc.y = fmaf(w, v.y, acc.y), acc.z = fmaf(w, v.z, acc.z), acc.w = fmaf(w, v.w, acc.w);
    }
    const float inv = L == 0.f ? 0.f : 1.f / L;
    store_out4<T>(out + 4 * lane, acc.x * inv, acc.y * inv, acc.z * inv, acc.w * inv);
}

// The first few_ctas CTAs take 8 of the up to 16 rows of a pair that was
// attend_rows_kernel's, the others the rows of split row tiles in turn, one a warp.
// Until grid_dependency_wait only the call's own arguments are read; every
// thread waits, so this grid ends last.
template <typename T>
__global__ void __launch_bounds__(256) attend_combine_kernel(const __grid_constant__ ChunkParams p, int few_ctas) {
    const int warp = threadIdx.x >> 5;
    T *out = static_cast<T *>(p.out);
    if ((int)blockIdx.x < few_ctas) {
        const int pair = blockIdx.x >> 1, r = (blockIdx.x & 1) * 8 + warp, s = pair / p.hkv, kvh = pair % p.hkv;
        const int rows = sequence_tokens(p, s) * p.group;
        int before, splits = 1, first = 0;
        bool late = false;  // the first part lies in its CTA's second place
        const FewWork work_of = few_work(p, s, &before);
        if (r < rows && rows <= p.few_rows) {
            const int units = few_pair(p, s);
            before += kvh * units;
            first = few_owner(work_of, before + kFewStart);
            splits = few_owner(work_of, before + units - 1) - first + 1;
            late = few_begin(work_of, first) < before;
        }
        grid_dependency_wait();
        if (splits > 1)
            combine_row<T>(out + ((size_t)(p.q_start[s] + r / p.group) * p.hq + kvh * p.group + r % p.group) * kHeadDim, p.few_o,
                           p.few_ml, splits,
                           [&](int c) { return (size_t)(2 * (first + c) + (c == 0 && late)) * kFewRows + r; });
        return;
    }
    int mine;
    const ChunkWork work_of = chunk_work(p, &mine);
    const int rows = work_of.pieces > 1 ? (work_of.pairs - work_of.whole) << p.tile_shift : 0;
    const int warps = (gridDim.x - few_ctas) * 8, first = (blockIdx.x - few_ctas) * 8 + warp;
    grid_dependency_wait();
#pragma unroll 1
    for (int i = first; i < rows; i += warps) {
        const int tail = i >> p.tile_shift, r = i & (p.tile_rows - 1), rank = work_of.whole + tail;
        int tile = work_of.tiles - 1 - rank / p.hkv;
        const int seq = chunk_sequence(p, mine, &tile);
        const RowTile rt = row_tile(p, seq, tile, p.tile_rows, work_of.pieces);
        if (r >= rt.rows || rt.splits == 1) continue;
        const int row = tile * p.tile_rows + r;
        combine_row<T>(out + ((size_t)(rt.begin + row / p.group) * p.hq + rank % p.hkv * p.group + row % p.group) * kHeadDim,
                       p.part_o, p.part_ml, rt.splits,
                       [&](int c) { return ((size_t)tail * work_of.pieces + c) * p.tile_rows + r; });
    }
}

int key_tiles(int max_pages) { return (max_pages + kTilePages - 1) / kTilePages; }

// Pieces of one row tile, and of the row tiles of a call that are split: two
// turns of the SMs where there are no more row tiles than SMs, else three.
int most_splits(int max_pages) { return std::max(1, key_tiles(max_pages) / kMinChunk); }
long long most_pieces(long long pairs) { return (pairs <= sm_count() ? 2LL : 3LL) * sm_count(); }
int few_ctas(bool fp32) { return (fp32 ? kFewCtas<true> : kFewCtas<false>) * sm_count(); }

// A launch that may start while the one before it in the stream runs.
template <typename... Args>
int launch_beside(void (*kern)(Args...), dim3 grid, int threads, int smem, cudaStream_t st, const Args &...args) {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
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

// attend_chunk_kernel, attend_rows_kernel beside it, and the combine when keys
// are split.  Only the device knows the sequences' lengths, so both kernels
// are launched unless the sizes rule one out: every row in sequences of at
// most 16 (few enough rows in all), or a single longer sequence.
template <typename T, bool kSplit>
int launch_attend(ChunkParams &p, void *workspace, cudaStream_t st) {
    auto kern = attend_chunk_kernel<T, kSplit>;
    static std::atomic<bool> attr_done[kMaxDevices];
    if (ensure_smem_attr(attr_done, kern, kChunkSmem) != KVX_OK) return KVX_ECUDA;
    auto few_kern = attend_rows_kernel<T, kSplit>;
    constexpr int few_smem = sizeof(FewShared<kSplit>);
    static std::atomic<bool> few_attr_done[kMaxDevices];
    if (ensure_smem_attr(few_attr_done, few_kern, few_smem) != KVX_OK) return KVX_ECUDA;
    const long long rows = (long long)p.total * p.group;
    const bool chunk = rows > kFewRows, few = p.batch > 1 || rows <= kFewRows;
    p.few_rows = few ? kFewRows : 0;
    // row tiles: a sequence of more than 16 rows has one tile beside its whole ones
    auto row_tiles = [&](int tile_rows) {
        return rows / tile_rows + (few ? std::min<long long>(p.batch, rows / (kFewRows + 1)) : p.batch);
    };
    // Rows of a CTA (fp16): 256, which converts each key tile for twice the
    // rows (3.6 us a key tile, 128: 2.0), or 128, which fills the SMs better.
    // Behind many keys (four times the new tokens, as far as the block table
    // tells) the lesser cost by the model that also splits the row tiles;
    // prompts have tiles of all lengths: 128 while CTAs of 256 would leave SMs
    // idle.  24 q-heads on 8, 128 against 256: 1001 tokens 32 and 40 us, 1500:
    // 47 and 53, 2600: 105 and 85; behind 8000 500: 113 and 97, 1500: 273 and
    // 261; 100 behind 30000: 89 and 105.  A block table wider than the lengths
    // (2048 pages) makes a prompt count as one behind many keys: 1001 tokens 40
    // us, 1500: 53, 2 x 700: 36 against 38.
    auto cost = [&](int tile_rows) {
        const long long pairs = row_tiles(tile_rows) * p.hkv, rest = pairs % sm_count(), keys = key_tiles(p.max_pages);
        long long tail = rest ? 64 * (keys + piece_start(tile_rows)) : 0;
        const long long most = rest ? std::min<long long>({most_splits(p.max_pages), most_pieces(pairs) / rest, 32}) : 1;  // an estimate
        for (long long n = 2; n <= most; ++n)
            tail = std::min(tail, 64 * ((rest * n + sm_count() - 1) / sm_count()) * ((keys + n - 1) / n + piece_start(tile_rows)) +
                                      rest * n + 128);
        return (tile_rows == 256 ? 12 : 7) * (64 * (pairs / sm_count()) * (keys + piece_start(tile_rows)) + tail);
    };
    const long long wide = row_tiles(256) * p.hkv;
    const bool far = (long long)p.max_pages * kPageTokens >= 4LL * p.total / p.batch;
    p.tile_rows = kSplit || (wide <= 2LL * sm_count() && (far ? cost(128) < cost(256) : wide <= sm_count())) ? 128 : 256;
    p.tile_shift = p.tile_rows == 256 ? 8 : 7;
    p.max_tiles = (int)row_tiles(p.tile_rows);
    const long long pairs = (long long)p.max_tiles * p.hkv;  // at most
    p.sms = sm_count();
    p.max_splits = most_splits(p.max_pages);
    // A prompt from (nearly) its start on more row tiles than SMs: its last
    // turn are its shortest tiles, not worth a combine (1001 tokens, 24 q-heads
    // on 8: 32 us, and 37 with the launches that may split them).
    if (p.causal && p.batch == 1 && pairs > p.sms && (long long)p.max_pages * kPageTokens - p.total < 2 * kMinChunk * kTileKeys)
        p.max_splits = 1;
    p.max_pieces = (int)most_pieces(pairs);
    // at most the whole pairs and the pieces, or all pairs in as many pieces as one may have
    const long long grid_x = std::min(pairs * p.max_splits, pairs <= p.sms ? std::max(pairs, (long long)p.max_pieces) : pairs + p.max_pieces);
    const size_t few_all = (size_t)few_ctas(kSplit) * 2 * kFewRows;
    p.few_ctas = few_ctas(kSplit);
    p.few_keys = kFewWarps<kSplit> == 8 ? 7 : 6;
    static_assert(kFewWarps<kSplit> == 8 || kFewWarps<kSplit> == 4);
    p.few_o = static_cast<float *>(workspace);
    p.few_ml = reinterpret_cast<float2 *>(p.few_o + few_all * kHeadDim);
    p.part_o = p.few_o + (few ? few_all * (kHeadDim + 2) : 0);
    p.part_ml = reinterpret_cast<float2 *>(p.part_o + (size_t)std::min<long long>(pairs * p.max_splits, p.max_pieces) * p.tile_rows * kHeadDim);
    const bool split = chunk && p.max_splits > 1;
    p.followed = few || split;
    int rc = KVX_OK;
    if (chunk) {
        kern<<<(unsigned)grid_x, kChunkThreads, kChunkSmem, st>>>(p);
        rc = launch_status();
    }
    if (few && rc == KVX_OK) {
        const dim3 grid((unsigned)p.few_ctas);
        if (chunk) {
            rc = launch_beside(few_kern, grid, kFewWarps<kSplit> * 32, few_smem, st, p);
        } else {
            few_kern<<<grid, kFewWarps<kSplit> * 32, few_smem, st>>>(p);
            rc = launch_status();
        }
    }
    if (rc != KVX_OK || (!split && !few)) return rc;
    const int few_grid = few ? p.batch * p.hkv * (kFewRows / 8) : 0;
    const unsigned grid = few_grid + (split ? (unsigned)std::min<long long>(std::min<long long>(pairs, p.sms) * (p.tile_rows / 8), 4 * p.sms) : 0);
    return launch_beside(attend_combine_kernel<T>, dim3(grid), 256, 0, st, p, few_grid);
}

}  // namespace
}  // namespace kvx

using namespace kvx;

// For every call of at most this many sequences, tokens and pages: the pieces
// of split row tiles, and a row tile and kv-head has at most 256 rows more
// than its sequence.
extern "C" KVX_API size_t kvx_attend_chunk_workspace_bytes(int32_t batch, int32_t total_tokens, int32_t num_q_heads,
                                                           int32_t num_kv_heads, int32_t max_pages) {
    if (batch <= 0 || total_tokens <= 0 || num_q_heads <= 0 || num_kv_heads <= 0 || num_q_heads % num_kv_heads ||
        max_pages <= 0)
        return 0;
    long long rows = 2LL * few_ctas(true) * kFewRows;
    const long long splits = most_splits(max_pages), padded = (long long)total_tokens * num_q_heads + 256LL * batch * num_kv_heads;
    if (splits > 1) rows += std::min(splits * padded, 3LL * sm_count() * 256);
    return (size_t)rows * (kHeadDim + 2) * sizeof(float) + 16;
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
        (long long)total_tokens * num_q_heads > 0x3fffffff ||
        (long long)batch * kv->num_kv_heads * (max_pages / kFewWarps<true> + kFewStart + 1) > 0x7fffffff)
        return KVX_EUNSUPPORTED;  // grid, key, row and unit counts fit an int
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
