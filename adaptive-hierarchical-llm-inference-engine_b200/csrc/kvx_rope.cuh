// kvx_rope.cuh -- rotation of one (token, pair) and of 16-byte vectors of a
// row, shared by kvx_rope and kvx_rope_append.
#pragma once

#include "kvx_common.cuh"

namespace kvx {

// (cos, sin) of position * f, f = turns * 2^-64 turns per position.  The
// product modulo 2^64 is the fraction of a turn, exact at any position; it
// is folded to the nearest quarter, so that the float argument (half turns,
// |x| <= 1/4) keeps 24 bits of the remainder: about 2^-26 radians of error,
// below the rounding of the cosine itself.
__device__ __forceinline__ float2 rope_turn(uint64_t turns, int64_t pos, float amplitude) {
    const uint64_t phase = turns * (uint64_t)pos;
    const uint32_t quarter = (uint32_t)((phase + (1ull << 61)) >> 62);
    const int64_t rest = (int64_t)(phase - ((uint64_t)quarter << 62));  // [-2^61, 2^61)
    float s, c;
    sincospif((float)(int32_t)(rest >> 30) * 0x1p-33f, &s, &c);
    const float co = quarter & 1 ? -s : c, si = quarter & 1 ? c : s;
    const float a = quarter & 2 ? -amplitude : amplitude;
    return make_float2(co * a, si * a);
}

// The rounding of both products is fixed here (one product rounded, the
// other fused), so that every kernel gives a rotated row the same bits.
__device__ __forceinline__ void rope_pair(float &a, float &b, float2 cs) {
    const float ra = fmaf(a, cs.x, -__fmul_rn(b, cs.y));
    b = fmaf(b, cs.x, __fmul_rn(a, cs.y));
    a = ra;
}

template <typename T> constexpr int kRopeVec = 16 / (int)sizeof(T);  // elements of a 16-byte vector

template <typename T> __device__ __forceinline__ void rope_unpack(const uint4 &w, float *f);
template <> __device__ __forceinline__ void rope_unpack<float>(const uint4 &w, float *f) {
    f[0] = __uint_as_float(w.x), f[1] = __uint_as_float(w.y), f[2] = __uint_as_float(w.z), f[3] = __uint_as_float(w.w);
}
template <> __device__ __forceinline__ void rope_unpack<__half>(const uint4 &w, float *f) {
    const float2 a = h2_to_f2(w.x), b = h2_to_f2(w.y), c = h2_to_f2(w.z), d = h2_to_f2(w.w);
    f[0] = a.x, f[1] = a.y, f[2] = b.x, f[3] = b.y, f[4] = c.x, f[5] = c.y, f[6] = d.x, f[7] = d.y;
}
template <typename T> __device__ __forceinline__ uint4 rope_pack(const float *f);
template <> __device__ __forceinline__ uint4 rope_pack<float>(const float *f) {
    return make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3]));
}
template <> __device__ __forceinline__ uint4 rope_pack<__half>(const float *f) {
    uint32_t u[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const __half2 h = __floats2half2_rn(f[2 * k], f[2 * k + 1]);
        u[k] = *reinterpret_cast<const uint32_t *>(&h);
    }
    return make_uint4(u[0], u[1], u[2], u[3]);
}

// A row's elements are dealt out as items, so that a thread keeps the same
// item (and its cosines) over many rows:
//   half layout         rotary/2 / E items of the two vectors that pair up
//   interleaved layout  rotary / E items of one vector of whole pairs
//   behind rotary_dim   one vector, passed unchanged
// E: elements of a 16-byte vector, or 1 (a pair of two in the interleaved
// layout) where sizes or addresses do not allow vectors.
__host__ __device__ inline int rope_items(int head_dim, int rotary, bool half, int e) {
    const int turning = half ? rotary / 2 / e : (e == 1 ? rotary / 2 : rotary / e);
    return turning + (head_dim - rotary) / e;
}

// Whether vectors fit a row's sizes (addresses are the caller's matter).
inline bool rope_vector_sizes(int head_dim, int rotary, bool half, int e) {
    return (half ? rotary / 2 : rotary) % e == 0 && (head_dim - rotary) % e == 0;
}

// One thread's item: which elements, and how they turn.
template <typename T, bool kHalf, bool kVec>
struct RopeItem {
    static constexpr int E = kVec ? kRopeVec<T> : 1;
    static constexpr int kPairs = kHalf ? E : (kVec ? E / 2 : 1);
    static constexpr int kWords = kVec ? (kHalf ? 2 : 1) : 2;  // vectors (or elements) moved
    int first, second;  // element offsets (second: half layout, or the odd element when scalar)
    bool turns;
    float2 cs[kPairs];

    __device__ __forceinline__ RopeItem(int item, int rotary) {
        const int half = rotary / 2;
        const int turning = kHalf ? half / E : (kVec ? rotary / E : half);
        turns = item < turning;
        if (turns) {
            first = kHalf ? item * E : (kVec ? item * E : 2 * item);
            second = kHalf ? first + half : first + 1;
        } else {
            first = rotary + (item - turning) * E;
            second = -1;
        }
    }
    // cs_row: (cos, sin) of the token's pairs, in shared memory
    __device__ __forceinline__ void cosines(const float2 *cs_row) {
        if (turns)
#pragma unroll
            for (int k = 0; k < kPairs; ++k) cs[k] = cs_row[(kHalf ? first : first / 2) + k];
    }

    struct Data {
        uint4 w[kVec ? kWords : 1];
        T x[kVec ? 1 : 2];
    };
    __device__ __forceinline__ void load(const T *row, Data &d) const {
        if constexpr (kVec) {
            d.w[0] = *reinterpret_cast<const uint4 *>(row + first);
            if constexpr (kHalf)
                if (turns) d.w[1] = *reinterpret_cast<const uint4 *>(row + second);
        } else {
            d.x[0] = row[first];
            if (turns) d.x[1] = row[second];
        }
    }
    __device__ __forceinline__ void turn(Data &d) const {
        if (!turns) return;
        if constexpr (kVec && kHalf) {
            float a[E], b[E];
            rope_unpack<T>(d.w[0], a);
            rope_unpack<T>(d.w[1], b);
#pragma unroll
            for (int k = 0; k < E; ++k) rope_pair(a[k], b[k], cs[k]);
            d.w[0] = rope_pack<T>(a);
            d.w[1] = rope_pack<T>(b);
        } else if constexpr (kVec) {
            float a[E];
            rope_unpack<T>(d.w[0], a);
#pragma unroll
            for (int k = 0; k < E / 2; ++k) rope_pair(a[2 * k], a[2 * k + 1], cs[k]);
            d.w[0] = rope_pack<T>(a);
        } else {
            float a = io_traits<T>::load(&d.x[0]), b = io_traits<T>::load(&d.x[1]);
            rope_pair(a, b, cs[0]);
            io_traits<T>::store(&d.x[0], a);
            io_traits<T>::store(&d.x[1], b);
        }
    }
    __device__ __forceinline__ void store(T *row, const Data &d) const {
        if constexpr (kVec) {
            *reinterpret_cast<uint4 *>(row + first) = d.w[0];
            if constexpr (kHalf)
                if (turns) *reinterpret_cast<uint4 *>(row + second) = d.w[1];
        } else {
            row[first] = d.x[0];
            if (turns) row[second] = d.x[1];
        }
    }
};

}  // namespace kvx
