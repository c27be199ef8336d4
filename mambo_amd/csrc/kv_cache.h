// The paged 8-bit cache of keys and values: its layout, the sequences of a call, and rotary angles.
#pragma once
#include "experts.h"

// A cache holds pages of page_size tokens, each `heads` x (page_size / 32) blocks: 32 tokens of one
// head, first the keys' codes, then the values', 32 x kv_padded(head_dim) E4M3 bytes each, and beside
// them two E8M0 bytes (keys, values): a value is code * 2^(byte - 127).
//
// The order inside a block is the operand order of v_mfma_f32_16x16x32_bf16 once the bytes are
// widened to bf16, so that one token's attention needs no lane to hand anything to another. For each 32 of
// the head (ds = d / 32), lane l = 16 kk + i has 16 bytes at 1024 ds + 16 l:
//   keys    tokens 8 (i / 4) + i % 4 and 4 more, each 8 bytes of d = 32 ds + 8 kk ..
//   values  d = 32 ds + i and 16 more, each 8 bytes of tokens 8 kk ..
// The scores of both key tiles then leave lane 16 kk + i with tokens 8 kk .. 8 kk + 7 of query i,
// which is what the product with the values wants of it.
constexpr int kKvBlock = 32;
constexpr int kKvLowest = -100; // lowest exponent: what an empty or all-zero block has
// The largest float32 has the exponent 120, where the code after 240 would stand for 2^128.
constexpr int kKvHighest = 120;
constexpr float kKvMostThere = 240.0f;

__host__ __device__ constexpr int kv_padded(int dim) { return (dim + 31) & ~31; }
__host__ __device__ constexpr int kv_key_byte(int token, int d)
{
    return (d >> 5) * 1024 + ((((d >> 3) & 3) << 4) + ((token >> 3) << 2) + (token & 3)) * 16 + ((token >> 2) & 1) * 8 + (d & 7);
}
__host__ __device__ constexpr int kv_value_byte(int token, int d)
{
    return (d >> 5) * 1024 + (((token >> 3) << 4) + (d & 15)) * 16 + ((d >> 4) & 1) * 8 + (token & 7);
}

struct KvCache {
    uint8_t *codes, *scales;
    int pages, heads, dim, shift; // blocks of a page: 1 << shift
    // Index of a block, for 2 * 32 * padded bytes of codes and 2 of scales; page within [0, pages). 32 bits: so many
    // blocks are 4 TiB and more, and refused.
    __device__ uint32_t block(int page, int head, int b) const
    {
        return ((uint32_t)(page * heads + head) << shift) + (uint32_t)(b & ((1 << shift) - 1));
    }
};

// The sequences of a call. Whatever the device's arrays hold, what is made of them stays in range:
// rows within the call's tokens, cached tokens within the tables, pages (checked where they are read).
// Positions are those of the length that was given: past the table's end they are nobody's place.
struct KvBatch {
    const int32_t *tables, *lengths, *offsets; // offsets NULL: `each` rows a sequence
    int64_t ldt;
    int width, seqs, tokens, each, capacity; // capacity: width * page_size

    __device__ int offset(int s) const
    {
        return offsets ? min(max(offsets[s], 0), tokens) : s * each;
    }
    __device__ int length(int s) const { return max(lengths[s], 0); }
    __device__ int page(int s, int column) const { return tables[s * ldt + column]; }
};

__device__ __forceinline__ int lane_id()
{
    return (int)__builtin_amdgcn_mbcnt_hi(~0u, __builtin_amdgcn_mbcnt_lo(~0u, 0u));
}

// The sequence that has slot `slot`, where sequence s has the slots from first(s) on, first rising
// from first(0) == 0: every wave looks at 64 sequences at a time.
template <typename F>
__device__ __forceinline__ int find_slot(int seqs, int64_t slot, F first)
{
    const int lane = lane_id();
    int found = 0;
    for (int s0 = 0; s0 < seqs; s0 += 64) {
        const int s = min(s0 + lane, seqs - 1);
        const uint64_t begun = __ballot(first(s) <= slot && s0 + lane < seqs);
        if (begun)
            found = s0 + 63 - __builtin_clzll(begun);
        if (begun != ~0ull)
            break;
    }
    return __builtin_amdgcn_readfirstlane(found);
}

// ----------------------------------------------------------------------------- rotary angles
struct RotaryTable {
    const uint64_t *turns; // of pair i: the fraction of a turn that a position adds, times 2^64
    int size, interleaved; // values of a head that are rotated, in pairs (i, i + size / 2) or (2i, 2i + 1)
    double magnitude;
};

// Magnitude times cosine and sine of position * turns, each rounded once from 64 bits. The product wraps
// at 2^64 as the angle does at a turn, so far positions lose nothing; the nearest quarter of a turn is taken off as an
// integer, and what is left, up to pi / 4, goes into the Taylor series of sine and cosine (the first terms left
// out, x^13 / 13! and x^14 / 14!, are below 2^-36). 13 multiply-adds of half the float32 rate: no more than the
// library's float32 functions take, whose angle is off by 2^-24 of up to pi and which moves a code's rounding
// for 2.5 times as many keys.
__device__ __forceinline__ float2 rotary_angle(const RotaryTable &t, int position, int i)
{
    const uint64_t phase = (uint64_t)(int64_t)position * t.turns[i];
    const uint32_t quarter = (uint32_t)((phase + (1ull << 61)) >> 62);
    const double x = (double)(int64_t)(phase - ((uint64_t)quarter << 62)) * (6.283185307179586 * 0x1p-64), y = x * x;
    double s = -1.0 / 39916800.0, c = 1.0 / 479001600.0;
    s = __builtin_fma(s, y, 1.0 / 362880.0);
    c = __builtin_fma(c, y, -1.0 / 3628800.0);
    s = __builtin_fma(s, y, -1.0 / 5040.0);
    c = __builtin_fma(c, y, 1.0 / 40320.0);
    s = __builtin_fma(s, y, 1.0 / 120.0);
    c = __builtin_fma(c, y, -1.0 / 720.0);
    s = __builtin_fma(s, y, -1.0 / 6.0);
    c = __builtin_fma(c, y, 1.0 / 24.0);
    s = __builtin_fma(s * y, x, x);
    c = __builtin_fma(c, y, -0.5);
    c = __builtin_fma(c, y, 1.0);
    const float cos = (float)(t.magnitude * (quarter & 1 ? s : c)), sin = (float)(t.magnitude * (quarter & 1 ? c : s));
    return make_float2((quarter + 1) & 2 ? -cos : cos, quarter & 2 ? -sin : sin);
}

// A pair by an angle. Written out as it is rounded (one product, then one multiply-add), so that every kernel
// and every form of one gives the same bits.
__device__ __forceinline__ float turn_low(float a, float b, float2 t) { return __builtin_fmaf(a, t.x, -(b * t.y)); }
__device__ __forceinline__ float turn_high(float a, float b, float2 t) { return __builtin_fmaf(a, t.y, b * t.x); }

inline bool kv_dim_ok(int64_t dim) { return dim >= 8 && dim <= MAMBO_KV_MAX_DIM && dim % 8 == 0; }

// Checks shared by the entry points that take a cache and sequences; what they make of the two.
int kv_check_cache(const mambo_kv_cache *cache, KvCache *out);
int kv_check_batch(const mambo_kv_batch *batch, int64_t tokens, const mambo_kv_cache *cache, KvBatch *out);
