// Rows grouped by expert: what the grouped products are told of them, the search of a workgroup's
// rows, and the stores of f32 sums as f32 or bf16.
#pragma once
#include <type_traits>

#include "mambo_common.h"

// r output rows, expert e's at [offsets[e], offsets[e+1]); row i reads row rows[i] (NULL: i) of the m
// input rows. offsets NULL: one weight, every row its own.
struct ExpertRows {
    const int32_t *offsets;
    const int32_t *rows;
    int64_t r, m;
    int experts;
};

// Rows [row0, row0 + count) of one expert; expert == experts: rows of none, which come out as zeros.
struct RowTile {
    int expert, count;
    int64_t row0;
};

// Most tiles of `tile` rows that r rows of `experts` experts and the rows of none can take.
inline int64_t expert_row_tiles(int64_t r, int64_t experts, int64_t tile)
{
    return r / tile + (r < experts ? r : experts) + 1;
}

// Tile t of the rows in tiles of `tile`, counted expert by expert, then the rows of none; false:
// there is no such tile. Every wave searches for itself: 64 experts at a time, a lane each, with a
// scan over the lanes of the tiles that they take (about 1 us beside a launch's weights; a table of
// tiles would have to be another launch's work). Offsets are held within [0, r], whatever they are.
__device__ __forceinline__ bool find_row_tile(const ExpertRows &er, int tile, int t, RowTile *out)
{
    const int lane = (int)__builtin_amdgcn_mbcnt_hi(~0u, __builtin_amdgcn_mbcnt_lo(~0u, 0u));
    const int r = (int)er.r;
    int base = 0;
    for (int e0 = 0; e0 <= er.experts; e0 += 64) {
        const int e = e0 + lane;
        int lo = er.offsets[min(e, er.experts)];
        int hi = e < er.experts ? er.offsets[min(e + 1, er.experts)] : r;
        lo = min(max(lo, 0), r);
        hi = min(max(hi, lo), r);
        const int tiles = e <= er.experts ? (int)(((uint32_t)(hi - lo) + (uint32_t)tile - 1) / (uint32_t)tile) : 0;
        int incl = tiles;
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
            const int up = __shfl_up(incl, d);
            incl += lane >= d ? up : 0;
        }
        const uint64_t past = __ballot(base + incl > t);
        if (past) {
            const int src = __builtin_ctzll(past);
            const int first = t - base - (__builtin_amdgcn_readlane(incl, src) - __builtin_amdgcn_readlane(tiles, src));
            const int begin = __builtin_amdgcn_readlane(lo, src) + first * tile;
            out->expert = e0 + src;
            out->row0 = begin;
            out->count = min(tile, __builtin_amdgcn_readlane(hi, src) - begin);
            return true;
        }
        base += __builtin_amdgcn_readlane(incl, 63);
    }
    return false;
}

// Input row of output row i.
__device__ __forceinline__ int64_t source_row(const ExpertRows &er, int64_t i)
{
    if (!er.rows)
        return i;
    const int64_t s = er.rows[i];
    return s < 0 ? 0 : s >= er.m ? er.m - 1 : s;
}

// Host checks that the grouped products share.
inline int check_expert_rows(int64_t m, const int32_t *rows, int64_t r, const int32_t *offsets, int64_t experts)
{
    MAMBO_REQUIRE(experts >= 1 && experts <= MAMBO_MAX_EXPERTS, MAMBO_ERR_VALUE,
                  "experts must be in [1, %d] (got %lld)", MAMBO_MAX_EXPERTS, (long long)experts);
    MAMBO_REQUIRE(r >= 0 && r <= 0x7FFFFFFF, MAMBO_ERR_VALUE, "rows must number 0 to 2^31 - 1 (got %lld)", (long long)r);
    MAMBO_REQUIRE(rows ? m >= (r ? 1 : 0) : m == r, MAMBO_ERR_VALUE,
                  "without rows every output row has an input row of its own (got %lld and %lld)", (long long)r, (long long)m);
    MAMBO_REQUIRE(r == 0 || offsets != nullptr, MAMBO_ERR_VALUE, "null pointer");
    return MAMBO_OK;
}

// ----------------------------------------------------------------------------- f32 and bf16 values
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));

// Element type of rows that are f32 or bf16.
template <bool kBf16>
using row_t = std::conditional_t<kBf16, __bf16, float>;

// Four consecutive sums of a row, n of them past the row's end left out. kVec: the row is aligned
// for one store. Rounded once, to nearest even.
template <bool kBf16>
__device__ __forceinline__ void store_row4(void *out, int64_t at, v4f v, int64_t left, bool vec)
{
    row_t<kBf16> *o = reinterpret_cast<row_t<kBf16> *>(out) + at;
    if (vec && left >= 4) {
        if constexpr (kBf16)
            __builtin_nontemporal_store(__builtin_convertvector(v, bf16x4), reinterpret_cast<bf16x4 *>(o));
        else
            __builtin_nontemporal_store(v, reinterpret_cast<v4f *>(o));
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (i < left)
                o[i] = (row_t<kBf16>)v[i];
    }
}

// 16 bytes of a row, those past its end (`left` elements on) left out.
template <bool kBf16>
__device__ __forceinline__ void store_chunk(void *out, int64_t at, uint4 v, int64_t left, bool vec)
{
    constexpr int n = kBf16 ? 8 : 4;
    row_t<kBf16> *o = reinterpret_cast<row_t<kBf16> *>(out) + at;
    if (vec && left >= n) {
        *reinterpret_cast<uint4 *>(o) = v;
    } else {
        struct Values {
            row_t<kBf16> v[n];
        };
        const Values e = __builtin_bit_cast(Values, v);
#pragma unroll
        for (int i = 0; i < n; ++i)
            if (i < left)
                o[i] = e.v[i];
    }
}

// Whether a row of f32 or bf16 outputs takes 16 bytes in one store.
inline bool rows_take_vectors(const void *out, int64_t ldo, int dtype)
{
    return (uintptr_t)out % 16 == 0 && ldo % (dtype == MAMBO_DTYPE_BF16 ? 8 : 4) == 0;
}
