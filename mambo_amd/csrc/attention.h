// Attention over the paged 8-bit cache: what its two kernels and the joins share.
#pragma once
#include "kv_cache.h"

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

struct Attention {
    const __bf16 *q;
    int64_t ldqt, ldqh;
    KvCache cache;
    KvBatch b;
    int group; // query heads of a key/value head
    float scale; // of the scores, times log2(e): softmax in powers of two
    int causal, window;
    __bf16 *out;
    int64_t ldot, ldoh;
    float *lse;
    int few_rows; // sequences of up to so many rows (queries x group) are attend_rows' work, others attend_tiles'
    int slots;    // attend_rows: workgroups of a head; 0: attend_short takes its place
    int parts, tiles_each; // attend_tiles: parts of the keys; tiles of a sequence of a uniform batch
    float *rows_o, *rows_ml; // partial sums, their largest scores and totals
    int32_t *begins;         // first block of each sequence in the row kernel's order, and the total
    float *tiles_o, *tiles_ml;
};

// A sequence's rows [first, first + n), the last at position end - 1, its cached tokens [0, len) and the blocks [lo, hi) of
// them that any row sees (none: lo >= hi).
struct Sequence {
    int first, n, end, len, lo, hi;
};

__device__ __forceinline__ Sequence sequence(const Attention &a, int s)
{
    Sequence q;
    q.first = a.b.offset(s);
    q.n = max(0, (a.b.offsets ? a.b.offset(s + 1) : q.first + a.b.each) - q.first);
    q.end = a.b.length(s);
    q.len = min(q.end, a.b.capacity);
    q.lo = a.window ? max(0, q.end - q.n + 1 - a.window) / kKvBlock : 0;
    q.hi = (q.len + kKvBlock - 1) / kKvBlock;
    return q;
}

// What row (query i of n) sees: keys in [from, to).
__device__ __forceinline__ int sees_to(const Attention &a, const Sequence &q, int i)
{
    return a.causal ? min(q.end - q.n + i + 1, q.len) : q.len;
}
__device__ __forceinline__ int sees_from(const Attention &a, const Sequence &q, int i)
{
    return a.window ? q.end - q.n + i + 1 - a.window : 0;
}

// Eight E4M3 codes times a power of two as bf16, which holds them exactly (4 of its 8 bits).
__device__ __forceinline__ bf16x8 widen(uint32_t lo, uint32_t hi, float scale)
{
    const bf16x2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, scale, false);
    const bf16x2 b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, scale, true);
    const bf16x2 c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, scale, false);
    const bf16x2 d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, scale, true);
    return bf16x8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

// 2^(byte - 127) of an E8M0 byte; the append makes bytes of 27 to 247.
__device__ __forceinline__ float e8m0(uint32_t byte) { return __uint_as_float(byte << 23); }

__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }

// Zero, in a vector register: an address that it is part of is one of each lane to the compiler, which otherwise
// brings a loaded value that all lanes share into a scalar register, and waits for it, right behind the load.
__device__ __forceinline__ int vector_zero()
{
    int zero;
    asm("v_mov_b32 %0, 0" : "=v"(zero));
    return zero;
}

// A word that every lane wants and no kernel writes while this one runs.
__device__ __forceinline__ int scalar_load(const int32_t *p)
{
    return *(const __attribute__((address_space(4))) int32_t *)p;
}

// Codes past the first `left` (of eight) become zeros: what a page holds behind a sequence's last token is
// anything, and a NaN there times a probability of zero would still be one.
__device__ __forceinline__ uint2 keep_tokens(uint32_t lo, uint32_t hi, int left)
{
    const uint64_t mask = left >= 8 ? ~0ull : left <= 0 ? 0ull : (1ull << (8 * left)) - 1;
    return make_uint2(lo & (uint32_t)mask, hi & (uint32_t)(mask >> 32));
}

// Most rows that attend_rows takes, in tiles of 16: more than that attend_tiles is faster at (8 key/value heads: 4 x 64 rows of D = 128
// behind 20000 tokens 57 us, with four tiles here 75; 4 x 32 of 192 behind 10000 52, here 37; of 256 73, here 53).
constexpr int max_row_tiles(int padded) { return padded <= 64 ? 4 : 2; }

// Whether attend_short takes so many tiles of heads of 32 ds: its eight waves have not the registers for two of heads above 128,
// which always take the shares.
constexpr bool short_fits(int ds, int row_tiles) { return ds * row_tiles <= 9; }

// Waves of a workgroup of attend_tiles, each with 32 rows, by the head size in 32s. Eight, two a SIMD, while a wave's
// registers are enough, above that four with twice the registers. 4096 tokens of 32 heads with eight and with four: of 64 101 us
// and 117, of 96 119 and 219, of 160 213 and 278, of 192 285 and 299, of 224 530 and 355, of 256 1968 and 417; 8192 tokens of
// 128 498 and 814.
constexpr int tile_waves(int ds) { return ds <= 6 ? 8 : 4; }
constexpr int tile_rows(int ds) { return 32 * tile_waves(ds); }

// Blocks that a sequence has in the row kernel's order.
__device__ __forceinline__ int row_blocks(const Attention &a, const Sequence &q)
{
    return q.n > 0 && q.n <= a.few_rows / a.group ? max(0, q.hi - q.lo) : 0;
}

// The shares: workgroups that have any (at least four blocks each, one a wave), and where they begin.
__device__ __forceinline__ int shares(const Attention &a, int total) { return max(1, min(a.slots, (total + 3) / 4)); }
__device__ __forceinline__ int share_begin(int p, int total, int count) { return (int)((int64_t)p * total / count); }
__device__ __forceinline__ int share_of(int block, int total, int count)
{
    return (int)((((int64_t)block + 1) * count + total - 1) / total) - 1;
}

// A row's result: four values of it, and with the first of them its lse.
__device__ __forceinline__ void store_row(const Attention &a, int64_t t, int h, int d, v4f o, float top, float sum)
{
    o *= sum == 0.0f ? 0.0f : 1.0f / sum;
    if (d < a.cache.dim)
        store_row4<true>(a.out, t * a.ldot + h * a.ldoh + d, o, a.cache.dim - d,
                         a.ldot % 4 == 0 && a.ldoh % 4 == 0 && (uintptr_t)a.out % 8 == 0);
    if (a.lse && d == 0)
        a.lse[t * ((int64_t)a.group * a.cache.heads) + h] = sum == 0.0f ? -__builtin_inff() : (top + __log2f(sum)) * kLn2;
}

constexpr int kTileBlocks = 2; // blocks of 32 tokens of a tile

// The blocks [lo, hi) of keys of the rows from row0 on: what the first row sees of the window to what the last one sees.
// They are dealt evenly to several workgroups where there are five steps of the kernel and more for each.
struct Keys {
    int lo, hi, tiles, parts;
    __device__ int begin(int part) const { return lo + kTileBlocks * (int)((int64_t)tiles * part / parts); }
};
__device__ __forceinline__ Keys tile_keys(const Attention &a, const Sequence &seq, int row0, int tile_rows)
{
    const int i0 = row0 / a.group, i1 = (min(row0 + tile_rows, seq.n * a.group) - 1) / a.group;
    Keys k;
    k.lo = max(0, sees_from(a, seq, i0)) / kKvBlock;
    k.hi = (max(0, sees_to(a, seq, i1)) + kKvBlock - 1) / kKvBlock;
    k.tiles = max(0, k.hi - k.lo + kTileBlocks - 1) / kTileBlocks;
    k.parts = max(1, min(a.parts, k.tiles / 5));
    return k;
}

// What is joined: workgroups for rows of attend_tiles, each of join_tile_rows, then one for each of the row_count rows that a
// sequence and a head can have in attend_rows.
struct Join {
    int64_t tiles = 0, rows = 0;
    int row_count = 0;
};
constexpr int join_tile_rows(int ds) { return 256 / (8 * ds); }

int launch_attend_rows(const Attention &a, int row_tiles, hipStream_t s);
int launch_attend_tiles(const Attention &a, int64_t tiles, hipStream_t s);
int launch_attend_join(const Attention &a, int row_tiles, const Join &join, hipStream_t s);
