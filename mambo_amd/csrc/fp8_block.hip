// E4M3 products with an f32 scale for each block of 128: the quantizer of the rows, the private
// layout of the weights and the products, dense and grouped by expert.
//
//   out[m, n] = sum_g xs[m, g] * ws[n / 128, g] * sum_{k in group g} xv[m, k] * w[n, k]
//
// A group of K is one K = 128 of matrix work (V_MFMA_F32_16X16X128_F8F6F4, or two of
// V_MFMA_F32_32X32X64_F8F6F4), whose sums are scaled in f32: the scales are no powers of two, so
// the MFMA's own scales cannot carry them. The weight is the MFMA's A operand (its rows n) and the
// tokens the B operand (its columns), so a lane's sums belong to one token and its scale is one
// factor, xs * ws, of which ws is the same for the wave.
//
// An FP8 MFMA adds the products of eight consecutive K as multiples of 2^-13 of 2^E and cuts what is below,
// E being the largest sum of two codes' exponents among the eight (measured on gfx950: beside a product of 2^16
// one of 2^3 counts and one of 2^2 does not, of either sign, in the 16 x 16 x 128 and 32 x 32 x 64 shapes and in
// the older 16 x 16 x 32 and 32 x 32 x 16 alike; among other eights it does). At worst that leaves out seven
// products of the eight, 7 x 2^-13 = 8.5e-4 of the largest (measured 7.5e-4 of the sum of magnitudes); over codes of
// all exponents it is 5e-5 of the sums in the 2-norm, 2^-5 of what rounding them to bf16 takes, so bf16 outputs use
// it. Where a row's terms cancel, what is cut does not shrink with the result. f32 outputs are of f32 sums: the codes
// are widened to bf16, exactly, and multiplied by the bf16 MFMAs, which add without that loss (2.5e-7 on the same
// data), at half the matrix rate.
//
// Layout of a weight (mambo_fp8_block_pack): tiles of 32 rows x 128 of K, 4096 bytes, ordered
// [expert][n / 32][k / 128]; within a tile 16-byte chunk c of row i (K 16c .. 16c+15 of the group) at
// 512 c + 16 i. A wave's load of 16 bytes a lane is then 1 KiB in one piece, and lands as the
// operand: lane (i, h) of the 32 x 32 MFMA of K step s takes chunks 4s + h and 4s + 2 + h, of the 16 x
// 16 MFMA chunks h and 4 + h. Rows past n and K past k are zeros, so nothing else looks after the
// ends of a weight. (Any order of K serves that both operands share.)
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "experts.h"

namespace {

constexpr int kGroup = 128;      // K of one scale
constexpr int kTileN = 32;       // weight rows of a tile
constexpr int kFp8Tile = 4096;   // bytes of a tile
constexpr int64_t kMaxK = 1 << 26; // of a weight: a tile row's bytes in 31 bits
int64_t cdiv(int64_t a, int64_t b) { return (a + b - 1) / b; }

// ============================================================================ quantizer
// 16 lanes of eight elements a group, so a wave's loads cover 512 elements in one piece, and the
// group's maximum takes four lane swaps. Bound by HBM: k * (2 or 4) bytes read and k * 33/32
// written a row.
//
// A code is E4M3(x / s) with s = amax / 448 kept as f32. Dividing by that rounded s (or multiplying
// by its rounded inverse) would move values that lie half way between two codes, which rows of bf16
// often hold, to either side; 448 x / amax has no other rounding than its own. It is taken as
// (0.875 x) / (amax 2^-9), which neither overflows nor leaves the normal numbers, by the rounded
// inverse and one correction, which gives the correctly rounded quotient (Markstein, "Computation of
// elementary functions on the IBM RISC System/6000 processor", 1990).
constexpr float kSmallestScale = 0x1p-100f;

template <bool kBf16, bool kVec>
__device__ __forceinline__ void load8(const void *x, int64_t at, float (&v)[8])
{
    const row_t<kBf16> *p = reinterpret_cast<const row_t<kBf16> *>(x) + at;
    if constexpr (kVec) {
        typedef row_t<kBf16> row16 __attribute__((ext_vector_type(kBf16 ? 8 : 4)));
#pragma unroll
        for (int i = 0; i < 8; i += kBf16 ? 8 : 4) {
            const row16 r = __builtin_nontemporal_load(reinterpret_cast<const row16 *>(p + i));
#pragma unroll
            for (int j = 0; j < (kBf16 ? 8 : 4); ++j)
                v[i + j] = (float)r[j];
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            v[i] = (float)p[i];
    }
}

// R rows at a time, their loads issued before either is converted: 8192 x 4096 bf16 takes 26.9 us with one row, 22.2 (4.5
// TB/s of reads and writes) with two, 23.9 with four and 28.0 with eight; 512 x 4096 with one 4.3, with two 4.9.
template <bool kBf16, bool kVec, int R>
__global__ __launch_bounds__(256) void quantize_fp8_block_kernel(const void *__restrict__ x, int64_t ldx, int64_t m,
                                                                 int k, uint8_t *__restrict__ values, int64_t ldv,
                                                                 float *__restrict__ scales, int64_t lds, int64_t gss)
{
    const int at = (int)(blockIdx.x * 16 + (threadIdx.x >> 4)) * kGroup + 8 * (threadIdx.x & 15); // in the row
    const bool in = at < k; // k is a multiple of 16, so all eight or none
    for (int64_t row0 = (int64_t)blockIdx.y * R; row0 < m; row0 += (int64_t)gridDim.y * R) {
        float v[R][8] = {};
#pragma unroll
        for (int r = 0; r < R; ++r)
            if (in && row0 + r < m)
                load8<kBf16, kVec>(x, (row0 + r) * ldx + at, v[r]);
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const int64_t row = row0 + r;
            uint32_t amax = 0u; // over the magnitude bits: a NaN beats an infinity, that every number
#pragma unroll
            for (int i = 0; i < 8; ++i)
                amax = max(amax, abs_bits(v[r][i]));
#pragma unroll
            for (int d = 1; d < 16; d <<= 1)
                amax = max(amax, (uint32_t)__shfl_xor((int)amax, d));
            if (!in || row >= m)
                continue;
            const bool finite = amax < kNonFiniteBits;
            const float top = fmaxf(__uint_as_float(amax), 448.0f * kSmallestScale);
            const float b = top * 0x1p-9f, inv = 1.0f / b;
            float q[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float a = 0.875f * v[r][i], y = a * inv;
                q[i] = __builtin_copysignf(__builtin_fmaf(__builtin_fmaf(-y, b, a), inv, y), a); // -0 stays -0
            }
            uint2 codes;
            if (finite) {
                codes.x = pack4<kQuantHwCvt>(q[0], q[1], q[2], q[3]);
                codes.y = pack4<kQuantHwCvt>(q[4], q[5], q[6], q[7]);
            } else {
                codes.x = nan4(v[r][0], v[r][1], v[r][2], v[r][3]);
                codes.y = nan4(v[r][4], v[r][5], v[r][6], v[r][7]);
            }
            uint8_t *o = values + row * ldv + at;
            if constexpr (kVec) {
                *reinterpret_cast<uint2 *>(o) = codes; // read again by the product that follows
            } else {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    o[i] = (uint8_t)(codes.x >> (8 * i));
                    o[4 + i] = (uint8_t)(codes.y >> (8 * i));
                }
            }
            if ((threadIdx.x & 15) == 0)
                scales[row * lds + at / kGroup * gss] = finite ? top / 448.0f : __builtin_nanf("");
        }
    }
}

// ============================================================================ weight layout
// One workgroup per tile: 256 threads, a 16-byte chunk each, read along the rows. Bound by HBM (64 x 2048 x 4096: 185 us,
// 5.8 TB/s of reads and writes).
__global__ __launch_bounds__(256) void fp8_block_pack_kernel(const uint8_t *__restrict__ w, int64_t n, int64_t k,
                                                             int64_t stride_e, int64_t stride_n, int64_t ntiles,
                                                             int64_t groups, bool vec, uint8_t *__restrict__ packed)
{
    const int64_t tile = blockIdx.x;
    const int64_t e = tile / (ntiles * groups), rest = tile - e * ntiles * groups;
    const int i = threadIdx.x >> 3, c = threadIdx.x & 7;
    const int64_t row = rest / groups * kTileN + i, at = rest % groups * kGroup + 16 * c;
    uint4 v = {0u, 0u, 0u, 0u};
    if (row < n && at < k) {
        const uint8_t *p = w + e * stride_e + row * stride_n + at;
        if (vec) {
            v = *reinterpret_cast<const uint4 *>(p);
        } else {
            uint32_t d[4] = {};
#pragma unroll
            for (int j = 0; j < 16; ++j)
                d[j >> 2] |= (uint32_t)p[j] << (8 * (j & 3));
            v = uint4{d[0], d[1], d[2], d[3]};
        }
    }
    *reinterpret_cast<uint4 *>(packed + tile * kFp8Tile + 512 * c + 16 * i) = v;
}

// ============================================================================ products
struct Fp8Args {
    const uint8_t *xv;
    const float *xs;
    int64_t ldxv, ldxs, gsxs; // xs: strides of rows and of groups
    ExpertRows er;
    const uint8_t *packed;
    const float *ws;
    void *out;
    int64_t ldo;
    int n, k, groups, ntiles; // groups of K, tiles of 32 weight rows
    bool vec;                 // the outputs take one store of four
    uint32_t tiles, group, deal; // Order
};

// The row tile and the column tile of this workgroup. Workgroups go to the eight XCDs in turn, and each XCD has an L2 of its
// own: they are dealt to it `deal` at a time from an order of column groups (`group` columns wide), in a group row tile by row
// tile, in a row tile column by column. False: a workgroup past the last.
__device__ __forceinline__ bool place(const Fp8Args &a, int columns, int *tile, int *column)
{
    const uint32_t xcd = blockIdx.x & 7, i = blockIdx.x >> 3, round = i / a.deal;
    const uint32_t at = (round * 8 + xcd) * a.deal + (i - round * a.deal);
    if (at >= a.tiles * (uint32_t)columns)
        return false;
    const uint32_t span = a.group * a.tiles, group = at / span, rest = at - group * span;
    const uint32_t width = min(a.group, (uint32_t)columns - group * a.group);
    *tile = (int)(rest / width);
    *column = (int)(group * a.group + (rest - (uint32_t)*tile * width));
    return true;
}

template <bool kExperts>
__device__ __forceinline__ bool row_tile(const Fp8Args &a, int tile, int t, RowTile *rt)
{
    if constexpr (kExperts) {
        return find_row_tile(a.er, tile, t, rt);
    } else {
        rt->expert = 0;
        rt->row0 = (int64_t)t * tile;
        rt->count = (int)min<int64_t>(tile, a.er.r - rt->row0);
        return true;
    }
}

typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

__device__ __forceinline__ v8i operand(const uint4 &lo, const uint4 &hi)
{
    return v8i{(int)lo.x, (int)lo.y, (int)lo.z, (int)lo.w, (int)hi.x, (int)hi.y, (int)hi.z, (int)hi.w};
}

// Eight E4M3 codes as bf16, which holds each of them.
__device__ __forceinline__ bf16x8 widen(uint32_t lo, uint32_t hi)
{
    const bf16x2 v[4] = {__builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.0f, false),
                         __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.0f, true),
                         __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.0f, false),
                         __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.0f, true)};
    return __builtin_bit_cast(bf16x8, v);
}

// c + the products of 16 x 16 rows over K = 128, or 32 x 32 rows over K = 64: a lane's 32 codes of its
// weight row and of its token. kWide: through bf16.
template <bool kWide>
__device__ __forceinline__ v4f multiply(const uint4 (&w)[2], const uint4 (&x)[2], v4f c)
{
    if constexpr (!kWide) {
        return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(operand(w[0], w[1]), operand(x[0], x[1]), c, 0, 0, 0, 0, 0,
                                                                0); // both scales 0: the unscaled MFMA
    } else {
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(widen(w[j].x, w[j].y), widen(x[j].x, x[j].y), c, 0, 0, 0);
            c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(widen(w[j].z, w[j].w), widen(x[j].z, x[j].w), c, 0, 0, 0);
        }
        return c;
    }
}
template <bool kWide>
__device__ __forceinline__ v16f multiply(const uint4 (&w)[2], const uint4 (&x)[2], v16f c)
{
    if constexpr (!kWide) {
        return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(operand(w[0], w[1]), operand(x[0], x[1]), c, 0, 0, 0, 0, 0,
                                                               0);
    } else {
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            c = __builtin_amdgcn_mfma_f32_32x32x16_bf16(widen(w[j].x, w[j].y), widen(x[j].x, x[j].y), c, 0, 0, 0);
            c = __builtin_amdgcn_mfma_f32_32x32x16_bf16(widen(w[j].z, w[j].w), widen(x[j].z, x[j].w), c, 0, 0, 0);
        }
        return c;
    }
}

// Few rows: bound by the weights' bytes. A workgroup computes 16 tokens x 16 H weight rows; its W waves take the K groups in
// turn and every wave streams its own, the next group's weights and rows in flight while one is multiplied and no barrier
// before the end, where the waves' sums meet in LDS and are added in order. The weights pass the caches by (each byte is read
// once by one workgroup in a launch of few rows; 58 MB 13.1 -> 12.2 us, 117 MB 22.7 -> 20.4; weights that a cache still
// holds from before lose by it, 4 MB 4.6 -> 5.1). Three and four groups in flight were slower (58 MB 15.8 us).
typedef unsigned int u32x4 __attribute__((ext_vector_type(4)));

template <int H, int W, bool kExperts, bool kBf16>
__global__ __launch_bounds__(W * 64) void fp8_stream_kernel(Fp8Args a)
{
    constexpr int T = 16, kCols = 16 * H;
    constexpr int kPad = kCols + 4; // floats of a token's sums in LDS
    __shared__ __align__(16) float s_red[W * T * kPad];
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int tiles_n = (a.n + kCols - 1) / kCols;
    RowTile rt;
    int tile_m, nt;
    if (!place(a, tiles_n, &tile_m, &nt) || !row_tile<kExperts>(a, T, tile_m, &rt))
        return;
    const bool none = kExperts && rt.expert == a.er.experts;

    if (!none) {
        // lanes past the last row read it again: they feed sums that are not stored
        const int col = lane & 15, q = lane >> 4;
        const int64_t src = source_row(a.er, rt.row0 + min(col, rt.count - 1));
        const uint8_t *xp = a.xv + src * a.ldxv;
        const float *sp = a.xs + src * a.ldxs;
        // chunk q + 4 j of weight row 16 t + col: halves t of a tile of 32 rows, H 4: of this one and the next (the last
        // tile stands in for one past it)
        const int tile = nt * kCols / kTileN;
        const uint8_t *wp = a.packed + ((int64_t)rt.expert * a.ntiles + tile) * a.groups * kFp8Tile + 512 * q + 16 * col +
                            (H == 1 ? 256 * (nt & 1) : 0);
        const int64_t next = tile + 1 < a.ntiles ? (int64_t)a.groups * kFp8Tile : 0;
        const float *ws = a.ws + ((int64_t)rt.expert * ((a.n + kGroup - 1) / kGroup) + nt * kCols / kGroup) * a.groups;

        float acc[H][4] = {};
        struct Ring {
            uint4 w[H][2], x[2];
            float xs, ws;
        } ring[2];
        const int count = wave < a.groups ? (a.groups - wave + W - 1) / W : 0;
        auto load = [&](Ring &r, int i) {
            const int g = max(min(wave + min(i, count - 1) * W, a.groups - 1), 0); // past the last: any, scaled by 0
            const uint8_t *p = wp + (int64_t)g * kFp8Tile;
#pragma unroll
            for (int t = 0; t < H; ++t)
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    const u32x4 v = __builtin_nontemporal_load(
                        reinterpret_cast<const u32x4 *>(p + 2048 * j + 256 * (t & 1) + (t >> 1) * next));
                    r.w[t][j] = uint4{v[0], v[1], v[2], v[3]};
                }
            const int k0 = g * kGroup;
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const int at = k0 + 16 * (q + 4 * j); // a chunk past the row's end meets zero weights: any of the row does
                r.x[j] = *reinterpret_cast<const uint4 *>(xp + (at < a.k ? at : k0));
            }
            r.xs = sp[g * a.gsxs];
            r.ws = i < count ? ws[g] : 0.0f;
        };
        load(ring[0], 0);
        for (int i0 = 0; i0 < count; i0 += 2) {
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                load(ring[j ^ 1], i0 + j + 1);
                __builtin_amdgcn_sched_barrier(0);
                const Ring &r = ring[j];
                const float f = r.xs * r.ws;
#pragma unroll
                for (int t = 0; t < H; ++t) {
                    const v4f c = multiply<!kBf16>(r.w[t], r.x, v4f{});
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        acc[t][i] = __builtin_fmaf(c[i], f, acc[t][i]);
                }
                __builtin_amdgcn_sched_barrier(0);
            }
        }
        // the sums of a lane: token col, weight rows 16 t + 4 q .. 4 q + 3
        float *red = s_red + (wave * T + col) * kPad + 4 * q;
#pragma unroll
        for (int t = 0; t < H; ++t)
            *reinterpret_cast<v4f *>(red + 16 * t) = v4f{acc[t][0], acc[t][1], acc[t][2], acc[t][3]};
    }
    __syncthreads();
    for (int i = tid; i < T * 4 * H; i += W * 64) {
        const int token = i / (4 * H), n4 = 4 * (i % (4 * H)), at = nt * kCols + n4;
        if (token >= rt.count)
            break;
        v4f v = {0.0f, 0.0f, 0.0f, 0.0f};
        if (!none)
#pragma unroll
            for (int w = 0; w < W; ++w)
                v += *reinterpret_cast<const v4f *>(s_red + (w * T + token) * kPad + n4);
        if (at < a.n)
            store_row4<kBf16>(a.out, (rt.row0 + token) * a.ldo + at, v, a.n - at, a.vec);
    }
}

// LDS destination of the direct global-to-LDS copies.
typedef __attribute__((address_space(3))) void *lds_ptr;
typedef const __attribute__((address_space(4))) float *constant_floats; // read by scalar loads

__device__ __forceinline__ __amdgpu_buffer_rsrc_t open_rsrc(const void *base)
{
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<void *>(base), 0, (int)0xFFFFFFFFu, 0x00020000);
}

// Row i's 16-byte chunk c lies at slot c ^ slot_of(i) of its 128 bytes in LDS: the chunks c of 16 consecutive rows lie in
// different banks.
__device__ __forceinline__ int slot_of(int row) { return (row ^ ((row >> 3) & 3)) & 7; }

// More rows: a workgroup computes 32 MT tokens x 32 NB WN weight rows with KG groups of WN waves, each group taking a KG-th
// of K; a wave owns 32 NB weight rows and all the tokens. A K group's token rows are copied straight into LDS, double
// buffered, their scales beside them; the weights go to registers as they lie. Within a wave the MFMAs of one 32 x 32 tile
// and the f32 scalings of the one before alternate, and the LDS reads of the next 32 tokens go between; the next group's
// weights are asked for as this one's last MFMAs have them, and a wave that multiplies goes before one that waits (2048 x 4096
// x 14336 120.3 -> 118.1 us with both, 121.6 and 124.2 with either; 8192 x 14336 x 4096 417 -> 413). Bound by the matrix units
// where the launch fills the chip (128 x 256 tiles, 8192 x 14336 x 4096: 413 us, 2.33 PFLOP/s, 60 to 64% of the MFMA cycles
// busy; a library product with one scale takes 325), else by a step's own chain of LDS reads, MFMAs, scalings and a barrier
// (203 x 5003 x 2832 12.6 us; 64 x 4096 x 14336, on 128 CUs, 25: a CU fetches 43 and 55 GB/s there, and 53 where the launch
// fills the chip).
template <int MT, int NB, int WN, int KG, bool kExperts, bool kBf16>
__global__ __launch_bounds__(WN * KG * 64) __attribute__((amdgpu_waves_per_eu(2))) void fp8_tile_kernel(Fp8Args a)
{
    constexpr int kRows = 32 * MT;
    constexpr int kCopies = kRows / 8 / WN;            // of a wave, 1 KiB each: 8 rows
    constexpr int kScaleCopies = (kRows + 63) / 64;    // of a K group, 64 rows each
    constexpr int kRowBytes = kRows * kGroup;
    static_assert(kRows % (8 * WN) == 0 && kScaleCopies <= WN, "copies spread evenly over the waves");
    static_assert(WN == 2 || WN % 4 == 0, "a wave's copies lie 8 WN rows apart: slots of one kind, or of two in turn");
    __shared__ __align__(1024) uint8_t s_rows0[KG * kRowBytes];
    __shared__ __align__(1024) uint8_t s_rows1[KG * kRowBytes];
    __shared__ __align__(256) float s_scale0[KG * 64 * kScaleCopies];
    __shared__ __align__(256) float s_scale1[KG * 64 * kScaleCopies];
    const int tid = threadIdx.x, lane = tid & 63;
    const int wgwave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wave = wgwave % WN, kg = wgwave / WN; // wave within its K group
    const int col = lane & 31, h = lane >> 5;
    const int tiles_n = (a.ntiles + NB * WN - 1) / (NB * WN);
    RowTile rt;
    int tile_m, column;
    if (!place(a, tiles_n, &tile_m, &column) || !row_tile<kExperts>(a, kRows, tile_m, &rt))
        return;
    const int nt = column * (NB * WN) + wave * NB; // this wave's first tile of 32 weight rows
    float acc[MT][NB][16];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int nb = 0; nb < NB; ++nb)
#pragma unroll
            for (int i = 0; i < 16; ++i)
                acc[mt][nb][i] = 0.0f;

    if (!(kExperts && rt.expert == a.er.experts)) {
        const int G = a.groups, per = (G + KG - 1) / KG, g0 = kg * per, end = g0 + per; // G and more: scaled by 0
        // Copy j of a wave moves 8 rows, lane l chunk (l & 7) ^ slot_of(row) of row 8 (wave + WN j) + l / 8. Rows are told
        // by 32-bit offsets: from the first row of the tile, or of all input rows where they are gathered (the host
        // sees to it that these reach). Rows past the last one are the last one again.
        const int chunk = (lane & 7) ^ slot_of((8 * wave + (lane >> 3)) & 31); // of even copies; odd ones with WN == 2: ^ 2
        const __amdgpu_buffer_rsrc_t xr = open_rsrc(a.er.rows ? a.xv : a.xv + rt.row0 * a.ldxv);
        uint32_t xo[kCopies];
#pragma unroll
        for (int j = 0; j < kCopies; ++j) {
            const int row = min(8 * (wave + WN * j) + (lane >> 3), rt.count - 1);
            xo[j] = (uint32_t)(a.er.rows ? source_row(a.er, rt.row0 + row) : row) * (uint32_t)a.ldxv;
        }
        const __amdgpu_buffer_rsrc_t sr = open_rsrc(a.er.rows ? a.xs : a.xs + rt.row0 * a.ldxs);
        const uint32_t gs4 = 4u * (uint32_t)a.gsxs;
        const int srow = min(64 * (wave % kScaleCopies) + lane, rt.count - 1);
        const uint32_t so = 4u * (uint32_t)(a.er.rows ? source_row(a.er, rt.row0 + srow) : srow) * (uint32_t)a.ldxs;
        // tiles past the weight's last read it again: their sums are not stored
        __amdgpu_buffer_rsrc_t wp[NB];
#pragma unroll
        for (int nb = 0; nb < NB; ++nb)
            wp[nb] = open_rsrc(a.packed + ((int64_t)rt.expert * a.ntiles + min(nt + nb, a.ntiles - 1)) * G * kFp8Tile);
        const constant_floats ws = (constant_floats)(uintptr_t)(a.ws + ((int64_t)rt.expert * ((a.n + kGroup - 1) / kGroup) +
                                                                        min(nt, a.ntiles - 1) * kTileN / kGroup) * G);
        // a chunk past the row's end meets zero weights: any of the row does
        const uint32_t whole = 16u * chunk, last = (G - 1) * kGroup + 16 * chunk < a.k ? whole : 0u;
        const uint32_t whole1 = whole ^ 32u, last1 = (G - 1) * kGroup + (int)whole1 < a.k ? whole1 : 0u;

        auto stage = [&](uint8_t *rows, float *scale, int g) {
            const uint32_t off[2] = {g >= G - 1 ? last : whole, g >= G - 1 ? last1 : whole1};
            const int gc = min(g, G - 1);
#pragma unroll
            for (int j = 0; j < kCopies; ++j) {
                const uint32_t vo = xo[j] + off[WN == 2 ? j & 1 : 0]; // (the host pass drops the kernel with the element as an argument)
                __builtin_amdgcn_raw_ptr_buffer_load_lds(xr, (lds_ptr)(rows + kg * kRowBytes + 1024 * (wave + WN * j)), 16,
                                                         vo, gc * kGroup, 0, 0);
            }
            // waves past the last 64 rows repeat a copy (the same bytes): behind a branch the compiler could not count the
            // copies in flight
            __builtin_amdgcn_raw_ptr_buffer_load_lds(sr, (lds_ptr)(scale + 64 * (kg * kScaleCopies + wave % kScaleCopies)), 4,
                                                     so, gc * gs4, 0, 0);
        };
        uint4 w[NB][2][2]; // [tile][K step of 64][half]
        float wscale;
        uint32_t lane16 = 16 * lane;
        asm volatile("" : "+v"(lane16)); // or the compiler keeps a register for each of the four offsets below
        auto load_w = [&](int nb, int g) {
            const int gc = min(g, G - 1);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const auto v = __builtin_amdgcn_raw_buffer_load_b128(wp[nb], lane16 + 1024 * j, gc * kFp8Tile, 0);
                w[nb][j >> 1][j & 1] = uint4{v[0], v[1], v[2], v[3]};
            }
            if (nb == NB - 1)
                wscale = KG == 1 || g < G ? ws[gc] : 0.0f;
        };
        // chunk 4s + 2j + h of row r
        uint32_t slot[2][2];
#pragma unroll
        for (int j = 0; j < 4; ++j)
            slot[j >> 1][j & 1] = kg * kRowBytes + 128u * col + 16u * ((2 * j + h) ^ slot_of(col));

        // the weights of group `next` are asked for as the last tiles are done with this group's
        auto multiply_group = [&](const uint8_t *rows, const float *scale, int next) {
            v16f c[2];
            float f[2];
            uint4 x[2][2][2];
            auto load_x = [&](int mt) {
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    x[mt & 1][j >> 1][j & 1] = *reinterpret_cast<const uint4 *>(rows + 4096 * mt + slot[j >> 1][j & 1]);
                f[mt & 1] = scale[64 * kg * kScaleCopies + 32 * mt + col] * wscale;
            };
            load_x(0);
#pragma unroll
            for (int p = 0; p <= MT * NB; ++p) {
                const int mt = p / NB, nb = p % NB, q = p > 0 ? p - 1 : 0;
                const float fq = f[(q / NB) & 1];
                auto scale_sums = [&](int i0) {
                    if (p > 0)
#pragma unroll
                        for (int i = i0; i < i0 + 8; ++i)
                            acc[q / NB][q % NB][i] = __builtin_fmaf(c[q & 1][i], fq, acc[q / NB][q % NB][i]);
                    __builtin_amdgcn_sched_barrier(0);
                };
                if (p > MT * NB - NB) {
                    load_w(p - (MT * NB - NB) - 1, next);
                    __builtin_amdgcn_sched_barrier(0);
                }
                if (p < MT * NB) {
                    c[p & 1] = multiply<!kBf16>(w[nb][0], x[mt & 1][0], v16f{});
                    __builtin_amdgcn_sched_barrier(0);
                    if (nb == 0 && NB > 1 && mt + 1 < MT)
                        load_x(mt + 1);
                }
                scale_sums(0);
                if (p < MT * NB) {
                    c[p & 1] = multiply<!kBf16>(w[nb][1], x[mt & 1][1], c[p & 1]);
                    __builtin_amdgcn_sched_barrier(0);
                }
                scale_sums(8);
                if (NB == 1 && p < MT * NB && mt + 1 < MT)
                    load_x(mt + 1);
            }
        };
        constexpr int kVm = 0x0F70 | (4 * NB); // the copies are done, the weights behind them need not be
        stage(s_rows0, s_scale0, g0);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int nb = 0; nb < NB; ++nb)
            load_w(nb, g0);
        __builtin_amdgcn_sched_barrier(0);
        __builtin_amdgcn_s_waitcnt(kVm);
        __syncthreads();
        __builtin_amdgcn_sched_barrier(0);
        for (int g = g0; g < end; g += 2) {
            stage(s_rows1, s_scale1, g + 1);
            __builtin_amdgcn_sched_barrier(0);
            __builtin_amdgcn_s_setprio(1);
            multiply_group(s_rows0, s_scale0, g + 1);
            __builtin_amdgcn_sched_barrier(0);
            __builtin_amdgcn_s_setprio(0);
            __builtin_amdgcn_s_waitcnt(kVm);
            __syncthreads();
            __builtin_amdgcn_sched_barrier(0);
            if (g + 1 >= end)
                break;
            stage(s_rows0, s_scale0, g + 2);
            __builtin_amdgcn_sched_barrier(0);
            __builtin_amdgcn_s_setprio(1);
            multiply_group(s_rows1, s_scale1, g + 2);
            __builtin_amdgcn_sched_barrier(0);
            __builtin_amdgcn_s_setprio(0);
            __builtin_amdgcn_s_waitcnt(kVm);
            __syncthreads();
            __builtin_amdgcn_sched_barrier(0);
        }
        __builtin_amdgcn_s_waitcnt(0x0F70);
        // the K groups' sums, the upper half's added to the lower half's until one is left
        if constexpr (KG > 1) {
            static_assert(WN * 4096 * (KG / 2) <= KG * kRowBytes, "half the groups' sums of a tile fit a buffer");
#pragma unroll
            for (int half = KG / 2; half > 0; half /= 2)
#pragma unroll
                for (int t = 0; t < MT * NB; ++t) {
                    __syncthreads();
                    float *red = reinterpret_cast<float *>(t & 1 ? s_rows1 : s_rows0) + 1024 * (wave + WN * (kg % half));
                    float(&sum)[16] = acc[t / NB][t % NB];
                    if (kg >= half && kg < 2 * half)
#pragma unroll
                        for (int i = 0; i < 16; ++i)
                            red[64 * i + lane] = sum[i];
                    __syncthreads();
                    if (kg < half)
#pragma unroll
                        for (int i = 0; i < 16; ++i)
                            sum[i] += red[64 * i + lane];
                }
        }
    }
    __syncthreads(); // every wave has read its last rows
    if (kg)
        return;
    // A lane's sums are those of token col and weight rows 8 j + 4 h + 0 .. 3 of each 32: stored as they are, every store
    // would touch 32 lines with 16 bytes each. They go through LDS, 128 bytes a token at a time (chunk c of token t at slot
    // c ^ (t & 7), in a region of the wave's own), and out in whole lines.
    constexpr int kSpan = kBf16 && NB > 1 ? 64 : 32; // columns
    constexpr int kTiles = kSpan / kTileN;
    constexpr int kBytes = kSpan * (kBf16 ? 2 : 4), kChunks = kBytes / 16; // of a token
    static_assert(NB % kTiles == 0 && KG * kRowBytes >= kBytes * 32 * (WN / 2), "a region per wave");
    uint8_t *region = (wave & 1 ? s_rows1 : s_rows0) + 32 * kBytes * (wave >> 1);
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int nb = 0; nb < NB; nb += kTiles) {
#pragma unroll
            for (int t = 0; t < kTiles; ++t)
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const v4f v = {acc[mt][nb + t][4 * j], acc[mt][nb + t][4 * j + 1], acc[mt][nb + t][4 * j + 2],
                                   acc[mt][nb + t][4 * j + 3]};
                    const int c = kBf16 ? 4 * t + j : 2 * j + h;
                    uint8_t *to = region + kBytes * col + 16 * (c ^ (col & (kChunks - 1)));
                    if constexpr (kBf16)
                        *reinterpret_cast<bf16x4 *>(to + 8 * h) = __builtin_convertvector(v, bf16x4);
                    else
                        *reinterpret_cast<v4f *>(to) = v;
                }
            const int c = lane & (kChunks - 1), at = (nt + nb) * kTileN + c * (kSpan / kChunks);
#pragma unroll
            for (int p = 0; p < kChunks / 2; ++p) {
                const int t = 64 / kChunks * p + lane / kChunks, token = 32 * mt + t;
                const uint4 v = *reinterpret_cast<const uint4 *>(region + kBytes * t + 16 * (c ^ (t & (kChunks - 1))));
                if (token < rt.count)
                    store_chunk<kBf16>(a.out, (rt.row0 + token) * a.ldo + at, v, a.n - at, a.vec);
            }
        }
}

// The kernels of a product: tokens and weight rows of a workgroup, K groups of waves in it, workgroups that a CU holds, and
// microseconds: of a launch, of a round of workgroups on the busiest CU, of a step of a K group with 1, 2, .. of them on
// the CU, per million outputs and, beside these (the longer of the two hides most of the other: their squares add up), per
// million weights.
struct Fp8Kernel {
    int tokens, rows, kg, resident;
    double launch, round, step[4], outputs, weights;
};
// Fitted to 355 products a dense table (1 to 8192 tokens, 300 to 57344 rows, K 272 to 28672, weights rotated past the caches)
// and 174 by expert with bf16 outputs; float32 outputs by expert go by the dense table of theirs, and the kernel that it picks
// takes 3% more than the fastest on average over 100 products (1 to 512 rows of each of 4 to 128 experts), most 58% (64 rows of
// 8, 2880 x 2880). The kernel that they pick takes 0.8% more than the fastest of the nine on average (f32 0.9%, by
// expert, where they do not know how the rows fall, 3.3%; measured again, with 66 more by expert, 1.0%, 1.0% and 3.7%). None
// of the nine is spare: without it the fastest of the others takes 0.2 to 3% more on average and up to 1.11 to 1.63 times.
// Measured beside them: 128 x 128 tiles, 64 x 64 of eight K groups, 64 x 128 and 64 x 64 of one and two (no gain of 0.5%);
// a second and a third buffer for the weights and the rows (0 to 25% slower: a step is not bound by the latency of its
// loads).
constexpr Fp8Kernel kFp8Kernels[3][9] = {
    // float32 outputs
    {{16, 16, 8, 2, 2.601, 0.338, {0.707, 1.432}, 9.221, 0.000},
     {16, 32, 4, 4, 2.726, 0.394, {0.474, 0.952, 1.534, 1.873}, 2.753, 0.110},
     {16, 64, 4, 4, 2.533, 0.749, {0.750, 1.498, 2.334, 3.287}, 1.519, 0.144},
     {32, 64, 4, 3, 3.442, 0.230, {0.638, 1.208, 1.874}, 1.844, 0.166},
     {64, 64, 4, 2, 3.421, 1.014, {1.004, 2.267}, 2.027, 0.145},
     {64, 128, 2, 2, 4.146, 0.000, {0.965, 2.095}, 1.180, 0.136},
     {64, 256, 2, 1, 3.914, 0.791, {1.676}, 1.215, 0.137},
     {64, 256, 1, 2, 4.216, 0.000, {1.101, 1.726}, 0.644, 0.149},
     {0, 0, 0, 0, 0.0, 0.0, {}, 0.0, 0.0}}, // 128 x 256 tiles through bf16 spill
    // bfloat16 outputs
    {{16, 16, 8, 2, 2.617, 0.179, {0.729, 1.417}, 12.342, 0.000},
     {16, 32, 4, 4, 2.904, 0.000, {0.472, 0.943, 1.505, 1.882}, 3.222, 0.108},
     {16, 64, 4, 4, 3.040, 0.000, {0.726, 1.432, 2.188, 3.133}, 1.687, 0.134},
     {32, 64, 4, 3, 3.307, 0.320, {0.500, 1.100, 1.610}, 0.913, 0.180},
     {64, 64, 4, 2, 3.453, 0.669, {0.695, 1.476}, 0.996, 0.184},
     {64, 128, 2, 2, 3.595, 0.120, {0.595, 1.183}, 0.514, 0.179},
     {64, 256, 2, 1, 3.285, 1.096, {1.075}, 0.570, 0.182},
     {64, 256, 1, 2, 3.324, 0.000, {0.754, 1.005}, 0.381, 0.160},
     {128, 256, 1, 2, 3.501, 1.251, {1.049, 1.706}, 0.240, 0.150}},
    // bfloat16 outputs by expert
    {{16, 16, 8, 2, 4.761, 0.359, {0.334, 1.006}, 31.116, 0.066},
     {16, 32, 4, 4, 4.101, 0.000, {0.572, 0.893, 1.395, 1.797}, 9.507, 0.068},
     {16, 64, 4, 4, 3.539, 0.000, {1.028, 1.887, 2.402, 2.838}, 10.820, 0.086},
     {32, 64, 4, 3, 4.257, 0.000, {0.548, 1.371, 1.921}, 2.891, 0.138},
     {64, 64, 4, 2, 5.214, 0.000, {0.645, 1.406}, 3.692, 0.139},
     {64, 128, 2, 2, 4.246, 0.000, {0.560, 1.346}, 1.068, 0.155},
     {64, 256, 2, 1, 4.125, 0.000, {0.898}, 2.742, 0.162},
     {64, 256, 1, 2, 2.893, 0.000, {0.697, 1.118}, 0.775, 0.154},
     {128, 256, 1, 2, 4.436, 0.000, {1.007, 1.513}, 0.833, 0.139}}};
constexpr int kFirstTile = 3; // those from here on address rows by 32-bit offsets
constexpr int kThreads[9] = {512, 256, 256, 512, 512, 512, 512, 256, 256}; // of a workgroup
constexpr int64_t kCUs = 256;

double fp8_time(const Fp8Kernel &t, int64_t wgs, int64_t groups, double outputs, double weights)
{
    const int64_t per = cdiv(wgs, kCUs), full = per / t.resident, rem = per % t.resident;
    const double work = t.round * (double)(full + (rem ? 1 : 0)) + 1e-6 * t.outputs * outputs +
                        (double)cdiv(groups, t.kg) * ((double)full * t.step[t.resident - 1] + (rem ? t.step[rem - 1] : 0.0));
    return t.launch + std::hypot(work, 1e-6 * t.weights * weights);
}

// The order in which workgroups of `tokens` tokens, `tiles` x `columns` of them, go to the XCDs, and their number.
int64_t order_tiles(Fp8Args *a, int tokens, int64_t tiles, int64_t columns, double rows_of_expert)
{
    const int64_t total = tiles * columns;
    const bool grouped = a->er.offsets && a->er.experts > 1;
    const double reuse = rows_of_expert / tokens; // row tiles that read an expert's weight
    int64_t group = columns, deal = 1; // row tile by row tile, to the XCDs in turn
    if (!grouped) {
        // An eighth of all to each XCD, so that the row tiles that read a weight do it in one L2: 256 x 2880 x 5120 16.5 ->
        // 12.3 us, 768 x 7000 x 6144 81 -> 49, the more the less the columns are a multiple of eight by themselves. Of many
        // row tiles a few columns at a time, which share the rows (8192 x 14336 x 4096 468 -> 444).
        group = tiles >= 8 ? 4 : 1;
        deal = cdiv(total, 8);
    } else if (total >= 768 && reuse >= (columns % 8 ? 2.0 / 3.0 : 4.0)) {
        // 32 neighbours at a time, for which row tiles there are is not known: an eighth at a time, the last XCD would have
        // the tiles of no rows. From 768 workgroups on, 24 deals, three an XCD: fewer fall too unevenly (48 rows of 16, 2880 x
        // 2880, 348 workgroups, 30 -> 48 us; 96 of 8, 7000 x 4096, 588, 73 -> 83), though some would gain (192 of 32, 600 x 5120,
        // 645, 80 -> 56). Where the columns are a multiple of eight, an XCD has columns of its own in turn too, and
        // gains with many row tiles alone (65536 rows of 64 experts, 2048 x 4096 596 -> 569 us, 16384 188 -> 190, 4096 rows of
        // 16, 4096 x 4096 74 -> 77); else 8192 of 32, 600 x 5120 89 -> 62, 16384 of 128, 1536 x 2048 129 -> 119, 12000 111 ->
        // 100 (but 4096 of 32, 2880 x 2880 86 -> 97).
        group = 8;
        deal = 32;
    } else if (reuse > 1.0 && columns >= 8 && columns % 8) {
        group = 1; // every XCD has columns of its own
        deal = cdiv(total, 8);
    }
    a->tiles = (uint32_t)tiles;
    a->group = (uint32_t)std::min(group, columns);
    a->deal = (uint32_t)deal;
    return cdiv(total, 8 * deal) * 8 * deal;
}

// The kernel of a product, the order of its workgroups and their number. How the rows fall to the experts is not known here:
// the tiles that they take are counted for rows that fall to them at random, and the grid holds the most that they can take.
int fp8_plan(Fp8Args *a, bool bf16, int64_t *wgs)
{
    const ExpertRows &er = a->er;
    const bool far = a->ldxv * (er.rows ? er.m : 128) + a->k >= ((int64_t)1 << 32) ||
                     4 * (a->ldxs * (er.rows ? er.m : 128) + a->gsxs * a->groups) >= ((int64_t)1 << 32);
    const bool grouped = er.offsets && er.experts > 1; // one expert's rows take the kernel that they would take without
    const double r = (double)er.r, taken = grouped ? er.experts * -std::expm1(-r / er.experts) : 1.0;
    int best = -1;
    double least = 0.0;
    for (int i = 0; i < (far ? kFirstTile : 9); ++i) {
        const Fp8Kernel &t = kFp8Kernels[bf16 ? grouped ? 2 : 1 : 0][i];
        if (!t.tokens)
            continue;
        const int64_t columns = cdiv(a->n, t.rows), most = er.offsets ? expert_row_tiles(er.r, er.experts, t.tokens) : cdiv(er.r, t.tokens);
        if (!grid_takes(most * columns + 255, kThreads[i])) // with what the order rounds up to; place() adds in 32 bits
            continue;
        const double tiles = grouped ? std::fmax(taken, r / t.tokens + 0.5 * taken) : (double)cdiv(er.r, t.tokens);
        const double us = fp8_time(t, (int64_t)std::ceil(tiles) * columns, a->groups, r * a->n, taken * a->n * a->k);
        if (best < 0 || us < least) {
            best = i;
            least = us;
            *wgs = order_tiles(a, t.tokens, most, columns, r / taken);
        }
    }
    return best;
}

// Whether scales of m rows and `groups` groups at these strides lie apart: rows of groups, or groups of rows.
bool scales_apart(int64_t ld, int64_t gs, int64_t m, int64_t groups)
{
    return m == 0 || (ld >= 1 && gs >= 1 && (ld >= gs * groups || gs >= ld * m));
}

template <bool kExperts, bool kBf16>
int launch_products(const Fp8Args &a, int which, int64_t wgs, hipStream_t stream)
{
#define MAMBO_STREAM(I, H, W)                                                                                      \
    case I:                                                                                                        \
        static_assert(kThreads[I] == W * 64);                                                                      \
        MAMBO_LAUNCH((fp8_stream_kernel<H, W, kExperts, kBf16>), dim3((unsigned)wgs), dim3(W * 64), 0, stream, a); \
        break
#define MAMBO_TILE(I, MT, NB, WN, KG)                                                                              \
    case I:                                                                                                        \
        static_assert(kThreads[I] == WN * KG * 64);                                                                \
        MAMBO_LAUNCH((fp8_tile_kernel<MT, NB, WN, KG, kExperts, kBf16>), dim3((unsigned)wgs), dim3(WN * KG * 64), 0,     \
                     stream, a);                                                                                   \
        break
    switch (which) {
        MAMBO_STREAM(0, 1, 8);
        MAMBO_STREAM(1, 2, 4);
        MAMBO_STREAM(2, 4, 4);
        MAMBO_TILE(3, 1, 1, 2, 4);
        MAMBO_TILE(4, 2, 1, 2, 4);
        MAMBO_TILE(5, 2, 1, 4, 2);
        MAMBO_TILE(6, 2, 2, 4, 2);
        MAMBO_TILE(7, 2, 2, 4, 1);
    default:
        if constexpr (kBf16) {
            switch (which) {
                MAMBO_TILE(8, 4, 2, 4, 1);
            }
        }
    }
#undef MAMBO_STREAM
#undef MAMBO_TILE
    return mambo_check_launch("fp8_block_matmul");
}

int check_product(int64_t n, int64_t k, int out_dtype)
{
    MAMBO_REQUIRE(out_dtype == MAMBO_DTYPE_F32 || out_dtype == MAMBO_DTYPE_BF16, MAMBO_ERR_VALUE,
                  "outputs must be float32 or bfloat16");
    MAMBO_REQUIRE(n >= 1 && n <= 0x7FFFFF00 && k >= 16 && k <= kMaxK && k % 16 == 0, MAMBO_ERR_VALUE,
                  "weights must be [N,K] with N >= 1 and K a multiple of 16 up to 2^26 (got N=%lld K=%lld)", (long long)n, (long long)k);
    return MAMBO_OK;
}

int run_products(const uint8_t *xv, int64_t ldxv, const float *xs, int64_t ldxs, int64_t gsxs, const ExpertRows &er,
                 const uint8_t *packed, const float *ws, int64_t n, int64_t k, void *out, int out_dtype, int64_t ldo,
                 hipStream_t stream)
{
    const int rc = check_product(n, k, out_dtype);
    if (rc != MAMBO_OK)
        return rc;
    MAMBO_REQUIRE(ldxv >= k && ldo >= n && scales_apart(ldxs, gsxs, er.m, cdiv(k, kGroup)), MAMBO_ERR_VALUE,
                  "strides must cover the rows");
    if (er.r == 0)
        return MAMBO_OK;
    MAMBO_REQUIRE(xv && xs && packed && ws && out, MAMBO_ERR_VALUE, "null pointer");
    MAMBO_REQUIRE((uintptr_t)xv % 16 == 0 && ldxv % 16 == 0 && (uintptr_t)packed % 16 == 0, MAMBO_ERR_VALUE,
                  "rows and packed weights must be 16-byte aligned");
    MAMBO_REQUIRE((uintptr_t)xs % 4 == 0 && (uintptr_t)ws % 4 == 0 &&
                      (uintptr_t)out % (out_dtype == MAMBO_DTYPE_BF16 ? 2 : 4) == 0,
                  MAMBO_ERR_VALUE, "scales and outputs must be aligned to their type");
    Fp8Args a = {xv, xs, ldxv, ldxs, gsxs, er, packed, ws, out, ldo, (int)n, (int)k, (int)cdiv(k, kGroup), (int)cdiv(n, kTileN),
                 rows_take_vectors(out, ldo, out_dtype), 0, 0, 0};
    const bool bf16 = out_dtype == MAMBO_DTYPE_BF16;
    int64_t wgs = 0;
    const int which = fp8_plan(&a, bf16, &wgs);
    MAMBO_REQUIRE(which >= 0, MAMBO_ERR_VALUE, "too many rows and columns for one launch");
    if (er.offsets)
        return bf16 ? launch_products<true, true>(a, which, wgs, stream) : launch_products<true, false>(a, which, wgs, stream);
    return bf16 ? launch_products<false, true>(a, which, wgs, stream) : launch_products<false, false>(a, which, wgs, stream);
}

} // namespace

extern "C" int mambo_quantize_fp8_block(const void *x, int x_dtype, int64_t m, int64_t k, int64_t ldx, uint8_t *values,
                                        int64_t ldv, float *scales, int64_t lds, int64_t gss, mambo_stream_t stream)
{
    MAMBO_REQUIRE(x_dtype == MAMBO_DTYPE_F32 || x_dtype == MAMBO_DTYPE_BF16, MAMBO_ERR_VALUE,
                  "activation dtype must be float32 or bfloat16");
    MAMBO_REQUIRE(m >= 0 && k >= 16 && k <= 0x7FFFFF00 && k % 16 == 0, MAMBO_ERR_VALUE,
                  "activation must be [M,K] with K a multiple of 16 (got M=%lld K=%lld)", (long long)m, (long long)k);
    const int64_t groups = cdiv(k, kGroup);
    MAMBO_REQUIRE(ldx >= k && ldv >= k && scales_apart(lds, gss, m, groups), MAMBO_ERR_VALUE, "strides must cover K");
    if (m == 0)
        return MAMBO_OK;
    MAMBO_REQUIRE(x && values && scales, MAMBO_ERR_VALUE, "null pointer");
    const bool bf16 = x_dtype == MAMBO_DTYPE_BF16;
    MAMBO_REQUIRE((uintptr_t)x % (bf16 ? 2 : 4) == 0 && (uintptr_t)scales % 4 == 0, MAMBO_ERR_VALUE,
                  "rows and scales must be aligned to their type");
    const bool vec = (uintptr_t)x % 16 == 0 && ldx % (bf16 ? 8 : 4) == 0 && (uintptr_t)values % 8 == 0 && ldv % 8 == 0;
    const int at_once = m * cdiv(groups, 16) >= 4096 ? 2 : 1; // fewer do not fill the card twice
    const int64_t ry = cdiv(m, at_once);
    const dim3 grid((unsigned)cdiv(groups, 16), (unsigned)(ry < 65535 ? ry : 65535));
    hipStream_t s = (hipStream_t)stream;
#define MAMBO_QUANT(B, V, R)                                                                                       \
    if (bf16 == B && vec == V && at_once == R)                                                                     \
    MAMBO_LAUNCH((quantize_fp8_block_kernel<B, V, R>), grid, dim3(256), 0, s, x, ldx, m, (int)k, values, ldv, scales, lds, \
                 gss)
    MAMBO_QUANT(true, true, 1);
    MAMBO_QUANT(true, true, 2);
    MAMBO_QUANT(true, false, 1);
    MAMBO_QUANT(true, false, 2);
    MAMBO_QUANT(false, true, 1);
    MAMBO_QUANT(false, true, 2);
    MAMBO_QUANT(false, false, 1);
    MAMBO_QUANT(false, false, 2);
#undef MAMBO_QUANT
    return mambo_check_launch("quantize_fp8_block");
}

extern "C" int64_t mambo_fp8_block_packed_bytes(int64_t experts, int64_t n, int64_t k)
{
    if (experts < 1 || n < 1 || k < 1 || n > 0x7FFFFF00 || k > kMaxK || experts > MAMBO_MAX_EXPERTS)
        return 0;
    return experts * cdiv(n, kTileN) * cdiv(k, kGroup) * kFp8Tile;
}

extern "C" int mambo_fp8_block_pack(const uint8_t *w, int64_t experts, int64_t n, int64_t k, int64_t stride_e,
                                    int64_t stride_n, uint8_t *packed, mambo_stream_t stream)
{
    MAMBO_REQUIRE(experts >= 1 && experts <= MAMBO_MAX_EXPERTS && n >= 1 && n <= 0x7FFFFF00 && k >= 16 &&
                      k <= kMaxK && k % 16 == 0,
                  MAMBO_ERR_VALUE,
                  "weights must be [E,N,K] with E in [1, %d], N >= 1 and K a multiple of 16 up to 2^26 (got E=%lld N=%lld K=%lld)",
                  MAMBO_MAX_EXPERTS, (long long)experts, (long long)n, (long long)k);
    MAMBO_REQUIRE(w && packed, MAMBO_ERR_VALUE, "null pointer");
    MAMBO_REQUIRE((uintptr_t)packed % 16 == 0, MAMBO_ERR_VALUE, "packed must be 16-byte aligned");
    const int64_t ntiles = cdiv(n, kTileN), groups = cdiv(k, kGroup), tiles = experts * ntiles * groups;
    MAMBO_REQUIRE(grid_takes(tiles, 256), MAMBO_ERR_VALUE, "weights too large for one call");
    const bool vec = (uintptr_t)w % 16 == 0 && stride_e % 16 == 0 && stride_n % 16 == 0;
    MAMBO_LAUNCH(fp8_block_pack_kernel, dim3((unsigned)tiles), dim3(256), 0, (hipStream_t)stream, w, n, k, stride_e,
                 stride_n, ntiles, groups, vec, packed);
    return mambo_check_launch("fp8_block_pack");
}

extern "C" int mambo_fp8_block_matmul(const uint8_t *xv, int64_t ldxv, const float *xs, int64_t ldxs, int64_t gsxs,
                                      int64_t m, const uint8_t *packed, const float *ws, int64_t n, int64_t k, void *out,
                                      int out_dtype, int64_t ldo, mambo_stream_t stream)
{
    MAMBO_REQUIRE(m >= 0, MAMBO_ERR_VALUE, "rows must not be negative");
    const ExpertRows er = {nullptr, nullptr, m, m, 1};
    return run_products(xv, ldxv, xs, ldxs, gsxs, er, packed, ws, n, k, out, out_dtype, ldo, (hipStream_t)stream);
}

extern "C" int mambo_fp8_block_plan(int64_t m, int64_t r, int64_t experts, int64_t n, int64_t k, int64_t ldxv,
                                    int out_dtype, int32_t *plan)
{
    static const int32_t one = 0; // never read: that the plan is of rows by expert, or gathered
    const int32_t *rows = experts && m != r ? &one : nullptr, *offsets = experts ? &one : nullptr;
    int rc = check_product(n, k, out_dtype);
    if (rc == MAMBO_OK)
        rc = check_expert_rows(m, rows, experts ? r : m, experts ? offsets : &one, experts ? experts : 1);
    if (rc != MAMBO_OK)
        return rc;
    MAMBO_REQUIRE(ldxv >= k && plan && (experts ? r : m) >= 1, MAMBO_ERR_VALUE, "a plan is of one row or more");
    Fp8Args a = {};
    a.er = {offsets, rows, experts ? r : m, m, (int)(experts ? experts : 1)};
    a.ldxv = ldxv, a.ldxs = 1, a.gsxs = m;
    a.n = (int)n, a.k = (int)k, a.groups = (int)cdiv(k, kGroup);
    int64_t wgs = 0;
    const int which = fp8_plan(&a, out_dtype == MAMBO_DTYPE_BF16, &wgs);
    MAMBO_REQUIRE(which >= 0, MAMBO_ERR_VALUE, "too many rows and columns for one launch");
    const Fp8Kernel &t = kFp8Kernels[out_dtype == MAMBO_DTYPE_BF16][which]; // the sizes are the same by expert
    plan[0] = t.tokens, plan[1] = t.rows, plan[2] = t.kg;
    plan[3] = (int32_t)a.group, plan[4] = (int32_t)a.deal;
    return MAMBO_OK;
}

extern "C" int mambo_fp8_block_matmul_experts(const uint8_t *xv, int64_t ldxv, const float *xs, int64_t ldxs, int64_t gsxs,
                                              int64_t m, const int32_t *rows, int64_t r, const int32_t *offsets, int64_t experts,
                                              const uint8_t *packed, const float *ws, int64_t n, int64_t k, void *out,
                                              int out_dtype, int64_t ldo, mambo_stream_t stream)
{
    const int rc = check_expert_rows(m, rows, r, offsets, experts);
    if (rc != MAMBO_OK)
        return rc;
    const ExpertRows er = {offsets, rows, r, m, (int)experts};
    return run_products(xv, ldxv, xs, ldxs, gsxs, er, packed, ws, n, k, out, out_dtype, ldo, (hipStream_t)stream);
}
