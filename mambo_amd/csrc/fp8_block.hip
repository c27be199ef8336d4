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
// An FP8 MFMA aligns the products of eight consecutive K and keeps 14 bits below the largest of them
// (measured on gfx950: beside a product of 2^16 one of 2^3 counts and one of 2^2 does not, in the
// 16 x 16 x 128 and 32 x 32 x 64 shapes and in the older 16 x 16 x 32 and 32 x 32 x 16 alike), an error of
// up to 1.7e-4 of the sum of magnitudes, 5e-5 in the 2-norm over codes of all exponents. That is 2^-5 of
// what rounding to bf16 takes, so bf16 outputs use it. f32 outputs are of f32 sums: the codes are widened
// to bf16, exactly, and multiplied by the bf16 MFMAs, which add without that loss (2.5e-7 on the same
// data), at half the matrix rate.
//
// Layout of a weight (mambo_fp8_block_pack): tiles of 32 rows x 128 of K, 4096 bytes, ordered
// [expert][n / 32][k / 128]; within a tile 16-byte chunk c of row i (K 16c .. 16c+15 of the group) at
// 512 c + 16 i. A wave's load of 16 bytes a lane is then 1 KiB in one piece, and lands as the
// operand: lane (i, h) of the 32 x 32 MFMA of K step s takes chunks 4s + h and 4s + 2 + h, of the 16 x
// 16 MFMA chunks h and 4 + h. Rows past n and K past k are zeros, so nothing else looks after the
// ends of a weight. (Any order of K serves that both operands share.)
#include <type_traits>

#include "experts.h"

namespace {

constexpr int kGroup = 128;      // K of one scale
constexpr int kTileN = 32;       // weight rows of a tile
constexpr int kFp8Tile = 4096;   // bytes of a tile
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

template <bool kBf16, bool kVec>
__global__ __launch_bounds__(256) void quantize_fp8_block_kernel(const void *__restrict__ x, int64_t ldx, int64_t m,
                                                                 int k, uint8_t *__restrict__ values, int64_t ldv,
                                                                 float *__restrict__ scales, int64_t lds)
{
    const int at = (int)(blockIdx.x * 16 + (threadIdx.x >> 4)) * kGroup + 8 * (threadIdx.x & 15); // in the row
    const bool in = at < k; // k is a multiple of 16, so all eight or none
    for (int64_t row = blockIdx.y; row < m; row += gridDim.y) {
        float v[8] = {};
        if (in)
            load8<kBf16, kVec>(x, row * ldx + at, v);
        uint32_t amax = 0u; // over the magnitude bits: a NaN beats an infinity, that every number
#pragma unroll
        for (int i = 0; i < 8; ++i)
            amax = max(amax, abs_bits(v[i]));
#pragma unroll
        for (int d = 1; d < 16; d <<= 1)
            amax = max(amax, (uint32_t)__shfl_xor((int)amax, d));
        if (!in)
            continue;
        const bool finite = amax < kNonFiniteBits;
        const float top = fmaxf(__uint_as_float(amax), 448.0f * kSmallestScale);
        const float b = top * 0x1p-9f, inv = 1.0f / b;
        float q[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float a = 0.875f * v[i], y = a * inv;
            q[i] = __builtin_copysignf(__builtin_fmaf(__builtin_fmaf(-y, b, a), inv, y), a); // -0 stays -0
        }
        uint2 codes;
        if (finite) {
            codes.x = pack4<kQuantHwCvt>(q[0], q[1], q[2], q[3]);
            codes.y = pack4<kQuantHwCvt>(q[4], q[5], q[6], q[7]);
        } else {
            codes.x = nan4(v[0], v[1], v[2], v[3]);
            codes.y = nan4(v[4], v[5], v[6], v[7]);
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
            scales[row * lds + at / kGroup] = finite ? top / 448.0f : __builtin_nanf("");
    }
}

// ============================================================================ weight layout
// One workgroup per tile: 256 threads, a 16-byte chunk each, read along the rows.
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
    int64_t ldxv, ldxs;
    ExpertRows er;
    const uint8_t *packed;
    const float *ws;
    void *out;
    int64_t ldo;
    int n, k, groups, ntiles; // groups of K, tiles of 32 weight rows
    bool vec;                 // the outputs take one store of four
};

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

// Few rows: bound by the weights' bytes. A workgroup computes T tokens x 32 weight rows; its W waves
// take the K groups in turn and every wave streams its own, a ring of D groups of weights and rows in
// registers and no barrier before the end, where the waves' sums meet in LDS and are added in order.
template <int T, int W, int D, bool kExperts, bool kBf16>
__global__ __launch_bounds__(W * 64) void fp8_stream_kernel(Fp8Args a)
{
    constexpr int S = T < 32 ? 16 : 32;  // tokens of an MFMA
    constexpr int U = T / S;             // MFMAs side by side
    constexpr int kRegs = S == 16 ? 4 : 16; // sums per lane of an MFMA
    constexpr int kHalves = S == 16 ? 2 : 1; // MFMAs that 32 weight rows take
    constexpr int kPad = 36;             // floats of a token's 32 sums in LDS
    __shared__ __align__(16) float s_red[W * T * kPad];
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int nt = blockIdx.x % a.ntiles;
    RowTile rt;
    if (!row_tile<kExperts>(a, T, blockIdx.x / a.ntiles, &rt))
        return;
    const bool none = kExperts && rt.expert == a.er.experts;

    if (!none) {
        const int col = lane & (S - 1), h = lane / S;
        const uint8_t *xp[U];
        const float *sp[U];
#pragma unroll
        for (int u = 0; u < U; ++u) { // lanes past the last row read it again: they feed sums that are not stored
            const int64_t src = source_row(a.er, rt.row0 + min(S * u + col, rt.count - 1));
            xp[u] = a.xv + src * a.ldxv;
            sp[u] = a.xs + src * a.ldxs;
        }
        const int64_t wtile = (int64_t)rt.expert * a.ntiles + nt;
        const uint8_t *wp = a.packed + wtile * a.groups * kFp8Tile + (S == 16 ? 512 * h + 16 * col : 16 * lane);
        const float *ws = a.ws + ((int64_t)rt.expert * ((a.n + kGroup - 1) / kGroup) + nt * kTileN / kGroup) * a.groups;

        float acc[U][kHalves][kRegs];
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int t = 0; t < kHalves; ++t)
#pragma unroll
                for (int i = 0; i < kRegs; ++i)
                    acc[u][t][i] = 0.0f;

        // operands of one K group: weights [half or step][32 bytes], rows [step][32 bytes]
        constexpr int kSteps = S == 16 ? 1 : 2;
        struct Ring {
            uint4 w[2][2], x[U][kSteps][2];
            float xs[U], ws;
        } ring[D];
        const int count = wave < a.groups ? (a.groups - wave + W - 1) / W : 0;
        auto load = [&](Ring &r, int i) {
            const int g = min(wave + min(i, count - 1) * W, a.groups - 1); // count 0: any group, scaled by 0
            const int gc = max(g, 0);
            const uint8_t *p = wp + (int64_t)gc * kFp8Tile;
#pragma unroll
            for (int j = 0; j < 4; ++j) { // S 16: (half j >> 1, chunk h + 4 (j & 1)); else (step j >> 1, chunk 4s + 2 (j & 1) + h)
                const int off = S == 16 ? 2048 * (j & 1) + 256 * (j >> 1) : 1024 * j;
                r.w[j >> 1][j & 1] = *reinterpret_cast<const uint4 *>(p + off);
            }
            const int k0 = gc * kGroup;
#pragma unroll
            for (int u = 0; u < U; ++u) {
#pragma unroll
                for (int j = 0; j < 2 * kSteps; ++j) {
                    // a chunk past the row's end meets zero weights: any chunk of the row does
                    const int at = k0 + 16 * (S == 16 ? h + 4 * j : 2 * j + h);
                    r.x[u][j >> 1][j & 1] = *reinterpret_cast<const uint4 *>(xp[u] + (at < a.k ? at : k0));
                }
                r.xs[u] = sp[u][gc];
            }
            r.ws = i < count ? ws[gc] : 0.0f;
        };
#pragma unroll
        for (int j = 0; j < D - 1; ++j)
            load(ring[j], j);
        for (int i0 = 0; i0 < count; i0 += D) {
#pragma unroll
            for (int j = 0; j < D; ++j) {
                load(ring[(j + D - 1) % D], i0 + j + D - 1);
                __builtin_amdgcn_sched_barrier(0);
                const Ring &r = ring[j];
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    const float f = r.xs[u] * r.ws;
                    if constexpr (S == 16) {
#pragma unroll
                        for (int t = 0; t < 2; ++t) {
                            const v4f c = multiply<!kBf16>(r.w[t], r.x[u][0], v4f{});
#pragma unroll
                            for (int q = 0; q < 4; ++q)
                                acc[u][t][q] = __builtin_fmaf(c[q], f, acc[u][t][q]);
                        }
                    } else {
                        const v16f c = multiply<!kBf16>(r.w[1], r.x[u][1], multiply<!kBf16>(r.w[0], r.x[u][0], v16f{}));
#pragma unroll
                        for (int q = 0; q < 16; ++q)
                            acc[u][0][q] = __builtin_fmaf(c[q], f, acc[u][0][q]);
                    }
                }
                __builtin_amdgcn_sched_barrier(0);
            }
        }
        // the sums of a lane: token col, weight rows 4 h + .. (S 16, half t: 16 t more), 8 j + 4 h + .. (S 32)
        float *red = s_red + wave * T * kPad;
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int t = 0; t < kHalves; ++t)
#pragma unroll
                for (int j = 0; j < kRegs; j += 4)
                    *reinterpret_cast<v4f *>(red + (S * u + col) * kPad + 16 * t + 2 * j + 4 * h) =
                        v4f{acc[u][t][j], acc[u][t][j + 1], acc[u][t][j + 2], acc[u][t][j + 3]};
    }
    __syncthreads();
    for (int i = tid; i < T * 8; i += W * 64) {
        const int token = i >> 3, n4 = 4 * (i & 7);
        if (token >= rt.count)
            break;
        v4f v = {0.0f, 0.0f, 0.0f, 0.0f};
        if (!none)
#pragma unroll
            for (int w = 0; w < W; ++w)
                v += *reinterpret_cast<const v4f *>(s_red + (w * T + token) * kPad + n4);
        const int at = nt * kTileN + n4;
        if (at < a.n)
            store_row4<kBf16>(a.out, (rt.row0 + token) * a.ldo + at, v, a.n - at, a.vec);
    }
}

template <bool kExperts, bool kBf16>
int launch_products(const Fp8Args &a, hipStream_t stream)
{
    const int64_t per = kExperts ? cdiv(a.er.r, a.er.experts) : a.er.r; // rows of an expert on average
    const int tile = per <= 16 ? 16 : 32;
    const int64_t tiles = kExperts ? expert_row_tiles(a.er.r, a.er.experts, tile) : cdiv(a.er.r, tile);
    const int64_t wgs = tiles * a.ntiles;
    MAMBO_REQUIRE(wgs <= 0x7FFFFFFF, MAMBO_ERR_VALUE, "too many rows and columns for one launch");
    if (tile == 16)
        MAMBO_LAUNCH((fp8_stream_kernel<16, 8, 3, kExperts, kBf16>), dim3((unsigned)wgs), dim3(512), 0, stream, a);
    else
        MAMBO_LAUNCH((fp8_stream_kernel<32, 8, 3, kExperts, kBf16>), dim3((unsigned)wgs), dim3(512), 0, stream, a);
    return mambo_check_launch("fp8_block_matmul");
}

int run_products(const uint8_t *xv, int64_t ldxv, const float *xs, int64_t ldxs, const ExpertRows &er,
                 const uint8_t *packed, const float *ws, int64_t n, int64_t k, void *out, int out_dtype, int64_t ldo,
                 hipStream_t stream)
{
    MAMBO_REQUIRE(out_dtype == MAMBO_DTYPE_F32 || out_dtype == MAMBO_DTYPE_BF16, MAMBO_ERR_VALUE,
                  "outputs must be float32 or bfloat16");
    MAMBO_REQUIRE(n >= 1 && n <= 0x7FFFFF00 && k >= 16 && k <= 0x7FFFFF00 && k % 16 == 0, MAMBO_ERR_VALUE,
                  "weights must be [N,K] with N >= 1 and K a multiple of 16 (got N=%lld K=%lld)", (long long)n, (long long)k);
    MAMBO_REQUIRE(ldxv >= k && ldxs >= cdiv(k, kGroup) && ldo >= n, MAMBO_ERR_VALUE, "row strides must cover the rows");
    if (er.r == 0)
        return MAMBO_OK;
    MAMBO_REQUIRE(xv && xs && packed && ws && out, MAMBO_ERR_VALUE, "null pointer");
    MAMBO_REQUIRE((uintptr_t)xv % 16 == 0 && ldxv % 16 == 0 && (uintptr_t)packed % 16 == 0, MAMBO_ERR_VALUE,
                  "rows and packed weights must be 16-byte aligned");
    MAMBO_REQUIRE((uintptr_t)xs % 4 == 0 && (uintptr_t)ws % 4 == 0 &&
                      (uintptr_t)out % (out_dtype == MAMBO_DTYPE_BF16 ? 2 : 4) == 0,
                  MAMBO_ERR_VALUE, "scales and outputs must be aligned to their type");
    Fp8Args a = {xv, xs, ldxv, ldxs, er, packed, ws, out, ldo, (int)n, (int)k, (int)cdiv(k, kGroup), (int)cdiv(n, kTileN),
                 rows_take_vectors(out, ldo, out_dtype)};
    const bool bf16 = out_dtype == MAMBO_DTYPE_BF16;
    if (er.offsets)
        return bf16 ? launch_products<true, true>(a, stream) : launch_products<true, false>(a, stream);
    return bf16 ? launch_products<false, true>(a, stream) : launch_products<false, false>(a, stream);
}

} // namespace

extern "C" int mambo_quantize_fp8_block(const void *x, int x_dtype, int64_t m, int64_t k, int64_t ldx, uint8_t *values,
                                        int64_t ldv, float *scales, int64_t lds, mambo_stream_t stream)
{
    MAMBO_REQUIRE(x_dtype == MAMBO_DTYPE_F32 || x_dtype == MAMBO_DTYPE_BF16, MAMBO_ERR_VALUE,
                  "activation dtype must be float32 or bfloat16");
    MAMBO_REQUIRE(m >= 0 && k >= 16 && k <= 0x7FFFFF00 && k % 16 == 0, MAMBO_ERR_VALUE,
                  "activation must be [M,K] with K a multiple of 16 (got M=%lld K=%lld)", (long long)m, (long long)k);
    const int64_t groups = cdiv(k, kGroup);
    MAMBO_REQUIRE(ldx >= k && ldv >= k && lds >= groups, MAMBO_ERR_VALUE, "row strides must cover K");
    if (m == 0)
        return MAMBO_OK;
    MAMBO_REQUIRE(x && values && scales, MAMBO_ERR_VALUE, "null pointer");
    const bool bf16 = x_dtype == MAMBO_DTYPE_BF16;
    MAMBO_REQUIRE((uintptr_t)x % (bf16 ? 2 : 4) == 0 && (uintptr_t)scales % 4 == 0, MAMBO_ERR_VALUE,
                  "rows and scales must be aligned to their type");
    const bool vec = (uintptr_t)x % 16 == 0 && ldx % (bf16 ? 8 : 4) == 0 && (uintptr_t)values % 8 == 0 && ldv % 8 == 0;
    const dim3 grid((unsigned)cdiv(groups, 16), (unsigned)(m < 65535 ? m : 65535));
    hipStream_t s = (hipStream_t)stream;
#define MAMBO_QUANT(B, V)                                                                                          \
    if (bf16 == B && vec == V)                                                                                     \
    MAMBO_LAUNCH((quantize_fp8_block_kernel<B, V>), grid, dim3(256), 0, s, x, ldx, m, (int)k, values, ldv, scales, lds)
    MAMBO_QUANT(true, true);
    MAMBO_QUANT(true, false);
    MAMBO_QUANT(false, true);
    MAMBO_QUANT(false, false);
#undef MAMBO_QUANT
    return mambo_check_launch("quantize_fp8_block");
}

extern "C" int64_t mambo_fp8_block_packed_bytes(int64_t experts, int64_t n, int64_t k)
{
    if (experts < 1 || n < 1 || k < 1 || n > 0x7FFFFF00 || k > 0x7FFFFF00 || experts > MAMBO_MAX_EXPERTS)
        return 0;
    return experts * cdiv(n, kTileN) * cdiv(k, kGroup) * kFp8Tile;
}

extern "C" int mambo_fp8_block_pack(const uint8_t *w, int64_t experts, int64_t n, int64_t k, int64_t stride_e,
                                    int64_t stride_n, uint8_t *packed, mambo_stream_t stream)
{
    MAMBO_REQUIRE(experts >= 1 && experts <= MAMBO_MAX_EXPERTS && n >= 1 && n <= 0x7FFFFF00 && k >= 16 &&
                      k <= 0x7FFFFF00 && k % 16 == 0,
                  MAMBO_ERR_VALUE,
                  "weights must be [E,N,K] with E in [1, %d], N >= 1 and K a multiple of 16 (got E=%lld N=%lld K=%lld)",
                  MAMBO_MAX_EXPERTS, (long long)experts, (long long)n, (long long)k);
    MAMBO_REQUIRE(w && packed, MAMBO_ERR_VALUE, "null pointer");
    MAMBO_REQUIRE((uintptr_t)packed % 16 == 0, MAMBO_ERR_VALUE, "packed must be 16-byte aligned");
    const int64_t ntiles = cdiv(n, kTileN), groups = cdiv(k, kGroup), tiles = experts * ntiles * groups;
    MAMBO_REQUIRE(tiles <= 0x7FFFFFFF, MAMBO_ERR_VALUE, "weights too large for one call");
    const bool vec = (uintptr_t)w % 16 == 0 && stride_e % 16 == 0 && stride_n % 16 == 0;
    MAMBO_LAUNCH(fp8_block_pack_kernel, dim3((unsigned)tiles), dim3(256), 0, (hipStream_t)stream, w, n, k, stride_e,
                 stride_n, ntiles, groups, vec, packed);
    return mambo_check_launch("fp8_block_pack");
}

extern "C" int mambo_fp8_block_matmul(const uint8_t *xv, int64_t ldxv, const float *xs, int64_t ldxs, int64_t m,
                                      const uint8_t *packed, const float *ws, int64_t n, int64_t k, void *out,
                                      int out_dtype, int64_t ldo, mambo_stream_t stream)
{
    MAMBO_REQUIRE(m >= 0, MAMBO_ERR_VALUE, "rows must not be negative");
    const ExpertRows er = {nullptr, nullptr, m, m, 1};
    return run_products(xv, ldxv, xs, ldxs, er, packed, ws, n, k, out, out_dtype, ldo, (hipStream_t)stream);
}

extern "C" int mambo_fp8_block_matmul_experts(const uint8_t *xv, int64_t ldxv, const float *xs, int64_t ldxs, int64_t m,
                                              const int32_t *rows, int64_t r, const int32_t *offsets, int64_t experts,
                                              const uint8_t *packed, const float *ws, int64_t n, int64_t k, void *out,
                                              int out_dtype, int64_t ldo, mambo_stream_t stream)
{
    const int rc = check_expert_rows(m, rows, r, offsets, experts);
    if (rc != MAMBO_OK)
        return rc;
    const ExpertRows er = {offsets, rows, r, m, (int)experts};
    return run_products(xv, ldxv, xs, ldxs, er, packed, ws, n, k, out, out_dtype, ldo, (hipStream_t)stream);
}
