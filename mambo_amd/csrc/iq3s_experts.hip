// IQ3_S x MXFP8 products grouped by expert.
//
// Few rows an expert: a workgroup computes 16 tokens, or 4, x 32 weight rows; its W waves take the K blocks
// in turn and each streams its own through a ring of two blocks in registers. The waves' sums meet in
// LDS at the end and are added in order. More rows: the 32 x 32 MFMA kernel (iq3s_wide.h).
#include <cmath>

#include "iq3s_dense.h"
#include "iq3s_wide.h"

namespace {

struct Iq3sArgs {
    const uint8_t *xv, *xs;
    int64_t ldxv, ldxs;
    ExpertRows er;
    const uint8_t *packed;
    int64_t expert_stride;
    void *out;
    int64_t ldo;
    int n, blocks, ntiles; // ntiles: pairs of 16-row tiles
    bool vec;
};

// kDiag false: 16 tokens, every weight as an exact pair of E4M3 terms (iq3s_dense.h), four MFMAs a block and 16 rows.
// kDiag true: 4 tokens, whose rows fill the MFMA's 16 by its four blocks of K (ALane), so that a weight is its codebook
// word alone and its scale multiplies the sums: two MFMAs and 88 vector instructions a block and 16 rows against 120.
// Both are bound by those instructions (16 lookups, signs, addresses), not by the weights' bytes: 8 experts of 14336 x 4096,
// of which 6 have rows, 151 MB: 4 tokens each at most 33.9 us (4.5 TB/s), 16 36.3 (with four waves a workgroup 34.4 and
// 41.4). More copies of the codebook in LDS, against bank conflicts, gained nothing; a workgroup of several
// columns (which share the codebook) neither; 16 weight rows a wave instead of 32 lost 20%, 64 lost 5%.
template <bool kDiag, int W, bool kBf16>
__global__ __launch_bounds__(W * 64) __attribute__((amdgpu_waves_per_eu(2))) void iq3s_expert_stream_kernel(Iq3sArgs a)
{
    constexpr int T = kDiag ? 4 : 16, NT = 2, kPad = 16 * NT + 4, kQuads = 4 * NT;
    __shared__ __align__(16) uint32_t s_lut[512];
    __shared__ uint4 s_split[16];
    __shared__ __align__(16) float s_red[W * T * kPad];
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int tiles = (a.n + kTileRows - 1) / kTileRows, nt = blockIdx.x % a.ntiles;
    RowTile rt;
    if (!find_row_tile(a.er, T, blockIdx.x / a.ntiles, &rt))
        return;
    const bool none = rt.expert == a.er.experts;
    if (!none) {
        const int col = lane & 15, q = lane >> 4, B = a.blocks;
        const uint8_t *weight = a.packed + (int64_t)rt.expert * a.expert_stride;
        __amdgpu_buffer_rsrc_t wt[NT];
#pragma unroll
        for (int t = 0; t < NT; ++t)
            wt[t] = byte_rsrc(weight + (int64_t)min(NT * nt + t, tiles - 1) * B * kTileBytes);
        const int count = wave < B ? (B - wave + W - 1) / W : 0;
        const int token = kDiag ? lane & 3 : col;
        const int64_t src = source_row(a.er, rt.row0 + min(token, rt.count - 1));
        const uint8_t *xrow = a.xv + src * a.ldxv, *srow = a.xs + src * a.ldxs;
        const ALane al[1] = {a_lane<false>(lane, token < rt.count, xrow, srow, g_zero_chunk, g_unit_scales)};
        // the bytes and the scale of this lane's token (compute_dense, load_a_dense)
        const uint8_t *xp = xrow + 32 * (4 * (q >> 1)) + 16 * (q & 1), *sp = srow + 4 * (q & 1) + 2 * (q >> 1);
        struct Ring {
            WTile w[NT];
            ATile<1> x;
        } ring[2];
        auto load = [&](Ring &r, int i) {
            const int b = min(wave + max(min(i, count - 1), 0) * W, B - 1);
#pragma unroll
            for (int t = 0; t < NT; ++t)
                r.w[t] = load_w_rsrc(wt[t], (uint32_t)b * kTileBytes, lane, col);
            if constexpr (kDiag) {
                load_a<1>(r.x, al, b, g_zero_chunk);
            } else {
                const uint8_t *p = xp + 256 * (int64_t)b;
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const uint4 l = *reinterpret_cast<const uint4 *>(p + 32 * h), u = *reinterpret_cast<const uint4 *>(p + 32 * h + 64);
                    r.x.a[0][h] = v8i{(int)l.x, (int)l.y, (int)l.z, (int)l.w, (int)u.x, (int)u.y, (int)u.z, (int)u.w};
                }
                r.x.s[0] = *reinterpret_cast<const uint16_t *>(sp + 8 * (int64_t)b);
            }
        };
        load(ring[0], 0);
        if constexpr (kDiag) {
            for (int i = tid; i < 128; i += W * 64)
                reinterpret_cast<uint4 *>(s_lut)[i] = reinterpret_cast<const uint4 *>(rep_grid<0>())[i];
        } else {
            for (int i = tid; i < 512; i += W * 64)
                s_lut[i] = c_grid.level[i];
            if (tid < 16)
                s_split[tid] = uint4{c_split.w[tid][0], c_split.w[tid][1], c_split.w[tid][2], c_split.w[tid][3]};
        }
        const uint8_t *lut = reinterpret_cast<const uint8_t *>(s_lut);
        float acc[NT][1][4] = {};
        __syncthreads();
        for (int i0 = 0; i0 < count; i0 += 2) {
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                load(ring[j ^ 1], i0 + j + 1);
                __builtin_amdgcn_sched_barrier(0);
                const Ring &r = ring[j];
#pragma unroll
                for (int t = 0; t < NT; ++t) {
                    if constexpr (kDiag) {
                        compute_block<1, 0>(r.w[t], r.x, lut, 0, acc[t], i0 + j < count);
                    } else {
                        v8i bh[2], bl[2];
                        decode_block(r.w[t], lut, s_split, bh, bl);
                        const float d = i0 + j < count ? half_bits_to_float(r.w[t].dh) : 0.0f;
                        v4f c = {0.0f, 0.0f, 0.0f, 0.0f};
                        const int s0 = r.x.s[0] & 255, s1 = r.x.s[0] >> 8;
                        c = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(r.x.a[0][0], bh[0], c, 0, 0, 0, s0, 0, 128);
                        c = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(r.x.a[0][0], bl[0], c, 0, 0, 0, s0, 0, 128);
                        c = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(r.x.a[0][1], bh[1], c, 0, 0, 0, s1, 0, 128);
                        c = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(r.x.a[0][1], bl[1], c, 0, 0, 0, s1, 0, 128);
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            acc[t][0][i] = __builtin_fmaf(c[i], d, acc[t][0][i]);
                    }
                }
                __builtin_amdgcn_sched_barrier(0);
            }
        }
        float *red = s_red + wave * T * kPad + col;
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                if constexpr (kDiag) {
                    const float v = lane_group_sum(acc[t][0][i]);
                    if (lane < 16)
                        red[i * kPad + 16 * t] = v;
                } else {
                    red[(4 * q + i) * kPad + 16 * t] = acc[t][0][i];
                }
            }
    }
    __syncthreads();
    for (int i = tid; i < T * kQuads; i += W * 64) {
        const int token = i / kQuads, n4 = 4 * (i % kQuads), at = nt * 16 * NT + n4;
        if (token >= rt.count || at >= a.n)
            continue;
        v4f v = {0.0f, 0.0f, 0.0f, 0.0f};
        if (!none)
#pragma unroll
            for (int w = 0; w < W; ++w)
                v += *reinterpret_cast<const v4f *>(s_red + (w * T + token) * kPad + n4);
        store_row4<kBf16>(a.out, (rt.row0 + token) * a.ldo + at, v, a.n - at, a.vec);
    }
}

// The kernel of a product: the 32 x 32 MFMA kernel's plan, or the tokens of a tile and the waves that share K.
struct Iq3sChoice {
    bool wide;
    WidePlan plan;
    int tokens, waves;
};

Iq3sChoice iq3s_choose(const ExpertRows &er, int64_t n, int64_t blocks, int64_t ldxv, int64_t ldxs)
{
    const int64_t r = er.r, experts = er.experts, ntiles = (n + 31) / 32, apart = er.rows ? er.m : 256;
    Iq3sChoice c = {};
    // How the rows fall is not known here: experts with rows and tiles are counted for rows that fall at random.
    const double taken = (double)experts * -std::expm1(-(double)r / (double)experts);
    auto tiles = [&](int t) { return std::fmax(taken, (double)r / t + 0.5 * taken); };
    // The 32 x 32 MFMA kernel from 14 rows of an expert on, where 16 tokens a tile fill the card four times: 64 experts of
    // 2048 x 4096 with 12 rows each take it 75.4 us (the 16-token kernel 72.5), with 16 76.1 (94.6), 4 experts of 1024 x
    // 4096 with 64 rows 24.8 (16.1). It tells rows by 32-bit offsets, and a grid takes 2^29 weight rows of it and 65535
    // row tiles: past these the 16-token kernel is what is left, at a fraction of the rate (8 experts of 4096 x 14336, 4096
    // rows, 1721 us and 487).
    c.wide = (double)r > 14.0 * taken && tiles(16) * ntiles >= 1024.0 && n < (1 << 29) &&
             apart * ldxv + 256 * blocks < ((int64_t)1 << 32) && apart * ldxs + 8 * blocks < ((int64_t)1 << 32) &&
             expert_row_tiles(r, experts, 64) <= 65535;
    if (c.wide) {
        double tiles_of[2] = {tiles(64), tiles(128)};
        mambo_wide_experts_plan(er, n, blocks, tiles_of, &c.plan);
        return c;
    }
    // 4 tokens a tile up to 2.5 rows of an expert: 64 experts of 2048 x 4096 with 2.3 rows take 43.4 us (16 tokens a tile
    // 47.6), with 4 62.5 (50.8).
    c.tokens = (double)r <= 2.5 * taken ? 4 : 16;
    // Waves that share a workgroup's K, two blocks each at least: one where workgroups fill the card, more where they do
    // not (8 x 14336 x 4096, 4 tokens a tile, 3136 workgroups: 40.0 us with one, 42.1 with two, 43.6 with four; 2 experts,
    // 896: 16.1, 14.5, 14.9; 2 of 4096 x 14336, 256: 34.8, 21.1, 14.7).
    const double expected = tiles(c.tokens) * ntiles;
    c.waves = expected >= 2560.0 || blocks < 4 ? 1 : expected >= 640.0 || blocks < 8 ? 2 : 4;
    return c;
}

int check_iq3s_product(int64_t n, int64_t blocks, int out_dtype)
{
    MAMBO_REQUIRE(out_dtype == MAMBO_DTYPE_F32 || out_dtype == MAMBO_DTYPE_BF16, MAMBO_ERR_VALUE,
                  "outputs must be float32 or bfloat16");
    MAMBO_REQUIRE(n >= 1 && n <= 0x7FFFFF00 && blocks >= 1 && blocks <= 2000000, MAMBO_ERR_VALUE,
                  "weights must be [N,K/256] blocks with N, K >= 1 (got %lld and %lld)", (long long)n, (long long)blocks);
    return MAMBO_OK;
}

} // namespace

extern "C" int mambo_iq3s_experts_plan(int64_t m, int64_t r, int64_t experts, int64_t n, int64_t blocks, int64_t ldxv,
                                       int64_t ldxs, int32_t *plan)
{
    static const int32_t one = 0; // never read: that the rows are gathered, or by expert
    const int32_t *rows = m != r ? &one : nullptr;
    int rc = check_iq3s_product(n, blocks, MAMBO_DTYPE_F32);
    if (rc == MAMBO_OK)
        rc = check_expert_rows(m, rows, r, &one, experts);
    if (rc != MAMBO_OK)
        return rc;
    MAMBO_REQUIRE(ldxv >= 256 * blocks && ldxs >= 8 * blocks && plan && r >= 1, MAMBO_ERR_VALUE, "a plan is of one row or more");
    const Iq3sChoice c = iq3s_choose({&one, rows, r, m, (int)experts}, n, blocks, ldxv, ldxs);
    MAMBO_REQUIRE(c.wide || grid_takes(expert_row_tiles(r, experts, c.tokens) * ((n + 31) / 32), 64 * c.waves), MAMBO_ERR_VALUE,
                  "too many rows and columns for one launch");
    plan[0] = c.wide ? 32 * c.plan.mt : c.tokens;
    plan[1] = c.wide ? 32 * c.plan.waves : 32;
    plan[2] = c.wide ? c.plan.kg : c.waves;
    return MAMBO_OK;
}

extern "C" int mambo_iq3s_fp8_matmul_experts(const uint8_t *xv, int64_t ldxv, const uint8_t *xs, int64_t ldxs, int64_t m,
                                             const int32_t *rows, int64_t r, const int32_t *offsets, int64_t experts,
                                             const uint8_t *packed, int64_t expert_stride, int64_t n, int64_t blocks,
                                             void *out, int out_dtype, int64_t ldo, mambo_stream_t stream)
{
    int rc = check_expert_rows(m, rows, r, offsets, experts);
    if (rc == MAMBO_OK)
        rc = check_iq3s_product(n, blocks, out_dtype);
    if (rc != MAMBO_OK)
        return rc;
    MAMBO_REQUIRE(ldxv >= 256 * blocks && ldxs >= 8 * blocks && ldo >= n, MAMBO_ERR_VALUE,
                  "row strides must cover the rows");
    MAMBO_REQUIRE(expert_stride >= mambo_iq3s_packed_bytes(n, blocks) && expert_stride % 16 == 0, MAMBO_ERR_VALUE,
                  "expert_stride must be a multiple of 16 that covers a weight");
    if (r == 0)
        return MAMBO_OK;
    MAMBO_REQUIRE(xv && xs && packed && out, MAMBO_ERR_VALUE, "null pointer");
    MAMBO_REQUIRE((uintptr_t)xv % 16 == 0 && ldxv % 16 == 0 && (uintptr_t)xs % 8 == 0 && ldxs % 8 == 0 &&
                      (uintptr_t)packed % 16 == 0,
                  MAMBO_ERR_VALUE, "rows and packed weights must be 16-byte aligned, scales 8-byte aligned");
    MAMBO_REQUIRE((uintptr_t)out % (out_dtype == MAMBO_DTYPE_BF16 ? 2 : 4) == 0, MAMBO_ERR_VALUE,
                  "outputs must be aligned to their type");
    const ExpertRows er = {offsets, rows, r, m, (int)experts};
    const bool bf16 = out_dtype == MAMBO_DTYPE_BF16;
    hipStream_t s = (hipStream_t)stream;
    const Iq3sArgs a = {xv, xs, ldxv, ldxs, er, packed, expert_stride, out, ldo, (int)n,
                        (int)blocks, (int)((n + 31) / 32), rows_take_vectors(out, ldo, out_dtype)};
    const Iq3sChoice choice = iq3s_choose(er, n, blocks, ldxv, ldxs);
    if (choice.wide)
        return mambo_wide_experts_launch(choice.plan, xv, ldxv, xs, ldxs, er, packed, expert_stride, n, blocks, out, bf16, ldo, s);
    const bool diag = choice.tokens == 4;
    const int waves = choice.waves;
    const int64_t wgs = expert_row_tiles(r, experts, choice.tokens) * a.ntiles;
    MAMBO_REQUIRE(grid_takes(wgs, 64 * waves), MAMBO_ERR_VALUE, "too many rows and columns for one launch");
#define MAMBO_IQ3S(D, W, B)                                                                                            \
    if (diag == D && waves == W && bf16 == B)                                                                          \
    MAMBO_LAUNCH((iq3s_expert_stream_kernel<D, W, B>), dim3((unsigned)wgs), dim3(W * 64), 0, s, a)
#define MAMBO_IQ3S_WAVES(D, B) \
    MAMBO_IQ3S(D, 1, B);       \
    MAMBO_IQ3S(D, 2, B);       \
    MAMBO_IQ3S(D, 4, B)
    MAMBO_IQ3S_WAVES(false, false);
    MAMBO_IQ3S_WAVES(false, true);
    MAMBO_IQ3S_WAVES(true, false);
    MAMBO_IQ3S_WAVES(true, true);
#undef MAMBO_IQ3S_WAVES
#undef MAMBO_IQ3S
    return mambo_check_launch("iq3s_fp8_matmul_experts");
}
