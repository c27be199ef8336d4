// IQ3_S x MXFP8 products grouped by expert.
//
// Few rows an expert: the weights' bytes bound it. A workgroup computes 16 tokens x 32 weight rows;
// its W waves take the K blocks in turn and each streams its own through a ring of two blocks in
// registers, decoded as the dense kernel's (iq3s_dense.h): exact two-term E4M3 operands in the order of
// the dense MFMA, four MFMAs a block and 16 rows, the block's fp16 d in f32. The waves' sums meet in
// LDS at the end and are added in order.
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

template <int W, bool kBf16>
__global__ __launch_bounds__(W * 64) __attribute__((amdgpu_waves_per_eu(2))) void iq3s_expert_stream_kernel(Iq3sArgs a)
{
    constexpr int T = 16, NT = 2, kPad = 36;
    __shared__ uint32_t s_lvl[512];
    __shared__ uint4 s_split[16];
    __shared__ __align__(16) float s_red[W * T * kPad];
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int nt = blockIdx.x % a.ntiles;
    RowTile rt;
    if (!find_row_tile(a.er, T, blockIdx.x / a.ntiles, &rt))
        return;
    const bool none = rt.expert == a.er.experts;
    if (!none) {
        for (int i = tid; i < 512; i += W * 64)
            s_lvl[i] = c_grid.level[i];
        if (tid < 16)
            s_split[tid] = uint4{c_split.w[tid][0], c_split.w[tid][1], c_split.w[tid][2], c_split.w[tid][3]};
        const int col = lane & 15, q = lane >> 4;
        const int B = a.blocks, tiles = (a.n + kTileRows - 1) / kTileRows;
        const uint8_t *weight = a.packed + (int64_t)rt.expert * a.expert_stride;
        __amdgpu_buffer_rsrc_t wt[NT];
#pragma unroll
        for (int t = 0; t < NT; ++t)
            wt[t] = byte_rsrc(weight + (int64_t)min(NT * nt + t, tiles - 1) * B * kTileBytes);
        // the bytes and the scale of this lane's token (compute_dense, load_a_dense)
        const int64_t src = source_row(a.er, rt.row0 + min(col, rt.count - 1));
        const uint8_t *xp = a.xv + src * a.ldxv + 32 * (4 * (q >> 1)) + 16 * (q & 1);
        const uint8_t *sp = a.xs + src * a.ldxs + 4 * (q & 1) + 2 * (q >> 1);
        const uint8_t *lvl = reinterpret_cast<const uint8_t *>(s_lvl);
        const int count = wave < B ? (B - wave + W - 1) / W : 0;
        struct Ring {
            WTile w[NT];
            uint4 x[4];
            uint16_t s;
        } ring[2];
        auto load = [&](Ring &r, int i) {
            const int b = min(wave + max(min(i, count - 1), 0) * W, B - 1);
#pragma unroll
            for (int t = 0; t < NT; ++t)
                r.w[t] = load_w_rsrc(wt[t], (uint32_t)b * kTileBytes, lane, col);
            const uint8_t *p = xp + 256 * (int64_t)b;
#pragma unroll
            for (int j = 0; j < 4; ++j)
                r.x[j] = *reinterpret_cast<const uint4 *>(p + 32 * (j >> 1) + 64 * (j & 1));
            r.s = *reinterpret_cast<const uint16_t *>(sp + 8 * (int64_t)b);
        };
        float acc[NT][4] = {};
        load(ring[0], 0);
        __syncthreads();
        for (int i0 = 0; i0 < count; i0 += 2) {
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                load(ring[j ^ 1], i0 + j + 1);
                __builtin_amdgcn_sched_barrier(0);
                const Ring &r = ring[j];
                v8i x[2];
#pragma unroll
                for (int h = 0; h < 2; ++h)
                    x[h] = v8i{(int)r.x[2 * h].x,     (int)r.x[2 * h].y,     (int)r.x[2 * h].z,     (int)r.x[2 * h].w,
                               (int)r.x[2 * h + 1].x, (int)r.x[2 * h + 1].y, (int)r.x[2 * h + 1].z, (int)r.x[2 * h + 1].w};
#pragma unroll
                for (int t = 0; t < NT; ++t) {
                    v8i bh[2], bl[2];
                    decode_block(r.w[t], lvl, s_split, bh, bl);
                    const float d = i0 + j < count ? half_bits_to_float(r.w[t].dh) : 0.0f;
                    v4f c = {0.0f, 0.0f, 0.0f, 0.0f};
                    const int s0 = r.s & 255, s1 = r.s >> 8;
                    c = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(x[0], bh[0], c, 0, 0, 0, s0, 0, 128);
                    c = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(x[0], bl[0], c, 0, 0, 0, s0, 0, 128);
                    c = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(x[1], bh[1], c, 0, 0, 0, s1, 0, 128);
                    c = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(x[1], bl[1], c, 0, 0, 0, s1, 0, 128);
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        acc[t][i] = __builtin_fmaf(c[i], d, acc[t][i]);
                }
                __builtin_amdgcn_sched_barrier(0);
            }
        }
        // the sums of a lane: tokens 4q .. 4q + 3, weight row col of each tile
        float *red = s_red + (wave * T + 4 * q) * kPad + col;
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int i = 0; i < 4; ++i)
                red[i * kPad + 16 * t] = acc[t][i];
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
        const int at = nt * 32 + n4;
        if (at < a.n)
            store_row4<kBf16>(a.out, (rt.row0 + token) * a.ldo + at, v, a.n - at, a.vec);
    }
}

} // namespace

extern "C" int mambo_iq3s_fp8_matmul_experts(const uint8_t *xv, int64_t ldxv, const uint8_t *xs, int64_t ldxs, int64_t m,
                                             const int32_t *rows, int64_t r, const int32_t *offsets, int64_t experts,
                                             const uint8_t *packed, int64_t expert_stride, int64_t n, int64_t blocks,
                                             void *out, int out_dtype, int64_t ldo, mambo_stream_t stream)
{
    const int rc = check_expert_rows(m, rows, r, offsets, experts);
    if (rc != MAMBO_OK)
        return rc;
    MAMBO_REQUIRE(out_dtype == MAMBO_DTYPE_F32 || out_dtype == MAMBO_DTYPE_BF16, MAMBO_ERR_VALUE,
                  "outputs must be float32 or bfloat16");
    MAMBO_REQUIRE(n >= 1 && n <= 0x7FFFFF00 && blocks >= 1 && blocks <= 2000000, MAMBO_ERR_VALUE,
                  "weights must be [N,K/256] blocks with N, K >= 1 (got %lld and %lld)", (long long)n, (long long)blocks);
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
    // the 32 x 32 MFMA kernel from 17 rows of an expert on; it tells rows by 32-bit offsets
    const double taken = (double)experts * -std::expm1(-(double)r / (double)experts);
    if ((double)r > 16.0 * taken && (rows ? m : 256) * ldxv + 256 * blocks < ((int64_t)1 << 32) &&
        (rows ? m : 256) * ldxs + 8 * blocks < ((int64_t)1 << 32) && expert_row_tiles(r, experts, 64) <= 65535) {
        double tiles_of[2];
        for (int i = 0; i < 2; ++i)
            tiles_of[i] = std::fmax(taken, (double)r / (64 << i) + 0.5 * taken);
        WidePlan plan;
        mambo_wide_experts_plan(er, n, blocks, tiles_of, &plan);
        return mambo_wide_experts_launch(plan, xv, ldxv, xs, ldxs, er, packed, expert_stride, n, blocks, out, bf16, ldo, s);
    }
    const Iq3sArgs a = {xv, xs, ldxv, ldxs, er, packed, expert_stride, out, ldo, (int)n,
                        (int)blocks, (int)((n + 31) / 32), rows_take_vectors(out, ldo, out_dtype)};
    const int64_t wgs = expert_row_tiles(r, experts, 16) * a.ntiles;
    MAMBO_REQUIRE(wgs <= 0x7FFFFFFF, MAMBO_ERR_VALUE, "too many rows and columns for one launch");
    if (bf16)
        MAMBO_LAUNCH((iq3s_expert_stream_kernel<4, true>), dim3((unsigned)wgs), dim3(256), 0, s, a);
    else
        MAMBO_LAUNCH((iq3s_expert_stream_kernel<4, false>), dim3((unsigned)wgs), dim3(256), 0, s, a);
    return mambo_check_launch("iq3s_fp8_matmul_experts");
}
