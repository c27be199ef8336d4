// Attention of many rows (prompts, pieces of prompts): bound by the matrix units and the exponentials.
//
// A workgroup takes 256 rows (queries x heads of one key/value head, 32 a wave) and goes through their keys
// 64 at a time. The tile's codes are widened to bf16 once, on their way from registers into LDS, and every
// wave reads them from there: S^T = K Q^T in 32 x 32 x 16 MFMAs, softmax in registers (a lane has one
// query), O^T += V^T P^T. The key rows lie in LDS in such an order that the scores come out
// of the first product as the operand of the second. Two buffers: the next tile's codes are asked for before
// a tile is worked on and widened after it.
#include "attention.h"

namespace {

constexpr int kWaves = kTileRowsWg / 32;
constexpr int kThreads = 64 * kWaves;
constexpr int kTileBlocks = 2; // blocks of 32 tokens of a tile

__device__ __forceinline__ float halves_max(float x)
{
    auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
__device__ __forceinline__ float halves_sum(float x)
{
    auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return __uint_as_float(b[0]) + __uint_as_float(b[1]);
}

// Tiles of the sequences before s: at least as many as their rows fill.
__device__ __forceinline__ int64_t tiles_before(const Attention &a, int s)
{
    return (int64_t)a.b.offset(s) * a.group / kTileRowsWg + s;
}

template <int DS>
__global__ __launch_bounds__(kThreads, 2) void attend_tiles_kernel(const Attention a)
{
    constexpr int DP = 32 * DS, kSteps = DP / 16;
    constexpr int kPieces = kTileBlocks * DS * 64;               // 16-byte pieces of the keys of a tile, and of its values
    constexpr int kEach = (kPieces + kThreads - 1) / kThreads;   // of a thread
    // keys: [8 values of the head][64 rows of the first product]; values: [8 tokens][value of the head]
    __shared__ bf16x8 keys[2][DP / 8][32 * kTileBlocks];
    __shared__ bf16x8 values[2][4 * kTileBlocks][DP];

    const int tid = (int)threadIdx.x, lane = lane_id(), half = lane >> 5, col = lane & 31;
    const int wave = __builtin_amdgcn_readfirstlane(tid / 64);
    // neighbouring workgroups, which go to different XCDs, have different heads: a head's keys stay in one L2.
    // The last tiles, with the most keys, go first.
    const int head = (int)(blockIdx.x % (unsigned)a.cache.heads);
    const int tile = (int)(gridDim.x / (unsigned)a.cache.heads) - 1 - (int)(blockIdx.x / (unsigned)a.cache.heads);
    int s, part_tile;
    if (a.b.offsets) {
        s = find_slot(a.b.seqs, tile, [&](int i) { return tiles_before(a, i); });
        part_tile = tile - (int)tiles_before(a, s);
    } else {
        s = tile / a.tiles_each;
        part_tile = tile % a.tiles_each;
    }
    const Sequence seq = sequence(a, s);
    const int64_t rows64 = (int64_t)seq.n * a.group, row0_64 = (int64_t)part_tile * kTileRowsWg;
    if (part_tile < 0 || row0_64 >= rows64 || rows64 <= a.few_rows)
        return;
    const int rows = (int)rows64, row0 = (int)row0_64;

    // the tile's keys: what its first row sees of the window to what its last one sees
    const int i0 = row0 / a.group, i1 = (min(row0 + kTileRowsWg, rows) - 1) / a.group;
    int lo = max(0, sees_from(a, seq, i0)) / kKvBlock, hi = (max(0, sees_to(a, seq, i1)) + kKvBlock - 1) / kKvBlock;
    if (a.parts > 1) { // an even share of them
        const int tiles = (hi - lo + kTileBlocks - 1) / kTileBlocks, part = (int)blockIdx.y;
        const int begin = lo + kTileBlocks * (int)((int64_t)tiles * part / a.parts);
        hi = min(hi, lo + kTileBlocks * (int)((int64_t)tiles * (part + 1) / a.parts));
        lo = begin;
    }

    // this wave's rows: column col
    const int row = row0 + 32 * wave + col, i = row / a.group, h = head * a.group + row % a.group;
    const bool some = row < rows;
    const int to = some ? sees_to(a, seq, i) : 0, from = some ? sees_from(a, seq, i) : 0;
    const int wave_row0 = min(row0 + 32 * wave, rows - 1), wave_row1 = min(row0 + 32 * wave + 31, rows - 1);
    // keys that all of the wave's rows see, and that any does
    const int all_to = sees_to(a, seq, wave_row0 / a.group), all_from = sees_from(a, seq, wave_row1 / a.group);
    const int any_to = row0 + 32 * wave < rows ? sees_to(a, seq, wave_row1 / a.group) : 0;
    const int any_from = sees_from(a, seq, wave_row0 / a.group);

    bf16x8 q[kSteps];
    const __bf16 *x = a.q + (int64_t)(seq.first + i) * a.ldqt + h * a.ldqh;
#pragma unroll
    for (int d = 0; d < kSteps; ++d) {
        q[d] = bf16x8{};
        if (some && 16 * d + 8 * half < a.cache.dim)
            q[d] = *reinterpret_cast<const bf16x8 *>(x + 16 * d + 8 * half);
    }

    v16f o[DS];
#pragma unroll
    for (int d = 0; d < DS; ++d)
#pragma unroll
        for (int r = 0; r < 16; ++r)
            o[d][r] = 0.0f;
    float m = -__builtin_inff(), l = 0.0f;

    uint4 kc[kEach], vc[kEach];
    uint32_t sc[kEach]; // scales of the piece's block; bit 16: there is no such page
    const auto load = [&](int blk0) {
#pragma unroll
        for (int e = 0; e < kEach; ++e) {
            const int piece = tid + kThreads * e, blk = blk0 + piece / (64 * DS);
            kc[e] = vc[e] = make_uint4(0u, 0u, 0u, 0u);
            sc[e] = 1u << 16;
            if (piece >= kPieces || blk >= hi)
                continue;
            const int page = a.b.page(s, blk >> a.cache.shift);
            if (page < 0 || page >= a.cache.pages)
                continue;
            const int64_t at = a.cache.block(page, head, blk);
            const uint4 *codes = reinterpret_cast<const uint4 *>(a.cache.codes + at * (2 * kKvBlock * DP)) + piece % (64 * DS);
            kc[e] = codes[0];
            vc[e] = codes[64 * DS];
            sc[e] = *reinterpret_cast<const uint16_t *>(a.cache.scales + 2 * at);
        }
    };
    // Piece (block b, 32 values ds, lane 16 kk + j) has, of the keys, tokens 8 (j / 4) + j % 4 and 4 more, which are
    // rows 16 (j / 8) + 4 (j / 4 % 2) + j % 4 and 8 more of the first product.
    const auto widen_tile = [&](int blk0, int buf) {
#pragma unroll
        for (int e = 0; e < kEach; ++e) {
            const int piece = tid + kThreads * e;
            if (kPieces % kThreads && piece >= kPieces)
                continue;
            const int b = piece / (64 * DS), ds = piece / 64 % DS, kk = piece >> 4 & 3, j = piece & 15;
            const bool none = sc[e] >> 16;
            const float ks = none ? 1.0f : e8m0(sc[e] & 255), vs = none ? 1.0f : e8m0(sc[e] >> 8);
            const int at = 32 * b + 16 * (j >> 3) + 4 * (j >> 2 & 1) + (j & 3);
            keys[buf][4 * ds + kk][at] = widen(kc[e].x, kc[e].y, ks);
            keys[buf][4 * ds + kk][at + 8] = widen(kc[e].z, kc[e].w, ks);
            uint2 v0 = make_uint2(vc[e].x, vc[e].y), v1 = make_uint2(vc[e].z, vc[e].w);
            const int left = seq.len - (blk0 + b) * kKvBlock - 8 * kk;
            if (left < 8) {
                v0 = keep_tokens(v0.x, v0.y, left);
                v1 = keep_tokens(v1.x, v1.y, left);
            }
            values[buf][4 * b + kk][32 * ds + j] = widen(v0.x, v0.y, vs);
            values[buf][4 * b + kk][32 * ds + 16 + j] = widen(v1.x, v1.y, vs);
        }
    };
    // Pages that a table does not have: their tokens are left out (bit b: block b of the tile).
    const auto missing = [&](int blk0) {
        uint32_t gone = 0;
#pragma unroll
        for (int b = 0; b < kTileBlocks; ++b)
            if (blk0 + b < hi) {
                const int page = a.b.page(s, (blk0 + b) >> a.cache.shift);
                gone |= (page < 0 || page >= a.cache.pages) ? 1u << b : 0u;
            } else {
                gone |= 1u << b;
            }
        return (uint32_t)__builtin_amdgcn_readfirstlane(gone);
    };

    if (lo < hi) {
        load(lo);
        widen_tile(lo, 0);
    }
    __syncthreads();
    for (int blk = lo, buf = 0; blk < hi; blk += kTileBlocks, buf ^= 1) {
        const bool more = blk + kTileBlocks < hi;
        if (more)
            load(blk + kTileBlocks);
        const int token0 = blk * kKvBlock;
        if (token0 < any_to && token0 + 32 * kTileBlocks > any_from) { // of the wave's rows some see some
            const uint32_t gone = missing(blk);
            v16f sx[kTileBlocks];
#pragma unroll
            for (int b = 0; b < kTileBlocks; ++b)
#pragma unroll
                for (int r = 0; r < 16; ++r)
                    sx[b][r] = 0.0f;
#pragma unroll
            for (int d = 0; d < kSteps; ++d)
#pragma unroll
                for (int b = 0; b < kTileBlocks; ++b)
                    sx[b] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(keys[buf][2 * d + half][32 * b + col], q[d], sx[b], 0, 0, 0);
            const bool edge = token0 + 32 * kTileBlocks > all_to || token0 < all_from || gone;
            // score r of a block is of its token 16 (r / 8) + 8 half + r % 8
            float top = -__builtin_inff();
            if (edge) {
#pragma unroll
                for (int b = 0; b < kTileBlocks; ++b)
#pragma unroll
                    for (int r = 0; r < 16; ++r) {
                        const int token = token0 + 32 * b + 16 * (r >> 3) + 8 * half + (r & 7);
                        if (!(token < to && token >= from) || (gone >> b & 1))
                            sx[b][r] = -__builtin_inff();
                    }
            }
#pragma unroll
            for (int b = 0; b < kTileBlocks; ++b)
#pragma unroll
                for (int r = 0; r < 16; ++r)
                    top = fmaxf(top, sx[b][r]);
            top = halves_max(top);
            top *= a.scale;
            if (__any(top > m)) {
                const float grown = fmaxf(m, top);
                const float by = m == -__builtin_inff() ? 0.0f : exp2_fast(m - grown);
                m = grown;
                l *= by;
#pragma unroll
                for (int d = 0; d < DS; ++d)
                    o[d] *= by;
            }
            const float less = m == -__builtin_inff() ? 0.0f : m;
            bf16x8 p[2 * kTileBlocks];
#pragma unroll
            for (int b = 0; b < kTileBlocks; ++b)
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    const float y = exp2_fast(__builtin_fmaf(sx[b][r], a.scale, -less));
                    l += y;
                    p[2 * b + (r >> 3)][r & 7] = (__bf16)y;
                }
#pragma unroll
            for (int k = 0; k < 2 * kTileBlocks; ++k)
#pragma unroll
                for (int d = 0; d < DS; ++d)
                    o[d] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(values[buf][2 * k + half][32 * d + col], p[k], o[d], 0, 0, 0);
        }
        if (more)
            widen_tile(blk + kTileBlocks, buf ^ 1);
        __syncthreads();
    }

    l = halves_sum(l);
    if (!some)
        return;
    const int64_t t = seq.first + i, q_heads = (int64_t)a.group * a.cache.heads;
    if (a.parts > 1) {
        const int64_t entry = ((int64_t)blockIdx.y * a.b.tokens + t) * q_heads + h;
#pragma unroll
        for (int d = 0; d < DS; ++d)
#pragma unroll
            for (int r = 0; r < 16; r += 4)
                *reinterpret_cast<v4f *>(a.tiles_o + entry * DP + 32 * d + 2 * r + 4 * half) =
                    v4f{o[d][r], o[d][r + 1], o[d][r + 2], o[d][r + 3]};
        if (half == 0)
            *reinterpret_cast<float2 *>(a.tiles_ml + entry * 2) = make_float2(m, l);
        return;
    }
    const float by = l == 0.0f ? 0.0f : 1.0f / l;
    const bool vec = a.ldot % 4 == 0 && a.ldoh % 4 == 0 && (uintptr_t)a.out % 8 == 0;
#pragma unroll
    for (int d = 0; d < DS; ++d)
#pragma unroll
        for (int r = 0; r < 16; r += 4) {
            const int at = 32 * d + 2 * r + 4 * half;
            if (at < a.cache.dim)
                store_row4<true>(a.out, t * a.ldot + h * a.ldoh + at,
                                 v4f{o[d][r] * by, o[d][r + 1] * by, o[d][r + 2] * by, o[d][r + 3] * by}, a.cache.dim - at, vec);
        }
    if (a.lse && half == 0)
        a.lse[t * q_heads + h] = l == 0.0f ? -__builtin_inff() : (m + __log2f(l)) * kLn2;
}

// Rows whose keys were dealt to several workgroups: their sums weighted by the largest scores, in order.
template <int DS>
__global__ __launch_bounds__(256) void join_tiles_kernel(const Attention a)
{
    constexpr int DP = 32 * DS, kWide = DP / 4, kRows = 256 / kWide;
    const int64_t q_heads = (int64_t)a.group * a.cache.heads, all = a.b.tokens * q_heads;
    const int64_t entry = (int64_t)blockIdx.x * kRows + (int)threadIdx.x / kWide;
    const int d = 4 * ((int)threadIdx.x % kWide);
    if ((int)threadIdx.x >= kRows * kWide || entry >= all)
        return;
    const int64_t t = entry / q_heads, h = entry % q_heads;
    if (a.b.offsets) { // rows of sequences that this kernel has, and no others
        if (t < a.b.offset(0) || t >= a.b.offset(a.b.seqs))
            return;
        int lo = 0, hi = a.b.seqs - 1; // the last sequence that begins at or before t
        while (lo < hi) {
            const int mid = (lo + hi + 1) / 2;
            if (a.b.offset(mid) <= t)
                lo = mid;
            else
                hi = mid - 1;
        }
        const Sequence seq = sequence(a, lo);
        if (t >= seq.first + seq.n || (int64_t)seq.n * a.group <= a.few_rows)
            return;
    }
    float m = -__builtin_inff(), l = 0.0f;
    v4f o = {0.0f, 0.0f, 0.0f, 0.0f};
    for (int p = 0; p < a.parts; ++p) {
        const float2 ml = *reinterpret_cast<const float2 *>(a.tiles_ml + (p * all + entry) * 2);
        const v4f x = *reinterpret_cast<const v4f *>(a.tiles_o + (p * all + entry) * DP + d);
        const float top = fmaxf(m, ml.x), less = top == -__builtin_inff() ? 0.0f : top;
        const float f = exp2_fast(m - less), e = exp2_fast(ml.x - less);
        o = o * f + x * e;
        l = l * f + ml.y * e;
        m = top;
    }
    o *= l == 0.0f ? 0.0f : 1.0f / l;
    if (d < a.cache.dim)
        store_row4<true>(a.out, t * a.ldot + h * a.ldoh + d, o, a.cache.dim - d, a.ldot % 4 == 0 && a.ldoh % 4 == 0 && (uintptr_t)a.out % 8 == 0);
    if (a.lse && d == 0)
        a.lse[entry] = l == 0.0f ? -__builtin_inff() : (m + __log2f(l)) * kLn2;
}

template <int DS>
void launch_tiles(const Attention &a, int64_t tiles, hipStream_t s)
{
    MAMBO_LAUNCH((attend_tiles_kernel<DS>), dim3((unsigned)(tiles * a.cache.heads), (unsigned)a.parts), dim3(kThreads), 0, s, a);
    if (a.parts > 1) {
        const int64_t rows = (int64_t)a.b.tokens * a.group * a.cache.heads, each = 256 / (8 * DS);
        MAMBO_LAUNCH((join_tiles_kernel<DS>), dim3((unsigned)((rows + each - 1) / each)), dim3(256), 0, s, a);
    }
}

} // namespace

int launch_attend_tiles(const Attention &a, int64_t tiles, hipStream_t s)
{
    switch (kv_padded(a.cache.dim) / 32) {
    case 1: launch_tiles<1>(a, tiles, s); break;
    case 2: launch_tiles<2>(a, tiles, s); break;
    case 3: launch_tiles<3>(a, tiles, s); break;
    case 4: launch_tiles<4>(a, tiles, s); break;
    case 5: launch_tiles<5>(a, tiles, s); break;
    case 6: launch_tiles<6>(a, tiles, s); break;
    case 7: launch_tiles<7>(a, tiles, s); break;
    default: launch_tiles<8>(a, tiles, s); break;
    }
    return mambo_check_launch("kv_attention");
}
