// Attention of many rows (prompts, pieces of prompts): bound by the matrix units and the exponentials.
//
// A workgroup takes 256 rows (128 of large heads; queries x heads of one key/value head, 32 a wave) and goes through their keys
// 64 at a time. The tile's codes are widened to bf16 once, on their way from registers into LDS, and every
// wave reads them from there: S^T = K Q^T in 32 x 32 x 16 MFMAs, softmax in registers (a lane has one
// query), O^T += V^T P^T. The key rows lie in LDS in such an order that the scores come out
// of the first product as the operand of the second. Two buffers of each: while a tile is worked on, the codes of the
// keys two tiles ahead and of the values one ahead are widened into the places that its predecessor has left.
// Probabilities are rounded to bf16 for the second product, while the total adds them as they are: a second bf16 term would bring
// the outputs' error against 64 bits from 1.3 to 1.4 times that of their own rounding down to it, and takes 690 us for the 498 below.
// How the vector unit's work is dealt to the products is balanced at heads of 128: 4096 tokens of 32/8 heads take 1.4 times what
// the multiply-adds alone would at the best rate of a product (1.45 PFLOP/s), at 96 1.6, 64 2.1, where the exponentials are as many and the products half,
// 160 and 192 1.8 and 2.0, 224 and 256 (one wave a SIMD) 2.1 and 2.2.
// 8192 tokens of 32/8 heads of 128: 497 us, 1.11 PFLOP/s, half of the matrix units' cycles; a large library product of bf16
// reaches 1.2 to 1.45.
#include "attention.h"

namespace {

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

// Nothing is moved across: between two of these stand one matrix instruction, the read of a later one's operand and
// the vector instructions for which its 32 cycles leave time.
#define MAMBO_FIXED_ORDER() __builtin_amdgcn_sched_barrier(0)
constexpr int kAhead = 4; // operands read ahead

// Tiles of the sequences before s: at least as many as their rows fill.
__device__ __forceinline__ int64_t tiles_before(const Attention &a, int tile_rows, int s)
{
    return (int64_t)a.b.offset(s) * a.group / tile_rows + s;
}

template <int DS>
__global__ __launch_bounds__(64 * tile_waves(DS), tile_waves(DS) / 4) void attend_tiles_kernel(const Attention a)
{
    constexpr int kWaves = tile_waves(DS), kTileRows = 32 * kWaves;
    constexpr int DP = 32 * DS, kSteps = DP / 16;
    constexpr int kUnits = kTileBlocks * DS, kEach = (kUnits + kWaves - 1) / kWaves; // staged by all waves, and by one
    // keys: [8 values of the head][64 rows of the first product]; values: [8 tokens][value of the head]
    struct Staged {
        bf16x8 keys[2][DP / 8][32 * kTileBlocks];
        bf16x8 values[2][4 * kTileBlocks][DP];
    };
    __shared__ Staged staged;
    auto &keys = staged.keys;
    auto &values = staged.values;

    const int tid = (int)threadIdx.x, lane = lane_id(), half = lane >> 5, col = lane & 31;
    const int wave = __builtin_amdgcn_readfirstlane(tid / 64);
    // neighbouring workgroups, which go to different XCDs, have different heads: a head's keys stay in one L2.
    // The last tiles, with the most keys, go first.
    const int head = (int)(blockIdx.x % (unsigned)a.cache.heads);
    const int tile = (int)(gridDim.x / (unsigned)a.cache.heads) - 1 - (int)(blockIdx.x / (unsigned)a.cache.heads);
    int s, part_tile;
    if (a.b.offsets) {
        s = find_slot(a.b.seqs, tile, [&](int i) { return tiles_before(a, kTileRows, i); });
        part_tile = tile - (int)tiles_before(a, kTileRows, s);
    } else {
        s = tile / a.tiles_each;
        part_tile = tile % a.tiles_each;
    }
    const Sequence seq = sequence(a, s);
    const int64_t rows64 = (int64_t)seq.n * a.group, row0_64 = (int64_t)part_tile * kTileRows;
    if (part_tile < 0 || row0_64 >= rows64 || rows64 <= a.few_rows)
        return;
    const int rows = (int)rows64, row0 = (int)row0_64;

    const Keys keys_of = tile_keys(a, seq, row0, kTileRows);
    const int part = (int)blockIdx.y;
    if (part >= keys_of.parts)
        return;
    const int lo = keys_of.begin(part), hi = min(keys_of.hi, keys_of.begin(part + 1));

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
    float m = -__builtin_inff(), l[2] = {0.0f, 0.0f};

    const int zero = vector_zero();
    const int32_t *table = a.b.tables + s * a.b.ldt;
    // Staging: unit u of a tile is 32 values of the head of one of its blocks, a wave's 64 pieces of 16 bytes.
    // Its blocks' pages are read a tile ahead of its codes, by scalar loads that nothing waits for in between.
    struct Pages {
        int of[kTileBlocks];
        uint32_t gone; // bit b: there is no page for block b
    };
    const auto pages_of = [&](int blk0) {
        Pages p;
#pragma unroll
        for (int b = 0; b < kTileBlocks; ++b)
            p.of[b] = scalar_load(table + (min(blk0 + b, hi - 1) >> a.cache.shift));
        return p;
    };
    const auto checked = [&](int blk0, Pages p) {
        p.gone = 0;
#pragma unroll
        for (int b = 0; b < kTileBlocks; ++b)
            if (blk0 + b >= hi || (uint32_t)p.of[b] >= (uint32_t)a.cache.pages) {
                p.of[b] = 0;
                p.gone |= 1u << b;
            }
        return p;
    };
    // Loads and what is made of them have no branch between, whose end would wait for them: codes of a block that is
    // not there are some other block's.
    struct Codes {
        uint4 c[kEach];
        uint32_t scale[kEach]; // E8M0
    };
    struct Place {
        int64_t at[kEach]; // of the unit's block, twice, and one more for its values
    };
    const auto place_of = [&](int blk0, const Pages &p, int of_values) {
        Place x;
#pragma unroll
        for (int e = 0; e < kEach; ++e) {
            const int b = min(wave + kWaves * e, kUnits - 1) / DS;
            x.at[e] = 2 * (int64_t)a.cache.block(b ? p.of[1] : p.of[0], head, blk0 + b) + of_values;
        }
        return x;
    };
    const auto load = [&](const Place &p, Codes &x) {
#pragma unroll
        for (int e = 0; e < kEach; ++e) {
            const int ds = min(wave + kWaves * e, kUnits - 1) % DS;
            x.c[e] = reinterpret_cast<const uint4 *>(a.cache.codes + p.at[e] * (kKvBlock * DP))[64 * ds + lane];
            x.scale[e] = a.cache.scales[p.at[e] + zero];
        }
    };
    // Piece 16 kk + j has, of the keys, tokens 8 (j / 4) + j % 4 and 4 more, which are rows 16 (j / 8) + 4 (j / 4 % 2) +
    // j % 4 and 8 more of the first product.
    const int kk = lane >> 4, j16 = lane & 15, key_row = 16 * (j16 >> 3) + 4 * (j16 >> 2 & 1) + (j16 & 3);
    // Half h of piece e; a wave without a unit of its own does another's once more.
    const auto widen_keys = [&](const Codes &x, int e, int h, int buf) {
        const int u = min(wave + kWaves * e, kUnits - 1), b = u / DS, ds = u % DS;
        keys[buf][4 * ds + kk][32 * b + key_row + 8 * h] =
            widen(h ? x.c[e].z : x.c[e].x, h ? x.c[e].w : x.c[e].y, e8m0(x.scale[e]));
    };
    const auto widen_values = [&](const Codes &x, int e, int h, int buf) {
        const int u = min(wave + kWaves * e, kUnits - 1), b = u / DS, ds = u % DS;
        values[buf][4 * b + kk][32 * ds + 16 * h + j16] = widen(h ? x.c[e].z : x.c[e].x, h ? x.c[e].w : x.c[e].y, e8m0(x.scale[e]));
    };
    // Values behind the sequence's last token, and of a block without a page, become zeros.
    const auto trim_values = [&](Codes &x, int blk0, const Pages &p) {
#pragma unroll
        for (int e = 0; e < kEach; ++e) {
            const int u = min(wave + kWaves * e, kUnits - 1), b = u / DS;
            const bool there = !(p.gone >> b & 1);
            if ((blk0 + b + 1) * kKvBlock > seq.len || !there) {
                const int left = there ? seq.len - (blk0 + b) * kKvBlock - 8 * kk : 0;
                const uint2 v0 = keep_tokens(x.c[e].x, x.c[e].y, left), v1 = keep_tokens(x.c[e].z, x.c[e].w, left);
                x.c[e] = make_uint4(v0.x, v0.y, v1.x, v1.y);
                x.scale[e] = there ? x.scale[e] : 127u; // a scale of anything would make NaN of zeros
            }
        }
    };

    struct Scores {
        v16f x[kTileBlocks];
    };
    v16f zeros;
#pragma unroll
    for (int r = 0; r < 16; ++r)
        zeros[r] = 0.0f;
    const auto first_product = [&](Scores &sx, int buf) {
#pragma unroll
        for (int d = 0; d < kSteps; ++d)
#pragma unroll
            for (int b = 0; b < kTileBlocks; ++b)
                sx.x[b] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(keys[buf][2 * d + half][32 * b + col], q[d],
                                                                  d ? sx.x[b] : zeros, 0, 0, 0);
    };
    // Whether any row of the wave sees any token of the tile.
    const auto seen = [&](int blk0) { return blk0 * kKvBlock < any_to && (blk0 + kTileBlocks) * kKvBlock > any_from; };

    // Leaves out what a row does not see and tokens without a page.
    const auto mask = [&](int blk0, const Pages &pages, Scores &sx) {
        const int token0 = blk0 * kKvBlock;
        if (token0 + 32 * kTileBlocks > all_to || token0 < all_from || pages.gone) {
            // score r of a block is of its token 16 (r / 8) + 8 half + r % 8
#pragma unroll
            for (int b = 0; b < kTileBlocks; ++b)
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    const int token = token0 + 32 * b + 16 * (r >> 3) + 8 * half + (r & 7);
                    if (!(token < to && token >= from) || (pages.gone >> b & 1))
                        sx.x[b][r] = -__builtin_inff();
                }
        }
    };
    const auto largest = [&](const Scores &sx) {
        float top = -__builtin_inff();
#pragma unroll
        for (int b = 0; b < kTileBlocks; ++b)
#pragma unroll
            for (int r = 0; r < 16; ++r)
                top = fmaxf(top, sx.x[b][r]);
        return top;
    };

    Pages p1, p2; // of the next tile and the one after it
    Codes kc, vc; // keys two tiles ahead, values one
    Scores even, odd;
    float top = -__builtin_inff(); // of the scores at hand, before the halves of a row are put together
    if (lo < hi) {
        Codes k0, v0;
        Pages p0 = pages_of(lo);
        p1 = pages_of(lo + kTileBlocks), p2 = pages_of(lo + 2 * kTileBlocks);
        p0 = checked(lo, p0), p1 = checked(lo + kTileBlocks, p1), p2 = checked(lo + 2 * kTileBlocks, p2);
        load(place_of(lo, p0, 0), k0);
        load(place_of(lo, p0, 1), v0);
        load(place_of(lo + kTileBlocks, p1, 0), kc);
        trim_values(v0, lo, p0);
#pragma unroll
        for (int i = 0; i < 2 * kEach; ++i) {
            widen_keys(k0, i / 2, i % 2, 0);
            widen_values(v0, i / 2, i % 2, 0);
            widen_keys(kc, i / 2, i % 2, 1);
        }
        load(place_of(lo + 2 * kTileBlocks, p2, 0), kc);
        load(place_of(lo + kTileBlocks, p1, 1), vc);
        __syncthreads();
        if (seen(lo)) {
            first_product(even, 0);
            mask(lo, p0, even);
            top = largest(even);
        }
    }
    // Tile at blk, whose scores are in `sx`: the next one's scores go into `next` by matrix instructions that the
    // exponentials of this one run beside, and its largest are found beside the second product. Keys are staged a
    // tile further ahead than values, so that of each two buffers and one barrier a tile do: what is written was
    // last read before the barrier.
    const auto step = [&](int blk, int buf, Scores &sx, Scores &next) {
        __syncthreads();
        Pages p3 = pages_of(blk + 3 * kTileBlocks);
        trim_values(vc, blk + kTileBlocks, p1);
        const auto widen_part = [&](int i) { // of 4 kEach
            if (i < 2 * kEach)
                widen_keys(kc, i / 2, i % 2, buf);
            else
                widen_values(vc, i / 2 - kEach, i % 2, buf ^ 1);
        };
        Place next_keys, next_values;
        const auto find_next = [&] {
            p3 = checked(blk + 3 * kTileBlocks, p3);
            next_keys = place_of(blk + 3 * kTileBlocks, p3, 0);
            next_values = place_of(blk + 2 * kTileBlocks, p2, 1);
        };
        if (seen(blk)) {
            bf16x8 p[2 * kTileBlocks], ahead[kAhead];
            constexpr int kFirst = kTileBlocks * kSteps, kSecond = 2 * kTileBlocks * DS;
            const auto key = [&](int n) { return keys[buf ^ 1][2 * (n / kTileBlocks) + half][32 * (n % kTileBlocks) + col]; };
            const auto value = [&](int n) { return values[buf][2 * (n / DS) + half][32 * (n % DS) + col]; };
#pragma unroll
            for (int n = 0; n < kAhead; ++n)
                ahead[n] = key(n);
            MAMBO_FIXED_ORDER();
            top = halves_max(top) * a.scale;
            // The running largest may lag by 2^8: probabilities up to there are as exact, and sums are far from
            // overflow; most tiles then leave the sums as they are.
            if (__any(top > m + 8.0f || m == -__builtin_inff())) {
                const float grown = fmaxf(m, top);
                const float by = m == -__builtin_inff() ? 0.0f : exp2_fast(m - grown);
                m = grown;
                l[0] *= by;
                l[1] *= by;
#pragma unroll
                for (int d = 0; d < DS; ++d)
                    o[d] *= by;
            }
            const float less = m == -__builtin_inff() ? 0.0f : m;
            // Of the 32 probabilities of a lane 20 are worked out beside the first product, 12 beside the first half of
            // the second (whose operands they are later), the next tile's largest and the widening of what was loaded for
            // later ones beside the other half: about as much for the vector unit in all of them.
            constexpr int kEarly = 10 * kTileBlocks, kLate = 6 * kTileBlocks;
            const auto probability = [&](int i) {
                const float y = exp2_fast(__builtin_fmaf(sx.x[i / 16][i % 16], a.scale, -less));
                l[i & 1] += y;
                p[i / 8][i % 8] = (__bf16)y;
                if (i % 8 == 7 || i == kEarly - 1) // here, and not where it is used
                    asm volatile("" : "+v"(p[i / 8]), "+v"(l[0]), "+v"(l[1]));
            };
#pragma unroll
            for (int n = 0; n < kFirst; ++n) {
                MAMBO_FIXED_ORDER();
                v16f &x = next.x[n % kTileBlocks];
                x = __builtin_amdgcn_mfma_f32_32x32x16_bf16(ahead[n % kAhead], q[n / kTileBlocks], n < kTileBlocks ? zeros : x,
                                                            0, 0, 0);
                if (n + kAhead < kFirst)
                    ahead[n % kAhead] = key(n + kAhead);
                else
                    ahead[n % kAhead] = value(n + kAhead - kFirst);
#pragma unroll
                for (int i = n * kEarly / kFirst; i < (n + 1) * kEarly / kFirst; ++i)
                    probability(i);
            }
            MAMBO_FIXED_ORDER();
            mask(blk + kTileBlocks, p1, next);
            top = -__builtin_inff();
#pragma unroll
            for (int n = 0; n < kSecond; ++n) {
                MAMBO_FIXED_ORDER();
                o[n % DS] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(ahead[(kFirst + n) % kAhead], p[n / DS], o[n % DS], 0, 0, 0);
                if (n + kAhead < kSecond)
                    ahead[(kFirst + n) % kAhead] = value(n + kAhead);
                constexpr int kHalf = kSecond / 2;
                if (n < kHalf) {
#pragma unroll
                    for (int i = n * kLate / kHalf; i < (n + 1) * kLate / kHalf; ++i)
                        probability(kEarly + i);
                } else {
#pragma unroll
                    for (int i = (n - kHalf) * 16 * kTileBlocks / kHalf; i < (n - kHalf + 1) * 16 * kTileBlocks / kHalf; ++i)
                        top = fmaxf(top, next.x[i / 16][i % 16]);
#pragma unroll
                    for (int i = (n - kHalf) * 4 * kEach / kHalf; i < (n - kHalf + 1) * 4 * kEach / kHalf; ++i)
                        widen_part(i);
                    if (n == kSecond - 2)
                        find_next();
                }
            }
            MAMBO_FIXED_ORDER();
        } else {
            if (seen(blk + kTileBlocks)) {
                first_product(next, buf ^ 1);
                mask(blk + kTileBlocks, p1, next);
                top = largest(next);
            }
#pragma unroll
            for (int i = 0; i < 4 * kEach; ++i)
                widen_part(i);
            find_next();
        }
        load(next_keys, kc);
        load(next_values, vc);
        p1 = p2, p2 = p3;
    };
    for (int blk = lo; blk < hi; blk += 2 * kTileBlocks) {
        step(blk, 0, even, odd);
        if (blk + kTileBlocks >= hi)
            break;
        step(blk + kTileBlocks, 1, odd, even);
    }

    const float sum = halves_sum(l[0] + l[1]);
    const int64_t t = seq.first + i, q_heads = (int64_t)a.group * a.cache.heads;
    if (keys_of.parts > 1) {
        if (!some)
            return;
        const int64_t entry = ((int64_t)blockIdx.y * a.b.tokens + t) * q_heads + h;
#pragma unroll
        for (int d = 0; d < DS; ++d)
#pragma unroll
            for (int r = 0; r < 16; r += 4)
                *reinterpret_cast<v4f *>(a.tiles_o + entry * DP + 32 * d + 2 * r + 4 * half) =
                    v4f{o[d][r], o[d][r + 1], o[d][r + 2], o[d][r + 3]};
        if (half == 0)
            *reinterpret_cast<float2 *>(a.tiles_ml + entry * 2) = make_float2(m, sum);
        return;
    }
    const float by = sum == 0.0f ? 0.0f : 1.0f / sum;
    if (a.lse && half == 0 && some)
        a.lse[t * q_heads + h] = sum == 0.0f ? -__builtin_inff() : (m + __log2f(sum)) * kLn2;
    const int64_t to_row = t * a.ldot + h * a.ldoh;
    if ((uintptr_t)a.out % 16 == 0 && a.ldot % 8 == 0 && a.ldoh % 8 == 0) {
        // A lane has four values here and there of its row: whole rows are written from LDS, each chunk of 8 values as many
        // places on as its row's number, so that rows do not meet in a bank (8192 tokens 497 us for 529 with what a lane has
        // written as it is, 16 prompts of 64 tokens 14 for 21).
        constexpr int kChunks = DP / 8;
        __syncthreads(); // all waves have read their last operands
        __bf16 *const rows_of_wave = reinterpret_cast<__bf16 *>(&staged) + wave * (32 * DP);
#pragma unroll
        for (int d = 0; d < DS; ++d)
#pragma unroll
            for (int r = 0; r < 16; r += 4) {
                const int chunk = (4 * d + r / 4 + col) % kChunks;
                *reinterpret_cast<bf16x4 *>(rows_of_wave + col * DP + 8 * chunk + 4 * half) =
                    __builtin_convertvector(v4f{o[d][r] * by, o[d][r + 1] * by, o[d][r + 2] * by, o[d][r + 3] * by}, bf16x4);
            }
        __builtin_amdgcn_wave_barrier();
        for (int item = lane; item < 32 * kChunks; item += 64) {
            const int r = item / kChunks, chunk = item % kChunks;
            const int64_t to = ((int64_t)__shfl((int)(to_row >> 32), r) << 32) | (uint32_t)__shfl((int)to_row, r);
            if (row0 + 32 * wave + r < rows && 8 * chunk < a.cache.dim)
                *reinterpret_cast<uint4 *>(a.out + to + 8 * chunk) =
                    *reinterpret_cast<const uint4 *>(rows_of_wave + r * DP + 8 * ((chunk + r) % kChunks));
        }
        return;
    }
    if (!some)
        return;
    const bool vec = a.ldot % 4 == 0 && a.ldoh % 4 == 0 && (uintptr_t)a.out % 8 == 0;
#pragma unroll
    for (int d = 0; d < DS; ++d)
#pragma unroll
        for (int r = 0; r < 16; r += 4) {
            const int at = 32 * d + 2 * r + 4 * half;
            if (at < a.cache.dim)
                store_row4<true>(a.out, to_row + at, v4f{o[d][r] * by, o[d][r + 1] * by, o[d][r + 2] * by, o[d][r + 3] * by},
                                 a.cache.dim - at, vec);
        }
}

template <int DS>
void launch_tiles(const Attention &a, int64_t tiles, hipStream_t s)
{
    MAMBO_LAUNCH((attend_tiles_kernel<DS>), dim3((unsigned)(tiles * a.cache.heads), (unsigned)a.parts),
                 dim3(64 * tile_waves(DS)), 0, s, a);
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
