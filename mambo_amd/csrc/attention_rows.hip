// Attention of few rows (a token's heads, a short draft) over long caches: bound by the codes' bytes.
//
// The row kernel takes the blocks of 32 cached tokens of all its sequences, one after the other, in equal
// shares, so that one long sequence among short ones keeps no workgroup longer than the others. A
// workgroup's four waves take blocks in turn; a wave holds the scores of a block
//     S^T = K Q^T  (16 x 16 x 32 MFMAs over two tiles of 16 tokens)
// in such an order that lane 16 kk + i has query i's probabilities of the tokens 8 kk .. 8 kk + 7, the
// operand that  O^T += V^T P^T  wants of it: nothing goes through LDS or other lanes but the largest
// score. The running largest and total are f32; the codes are widened to bf16, which holds them exactly, and the
// probabilities are rounded to bf16 (2^-8 of each at most, beside the outputs' own): the other operand needs the exponents of bf16.
// What that costs is 13 to 28% of the error against 64 bits, which is the outputs' rounding otherwise (one token at 131150 2.03e-3 in
// the 2-norm for 1.68e-3). A second bf16 term of each probability takes it away, for 49.0 us in the place of 46.9 there, 112.5 of
// 111.1 for 64 users of up to 8192, and 690 of 498 for 8192 tokens by the kernel for many rows: left out in both, so that a row is as
// exact whichever takes it.
// One token at 131150 of 8 heads of 128: 43 us, 6.3 TB/s of codes; a large read reaches 6.4.
#include "attention.h"

namespace {

// Largest of the four lanes that share a query: rows of 16 lanes, then halves of the wave, exchanged.
__device__ __forceinline__ float across_max(float x)
{
    auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
    auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
__device__ __forceinline__ float across_sum(float x)
{
    auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = __uint_as_float(a[0]) + __uint_as_float(a[1]);
    auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return __uint_as_float(b[0]) + __uint_as_float(b[1]);
}

// The sequences' blocks added up by every wave for itself, 256 sequences at a time, four a lane (0.7 us up
// to 256, 1 us for every 256 more; a table of them would be a launch of its own).
struct Scan {
    const Attention &a;
    int w[4], before, through; // of this lane's sequences, and the blocks before them and through them
    int s0;

    __device__ Scan(const Attention &args) : a(args), s0(-1) {}
    __device__ void strip(int from, int base)
    {
        s0 = from;
        int sum = 0;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int s = from + 4 * lane_id() + j;
            w[j] = 0;
            if (s < a.b.seqs)
                w[j] = row_blocks(a, sequence(a, s));
            sum += w[j];
        }
        through = sum;
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
            const int up = __shfl_up(through, d);
            through += lane_id() >= d ? up : 0;
        }
        through += base;
        before = through - sum;
    }
    __device__ int end() const { return __builtin_amdgcn_readlane(through, 63); }
    // All blocks; where each sequence's begin, if asked for.
    __device__ int total(int32_t *begins)
    {
        int base = 0;
        for (int from = 0; from < a.b.seqs; from += 256) {
            strip(from, base);
            if (begins) {
                int at = before;
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const int s = from + 4 * lane_id() + j;
                    if (s < a.b.seqs)
                        begins[s] = at;
                    at += w[j];
                }
            }
            base = end();
        }
        if (begins && lane_id() == 0)
            begins[a.b.seqs] = base;
        return base;
    }
    // The sequence that has `block` (below the total), and its first block.
    __device__ void find(int block, int *sequence, int *first)
    {
        if (a.b.seqs > 256 || s0 < 0) {
            int base = 0;
            for (int from = 0; from < a.b.seqs; from += 256) {
                strip(from, base);
                base = end();
                if (base > block)
                    break;
            }
        }
        const uint64_t past = __ballot(through > block);
        const int src = past ? __builtin_ctzll(past) : 63;
        int s = s0 + 4 * lane_id(), at = before;
#pragma unroll
        for (int j = 0; j < 3; ++j)
            if (at + w[j] <= block && s == s0 + 4 * lane_id() + j) {
                at += w[j];
                ++s;
            }
        *sequence = __builtin_amdgcn_readlane(s, src);
        *first = __builtin_amdgcn_readlane(at, src);
    }
};

// A sequence's rows of a head over the blocks [first, last) of its keys.
struct Stretch {
    Sequence seq;
    int s, first, last;
};

// Such a stretch, whose blocks the workgroup's waves take in turn; what they found is left in LDS.
template <int DS, int RT, int NW>
struct Rows {
    static constexpr int DP = 32 * DS;
    struct Shared {
        float o[4][16 * RT][DP + 4];
        float m[4][16 * RT], l[4][16 * RT];
    };
    struct Block {
        uint4 k[DS], v[DS];
        uint32_t scales;
        int page;
    };
    // Blocks that a wave holds, all but one of them on their way.
    static constexpr int NB = NW == 8 && DS * RT <= 4 ? 3 : 2;

    // Blocks of a stretch that are on their way to this wave.
    struct Held {
        Block b[NB];
        int blk, next_page;
    };

    // Pages come by scalar loads, one block ahead of the codes; the last block's stands for those behind it, the first of
    // the table for those of no blocks at all.
    __device__ static int page_of(const Attention &a, const Stretch &st, int blk)
    {
        return scalar_load(a.b.tables + st.s * a.b.ldt + (max(min(blk, st.last - 1), 0) >> a.cache.shift));
    }
    __device__ static bool there(const Attention &a, int page) { return (uint32_t)page < (uint32_t)a.cache.pages; }

    // No branch ends between a load and its use, where the compiler would wait for it.
    __device__ static void load(const Attention &a, const Stretch &st, int head, int zero, int blk, int page, Block &b)
    {
        if (blk >= st.last)
            return;
        b.page = page;
        const int64_t at = a.cache.block(there(a, page) ? page : 0, head, blk);
        const uint4 *codes = reinterpret_cast<const uint4 *>(a.cache.codes + at * (2 * kKvBlock * DP)) + lane_id();
        b.scales = *reinterpret_cast<const uint16_t *>(a.cache.scales + 2 * (at + zero));
#pragma unroll
        for (int d = 0; d < DS; ++d)
            b.k[d] = codes[64 * d];
#pragma unroll
        for (int d = 0; d < DS; ++d)
            b.v[d] = codes[64 * (DS + d)];
    }

    __device__ static void begin(const Attention &a, const Stretch &st, int head, int zero, Held &held)
    {
        held.blk = st.first + __builtin_amdgcn_readfirstlane((int)threadIdx.x / 64);
#pragma unroll
        for (int j = 0; j < NB - 1; ++j)
            load(a, st, head, zero, held.blk + j * NW, page_of(a, st, held.blk + j * NW), held.b[j]);
        held.next_page = page_of(a, st, held.blk + (NB - 1) * NW);
    }

    __device__ static void attend(const Attention &a, const Stretch &st, int head, Shared &sh)
    {
        const Sequence &seq = st.seq;
        const int lane = lane_id(), kk = lane >> 4, col = lane & 15, zero = vector_zero();
        const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x / 64), rows = seq.n * a.group;
        Held held;
        begin(a, st, head, zero, held);

        bf16x8 q[RT][DS];
        int to[RT], from[RT];
#pragma unroll
        for (int r = 0; r < RT; ++r) {
            const int row = 16 * r + col, i = row / a.group, h = head * a.group + row % a.group;
            const bool some = row < rows;
            to[r] = some ? sees_to(a, seq, i) : 0;
            from[r] = some ? sees_from(a, seq, i) : 0;
            const __bf16 *x = a.q + (int64_t)(seq.first + i) * a.ldqt + h * a.ldqh;
#pragma unroll
            for (int d = 0; d < DS; ++d) {
                const int at_d = 32 * d + 8 * kk;
                q[r][d] = bf16x8{};
                if (some && at_d < a.cache.dim)
                    q[r][d] = *reinterpret_cast<const bf16x8 *>(x + at_d);
            }
        }
        // where no row's limits can be inside a block
        const int all_to = sees_to(a, seq, 0), all_from = sees_from(a, seq, seq.n - 1);

        v4f o[RT][2 * DS];
        float m[RT], l[RT];
#pragma unroll
        for (int r = 0; r < RT; ++r) {
            m[r] = -__builtin_inff();
            l[r] = 0.0f;
#pragma unroll
            for (int d = 0; d < 2 * DS; ++d)
                o[r][d] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
        }

        const auto take = [&](int blk, const Block &b) {
            if (!there(a, b.page))
                return;
            const float ks = e8m0(b.scales & 255), vs = e8m0(b.scales >> 8);
            v4f x[RT][2];
#pragma unroll
            for (int r = 0; r < RT; ++r)
                x[r][0] = x[r][1] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int d = 0; d < DS; ++d) {
                const bf16x8 k0 = widen(b.k[d].x, b.k[d].y, ks), k1 = widen(b.k[d].z, b.k[d].w, ks);
#pragma unroll
                for (int r = 0; r < RT; ++r) {
                    x[r][0] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(k0, q[r][d], x[r][0], 0, 0, 0);
                    x[r][1] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(k1, q[r][d], x[r][1], 0, 0, 0);
                }
            }
            const int token = blk * kKvBlock + 8 * kk;
            const bool edge = (blk + 1) * kKvBlock > all_to || blk * kKvBlock < all_from;
            bf16x8 p[RT];
#pragma unroll
            for (int r = 0; r < RT; ++r) {
                float y[8], top = -__builtin_inff();
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    y[j] = x[r][j >> 2][j & 3] * a.scale;
                    if (edge)
                        y[j] = token + j < to[r] && token + j >= from[r] ? y[j] : -__builtin_inff();
                    top = fmaxf(top, y[j]);
                }
                top = across_max(top);
                if (__any(top > m[r])) { // else nothing grows
                    const float grown = fmaxf(m[r], top);
                    const float by = m[r] == -__builtin_inff() ? 0.0f : exp2_fast(m[r] - grown);
                    m[r] = grown;
                    l[r] *= by;
#pragma unroll
                    for (int d = 0; d < 2 * DS; ++d)
                        o[r][d] *= by;
                }
                const float less = m[r] == -__builtin_inff() ? 0.0f : m[r];
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    y[j] = exp2_fast(y[j] - less);
                    l[r] += y[j];
                    p[r][j] = (__bf16)y[j];
                }
            }
            const int left = seq.len - token;
            const bool tail = (blk + 1) * kKvBlock > seq.len;
#pragma unroll
            for (int d = 0; d < DS; ++d) {
                uint2 v0 = make_uint2(b.v[d].x, b.v[d].y), v1 = make_uint2(b.v[d].z, b.v[d].w);
                if (tail) {
                    v0 = keep_tokens(v0.x, v0.y, left);
                    v1 = keep_tokens(v1.x, v1.y, left);
                }
                const bf16x8 w0 = widen(v0.x, v0.y, vs), w1 = widen(v1.x, v1.y, vs);
#pragma unroll
                for (int r = 0; r < RT; ++r) {
                    o[r][2 * d] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(w0, p[r], o[r][2 * d], 0, 0, 0);
                    o[r][2 * d + 1] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(w1, p[r], o[r][2 * d + 1], 0, 0, 0);
                }
            }
        };

        while (held.blk < st.last) {
#pragma unroll
            for (int j = 0; j < NB; ++j) {
                if (held.blk < st.last) {
                    load(a, st, head, zero, held.blk + (NB - 1) * NW, held.next_page, held.b[(j + NB - 1) % NB]);
                    held.next_page = page_of(a, st, held.blk + NB * NW);
                    take(held.blk, held.b[j]);
                }
                held.blk += NW;
            }
        }
        const auto leave = [&](int w) {
#pragma unroll
            for (int r = 0; r < RT; ++r) {
                const float sum = across_sum(l[r]);
                if (kk == 0) {
                    sh.m[w][16 * r + col] = m[r];
                    sh.l[w][16 * r + col] = sum;
                }
#pragma unroll
                for (int d = 0; d < 2 * DS; ++d)
                    *reinterpret_cast<v4f *>(&sh.o[w][16 * r + col][16 * d + 4 * kk]) = o[r][d];
            }
        };
        if constexpr (NW == 8) { // the second four through the places of the first
            if (wave >= 4)
                leave(wave - 4);
            __syncthreads();
            if (wave < 4) {
#pragma unroll
                for (int r = 0; r < RT; ++r) {
                    const float other = sh.m[wave][16 * r + col], top = fmaxf(m[r], other);
                    const float less = top == -__builtin_inff() ? 0.0f : top;
                    const float f = exp2_fast(m[r] - less), g = exp2_fast(other - less);
                    // a quarter of the other total for each of the lanes that add theirs up
                    l[r] = l[r] * f + 0.25f * sh.l[wave][16 * r + col] * g;
                    m[r] = top;
#pragma unroll
                    for (int d = 0; d < 2 * DS; ++d)
                        o[r][d] = o[r][d] * f + *reinterpret_cast<const v4f *>(&sh.o[wave][16 * r + col][16 * d + 4 * kk]) * g;
                }
                leave(wave);
            }
        } else {
            leave(wave);
        }
        __syncthreads();
    }

    // Four values of a row over all waves; its largest score and total.
    __device__ static v4f collect(const Shared &sh, int row, int d, float *top, float *sum)
    {
        *top = sh.m[0][row];
#pragma unroll
        for (int w = 1; w < 4; ++w)
            *top = fmaxf(*top, sh.m[w][row]);
        const float less = *top == -__builtin_inff() ? 0.0f : *top;
        *sum = 0.0f;
        v4f y = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            const float f = exp2_fast(sh.m[w][row] - less);
            *sum += f * sh.l[w][row];
            y += f * *reinterpret_cast<const v4f *>(&sh.o[w][row][d]);
        }
        return y;
    }
};

// Two waves a SIMD while a wave's registers are enough.
constexpr int rows_occupancy(int ds, int rt) { return ds * rt <= 4 ? 2 : 1; }

// 16 RT rows by 32 DS values a head, the blocks of all sequences in equal shares.
template <int DS, int RT>
__global__ __launch_bounds__(256, rows_occupancy(DS, RT)) void attend_rows_kernel(const Attention a)
{
    using R = Rows<DS, RT, 4>;
    constexpr int DP = 32 * DS;
    __shared__ typename R::Shared sh;
    const int tid = (int)threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid / 64);
    const int head = (int)(blockIdx.x % (unsigned)a.cache.heads), slot = (int)(blockIdx.x / (unsigned)a.cache.heads);
    Scan scan(a);
    const int total = scan.total(blockIdx.x == 0 && wave == 0 ? a.begins : nullptr);
    const int count = shares(a, total);
    if (slot >= count || total == 0)
        return;
    int at = share_begin(slot, total, count);
    const int end = share_begin(slot + 1, total, count);
    int s = 0, base = 0; // the sequence that `at` is in, and its first block in the order
    scan.find(at, &s, &base);

    while (at < end) {
        const Sequence seq = sequence(a, s);
        const int blocks = row_blocks(a, seq);
        if (at >= base + blocks) { // sequences without blocks between
            scan.find(at, &s, &base);
            continue;
        }
        const int stop = min(end, base + blocks);
        R::attend(a, {seq, s, seq.lo + at - base, seq.lo + stop - base}, head, sh);
        const bool whole = at == base && stop == base + blocks;
        const int which = at == base ? 1 : 0; // a share ends with a sequence that goes on, or begins with one
        const int64_t entry = ((int64_t)head * a.slots + slot) * 2 + which;
        for (int item = tid; item < seq.n * a.group * (DP / 4); item += 256) {
            const int row = item / (DP / 4), d = 4 * (item % (DP / 4));
            float top, sum;
            const v4f y = R::collect(sh, row, d, &top, &sum);
            if (whole) {
                store_row(a, seq.first + row / a.group, head * a.group + row % a.group, d, y, top, sum);
            } else {
                *reinterpret_cast<v4f *>(a.rows_o + (entry * (16 * RT) + row) * DP + d) = y;
                if (d == 0)
                    *reinterpret_cast<float2 *>(a.rows_ml + (entry * (16 * RT) + row) * 2) = make_float2(top, sum);
            }
        }
        at = stop;
        if (at < end) {
            base += blocks;
            ++s;
            __syncthreads();
        }
    }
}

// The same where no sequence has many blocks: one workgroup for all of a sequence and a head, nothing to join.
template <int DS, int RT>
__global__ __launch_bounds__(512, rows_occupancy(DS, RT)) void attend_short_kernel(const Attention a)
{
    using R = Rows<DS, RT, 8>;
    constexpr int DP = 32 * DS;
    __shared__ typename R::Shared sh;
    const int head = (int)(blockIdx.x % (unsigned)a.cache.heads), s = (int)(blockIdx.x / (unsigned)a.cache.heads);
    const Sequence seq = sequence(a, s);
    const int rows = seq.n * a.group;
    if (seq.n <= 0 || seq.n > a.few_rows / a.group)
        return;
    R::attend(a, {seq, s, seq.lo, seq.hi}, head, sh);
    for (int item = (int)threadIdx.x; item < rows * (DP / 4); item += 512) {
        const int row = item / (DP / 4), d = 4 * (item % (DP / 4));
        float top, sum;
        const v4f y = R::collect(sh, row, d, &top, &sum);
        store_row(a, seq.first + row / a.group, head * a.group + row % a.group, d, y, top, sum);
    }
}

template <int DS, int RT>
void launch_rows(const Attention &a, hipStream_t s)
{
    if constexpr (RT <= max_row_tiles(32 * DS)) {
        if (a.slots)
            MAMBO_LAUNCH((attend_rows_kernel<DS, RT>), dim3((unsigned)(a.slots * a.cache.heads)), dim3(256), 0, s, a);
        else if constexpr (short_fits(DS, RT))
            MAMBO_LAUNCH((attend_short_kernel<DS, RT>), dim3((unsigned)(a.b.seqs * a.cache.heads)), dim3(512), 0, s, a);
    }
}

} // namespace

int launch_attend_rows(const Attention &a, int row_tiles, hipStream_t s)
{
    const int ds = kv_padded(a.cache.dim) / 32;
#define MAMBO_ROWS(DS)                                                                                             \
    if (ds == DS)                                                                                                  \
    row_tiles == 1 ? launch_rows<DS, 1>(a, s) : row_tiles == 2 ? launch_rows<DS, 2>(a, s) : launch_rows<DS, 4>(a, s)
    MAMBO_ROWS(1);
    MAMBO_ROWS(2);
    MAMBO_ROWS(3);
    MAMBO_ROWS(4);
    MAMBO_ROWS(5);
    MAMBO_ROWS(6);
    MAMBO_ROWS(7);
    MAMBO_ROWS(8);
#undef MAMBO_ROWS
    return mambo_check_launch("kv_attention");
}
