// Rotary positions, the append to the paged 8-bit cache with the rotation on the way, and reading it back.
#include <algorithm>

#include "kv_cache.h"

namespace {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

// Eight consecutive values of a row as f32; kVec: the row is 16-byte aligned.
template <bool kBf16, bool kVec>
__device__ __forceinline__ void load8(const void *x, int64_t at, float (&v)[8])
{
    const row_t<kBf16> *p = reinterpret_cast<const row_t<kBf16> *>(x) + at;
    if constexpr (kVec && kBf16) {
        const bf16x8 w = *reinterpret_cast<const bf16x8 *>(p);
#pragma unroll
        for (int j = 0; j < 8; ++j)
            v[j] = (float)w[j];
    } else if constexpr (kVec) {
        const v4f a = reinterpret_cast<const v4f *>(p)[0], b = reinterpret_cast<const v4f *>(p)[1];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            v[j] = a[j];
            v[4 + j] = b[j];
        }
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j)
            v[j] = (float)p[j];
    }
}

template <bool kBf16, bool kVec>
__device__ __forceinline__ void store8(void *x, int64_t at, const float (&v)[8])
{
    row_t<kBf16> *p = reinterpret_cast<row_t<kBf16> *>(x) + at;
    if constexpr (kVec && kBf16) {
        bf16x8 w;
#pragma unroll
        for (int j = 0; j < 8; ++j)
            w[j] = (__bf16)v[j];
        *reinterpret_cast<bf16x8 *>(p) = w;
    } else if constexpr (kVec) {
        reinterpret_cast<v4f *>(p)[0] = v4f{v[0], v[1], v[2], v[3]};
        reinterpret_cast<v4f *>(p)[1] = v4f{v[4], v[5], v[6], v[7]};
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j)
            p[j] = (row_t<kBf16>)v[j];
    }
}

struct Rows {
    const void *x;
    int64_t ldt, ldh;
};

// --------------------------------------------------------------------------------- rotation
// Work on a head of `dim` values is cut into units, each of which reads all that it writes, so that a
// head may be rotated in place. Aligned rows whose pairs lie in whole chunks of 8 (kVec): two chunks that
// are each other's partners, or one chunk of neighbouring pairs or of values that are copied. Else
// one pair, or one value.
template <bool kVec>
__host__ __device__ __forceinline__ int rotary_units(int dim, int size, int interleaved)
{
    if (kVec)
        return interleaved ? dim / 8 : size / 16 + (dim - size) / 8;
    return size / 2 + dim - size;
}

// Unit u of the head at x, to out; cs: the cosines and sines of the token's size / 2 pairs.
template <bool kIn, bool kOut, bool kVec>
__device__ __forceinline__ void rotate_unit(const void *x, int64_t at, void *out, int64_t to, int u, int size,
                                            int interleaved, const float2 *cs)
{
    if constexpr (kVec) {
        float a[8], b[8];
        if (interleaved || u >= size / 16) {
            const int d = interleaved ? 8 * u : size + 8 * (u - size / 16);
            load8<kIn, true>(x, at + d, a);
            if (d < size)
#pragma unroll
                for (int j = 0; j < 8; j += 2) {
                    const float2 t = cs[(d + j) / 2];
                    const float p = a[j], q = a[j + 1];
                    a[j] = turn_low(p, q, t);
                    a[j + 1] = turn_high(p, q, t);
                }
            store8<kOut, true>(out, to + d, a);
        } else {
            load8<kIn, true>(x, at + 8 * u, a);
            load8<kIn, true>(x, at + size / 2 + 8 * u, b);
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const float2 t = cs[8 * u + j];
                const float p = a[j], q = b[j];
                a[j] = turn_low(p, q, t);
                b[j] = turn_high(p, q, t);
            }
            store8<kOut, true>(out, to + 8 * u, a);
            store8<kOut, true>(out, to + size / 2 + 8 * u, b);
        }
    } else {
        const row_t<kIn> *p = reinterpret_cast<const row_t<kIn> *>(x) + at;
        row_t<kOut> *o = reinterpret_cast<row_t<kOut> *>(out) + to;
        if (u < size / 2) {
            const int i = interleaved ? 2 * u : u, j = interleaved ? 2 * u + 1 : u + size / 2;
            const float2 t = cs[u];
            const float a = (float)p[i], b = (float)p[j];
            o[i] = (row_t<kOut>)turn_low(a, b, t);
            o[j] = (row_t<kOut>)turn_high(a, b, t);
        } else {
            const int i = u + size / 2;
            o[i] = (row_t<kOut>)(float)p[i];
        }
    }
}

struct Rotary {
    const void *x;
    void *out;
    int64_t ldt, ldh, ldot, ldoh;
    const int32_t *positions;
    RotaryTable table;
    int64_t tokens;
    int heads, dim, tile, heads_each; // tokens and heads of a workgroup
};

// A workgroup makes the angles of its tokens once in LDS (a sine and cosine are about 40 instructions, a
// rotation 4) for all of its heads; then a pass over the rows, bound by memory: 8192 x 32 heads of 128 in bf16 22.6 us, 5.9 TB/s.
template <bool kIn, bool kOut, bool kVec>
__global__ __launch_bounds__(256) void rotary_kernel(const Rotary a)
{
    extern __shared__ float2 angles[];
    const int half = a.table.size / 2, tid = (int)threadIdx.x;
    const int64_t t0 = (int64_t)blockIdx.x * a.tile;
    const int count = (int)min((int64_t)a.tile, a.tokens - t0);
    for (int i = tid; i < count * half; i += 256)
        angles[i] = rotary_angle(a.table, a.positions[t0 + i / half], i % half);
    __syncthreads();
    const int h0 = (int)blockIdx.y * a.heads_each, heads = min(a.heads_each, a.heads - h0);
    const int units = rotary_units<kVec>(a.dim, a.table.size, a.table.interleaved);
    const int wide = min(units, 256), step = 256 / wide;
    if (tid >= wide * step)
        return;
    int h = tid / wide, t = 0;
    t += h / heads;
    h %= heads;
    for (; t < count;) {
        for (int u = tid % wide; u < units; u += wide)
            rotate_unit<kIn, kOut, kVec>(a.x, (t0 + t) * a.ldt + (h0 + h) * a.ldh, a.out,
                                         (t0 + t) * a.ldot + (h0 + h) * a.ldoh, u, a.table.size, a.table.interleaved,
                                         angles + t * half);
        for (h += step; h >= heads; h -= heads)
            ++t;
    }
}

// ----------------------------------------------------------------------------------- append
struct Append {
    Rows k, v, q;
    void *q_out;
    int64_t ldot, ldoh;
    KvCache cache;
    KvBatch b;
    RotaryTable table; // size 0: keys as they are
    const int32_t *positions;
    int q_heads, q_parts; // workgroups that the queries of a block's tokens are dealt to
    int blocks_each;      // of a uniform batch: blocks that a sequence's rows can touch
};

// Largest magnitude (bits) over the workgroup of two values at once.
__device__ __forceinline__ uint2 largest(uint32_t a, uint32_t b, uint2 *scratch)
{
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        a = max(a, (uint32_t)__shfl_xor((int)a, d));
        b = max(b, (uint32_t)__shfl_xor((int)b, d));
    }
    if (lane_id() == 0)
        scratch[threadIdx.x / 64] = make_uint2(a, b);
    __syncthreads();
    uint2 m = scratch[0];
#pragma unroll
    for (int w = 1; w < 4; ++w)
        m = make_uint2(max(m.x, scratch[w].x), max(m.y, scratch[w].y));
    return m;
}

__device__ __forceinline__ int kv_exponent(uint32_t amax_bits)
{
    return amax_bits ? max(mxfp8_exponent(__uint_as_float(amax_bits)), kKvLowest) : kKvLowest;
}

// Four codes rounded again after a multiplication by 2^by (by < 0).
__device__ __forceinline__ uint32_t recode4(uint32_t w, int by)
{
    typedef float v2f __attribute__((ext_vector_type(2)));
    const v2f a = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, false), b = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, true);
    return pack4<true>(__builtin_ldexpf(a[0], by), __builtin_ldexpf(a[1], by), __builtin_ldexpf(b[0], by),
                       __builtin_ldexpf(b[1], by));
}

// One workgroup for each block that new tokens touch, of one key/value head: nobody else writes its scale. Others rotate the
// queries of the block's tokens, all heads of a token in one place, where its angles are worked out once.
// Keys: a thread has 8 neighbouring values of a token (P of them), values: two neighbouring ones of
// 8 tokens (PV of them), as the layout's 8-byte pieces want them, so that a long prompt is read and written in whole
// pieces; the rows stay in registers between the search for the largest and the rounding.
// Bound by memory: 8192 tokens of 8 key/value and 32 query heads of 128 in f32 60 us, 4.7 TB/s (71 with each head's queries in the
// workgroup of its keys, whose 2056 workgroups then are one round and a seventh).
// P: padded head size / 64, rounded up.
template <int P, bool kBf16, bool kVec>
__global__ __launch_bounds__(256) void append_kernel(const Append a)
{
    extern __shared__ float2 angles[];
    __shared__ uint2 scratch[4];
    __shared__ int bad[kKvBlock];
    const int tid = (int)threadIdx.x, head = (int)blockIdx.y, dim = a.cache.dim, padded = kv_padded(dim);
    int s, j;
    if (a.b.offsets) {
        s = find_slot(a.b.seqs, blockIdx.x, [&](int i) { return (int64_t)(a.b.offset(i) / kKvBlock) + 2 * i; });
        j = (int)blockIdx.x - a.b.offset(s) / kKvBlock - 2 * s;
    } else {
        s = (int)blockIdx.x / a.blocks_each;
        j = (int)blockIdx.x % a.blocks_each;
    }
    const int first = a.b.offset(s), n = (a.b.offsets ? a.b.offset(s + 1) : first + a.b.each) - first;
    const int len = a.b.length(s), start = len - n; // start: position of the first row
    const int from = max(start, 0), blk = from / kKvBlock + j;
    if (j < 0 || n <= 0 || j > n / kKvBlock + 1 || (j > 0 && blk > (len - 1) / kKvBlock))
        return;
    // positions of this block, none in the first where there are no rows that far
    const int base = blk * kKvBlock, lo = max(from, base), hi = base + min(kKvBlock, len - base);
    const int half = a.table.size / 2;
    const int64_t row0 = (int64_t)first - start; // row of position p: row0 + p

    const auto make_angles = [&](int p0, int count) {
        for (int i = tid; i < count * half; i += 256) {
            const int p = p0 + i / half;
            angles[i] = rotary_angle(a.table, a.positions ? a.positions[row0 + p] : p, i % half);
        }
    };
    if (head >= a.cache.heads) {
        const int part = head - a.cache.heads, each = kKvBlock / a.q_parts;
        const int units = rotary_units<kVec>(dim, a.table.size, a.table.interleaved); // at most 256
        const int step = 256 / units, row_step = step % a.q_heads, token_step = step / a.q_heads;
        // this block's tokens, and with the first also those before the sequence's start, which are not stored
        const int begin = j == 0 ? start : lo, rows = hi - begin;
        for (int done = part * each; done < rows; done += kKvBlock) {
            const int p0 = begin + done, count = min(each, rows - done);
            make_angles(p0, count);
            __syncthreads();
            int h = tid / units, t = h / a.q_heads;
            h %= a.q_heads;
            while (t < count && tid < units * step) {
                const int64_t row = row0 + p0 + t;
                rotate_unit<kBf16, true, kVec>(a.q.x, row * a.q.ldt + h * a.q.ldh, a.q_out, row * a.ldot + h * a.ldoh,
                                               tid % units, a.table.size, a.table.interleaved, angles + t * half);
                h += row_step;
                t += token_step;
                if (h >= a.q_heads) {
                    h -= a.q_heads;
                    ++t;
                }
            }
            __syncthreads();
        }
        return;
    }
    if (lo >= hi || base >= a.b.capacity) // whole blocks: a table's pages are
        return;
    make_angles(lo, hi - lo);
    if (tid < kKvBlock)
        bad[tid] = 0;
    __syncthreads();

    const int page = a.b.page(s, blk >> a.cache.shift);
    if ((uint32_t)page >= (uint32_t)a.cache.pages)
        return;
    const int64_t at = a.cache.block(page, head, blk);
    uint8_t *const keys = a.cache.codes + (int64_t)at * (2 * kKvBlock * padded), *const values = keys + kKvBlock * padded;
    uint8_t *const scale = a.cache.scales + 2 * (int64_t)at;

    const int chunks = padded / 8;
    float kx[P][8];
#pragma unroll
    for (int i = 0; i < P; ++i) {
        const int item = tid + 256 * i, t = item / chunks, d = 8 * (item % chunks), p = base + t;
#pragma unroll
        for (int e = 0; e < 8; ++e)
            kx[i][e] = 0.0f;
        if (t >= kKvBlock || d >= dim || p < lo || p >= hi)
            continue;
        const int64_t row = (row0 + p) * a.k.ldt + head * a.k.ldh;
        float x[8], y[8];
        load8<kBf16, kVec>(a.k.x, row + d, x);
        const int size = a.table.size;
        const float2 *cs = angles + (p - lo) * half;
        if (d >= size) {
#pragma unroll
            for (int e = 0; e < 8; ++e)
                y[e] = x[e];
        } else if (a.table.interleaved) {
#pragma unroll
            for (int e = 0; e < 8; e += 2) {
                const bool in = d + e < size;
                const float2 c = in ? cs[(d + e) / 2] : make_float2(1.0f, 0.0f);
                y[e] = turn_low(x[e], x[e + 1], c);
                y[e + 1] = turn_high(x[e], x[e + 1], c);
                if (!in) { // 0 * inf
                    y[e] = x[e];
                    y[e + 1] = x[e + 1];
                }
            }
        } else if (half % 8 == 0) {
            float z[8];
            const bool low = d < half;
            load8<kBf16, kVec>(a.k.x, row + (low ? d + half : d - half), z);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const float2 c = cs[(low ? d : d - half) + e];
                y[e] = low ? turn_low(x[e], z[e], c) : turn_high(z[e], x[e], c);
            }
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const int q = d + e;
                y[e] = x[e];
                if (q < size) {
                    const bool low = q < half;
                    const float z = (float)(reinterpret_cast<const row_t<kBf16> *>(a.k.x)[row + (low ? q + half : q - half)]);
                    const float2 c = cs[low ? q : q - half];
                    y[e] = low ? turn_low(x[e], z, c) : turn_high(z, x[e], c);
                }
            }
        }
        bool finite = true;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            kx[i][e] = y[e];
            finite &= abs_bits(y[e]) < kNonFiniteBits;
        }
        if (!finite)
            bad[t] = 1;
    }
    // values: piece (kk, d, d + 1)
    const int pairs = dim / 2;
    constexpr int PV = (P + 1) / 2;
    float vx[PV][8][2];
#pragma unroll
    for (int i = 0; i < PV; ++i) {
        const int item = tid + 256 * i, kk = item / pairs, d = 2 * (item % pairs);
#pragma unroll
        for (int t = 0; t < 8; ++t) {
            vx[i][t][0] = vx[i][t][1] = 0.0f;
            const int p = base + 8 * kk + t;
            if (kk >= kKvBlock / 8 || p < lo || p >= hi)
                continue;
            const row_t<kBf16> *x = reinterpret_cast<const row_t<kBf16> *>(a.v.x) + (row0 + p) * a.v.ldt + head * a.v.ldh + d;
            if constexpr (kVec) {
                typedef row_t<kBf16> pair_t __attribute__((ext_vector_type(2)));
                const pair_t w = *reinterpret_cast<const pair_t *>(x);
                vx[i][t][0] = (float)w[0];
                vx[i][t][1] = (float)w[1];
            } else {
                vx[i][t][0] = (float)x[0];
                vx[i][t][1] = (float)x[1];
            }
            if (abs_bits(vx[i][t][0]) >= kNonFiniteBits || abs_bits(vx[i][t][1]) >= kNonFiniteBits)
                bad[8 * kk + t] = 1;
        }
    }
    __syncthreads();
    uint32_t ka = 0u, va = 0u;
#pragma unroll
    for (int i = 0; i < P; ++i) {
        const int t = (tid + 256 * i) / chunks;
        if (t < kKvBlock && !bad[t])
#pragma unroll
            for (int e = 0; e < 8; ++e)
                ka = max(ka, abs_bits(kx[i][e]));
    }
#pragma unroll
    for (int i = 0; i < PV; ++i) {
        const int kk = (tid + 256 * i) / pairs;
#pragma unroll
        for (int e = 0; e < 8; ++e)
            if (kk < kKvBlock / 8 && !bad[8 * kk + e])
                va = max(va, max(abs_bits(vx[i][e][0]), abs_bits(vx[i][e][1])));
    }
    const bool fresh = lo == base;
    const int old_k = fresh ? kKvLowest : (int)scale[0] - 127, old_v = fresh ? kKvLowest : (int)scale[1] - 127;
    const uint2 amax = largest(ka, va, scratch); // its barrier: every wave has read the old exponents
    const int ke = max(old_k, kv_exponent(amax.x)), ve = max(old_v, kv_exponent(amax.y));
    const float k_most = ke >= kKvHighest ? kKvMostThere : 448.0f, v_most = ve >= kKvHighest ? kKvMostThere : 448.0f;
    __syncthreads();
    if (!fresh && (ke > old_k || ve > old_v)) {
        for (int i = tid; i < 2 * 2 * padded; i += 256) {
            uint4 *w = reinterpret_cast<uint4 *>(keys) + i;
            const int by = i < 2 * padded ? old_k - ke : old_v - ve;
            if (by < 0) {
                const uint4 c = *w;
                *w = make_uint4(recode4(c.x, by), recode4(c.y, by), recode4(c.z, by), recode4(c.w, by));
            }
        }
        __syncthreads(); // before the new tokens' bytes go to the same pieces
    }
    if (tid == 0) {
        scale[0] = (uint8_t)(ke + 127);
        scale[1] = (uint8_t)(ve + 127);
    }
#pragma unroll
    for (int i = 0; i < P; ++i) {
        const int item = tid + 256 * i, t = item / chunks, d = 8 * (item % chunks), p = base + t;
        if (t < kKvBlock && p >= lo && p < hi) {
            float y[8];
#pragma unroll
            for (int e = 0; e < 8; ++e)
                y[e] = fminf(fmaxf(__builtin_ldexpf(kx[i][e], -ke), -k_most), k_most);
            uint2 w = make_uint2(pack4<true>(y[0], y[1], y[2], y[3]), pack4<true>(y[4], y[5], y[6], y[7]));
            if (bad[t])
                w = make_uint2(0x7F7F7F7Fu, 0x7F7F7F7Fu);
            *reinterpret_cast<uint2 *>(keys + kv_key_byte(t, d)) = w;
        }
    }
#pragma unroll
    for (int i = 0; i < PV; ++i) {
        const int item = tid + 256 * i, kk = item / pairs, d = 2 * (item % pairs);
        if (kk >= kKvBlock / 8)
            continue;
        const int p = base + 8 * kk;
#pragma unroll
        for (int c = 0; c < 2; ++c) {
            float y[8];
#pragma unroll
            for (int e = 0; e < 8; ++e)
                y[e] = bad[8 * kk + e] ? 0.0f : fminf(fmaxf(__builtin_ldexpf(vx[i][e][c], -ve), -v_most), v_most);
            const uint2 w = make_uint2(pack4<true>(y[0], y[1], y[2], y[3]), pack4<true>(y[4], y[5], y[6], y[7]));
            uint8_t *to = values + kv_value_byte(8 * kk, d + c);
            if (p >= lo && p + 8 <= hi) {
                *reinterpret_cast<uint2 *>(to) = w;
            } else {
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    if (p + e >= lo && p + e < hi)
                        to[e] = (uint8_t)((e < 4 ? w.x : w.y) >> (8 * (e & 3)));
            }
        }
    }
}

// ------------------------------------------------------------------------------------- read
// 32 rows of one head a workgroup. Lanes side by side have rows side by side: of tokens that follow each other, eight use
// the eight bytes of one piece of the values, and four neighbouring pieces of the keys are one load. The rows are then
// written in whole from LDS (8192 tokens of 8 heads of 128 22.9 us with a row's values side by side).
__global__ __launch_bounds__(256) void read_kernel(const KvCache cache, const KvBatch b, const int32_t *sequences,
                                                   const int32_t *positions, int64_t n, __bf16 *k, __bf16 *v)
{
    extern __shared__ uint4 rows[]; // [2][32][dim / 8 + 1]
    typedef float v2f __attribute__((ext_vector_type(2)));
    const int chunks = cache.dim / 8, padded = kv_padded(cache.dim), head = (int)blockIdx.y, tid = (int)threadIdx.x;
    const int64_t first = (int64_t)blockIdx.x * 32, i = min(first + tid % 32, n - 1);
    const int s = sequences[i], p = positions[i], blk = p / kKvBlock, t = p % kKvBlock;
    const bool some = s >= 0 && s < b.seqs && p >= 0 && p < b.capacity;
    const int page = some ? b.page(s, blk >> cache.shift) : -1;
    const bool there = (uint32_t)page < (uint32_t)cache.pages;
    const int64_t at = there ? cache.block(page, head, blk) : 0;
    const uint8_t *keys = cache.codes + at * (2 * kKvBlock * padded), *values = keys + kKvBlock * padded;
    const int ke = (int)cache.scales[2 * at] - 127, ve = (int)cache.scales[2 * at + 1] - 127;
    for (int chunk = tid / 32; chunk < chunks; chunk += 8) {
        bf16x8 kv = {}, vv = {};
        if (there) {
            const int d = 8 * chunk;
            const uint2 w = *reinterpret_cast<const uint2 *>(keys + kv_key_byte(t, d));
            uint32_t c[8];
#pragma unroll
            for (int e = 0; e < 8; ++e)
                c[e] = values[kv_value_byte(t, d + e)];
#pragma unroll
            for (int e = 0; e < 8; e += 2) {
                const v2f x = __builtin_amdgcn_cvt_pk_f32_fp8((int)((e < 4 ? w.x : w.y) >> (8 * (e & 3))), false);
                const v2f y = __builtin_amdgcn_cvt_pk_f32_fp8((int)(c[e] | c[e + 1] << 8), false);
                kv[e] = (__bf16)__builtin_ldexpf(x[0], ke);
                kv[e + 1] = (__bf16)__builtin_ldexpf(x[1], ke);
                vv[e] = (__bf16)__builtin_ldexpf(y[0], ve);
                vv[e + 1] = (__bf16)__builtin_ldexpf(y[1], ve);
            }
        }
        rows[(tid % 32) * (chunks + 1) + chunk] = __builtin_bit_cast(uint4, kv);
        rows[(32 + tid % 32) * (chunks + 1) + chunk] = __builtin_bit_cast(uint4, vv);
    }
    __syncthreads();
    const int count = (int)min((int64_t)32, n - first);
    for (int item = tid; item < count * chunks; item += 256) {
        const int row = item / chunks, chunk = item % chunks;
        const int64_t to = ((first + row) * cache.heads + head) * cache.dim + 8 * chunk;
        *reinterpret_cast<uint4 *>(k + to) = rows[row * (chunks + 1) + chunk];
        *reinterpret_cast<uint4 *>(v + to) = rows[(32 + row) * (chunks + 1) + chunk];
    }
}

bool float_rows(int dtype) { return dtype == MAMBO_DTYPE_F32 || dtype == MAMBO_DTYPE_BF16; }
int64_t cdiv(int64_t a, int64_t b) { return (a + b - 1) / b; }

// Whether the rows can be read (or written) 16 bytes at a time.
bool vectors(const void *x, int64_t ldt, int64_t ldh, int dtype)
{
    const int64_t n = dtype == MAMBO_DTYPE_BF16 ? 8 : 4;
    return (uintptr_t)x % 16 == 0 && ldt % n == 0 && ldh % n == 0;
}

// Whether pairs lie in whole chunks of 8 of a head.
bool chunks(int64_t dim, const RotaryTable &t)
{
    return dim % 8 == 0 && t.size % (t.interleaved ? 8 : 16) == 0;
}

int check_table(const mambo_rotary_table *table, int64_t dim, RotaryTable *out)
{
    MAMBO_REQUIRE(table && table->turns, MAMBO_ERR_VALUE, "null pointer");
    MAMBO_REQUIRE(table->size >= 2 && table->size % 2 == 0 && table->size <= dim, MAMBO_ERR_VALUE,
                  "an even number of a head's %lld values is rotated (got %d)", (long long)dim, (int)table->size);
    MAMBO_REQUIRE((uintptr_t)table->turns % 8 == 0, MAMBO_ERR_VALUE, "the angles must be aligned to their type");
    *out = {table->turns, table->size, table->interleaved != 0, table->magnitude};
    return MAMBO_OK;
}

int check_rows(const void *x, int dtype, const char *what)
{
    MAMBO_REQUIRE(x != nullptr, MAMBO_ERR_VALUE, "null pointer (%s)", what);
    MAMBO_REQUIRE((uintptr_t)x % (dtype == MAMBO_DTYPE_BF16 ? 2 : 4) == 0, MAMBO_ERR_VALUE,
                  "%s must be aligned to their type", what);
    return MAMBO_OK;
}

} // namespace

int kv_check_cache(const mambo_kv_cache *c, KvCache *out)
{
    MAMBO_REQUIRE(c != nullptr, MAMBO_ERR_VALUE, "null pointer");
    MAMBO_REQUIRE(kv_dim_ok(c->head_dim), MAMBO_ERR_VALUE, "head_dim must be a multiple of 8 up to %d (got %d)",
                  MAMBO_KV_MAX_DIM, (int)c->head_dim);
    MAMBO_REQUIRE(c->page_size >= kKvBlock && c->page_size <= 65536 && (c->page_size & (c->page_size - 1)) == 0,
                  MAMBO_ERR_VALUE, "page_size must be a power of two from 32 to 65536 (got %d)", (int)c->page_size);
    MAMBO_REQUIRE(c->heads >= 1 && c->heads <= 16384 && c->pages >= 1 && c->pages <= 0x7FFFFFFF, MAMBO_ERR_VALUE,
                  "a cache has 1 to 2^31 - 1 pages of 1 to 16384 heads (got %lld of %d)", (long long)c->pages, (int)c->heads);
    MAMBO_REQUIRE(c->pages * c->heads * (c->page_size / kKvBlock) <= 0x7FFFFFFF, MAMBO_ERR_VALUE,
                  "a cache has at most 2^31 - 1 blocks of 32 tokens and a head (got %lld pages)", (long long)c->pages);
    MAMBO_REQUIRE(c->codes && c->scales, MAMBO_ERR_VALUE, "null pointer");
    MAMBO_REQUIRE((uintptr_t)c->codes % 16 == 0 && (uintptr_t)c->scales % 2 == 0, MAMBO_ERR_VALUE,
                  "codes must be 16-byte and scales 2-byte aligned");
    *out = {c->codes, c->scales, (int)c->pages, c->heads, c->head_dim, __builtin_ctz(c->page_size / kKvBlock)};
    return MAMBO_OK;
}

int kv_check_batch(const mambo_kv_batch *b, int64_t tokens, const mambo_kv_cache *cache, KvBatch *out)
{
    MAMBO_REQUIRE(b != nullptr, MAMBO_ERR_VALUE, "null pointer");
    MAMBO_REQUIRE(b->seqs >= 1 && b->seqs <= 0xFFFFFF, MAMBO_ERR_VALUE, "sequences must number 1 to 2^24 - 1 (got %lld)",
                  (long long)b->seqs);
    MAMBO_REQUIRE(tokens >= 0 && tokens <= 0x3FFFFFFF, MAMBO_ERR_VALUE, "rows must number 0 to 2^30 - 1 (got %lld)",
                  (long long)tokens);
    MAMBO_REQUIRE(b->offsets || tokens % b->seqs == 0, MAMBO_ERR_VALUE,
                  "without offsets every sequence has as many rows (got %lld of %lld)", (long long)tokens, (long long)b->seqs);
    MAMBO_REQUIRE(b->width >= 1 && b->width <= 0x3FFFFFFF / cache->page_size && b->ldt >= b->width, MAMBO_ERR_VALUE,
                  "tables must hold 1 to 2^30 - 1 tokens a sequence (got %lld pages, stride %lld)", (long long)b->width,
                  (long long)b->ldt);
    MAMBO_REQUIRE(b->tables && (b->lengths || tokens == 0), MAMBO_ERR_VALUE, "null pointer");
    *out = {b->tables, b->lengths, b->offsets, b->ldt, (int)b->width, (int)b->seqs, (int)tokens,
            (int)(tokens / b->seqs), (int)(b->width * cache->page_size)};
    return MAMBO_OK;
}

extern "C" int64_t mambo_kv_cache_bytes(int64_t pages, int64_t heads, int64_t head_dim, int64_t page_size)
{
    if (pages < 1 || pages > 0x7FFFFFFF || heads < 1 || heads > 16384 || !kv_dim_ok(head_dim) || page_size < kKvBlock ||
        page_size > 65536 || (page_size & (page_size - 1)) || pages * heads * (page_size / kKvBlock) > 0x7FFFFFFF)
        return 0;
    return pages * heads * page_size * 2 * kv_padded((int)head_dim);
}

extern "C" int mambo_rotary(const void *x, int x_dtype, int64_t tokens, int64_t heads, int64_t dim, int64_t ldt, int64_t ldh,
                            const int32_t *positions, const mambo_rotary_table *table, void *out, int out_dtype,
                            int64_t ldot, int64_t ldoh, mambo_stream_t stream)
{
    MAMBO_REQUIRE(float_rows(x_dtype) && float_rows(out_dtype), MAMBO_ERR_VALUE, "rows must be float32 or bfloat16");
    MAMBO_REQUIRE(tokens >= 0 && tokens <= 0x7FFFFFFF && heads >= 1 && heads <= 65535 && dim >= 2 && dim <= MAMBO_ROTARY_MAX_DIM,
                  MAMBO_ERR_VALUE, "got %lld tokens of %lld heads of %lld values", (long long)tokens, (long long)heads,
                  (long long)dim);
    Rotary a;
    if (const int rc = check_table(table, dim, &a.table))
        return rc;
    if (tokens == 0)
        return MAMBO_OK;
    MAMBO_REQUIRE(positions != nullptr, MAMBO_ERR_VALUE, "null pointer (positions)");
    if (const int rc = check_rows(x, x_dtype, "rows"))
        return rc;
    if (const int rc = check_rows(out, out_dtype, "rotated rows"))
        return rc;
    MAMBO_REQUIRE(ldot >= dim && ldoh >= dim, MAMBO_ERR_VALUE, "strides of the output must cover a head");
    a.x = x, a.out = out, a.ldt = ldt, a.ldh = ldh, a.ldot = ldot, a.ldoh = ldoh, a.positions = positions;
    a.tokens = tokens, a.heads = (int)heads, a.dim = (int)dim;
    // about a thousand workgroups, and eight tokens' angles at most
    a.tile = (int)std::max<int64_t>(1, std::min<int64_t>(8, tokens / 1024));
    a.heads_each = (int)std::min(heads, std::max<int64_t>(cdiv(heads * cdiv(tokens, a.tile), 1024), 4));
    const bool vec = chunks(dim, a.table) && vectors(x, ldt, ldh, x_dtype) && vectors(out, ldot, ldoh, out_dtype);
    const dim3 grid((unsigned)cdiv(tokens, a.tile), (unsigned)cdiv(heads, a.heads_each));
    const size_t lds = (size_t)a.tile * a.table.size * 4;
    hipStream_t s = (hipStream_t)stream;
    const bool in = x_dtype == MAMBO_DTYPE_BF16, to = out_dtype == MAMBO_DTYPE_BF16;
#define MAMBO_ROTARY(IN, OUT, VEC)                                                                                 \
    if (in == IN && to == OUT && vec == VEC)                                                                       \
    MAMBO_LAUNCH((rotary_kernel<IN, OUT, VEC>), grid, dim3(256), lds, s, a)
    MAMBO_ROTARY(true, true, true);
    MAMBO_ROTARY(true, false, true);
    MAMBO_ROTARY(false, true, true);
    MAMBO_ROTARY(false, false, true);
    MAMBO_ROTARY(true, true, false);
    MAMBO_ROTARY(true, false, false);
    MAMBO_ROTARY(false, true, false);
    MAMBO_ROTARY(false, false, false);
#undef MAMBO_ROTARY
    return mambo_check_launch("rotary");
}

extern "C" int mambo_kv_append(const mambo_kv_rows *rows, int64_t tokens, const mambo_kv_cache *cache, const mambo_kv_batch *batch,
                               const mambo_rotary_table *table, const int32_t *positions, mambo_stream_t stream)
{
    MAMBO_REQUIRE(rows != nullptr, MAMBO_ERR_VALUE, "null pointer");
    Append a;
    if (const int rc = kv_check_cache(cache, &a.cache))
        return rc;
    if (const int rc = kv_check_batch(batch, tokens, cache, &a.b))
        return rc;
    MAMBO_REQUIRE(float_rows(rows->dtype), MAMBO_ERR_VALUE, "rows must be float32 or bfloat16");
    const int64_t dim = cache->head_dim, heads = cache->heads;
    a.table = {};
    if (table)
        if (const int rc = check_table(table, dim, &a.table))
            return rc;
    MAMBO_REQUIRE(!rows->q || table, MAMBO_ERR_VALUE, "queries are taken to be rotated: they need a table");
    MAMBO_REQUIRE(!rows->q || (rows->q_heads >= heads && rows->q_heads % heads == 0 && rows->q_heads <= 65535), MAMBO_ERR_VALUE,
                  "%lld query heads are no multiple of %lld", (long long)rows->q_heads, (long long)heads);
    if (tokens == 0)
        return MAMBO_OK;
    if (const int rc = check_rows(rows->k, rows->dtype, "keys"))
        return rc;
    if (const int rc = check_rows(rows->v, rows->dtype, "values"))
        return rc;
    a.k = {rows->k, rows->ldkt, rows->ldkh};
    a.v = {rows->v, rows->ldvt, rows->ldvh};
    a.q = {nullptr, 0, 0};
    a.q_out = nullptr, a.ldot = a.ldoh = 0, a.q_heads = a.q_parts = 0, a.positions = positions;
    bool vec = vectors(rows->k, rows->ldkt, rows->ldkh, rows->dtype) && vectors(rows->v, rows->ldvt, rows->ldvh, rows->dtype);
    if (rows->q) {
        if (const int rc = check_rows(rows->q, rows->dtype, "queries"))
            return rc;
        if (const int rc = check_rows(rows->q_out, MAMBO_DTYPE_BF16, "rotated queries"))
            return rc;
        MAMBO_REQUIRE(rows->ldot >= dim && rows->ldoh >= dim, MAMBO_ERR_VALUE, "strides of the output must cover a head");
        a.q = {rows->q, rows->ldqt, rows->ldqh};
        a.q_out = rows->q_out, a.ldot = rows->ldot, a.ldoh = rows->ldoh, a.q_heads = (int)rows->q_heads;
        // eight tokens each, unless there are no more
        a.q_parts = a.b.offsets || a.b.each > 8 ? 4 : 1;
        vec = vec && chunks(dim, a.table) && vectors(rows->q, rows->ldqt, rows->ldqh, rows->dtype) &&
              vectors(rows->q_out, rows->ldot, rows->ldoh, MAMBO_DTYPE_BF16);
    }
    a.blocks_each = (a.b.each + kKvBlock - 2) / kKvBlock + 1;
    const int64_t slots = a.b.offsets ? tokens / kKvBlock + 2 * batch->seqs : batch->seqs * a.blocks_each;
    MAMBO_REQUIRE(grid_takes(slots, 256), MAMBO_ERR_VALUE, "too many rows for one launch");
    const dim3 grid((unsigned)slots, (unsigned)(heads + a.q_parts));
    const size_t lds = (size_t)kKvBlock * a.table.size * 4;
    hipStream_t s = (hipStream_t)stream;
    const bool bf16 = rows->dtype == MAMBO_DTYPE_BF16;
    const int parts = (int)cdiv(kv_padded((int)dim), 64);
#define MAMBO_APPEND(P, BF16, VEC)                                                                                 \
    if (parts == P && bf16 == BF16 && vec == VEC)                                                                  \
    MAMBO_LAUNCH((append_kernel<P, BF16, VEC>), grid, dim3(256), lds, s, a)
#define MAMBO_APPEND_ALL(P)                                                                                        \
    MAMBO_APPEND(P, true, true);                                                                                   \
    MAMBO_APPEND(P, true, false);                                                                                  \
    MAMBO_APPEND(P, false, true);                                                                                  \
    MAMBO_APPEND(P, false, false)
    MAMBO_APPEND_ALL(1);
    MAMBO_APPEND_ALL(2);
    MAMBO_APPEND_ALL(3);
    MAMBO_APPEND_ALL(4);
#undef MAMBO_APPEND_ALL
#undef MAMBO_APPEND
    return mambo_check_launch("kv_append");
}

extern "C" int mambo_kv_read(const mambo_kv_cache *cache, const mambo_kv_batch *batch, const int32_t *sequences,
                             const int32_t *positions, int64_t n, int64_t heads, int64_t dim, void *k, void *v,
                             mambo_stream_t stream)
{
    KvCache c;
    KvBatch b;
    if (const int rc = kv_check_cache(cache, &c))
        return rc;
    MAMBO_REQUIRE(batch != nullptr, MAMBO_ERR_VALUE, "null pointer");
    mambo_kv_batch tables = *batch;
    tables.offsets = nullptr;
    if (const int rc = kv_check_batch(&tables, 0, cache, &b))
        return rc;
    MAMBO_REQUIRE(heads == c.heads && dim == c.dim, MAMBO_ERR_VALUE, "the cache has %d heads of %d (got %lld of %lld)",
                  c.heads, c.dim, (long long)heads, (long long)dim);
    MAMBO_REQUIRE(n >= 0, MAMBO_ERR_VALUE, "a negative number of tokens");
    if (n == 0)
        return MAMBO_OK;
    MAMBO_REQUIRE(sequences && positions && k && v, MAMBO_ERR_VALUE, "null pointer");
    MAMBO_REQUIRE((uintptr_t)k % 16 == 0 && (uintptr_t)v % 16 == 0, MAMBO_ERR_VALUE, "keys and values must be 16-byte aligned");
    MAMBO_REQUIRE(grid_takes(n / 32 + 1, 256), MAMBO_ERR_VALUE, "too many rows for one launch");
    MAMBO_LAUNCH(read_kernel, dim3((unsigned)cdiv(n, 32), (unsigned)c.heads), dim3(256),
                 (size_t)64 * 16 * (c.dim / 8 + 1), (hipStream_t)stream, c, b,
                 sequences, positions, n, (__bf16 *)k, (__bf16 *)v);
    return mambo_check_launch("kv_read");
}
