// What several workgroups found of a row's keys, put together: of both attention kernels in one launch.
#include "attention.h"

namespace {

// The sum of a row's partial results, weighted by their largest scores; rows of sequences without keys become
// zeros. A workgroup a row: DP / 4 threads side by side, the parts dealt to 256 / (DP / 4) such groups, which
// are added in order.
template <int DS>
__device__ void join_rows(const Attention &a, int tile_rows, int row_count, int at)
{
    constexpr int DP = 32 * DS, kWide = DP / 4, kGroups = 256 / kWide;
    __shared__ v4f so[kGroups][kWide];
    __shared__ float sm[kGroups], sl[kGroups];
    const int row = at % row_count, pair = at / row_count, s = pair / a.cache.heads, head = pair % a.cache.heads;
    const int tid = (int)threadIdx.x, g = tid / kWide, d = 4 * (tid % kWide);
    const Sequence seq = sequence(a, s);
    if (seq.n <= 0 || seq.n > a.few_rows / a.group || row >= seq.n * a.group)
        return;
    const int blocks = seq.hi - seq.lo, total = a.begins[a.b.seqs], begin = a.begins[s];
    const int i = row / a.group, h = head * a.group + row % a.group;
    const int64_t t = seq.first + i;
    int p0 = 0, p1 = -1;
    if (blocks > 0) {
        const int count = shares(a, total);
        p0 = share_of(begin, total, count);
        p1 = share_of(begin + blocks - 1, total, count);
        if (p0 == p1)
            return; // written by the one that had all of it
    }
    float m = -__builtin_inff(), l = 0.0f;
    v4f o = {0.0f, 0.0f, 0.0f, 0.0f};
    if (g < kGroups) {
        for (int p = p0 + g; p <= p1; p += 4 * kGroups) { // four at a time on their way
            float2 ml[4];
            v4f x[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const int part = min(p + k * kGroups, p1);
                const int64_t entry = (((int64_t)head * a.slots + part) * 2 + (part == p0)) * tile_rows + row;
                ml[k] = *reinterpret_cast<const float2 *>(a.rows_ml + entry * 2);
                x[k] = *reinterpret_cast<const v4f *>(a.rows_o + entry * DP + d);
            }
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                if (p + k * kGroups > p1)
                    continue;
                const float top = fmaxf(m, ml[k].x), less = top == -__builtin_inff() ? 0.0f : top;
                const float f = exp2_fast(m - less), e = exp2_fast(ml[k].x - less);
                o = o * f + x[k] * e;
                l = l * f + ml[k].y * e;
                m = top;
            }
        }
        so[g][tid % kWide] = o;
        if (tid % kWide == 0) {
            sm[g] = m;
            sl[g] = l;
        }
    }
    __syncthreads();
    if (g > 0)
        return;
    m = sm[0];
#pragma unroll
    for (int k = 1; k < kGroups; ++k)
        m = fmaxf(m, sm[k]);
    const float less = m == -__builtin_inff() ? 0.0f : m;
    o = v4f{0.0f, 0.0f, 0.0f, 0.0f};
    l = 0.0f;
#pragma unroll
    for (int k = 0; k < kGroups; ++k) {
        const float f = exp2_fast(sm[k] - less);
        o += so[k][tid] * f;
        l += sl[k] * f;
    }
    store_row(a, t, h, d, o, m, l);
}

// Rows whose keys were dealt to several workgroups: their sums weighted by the largest scores, in order.
template <int DS>
__device__ void join_tiles(const Attention &a, int at)
{
    constexpr int DP = 32 * DS, kWide = DP / 4, kRows = join_tile_rows(DS);
    const int64_t q_heads = (int64_t)a.group * a.cache.heads, all = a.b.tokens * q_heads;
    const int64_t entry = (int64_t)at * kRows + (int)threadIdx.x / kWide;
    const int d = 4 * ((int)threadIdx.x % kWide);
    const int64_t t = min(entry, all - 1) / q_heads, h = min(entry, all - 1) % q_heads;
    int s = a.b.offsets ? 0 : (int)t / a.b.each;
    if (a.b.offsets) {
        // the last sequence that begins at or before the wave's first token, and from there on this thread's
        s = find_slot(a.b.seqs, __builtin_amdgcn_readfirstlane((int)t), [&](int i) { return (int64_t)a.b.offset(i); });
        while (s + 1 < a.b.seqs && a.b.offset(s + 1) <= t)
            ++s;
    }
    const Sequence seq = sequence(a, s);
    if ((int)threadIdx.x >= kRows * kWide || entry >= all || t < seq.first || t >= seq.first + seq.n ||
        (int64_t)seq.n * a.group <= a.few_rows)
        return; // rows of sequences that attend_tiles has, and no others
    const int row = ((int)t - seq.first) * a.group + (int)h % a.group;
    const int parts = tile_keys(a, seq, row / tile_rows(DS) * tile_rows(DS), tile_rows(DS)).parts;
    if (parts == 1)
        return; // written by the one that had all of them
    float m = -__builtin_inff(), l = 0.0f;
    v4f o = {0.0f, 0.0f, 0.0f, 0.0f};
    for (int p = 0; p < parts; ++p) {
        const float2 ml = *reinterpret_cast<const float2 *>(a.tiles_ml + (p * all + entry) * 2);
        const v4f x = *reinterpret_cast<const v4f *>(a.tiles_o + (p * all + entry) * DP + d);
        const float top = fmaxf(m, ml.x), less = top == -__builtin_inff() ? 0.0f : top;
        const float f = exp2_fast(m - less), e = exp2_fast(ml.x - less);
        o = o * f + x * e;
        l = l * f + ml.y * e;
        m = top;
    }
    store_row(a, t, (int)h, d, o, m, l);
}

// Workgroups below `rows_from` join the rows of attend_tiles, the others those of attend_rows.
template <int DS>
__global__ __launch_bounds__(256) void attend_join_kernel(const Attention a, int rows_from, int tile_rows, int row_count)
{
    const int at = (int)blockIdx.x;
    if (at < rows_from)
        join_tiles<DS>(a, at);
    else
        join_rows<DS>(a, tile_rows, row_count, at - rows_from);
}

template <int DS>
void launch_join(const Attention &a, int row_tiles, const Join &join, hipStream_t s)
{
    MAMBO_LAUNCH((attend_join_kernel<DS>), dim3((unsigned)(join.tiles + join.rows)), dim3(256), 0, s, a, (int)join.tiles,
                 16 * row_tiles, join.row_count);
}

} // namespace

int launch_attend_join(const Attention &a, int row_tiles, const Join &join, hipStream_t s)
{
    switch (kv_padded(a.cache.dim) / 32) {
    case 1: launch_join<1>(a, row_tiles, join, s); break;
    case 2: launch_join<2>(a, row_tiles, join, s); break;
    case 3: launch_join<3>(a, row_tiles, join, s); break;
    case 4: launch_join<4>(a, row_tiles, join, s); break;
    case 5: launch_join<5>(a, row_tiles, join, s); break;
    case 6: launch_join<6>(a, row_tiles, join, s); break;
    case 7: launch_join<7>(a, row_tiles, join, s); break;
    default: launch_join<8>(a, row_tiles, join, s); break;
    }
    return mambo_check_launch("kv_attention");
}
