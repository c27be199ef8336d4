// The router's plan and the join of the experts' rows.
#include <algorithm>
#include <type_traits>

#include "experts.h"

namespace {

int64_t cdiv(int64_t a, int64_t b) { return (a + b - 1) / b; }

// ============================================================================ router
// One wave per token, V logits a lane (experts V * lane .. + V - 1). A logit's key orders as the logit
// does (sign-folded bits, -0 as 0; 0: not to be chosen), so a choice is the largest key and, of equal
// ones, the lowest expert: a maximum over the lanes, the lowest lane that holds it and that lane's first.
// Each choice takes its key out; the softmax is taken of the choices at the end, one a lane. Bound by the
// vector instructions of a choice (about 20 + 5 V).
__device__ __forceinline__ uint32_t logit_key(float l)
{
    if (!(l > -__builtin_inff())) // -inf and NaN
        return 0u;
    const uint32_t u = __float_as_uint(l == 0.0f ? 0.0f : l);
    return (u >> 31) ? ~u : u | 0x80000000u;
}

__device__ __forceinline__ float key_logit(uint32_t key)
{
    return __uint_as_float((key >> 31) ? key & 0x7FFFFFFFu : ~key);
}

// exp(l - max), with 1 where both are infinite
__device__ __forceinline__ float softmax_term(float l, float max) { return l == max ? 1.0f : expf(l - max); }

// Maximum over the wave's lanes by DPP moves: pairs, fours, halves and whole rows of 16, then across rows.
template <int kCtrl>
__device__ __forceinline__ uint32_t max_dpp(uint32_t v)
{
    return ::max(v, (uint32_t)__builtin_amdgcn_update_dpp((int)v, (int)v, kCtrl, 0xF, 0xF, false));
}
__device__ __forceinline__ uint32_t wave_max(uint32_t v)
{
    v = max_dpp<0xB1>(v);  // quad_perm 1 0 3 2
    v = max_dpp<0x4E>(v);  // quad_perm 2 3 0 1
    v = max_dpp<0x141>(v); // row_half_mirror
    v = max_dpp<0x140>(v); // row_mirror
    const uint32_t a = ::max((uint32_t)__builtin_amdgcn_readlane((int)v, 0), (uint32_t)__builtin_amdgcn_readlane((int)v, 16));
    const uint32_t b = ::max((uint32_t)__builtin_amdgcn_readlane((int)v, 32), (uint32_t)__builtin_amdgcn_readlane((int)v, 48));
    return ::max(a, b);
}

// Sum over the wave's lanes.
__device__ __forceinline__ float wave_sum(float v)
{
#pragma unroll
    for (int d = 1; d < 64; d <<= 1)
        v += __shfl_xor(v, d);
    return v;
}

// The choices of one token by one wave: lane j < top_k gets choice j.
template <int V, bool kBf16>
__device__ __forceinline__ void choose(const void *logits, int64_t ld, int64_t token, int experts, int top_k,
                                       bool renormalize, int lane, int *id_out, float *weight_out)
{
    const row_t<kBf16> *row = reinterpret_cast<const row_t<kBf16> *>(logits) + token * ld;
    uint32_t key[V];
#pragma unroll
    for (int v = 0; v < V; ++v) {
        const int e = V * lane + v;
        key[v] = e < experts ? logit_key((float)row[e]) : 0u;
    }
    float all = 0.0f; // softmax terms of all experts
    uint32_t mine = 0u, first = 0u;
    int id = -1;
    for (int j = 0; j < top_k; ++j) {
        uint32_t best = key[0];
        int at = 0;
#pragma unroll
        for (int v = 1; v < V; ++v)
            if (key[v] > best) {
                best = key[v];
                at = v;
            }
        const uint32_t top = wave_max(best);
        if (top == 0u)
            break;
        if (j == 0) {
            first = top;
            if (!renormalize) {
                float t = 0.0f;
#pragma unroll
                for (int v = 0; v < V; ++v)
                    t += key[v] ? softmax_term(key_logit(key[v]), key_logit(top)) : 0.0f;
                all = wave_sum(t);
            }
        }
        const int holder = __builtin_ctzll(__ballot(best == top));
        const int slot = V == 1 ? 0 : __builtin_amdgcn_readlane(at, holder);
        if (lane == holder)
#pragma unroll
            for (int v = 0; v < V; ++v)
                if (v == slot)
                    key[v] = 0u;
        if (lane == j) {
            mine = top;
            id = V * holder + slot;
        }
    }
    const float term = id < 0 ? 0.0f : softmax_term(key_logit(mine), key_logit(first));
    if (renormalize)
        all = wave_sum(term);
    *id_out = id;
    *weight_out = id < 0 ? 0.0f : term / all;
}

template <int V, bool kBf16>
__global__ __launch_bounds__(256) void route_choose_kernel(const void *__restrict__ logits, int64_t ld, int64_t m,
                                                           int experts, int top_k, bool renormalize,
                                                           int32_t *__restrict__ ids, float *__restrict__ weights)
{
    const int lane = threadIdx.x & 63;
    const int64_t token = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (token >= m)
        return;
    int id;
    float weight;
    choose<V, kBf16>(logits, ld, token, experts, top_k, renormalize, lane, &id, &weight);
    if (lane < top_k) {
        ids[token * top_k + lane] = id;
        weights[token * top_k + lane] = weight;
    }
}

// c / top_k for choices c < 2^31 as c f >> 31 + s, with 2^s >= top_k and f = 2^(31 + s) / top_k rounded up: f top_k is less
// than top_k <= 2^s above 2^(31 + s), so c f / 2^(31 + s) is less than c / 2^31 / top_k < 1 / top_k above c / top_k. (The
// division took a third of the sort where an expert has many choices: 8192 x 8 of 64 experts, the call 24.6 -> 21.3 us.)
struct TokenOf {
    uint32_t factor;
    int shift;
};

inline TokenOf token_of(int64_t top_k)
{
    int s = 0;
    while ((int64_t)1 << s < top_k)
        ++s;
    return {(uint32_t)((((int64_t)1 << (31 + s)) + top_k - 1) / top_k), 31 + s};
}

// Workgroup e counts the choices of lower experts and its own, a stretch of the choices a wave, and puts
// its own down in their order: a sort that keeps the order of tokens, with no counter that workgroups share
// and the same result every time. e == experts: the choices of none, -1, which is after them all as an
// unsigned number. Every workgroup reads all choices, out of the caches, two vector instructions for 64 of
// them (65536 choices of 256 experts, 67 MB: 12.4 us; as 256 lanes with a stretch each 118).
constexpr int kSortWaves = 16;
constexpr int kSortLoads = 8; // of 64 choices each, in flight

__global__ __launch_bounds__(kSortWaves * 64) void route_sort_kernel(const uint32_t *__restrict__ ids, int count,
                                                                     TokenOf token_of, int experts, int32_t *__restrict__ offsets,
                                                                     int32_t *__restrict__ rows,
                                                                     int32_t *__restrict__ slots)
{
    __shared__ int s_less[kSortWaves], s_equal[kSortWaves];
    const int e = blockIdx.x, tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const uint32_t own = e < experts ? (uint32_t)e : 0xFFFFFFFFu;
    const int per = (int)(((int64_t)count + 64 * kSortWaves - 1) / (64 * kSortWaves)) * 64;
    const int lo = (int)min<int64_t>((int64_t)wave * per, count), hi = (int)min<int64_t>((int64_t)lo + per, count);
    // eight times 64 choices from i on; `last`: those past the stretch are of no expert, and not -1
    auto load = [&](uint32_t(&id)[kSortLoads], int i, bool last) {
#pragma unroll
        for (int j = 0; j < kSortLoads; ++j)
            id[j] = !last || 64 * j + lane < hi - i ? ids[i + 64 * j + lane] : 0xFFFFFFFEu;
    };
    constexpr int kStep = 64 * kSortLoads;
    int less = 0, equal = 0;
    auto tally = [&](int i, bool last) {
        uint32_t id[kSortLoads];
        load(id, i, last);
#pragma unroll
        for (int j = 0; j < kSortLoads; ++j) {
            less += __popcll(__ballot(id[j] < (uint32_t)e));
            equal += __popcll(__ballot(id[j] == own));
        }
    };
    int i = lo;
    for (; hi - i >= kStep; i += kStep) // (a sum would pass 2^31 in the last stretch of as many choices)
        tally(i, false);
    if (i < hi)
        tally(i, true);
    if (lane == 0) {
        s_less[wave] = less;
        s_equal[wave] = equal;
    }
    __syncthreads();
    int at = 0, begin = 0;
#pragma unroll
    for (int w = 0; w < kSortWaves; ++w) {
        begin += s_less[w];
        at += w < wave ? s_equal[w] : 0;
    }
    if (tid == 0)
        offsets[e] = begin;
    if (equal == 0)
        return;
    at += begin;
    const uint64_t lower = ((uint64_t)1 << lane) - 1;
    auto place = [&](int i, bool last) {
        uint32_t id[kSortLoads];
        load(id, i, last);
#pragma unroll
        for (int j = 0; j < kSortLoads; ++j) {
            const uint64_t here = __ballot(id[j] == own);
            if (here == 0)
                continue;
            if (id[j] == own) {
                const int slot = at + __popcll(here & lower), c = i + 64 * j + lane;
                rows[slot] = e < experts ? (int)((uint64_t)(uint32_t)c * token_of.factor >> token_of.shift) : -1;
                slots[c] = e < experts ? slot : -1;
            }
            at += __popcll(here);
        }
    };
    for (i = lo; hi - i >= kStep; i += kStep)
        place(i, false);
    if (i < hi)
        place(i, true);
}

// Few choices: both steps by one workgroup. A choice sets its bit among those of its expert, 64 choices a word, in
// LDS (whatever order the bits come in, the words are the same); an expert's count is the bits set, a scan of
// the counts the offsets, and a choice's row the offset and the lower bits set. One launch instead of two, the
// second of which costs more than this (16 tokens x 8 of 64 experts: 5.4 us, against 3.1 and 6.7).
constexpr int kFewChoices = 1024, kFewTokens = 64, kFewWords = 4096;

template <int V, bool kBf16>
__global__ __launch_bounds__(1024) void route_few_kernel(const void *__restrict__ logits, int64_t ld, int m, int experts,
                                                         int top_k, bool renormalize, int32_t *__restrict__ ids,
                                                         float *__restrict__ weights, int32_t *__restrict__ offsets,
                                                         int32_t *__restrict__ rows, int32_t *__restrict__ slots)
{
    __shared__ unsigned long long s_bits[kFewWords]; // [expert, the last one none][words]
    __shared__ int s_ids[kFewChoices], s_wave[16], s_begin[1025];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, count = m * top_k, words = (count + 63) / 64;
    for (int i = tid; i < (experts + 1) * words; i += 1024)
        s_bits[i] = 0;
    __syncthreads();
    for (int token = wave; token < m; token += 16) {
        int id;
        float weight;
        choose<V, kBf16>(logits, ld, token, experts, top_k, renormalize, lane, &id, &weight);
        if (lane < top_k) {
            const int c = token * top_k + lane, e = id < 0 ? experts : id;
            ids[c] = id;
            weights[c] = weight;
            s_ids[c] = e;
            atomicOr(&s_bits[e * words + (c >> 6)], 1ull << (c & 63));
        }
    }
    __syncthreads();
    int mine = 0;
    if (tid < experts)
        for (int w = 0; w < words; ++w)
            mine += __popcll(s_bits[tid * words + w]);
    int upto = mine; // of the wave's experts up to this one
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const int up = __shfl_up(upto, d);
        upto += lane >= d ? up : 0;
    }
    if (lane == 63)
        s_wave[wave] = upto;
    __syncthreads();
    int begin = upto - mine;
    for (int w = 0; w < wave; ++w)
        begin += s_wave[w];
    if (tid < experts) {
        offsets[tid] = begin;
        s_begin[tid] = begin;
        if (tid == experts - 1) {
            offsets[experts] = begin + mine;
            s_begin[experts] = begin + mine;
        }
    }
    __syncthreads();
    if (tid < count) {
        const int e = s_ids[tid];
        int row = s_begin[e] + __popcll(s_bits[e * words + (tid >> 6)] & ((1ull << (tid & 63)) - 1));
        for (int w = 0; w < tid >> 6; ++w)
            row += __popcll(s_bits[e * words + w]);
        rows[row] = e < experts ? tid / top_k : -1;
        slots[tid] = e < experts ? row : -1;
    }
}

// ============================================================================ join
// A thread adds 16 bytes' worth of columns of a token, the rows of four choices in flight, in the order of the choices.
// Bound by HBM: top_k rows read, one written (8192 tokens x 8 rows of 4096 bf16, 605 MB: 98 us).
template <bool kBf16, int N>
__device__ __forceinline__ void load_columns(const void *y, int64_t at, int64_t left, bool vec, float (&v)[N])
{
    const row_t<kBf16> *p = reinterpret_cast<const row_t<kBf16> *>(y) + at;
    if (vec && left >= N) {
        typedef row_t<kBf16> row16 __attribute__((ext_vector_type(kBf16 ? 8 : 4)));
#pragma unroll
        for (int i = 0; i < N; i += kBf16 ? 8 : 4) {
            const row16 r = __builtin_nontemporal_load(reinterpret_cast<const row16 *>(p + i));
#pragma unroll
            for (int j = 0; j < (kBf16 ? 8 : 4); ++j)
                v[i + j] = (float)r[j];
        }
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i)
            v[i] = i < left ? (float)p[i] : 0.0f;
    }
}

template <bool kYBf16, bool kBf16>
__global__ __launch_bounds__(256) void combine_kernel(const void *__restrict__ y, int64_t ldy, int64_t r,
                                                      const int32_t *__restrict__ slots,
                                                      const float *__restrict__ weights, int64_t m, int top_k, int64_t n,
                                                      void *__restrict__ out, int64_t ldo, bool in_vec, bool out_vec)
{
    constexpr int N = kYBf16 ? 8 : 4;
    const int64_t at = N * ((int64_t)blockIdx.x * blockDim.x + threadIdx.x);
    if (at >= n)
        return;
    for (int64_t token = blockIdx.y; token < m; token += gridDim.y) {
        float sum[N] = {};
        for (int j0 = 0; j0 < top_k; j0 += 4) {
            float v[4][N], w[4];
            bool some[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int64_t c = token * top_k + min(j0 + j, top_k - 1);
                const int64_t slot = slots[c];
                some[j] = j0 + j < top_k && slot >= 0 && slot < r;
                w[j] = weights[c];
                if (some[j])
                    load_columns<kYBf16, N>(y, slot * ldy + at, n - at, in_vec, v[j]);
            }
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (some[j])
#pragma unroll
                    for (int i = 0; i < N; ++i)
                        sum[i] = __builtin_fmaf(w[j], v[j][i], sum[i]);
        }
#pragma unroll
        for (int i = 0; i < N; i += 4)
            store_row4<kBf16>(out, token * ldo + at + i, v4f{sum[i], sum[i + 1], sum[i + 2], sum[i + 3]}, n - at - i, out_vec);
    }
}

bool float_rows(int dtype) { return dtype == MAMBO_DTYPE_F32 || dtype == MAMBO_DTYPE_BF16; }

struct Route {
    const void *logits;
    int64_t ld, m;
    int experts, top_k;
    bool renormalize;
    int32_t *ids;
    float *weights;
    int32_t *offsets, *rows, *slots;
};

// Tokens of a launch: four a workgroup, as many as a grid takes.
constexpr int64_t kChooseTokens = 4 * (kMaxGridThreads / 256);

template <int V, bool kBf16>
void launch_choose(const Route &a, bool few, hipStream_t s)
{
    if (few)
        MAMBO_LAUNCH((route_few_kernel<V, kBf16>), dim3(1), dim3(1024), 0, s, a.logits, a.ld, (int)a.m, a.experts, a.top_k,
                     a.renormalize, a.ids, a.weights, a.offsets, a.rows, a.slots);
    else
        for (int64_t t = 0; t < a.m; t += kChooseTokens)
            MAMBO_LAUNCH((route_choose_kernel<V, kBf16>), dim3((unsigned)cdiv(std::min(kChooseTokens, a.m - t), 4)), dim3(256), 0,
                         s, reinterpret_cast<const row_t<kBf16> *>(a.logits) + t * a.ld, a.ld, std::min(kChooseTokens, a.m - t),
                         a.experts, a.top_k, a.renormalize, a.ids + t * a.top_k, a.weights + t * a.top_k);
}

} // namespace

extern "C" int mambo_route_experts(const void *logits, int dtype, int64_t ld, int64_t m, int64_t experts, int64_t top_k,
                                   int renormalize, int32_t *ids, float *weights, int32_t *offsets, int32_t *rows,
                                   int32_t *slots, mambo_stream_t stream)
{
    MAMBO_REQUIRE(float_rows(dtype), MAMBO_ERR_VALUE, "logits must be float32 or bfloat16");
    MAMBO_REQUIRE(experts >= 1 && experts <= MAMBO_MAX_EXPERTS, MAMBO_ERR_VALUE,
                  "experts must be in [1, %d] (got %lld)", MAMBO_MAX_EXPERTS, (long long)experts);
    MAMBO_REQUIRE(top_k >= 1 && top_k <= experts && top_k <= MAMBO_MAX_TOP_K, MAMBO_ERR_VALUE,
                  "top_k must be in [1, min(experts, %d)] (got %lld)", MAMBO_MAX_TOP_K, (long long)top_k);
    MAMBO_REQUIRE(m >= 0 && m * top_k <= 0x7FFFFFFF && m <= 0x7FFFFFFF, MAMBO_ERR_VALUE,
                  "tokens times top_k must be below 2^31 (got %lld tokens)", (long long)m);
    MAMBO_REQUIRE(ld >= experts, MAMBO_ERR_VALUE, "row strides must cover the experts");
    MAMBO_REQUIRE(offsets && (m == 0 || (logits && ids && weights && rows && slots)), MAMBO_ERR_VALUE, "null pointer");
    hipStream_t s = (hipStream_t)stream;
    // one workgroup for both steps while every wave of it has at most four tokens and the bits fit its LDS
    const bool few = m > 0 && m <= kFewTokens && m * top_k <= kFewChoices && (experts + 1) * cdiv(m * top_k, 64) <= kFewWords;
    if (m > 0) {
        const Route a = {logits, ld, m, (int)experts, (int)top_k, renormalize != 0, ids, weights, offsets, rows, slots};
        const bool bf16 = dtype == MAMBO_DTYPE_BF16;
#define MAMBO_CHOOSE(V) (bf16 ? launch_choose<V, true>(a, few, s) : launch_choose<V, false>(a, few, s))
        if (experts <= 64)
            MAMBO_CHOOSE(1);
        else if (experts <= 128)
            MAMBO_CHOOSE(2);
        else if (experts <= 256)
            MAMBO_CHOOSE(4);
        else if (experts <= 512)
            MAMBO_CHOOSE(8);
        else
            MAMBO_CHOOSE(16);
#undef MAMBO_CHOOSE
        const int rc = mambo_check_launch("route_experts");
        if (rc != MAMBO_OK || few)
            return rc;
    }
    MAMBO_LAUNCH(route_sort_kernel, dim3((unsigned)(experts + 1)), dim3(kSortWaves * 64), 0, s, (const uint32_t *)ids, (int)(m * top_k),
                 token_of(top_k), (int)experts, offsets, rows, slots);
    return mambo_check_launch("route_experts");
}

extern "C" int mambo_combine_experts(const void *y, int y_dtype, int64_t ldy, int64_t r, const int32_t *slots,
                                     const float *weights, int64_t m, int64_t top_k, int64_t n, void *out, int out_dtype,
                                     int64_t ldo, mambo_stream_t stream)
{
    MAMBO_REQUIRE(float_rows(y_dtype) && float_rows(out_dtype), MAMBO_ERR_VALUE, "rows must be float32 or bfloat16");
    MAMBO_REQUIRE(m >= 0 && r >= 0 && n >= 1 && top_k >= 1 && top_k <= MAMBO_MAX_TOP_K, MAMBO_ERR_VALUE,
                  "got %lld tokens of %lld choices, %lld rows of %lld", (long long)m, (long long)top_k, (long long)r,
                  (long long)n);
    MAMBO_REQUIRE(ldy >= n && ldo >= n, MAMBO_ERR_VALUE, "row strides must cover the rows");
    if (m == 0)
        return MAMBO_OK;
    MAMBO_REQUIRE((y || r == 0) && slots && weights && out, MAMBO_ERR_VALUE, "null pointer");
    const bool yb = y_dtype == MAMBO_DTYPE_BF16, ob = out_dtype == MAMBO_DTYPE_BF16;
    MAMBO_REQUIRE((uintptr_t)y % (yb ? 2 : 4) == 0 && (uintptr_t)out % (ob ? 2 : 4) == 0, MAMBO_ERR_VALUE,
                  "rows must be aligned to their type");
    const int threads = n <= (yb ? 512 : 256) ? 64 : 256;
    const int64_t columns = cdiv(n, (yb ? 8 : 4) * threads);
    MAMBO_REQUIRE(grid_takes(columns, threads), MAMBO_ERR_VALUE, "rows too long");
    const dim3 grid((unsigned)columns, (unsigned)(m < 65535 ? m : 65535));
    const bool in_vec = rows_take_vectors(y, ldy, y_dtype), out_vec = rows_take_vectors(out, ldo, out_dtype);
    hipStream_t s = (hipStream_t)stream;
#define MAMBO_COMBINE(YB, OB)                                                                                      \
    if (yb == YB && ob == OB)                                                                                      \
    MAMBO_LAUNCH((combine_kernel<YB, OB>), grid, dim3(threads), 0, s, y, ldy, r, slots, weights, m, (int)top_k, n, out,  \
                 ldo, in_vec, out_vec)
    MAMBO_COMBINE(true, true);
    MAMBO_COMBINE(true, false);
    MAMBO_COMBINE(false, true);
    MAMBO_COMBINE(false, false);
#undef MAMBO_COMBINE
    return mambo_check_launch("combine_experts");
}
