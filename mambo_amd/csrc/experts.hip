// The router's plan and the join of the experts' rows.
#include <type_traits>

#include "experts.h"

namespace {

int64_t cdiv(int64_t a, int64_t b) { return (a + b - 1) / b; }

// ============================================================================ router
// One wave per token, V logits a lane (expert 64 v + lane). A logit's key orders as the logit does
// (sign-folded bits, -0 as 0; 0: not to be chosen), so a choice is the largest key and, of equal ones,
// the lowest expert: a maximum over the lanes, a ballot of those that hold it and the lowest index of
// these. Each choice takes its key out. Bound by the lane swaps: six a choice.
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

template <int V, bool kBf16>
__global__ __launch_bounds__(256) void route_choose_kernel(const void *__restrict__ logits, int64_t ld, int64_t m,
                                                           int experts, int top_k, bool renormalize,
                                                           int32_t *__restrict__ ids, float *__restrict__ weights)
{
    const int lane = threadIdx.x & 63;
    const int64_t token = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (token >= m)
        return;
    const row_t<kBf16> *row = reinterpret_cast<const row_t<kBf16> *>(logits) + token * ld;
    uint32_t key[V];
#pragma unroll
    for (int v = 0; v < V; ++v) {
        const int e = 64 * v + lane;
        key[v] = e < experts ? logit_key((float)row[e]) : 0u;
    }
    float max = 0.0f, sum = 0.0f, mine = 0.0f; // lane j keeps choice j
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
        uint32_t top = best;
#pragma unroll
        for (int d = 1; d < 64; d <<= 1)
            top = ::max(top, (uint32_t)__shfl_xor((int)top, d));
        if (top == 0u)
            break;
        int e = best == top ? 64 * at + lane : 0x7FFFFFFF; // a lane's lowest of equal keys
        const uint64_t holders = __ballot(best == top);
        if (holders & (holders - 1)) { // several lanes hold it
#pragma unroll
            for (int d = 1; d < 64; d <<= 1)
                e = min(e, __shfl_xor(e, d));
        } else {
            e = __builtin_amdgcn_readlane(e, __builtin_ctzll(holders));
        }
        if ((e & 63) == lane) {
#pragma unroll
            for (int v = 0; v < V; ++v)
                if (v == e >> 6) {
                    key[v] = 0u;
                }
        }
        const float l = key_logit(top);
        if (j == 0) {
            max = l;
            if (!renormalize) {
                float s = 0.0f;
#pragma unroll
                for (int v = 0; v < V; ++v) // the first choice's key is out already
                    s += key[v] ? softmax_term(key_logit(key[v]), max) : 0.0f;
#pragma unroll
                for (int d = 1; d < 64; d <<= 1)
                    s += __shfl_xor(s, d);
                sum = s + 1.0f;
            }
        }
        const float p = softmax_term(l, max);
        if (renormalize)
            sum += p;
        if (lane == j) {
            mine = p;
            id = e;
        }
    }
    if (lane < top_k) {
        ids[token * top_k + lane] = id;
        weights[token * top_k + lane] = id < 0 ? 0.0f : mine / sum;
    }
}

// Workgroup e counts the choices of lower experts and its own, a stretch of the choices a thread, and
// puts its own down in their order: a sort that keeps the order of tokens, with no counter that
// workgroups share and the same result every time. e == experts: the choices of none. The choices
// are read by every workgroup, out of the caches.
constexpr int kSortThreads = 256;

__global__ __launch_bounds__(kSortThreads) void route_sort_kernel(const int32_t *__restrict__ ids, int count, int top_k,
                                                                  int experts, int32_t *__restrict__ offsets,
                                                                  int32_t *__restrict__ rows, int32_t *__restrict__ slots)
{
    __shared__ int s_less[kSortThreads / 64], s_equal[kSortThreads / 64];
    const int e = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int per = (count + kSortThreads - 1) / kSortThreads;
    const int lo = (int)min<int64_t>((int64_t)tid * per, count), hi = min(lo + per, count);
    int less = 0, equal = 0;
    for (int i = lo; i < hi; ++i) {
        const int id = ids[i] < 0 ? experts : ids[i];
        less += id < e;
        equal += id == e;
    }
    int before = equal; // own choices of the lanes up to this one
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const int up = __shfl_up(before, d);
        before += lane >= d ? up : 0;
        less += __shfl_xor(less, d);
    }
    if (lane == 63) {
        s_equal[wave] = before;
        s_less[wave] = less;
    }
    __syncthreads();
    int at = before - equal, begin = 0;
#pragma unroll
    for (int w = 0; w < kSortThreads / 64; ++w) {
        begin += s_less[w];
        at += w < wave ? s_equal[w] : 0;
    }
    if (tid == 0)
        offsets[e] = begin;
    at += begin;
    for (int i = lo; i < hi; ++i) {
        const int id = ids[i] < 0 ? experts : ids[i];
        if (id == e) {
            rows[at] = e < experts ? i / top_k : -1;
            slots[i] = e < experts ? at : -1;
            ++at;
        }
    }
}

// ============================================================================ join
// A thread adds four columns of a token, choice by choice. Bound by HBM: top_k rows read, one written.
template <bool kYBf16, bool kVec>
__device__ __forceinline__ v4f load_row4(const void *y, int64_t at, int64_t left)
{
    const row_t<kYBf16> *p = reinterpret_cast<const row_t<kYBf16> *>(y) + at;
    if constexpr (kVec) {
        if (left >= 4) {
            if constexpr (kYBf16)
                return __builtin_convertvector(__builtin_nontemporal_load(reinterpret_cast<const bf16x4 *>(p)), v4f);
            else
                return __builtin_nontemporal_load(reinterpret_cast<const v4f *>(p));
        }
    }
    v4f v = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int i = 0; i < 4; ++i)
        if (i < left)
            v[i] = (float)p[i];
    return v;
}

template <bool kYBf16, bool kBf16, bool kVec>
__global__ __launch_bounds__(256) void combine_kernel(const void *__restrict__ y, int64_t ldy, int64_t r,
                                                      const int32_t *__restrict__ slots,
                                                      const float *__restrict__ weights, int64_t m, int top_k, int64_t n,
                                                      void *__restrict__ out, int64_t ldo, bool vec)
{
    const int64_t at = 4 * ((int64_t)blockIdx.x * 256 + threadIdx.x);
    if (at >= n)
        return;
    for (int64_t token = blockIdx.y; token < m; token += gridDim.y) {
        v4f sum = {0.0f, 0.0f, 0.0f, 0.0f};
        for (int j = 0; j < top_k; ++j) {
            const int64_t slot = slots[token * top_k + j];
            if (slot < 0 || slot >= r)
                continue;
            const float w = weights[token * top_k + j];
            const v4f v = load_row4<kYBf16, kVec>(y, slot * ldy + at, n - at);
#pragma unroll
            for (int i = 0; i < 4; ++i)
                sum[i] = __builtin_fmaf(w, v[i], sum[i]);
        }
        store_row4<kBf16>(out, token * ldo + at, sum, n - at, vec);
    }
}

bool float_rows(int dtype) { return dtype == MAMBO_DTYPE_F32 || dtype == MAMBO_DTYPE_BF16; }

template <int V>
void launch_choose(bool bf16, hipStream_t s, const void *logits, int64_t ld, int64_t m, int experts, int top_k,
                   bool renormalize, int32_t *ids, float *weights)
{
    const dim3 grid((unsigned)cdiv(m, 4));
    if (bf16)
        MAMBO_LAUNCH((route_choose_kernel<V, true>), grid, dim3(256), 0, s, logits, ld, m, experts, top_k, renormalize,
                     ids, weights);
    else
        MAMBO_LAUNCH((route_choose_kernel<V, false>), grid, dim3(256), 0, s, logits, ld, m, experts, top_k,
                     renormalize, ids, weights);
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
    if (m > 0) {
        const bool bf16 = dtype == MAMBO_DTYPE_BF16;
#define MAMBO_CHOOSE(V) launch_choose<V>(bf16, s, logits, ld, m, (int)experts, (int)top_k, renormalize != 0, ids, weights)
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
        if (rc != MAMBO_OK)
            return rc;
    }
    MAMBO_LAUNCH(route_sort_kernel, dim3((unsigned)(experts + 1)), dim3(kSortThreads), 0, s, ids, (int)(m * top_k),
                 (int)top_k, (int)experts, offsets, rows, slots);
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
    const int64_t columns = cdiv(n, 4 * 256);
    MAMBO_REQUIRE(columns <= 0x7FFFFFFF, MAMBO_ERR_VALUE, "rows too long");
    const dim3 grid((unsigned)columns, (unsigned)(m < 65535 ? m : 65535));
    const bool in_vec = rows_take_vectors(y, ldy, y_dtype), out_vec = rows_take_vectors(out, ldo, out_dtype);
    hipStream_t s = (hipStream_t)stream;
#define MAMBO_COMBINE(YB, OB, V)                                                                                   \
    if (yb == YB && ob == OB && in_vec == V)                                                                       \
    MAMBO_LAUNCH((combine_kernel<YB, OB, V>), grid, dim3(256), 0, s, y, ldy, r, slots, weights, m, (int)top_k, n, out, \
                 ldo, out_vec)
    MAMBO_COMBINE(true, true, true);
    MAMBO_COMBINE(true, true, false);
    MAMBO_COMBINE(true, false, true);
    MAMBO_COMBINE(true, false, false);
    MAMBO_COMBINE(false, true, true);
    MAMBO_COMBINE(false, true, false);
    MAMBO_COMBINE(false, false, true);
    MAMBO_COMBINE(false, false, false);
#undef MAMBO_COMBINE
    return mambo_check_launch("combine_experts");
}
