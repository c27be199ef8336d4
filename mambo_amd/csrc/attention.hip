// Attention over the paged 8-bit cache: which kernels a call takes, its workspace, and the entry points.
#include <algorithm>
#include <math.h>

#include "attention.h"

namespace {

int64_t cdiv(int64_t a, int64_t b) { return (a + b - 1) / b; }

struct Plan {
    int few_rows = 0, row_tiles = 0, slots = 0; // the kernel for few rows, 0: not launched
    int64_t tiles = 0;                          // the kernel for many, tiles of a head; 0: not launched
    int tiles_each = 1, parts = 1;
    int64_t rows_entries = 0, tiles_entries = 0, bytes = 0;
    Join join;
};

constexpr int kCus = 256;
// Keys of a sequence up to which one workgroup takes all of them. One user of 8 heads of 128, from a graph: 1000 tokens
// 9.7 us for 8.6 by two launches, whose second costs the host 3 us more, 2000 14.5 for 8.9; 32 users (a workgroup a CU)
// 1000 16.7 for 21.3, 2000 25.7 for 30.4.
constexpr int64_t kShortTokens = 1280, kShortTokensOfMany = 2048;
// Sequences from which the kernel for many rows takes those of 33 to 64 rows that no single workgroup takes: the shares of the
// other then end sequences too often. 36 rows of 8 heads of 64, by it and by the other: 32 x 2000 tokens 36.5 us for 52.3,
// 8 x 4000 25.0 for 30.7, 4 x 8000 26.4 for 28.7, 2 x 16000 29.1 for 27.9, 30000 32.8 for 27.3.
constexpr int kSeqsOfTiles = 4;

int64_t aligned(int64_t bytes) { return (bytes + 15) & ~(int64_t)15; }

Plan make_plan(const KvCache &c, const KvBatch &b, int group, int64_t window)
{
    Plan p;
    const int padded = kv_padded(c.dim);
    const int most = 16 * max_row_tiles(padded);
    const int64_t rows = (int64_t)(b.offsets ? b.tokens : b.each) * group; // of one sequence, at most
    const auto tiles_for = [](int64_t r) { return r <= 16 ? 1 : r <= 32 ? 2 : 4; };
    if (rows <= most)
        p.row_tiles = tiles_for(rows);
    else if (b.offsets && group <= most) // prompts and single tokens in one call: each has its kernel
        p.row_tiles = tiles_for(group);
    if (p.row_tiles) {
        p.few_rows = 16 * p.row_tiles;
        // blocks of a sequence at most; few enough, and one workgroup takes all of them
        int64_t seen = b.capacity;
        if (window)
            seen = std::min<int64_t>(seen, std::min(window, seen) + p.few_rows / group + kKvBlock);
        const int size = padded / 32 * p.row_tiles;
        const int64_t short_seen = (int64_t)b.seqs * c.heads >= kCus ? kShortTokensOfMany : kShortTokens;
        const bool short_ones = short_fits(padded / 32, p.row_tiles) && seen <= short_seen;
        if (!short_ones && p.row_tiles > 2 && !b.offsets && b.seqs >= kSeqsOfTiles) {
            p.row_tiles = p.few_rows = 0;
        } else if (!short_ones) {
            // A workgroup a CU, fewer where there is no work for them: the blocks that its waves have on their way are enough
            // (131149 tokens of 8 heads of 128 47.0 us, with two 49.6). Two of small heads (16 x 8000 of 8 heads of 64 28.7 us
            // for 35.4), and where a workgroup comes to the ends of several sequences, at which the other goes on (of 8 heads of
            // 128 64 sequences of up to 8192 109 us for 113, 32 of 4000 49.5 for 44.4).
            const int64_t blocks = (int64_t)b.seqs * (b.capacity / kKvBlock);
            const int per_cu = size <= 2 || (size <= 4 && (int64_t)b.seqs * c.heads >= 2 * kCus) ? 2 : 1;
            p.slots = (int)std::max<int64_t>(1, std::min<int64_t>(per_cu * kCus / c.heads, cdiv(blocks, 4)));
            p.rows_entries = (int64_t)c.heads * p.slots * 2 * p.few_rows;
            p.join.row_count = b.offsets ? p.few_rows : (int)rows;
            p.join.rows = (int64_t)b.seqs * c.heads * p.join.row_count;
        }
    }
    if (rows > most || !p.row_tiles) {
        const int tile = tile_rows(padded / 32);
        p.tiles_each = (int)cdiv(rows, tile);
        p.tiles = b.offsets ? (int64_t)b.tokens * group / tile + b.seqs : (int64_t)b.seqs * p.tiles_each;
        // A workgroup a CU, two of ragged sequences: the longest then have more parts than the others (pieces of six prompts 37 us
        // for 41; of sequences with as many rows each, 4 of 16 tokens of 32/8 heads of 128 behind 20000, 66 for 58).
        const int64_t places = (b.offsets ? 2 : 1) * kCus / (p.tiles * c.heads);
        p.parts = (int)std::max<int64_t>(1, std::min<int64_t>(places, cdiv(b.capacity, 512)));
        if (p.parts > 1) {
            const int64_t entries = (int64_t)b.tokens * group * c.heads;
            p.tiles_entries = p.parts * entries;
            p.join.tiles = cdiv(entries, join_tile_rows(padded / 32));
        }
    }
    p.bytes = aligned(p.rows_entries * (padded + 2) * 4) + aligned(p.slots ? ((int64_t)b.seqs + 1) * 4 : 0) +
              aligned(p.tiles_entries * (padded + 2) * 4);
    return p;
}

int check(const mambo_kv_cache *cache, const mambo_kv_batch *batch, int64_t tokens, int64_t q_heads, int64_t window,
          KvCache *c, KvBatch *b, Plan *p)
{
    if (const int rc = kv_check_cache(cache, c))
        return rc;
    if (const int rc = kv_check_batch(batch, tokens, cache, b))
        return rc;
    MAMBO_REQUIRE(q_heads >= c->heads && q_heads % c->heads == 0 && q_heads <= 65535, MAMBO_ERR_VALUE,
                  "%lld query heads are no multiple of %d", (long long)q_heads, c->heads);
    MAMBO_REQUIRE(window >= 0, MAMBO_ERR_VALUE, "a window is positive, and of causal attention");
    MAMBO_REQUIRE(tokens * q_heads <= 0x3FFFFFFF, MAMBO_ERR_VALUE, "tokens times query heads must be below 2^30 (got %lld)",
                  (long long)tokens);
    MAMBO_REQUIRE(batch->seqs * (int64_t)(b->capacity / kKvBlock) <= 0x7FFFFFF0, MAMBO_ERR_VALUE,
                  "tables must hold below 2^36 tokens together");
    *p = make_plan(*c, *b, (int)(q_heads / c->heads), window);
    const int64_t heads = c->heads;
    MAMBO_REQUIRE((p->row_tiles == 0 || p->slots || grid_takes(batch->seqs * heads, 512)) && grid_takes(p->tiles * heads, 512) &&
                      grid_takes(p->join.tiles + p->join.rows, 256),
                  MAMBO_ERR_VALUE, "too many rows for one launch");
    return MAMBO_OK;
}

} // namespace

extern "C" int64_t mambo_kv_attention_workspace(const mambo_kv_cache *cache, const mambo_kv_batch *batch, int64_t tokens,
                                                int64_t q_heads, int64_t window)
{
    KvCache c;
    KvBatch b;
    Plan p;
    if (const int rc = check(cache, batch, tokens, q_heads, window, &c, &b, &p))
        return rc;
    return p.bytes;
}

extern "C" int mambo_kv_attention_plan(const mambo_kv_cache *cache, const mambo_kv_batch *batch, int64_t tokens,
                                       int64_t q_heads, int64_t window, int32_t *plan)
{
    KvCache c;
    KvBatch b;
    Plan p;
    if (const int rc = check(cache, batch, tokens, q_heads, window, &c, &b, &p))
        return rc;
    MAMBO_REQUIRE(plan != nullptr, MAMBO_ERR_VALUE, "null pointer");
    plan[0] = p.few_rows;
    plan[1] = p.slots;
    plan[2] = p.tiles ? tile_rows(kv_padded(c.dim) / 32) : 0;
    plan[3] = p.parts;
    return MAMBO_OK;
}

extern "C" int mambo_kv_attention(const void *q, int64_t tokens, int64_t q_heads, int64_t dim, int64_t ldqt, int64_t ldqh,
                                  const mambo_kv_cache *cache,
                                  const mambo_kv_batch *batch, float scale, int causal, int64_t window, void *out,
                                  int64_t ldot, int64_t ldoh, float *lse, void *workspace, int64_t workspace_bytes,
                                  mambo_stream_t stream)
{
    Attention a;
    Plan p;
    if (const int rc = check(cache, batch, tokens, q_heads, window, &a.cache, &a.b, &p))
        return rc;
    MAMBO_REQUIRE(dim == a.cache.dim, MAMBO_ERR_VALUE, "the cache has heads of %d (got %lld)", a.cache.dim, (long long)dim);
    MAMBO_REQUIRE(scale * kLog2e > 0.0f && isfinite(scale * kLog2e), MAMBO_ERR_VALUE,
                  "the scale of the scores must be positive and finite");
    MAMBO_REQUIRE(window == 0 || causal, MAMBO_ERR_VALUE, "a window is positive, and of causal attention");
    if (tokens == 0)
        return MAMBO_OK;
    MAMBO_REQUIRE(q && out, MAMBO_ERR_VALUE, "null pointer");
    MAMBO_REQUIRE((uintptr_t)q % 16 == 0 && ldqt % 8 == 0 && ldqh % 8 == 0, MAMBO_ERR_VALUE, "queries must be 16-byte aligned");
    MAMBO_REQUIRE(ldot >= dim && ldoh >= dim, MAMBO_ERR_VALUE, "strides of the output must cover a head");
    MAMBO_REQUIRE((uintptr_t)out % 2 == 0 && (uintptr_t)lse % 4 == 0, MAMBO_ERR_VALUE, "outputs must be aligned to their type");
    MAMBO_REQUIRE(workspace_bytes >= p.bytes && (workspace || p.bytes == 0), MAMBO_ERR_VALUE,
                  "the workspace must hold %lld bytes (got %lld)", (long long)p.bytes, (long long)workspace_bytes);
    MAMBO_REQUIRE((uintptr_t)workspace % 16 == 0, MAMBO_ERR_VALUE, "the workspace must be 16-byte aligned");
    a.q = (const __bf16 *)q, a.ldqt = ldqt, a.ldqh = ldqh, a.group = (int)(q_heads / a.cache.heads);
    a.scale = scale * kLog2e, a.causal = causal != 0;
    a.window = (int)std::min<int64_t>(window, 0x3FFFFFFF);
    a.out = (__bf16 *)out, a.ldot = ldot, a.ldoh = ldoh, a.lse = lse;
    a.few_rows = p.few_rows, a.slots = p.slots, a.parts = p.parts, a.tiles_each = p.tiles_each;
    const int padded = kv_padded(a.cache.dim);
    char *at = (char *)workspace;
    a.rows_o = (float *)at, a.rows_ml = a.rows_o + p.rows_entries * padded;
    at += aligned(p.rows_entries * (padded + 2) * 4);
    a.begins = (int32_t *)at;
    at += aligned(p.slots ? ((int64_t)a.b.seqs + 1) * 4 : 0);
    a.tiles_o = (float *)at, a.tiles_ml = a.tiles_o + p.tiles_entries * padded;
    hipStream_t s = (hipStream_t)stream;
    if (p.tiles)
        if (const int rc = launch_attend_tiles(a, p.tiles, s))
            return rc;
    if (p.row_tiles)
        if (const int rc = launch_attend_rows(a, p.row_tiles, s))
            return rc;
    return p.join.tiles + p.join.rows ? launch_attend_join(a, p.row_tiles, p.join, s) : MAMBO_OK;
}
