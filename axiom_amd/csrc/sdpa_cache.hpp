// Attention of sequences of different lengths over packed keys or the pages of a cache: what its kernels share.
#pragma once

#include "divisor.hpp"
#include "sdpa.hpp"

namespace axhip {

int check_pages(const char *who, const AxhipKvPages &p); // cache.hip

// One run of queries against one run of keys for every entry (a sequence, or a group of sequences with one prefix).  A "row" is a token's
// query of one head: the rows of an entry and a key head are tokens * each, each = heads / kv_heads, row r being token r / each and head
// r % each of the key head's.  All of them read the same keys, so that a tile of keys is fetched once for `each` heads.
struct CacheArgs {
    const void *q, *k, *v;
    void *o;
    int dtype, heads, kv_heads, each, D, entries, causal;
    float scale_log2e;
    Divisor by_each;
    // the tokens of entry s: new_tokens of every sequence (decoding), or cu_q[s] .. cu_q[s + 1] - 1, at most total_q
    int new_tokens; // 0: by cu_q
    const int32_t *cu_q;
    int64_t total_q;
    int64_t qs[3], os[3]; // sequence (decoding), token, head; elements
    // its keys: cu_kv, or a table of pages
    const int32_t *cu_kv, *table, *lengths;
    int64_t total_kv, table_ld, n_pages;
    int page_shift;
    int64_t ks[3], vs[3]; // page, row, head; elements
    // prefixes (decoding): of groups of sequences
    int groups;
    const int32_t *group_starts, *prefix_table, *prefix_lengths;
    int64_t prefix_ld;
    // in parts: how many a prefix (decoding) or the keys of a block of rows (prompts) have, at most, and what they leave for the join, by row -- sequence, key head, row of it (decoding),
    // or token, head -- and part; the shares that a step's own keys are dealt out in, what they leave by slot (two to a share, then one to a sequence), key head and row, and for each
    // sequence the first of its slots and how many there are to join (0: it is finished)
    int parts, shares;
    float *part_out, *part_lse, *own_out, *own_lse;
    int2_t *parts_of;
};
// Work-groups of a step's own keys
inline int64_t own_blocks(const CacheArgs &a) { return (static_cast<int64_t>(a.new_tokens) * a.each + 15) / 16 * a.kv_heads * a.shares; }

constexpr int64_t MOST_KEYS = int64_t(1) << 30; // of a sequence

// The keys of an entry
struct KeyRun {
    const int32_t *table; // NULL: rows from `base` on
    int64_t base;
    int n;
};
__device__ __forceinline__ int clamped(int64_t v, int64_t lo, int64_t hi) { return static_cast<int>(v < lo ? lo : v > hi ? hi : v); }
__device__ __forceinline__ KeyRun keys_of(const CacheArgs &a, int s) {
    if (a.table) {
        const int64_t most = a.table_ld << a.page_shift;
        return {a.table + s * a.table_ld, 0, clamped(a.lengths[s], 0, most < MOST_KEYS ? most : MOST_KEYS)};
    }
    const int from = clamped(a.cu_kv[s], 0, a.total_kv);
    return {nullptr, from, clamped(a.cu_kv[s + 1], from, a.total_kv) - from};
}
__device__ __forceinline__ KeyRun prefix_of(const CacheArgs &a, int group) {
    const int64_t most = a.prefix_ld << a.page_shift;
    return {a.prefix_table + group * a.prefix_ld, 0, clamped(a.prefix_lengths[group], 0, most < MOST_KEYS ? most : MOST_KEYS)};
}
struct TokenRun { int from, n; };
__device__ __forceinline__ TokenRun tokens_of(const CacheArgs &a, int s) {
    if (a.new_tokens) return {0, a.new_tokens};
    const int from = clamped(a.cu_q[s], 0, a.total_q);
    return {from, clamped(a.cu_q[s + 1], from, a.total_q) - from};
}
// The group that sequence s belongs to, or -1: the last one that starts at or in front of it, if it does not end there
__device__ __forceinline__ int group_of(const CacheArgs &a, int s) {
    int lo = 0, hi = a.groups; // starts[lo - 1] <= s < starts[hi], as far as they are known
    while (lo < hi) {
        const int mid = (lo + hi) / 2;
        if (a.group_starts[mid] <= s) lo = mid + 1;
        else hi = mid;
    }
    return lo > 0 && a.group_starts[lo] > s ? lo - 1 : -1;
}

// The matrix-core kernels (16 bits) of rows found by cu_q: sdpa_tile.hpp; 4 or 8 waves of 32 rows
int launch_tile_bf16(const CacheArgs &a, int waves, hipStream_t s);
int launch_tile_f16(const CacheArgs &a, int waves, hipStream_t s);
// A decoding step with prefixes: sdpa_step.hpp; of fp32 the prefixes alone
int launch_step_bf16(const CacheArgs &a, hipStream_t s);
int launch_step_f16(const CacheArgs &a, hipStream_t s);
int launch_prefix_f32(const CacheArgs &a, hipStream_t s);
// Few rows and fp32: sdpa_rows.hpp
int launch_rows_own_bf16(const CacheArgs &a, hipStream_t s);
int launch_rows_own_f16(const CacheArgs &a, hipStream_t s);
int launch_rows_own_f32(const CacheArgs &a, hipStream_t s);
int launch_rows_packed_bf16(const CacheArgs &a, hipStream_t s);
int launch_rows_packed_f16(const CacheArgs &a, hipStream_t s);
int launch_rows_packed_f32(const CacheArgs &a, bool apart, hipStream_t s);
// .. whole sequences, prefix and own keys one behind the other: a step that is not divided
int launch_rows_whole_bf16(const CacheArgs &a, hipStream_t s);
int launch_rows_whole_f16(const CacheArgs &a, hipStream_t s);
int launch_rows_whole_f32(const CacheArgs &a, hipStream_t s);
int launch_join_bf16(const CacheArgs &a, hipStream_t s);
int launch_join_f16(const CacheArgs &a, hipStream_t s);
int launch_join_f32(const CacheArgs &a, hipStream_t s);

} // namespace axhip
