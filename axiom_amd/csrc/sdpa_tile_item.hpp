// Which rows and keys a work-group of the ragged attention kernels takes.
#pragma once

#include "sdpa_cache.hpp"

namespace axhip {

constexpr int TK = 64; // keys of a tile

// The last e < n with first(e) <= index (0 if there is none), by a wavefront: 64 candidates at a time.  Entry e gets the blocks from first(e) = rows in front of it / BM + e on, which is one
// more than it needs at most and never less, so that no lengths have to be added up.
template <class F> __device__ __forceinline__ int last_not_beyond(int n, int index, F first) {
    const int lane = threadIdx.x % WAVE;
    int lo = 0, hi = n;
    while (hi - lo > 1) {
        const int step = (hi - lo + WAVE - 1) / WAVE, e = lo + lane * step;
        const uint64_t below = __builtin_amdgcn_ballot_w64(e < hi && first(e) <= index);
        const int n_below = below ? 64 - __builtin_clzll(below) : 1;
        hi = min(hi, lo + n_below * step);
        lo = lo + (n_below - 1) * step;
    }
    return lo;
}

// Block `index` of BM rows of the groups' rows (those of their sequences, one behind the other): row row0 of the `rows` of group `group`, whose first sequence is `first`.  group < 0: no such block.
struct GroupItem { int group, row0, rows, first; };
template <int BM> __device__ __forceinline__ GroupItem group_item(const CacheArgs &a, int index) {
    const int per = a.new_tokens * a.each;
    auto start = [&](int e) { return clamped(a.group_starts[e], 0, a.entries); };
    auto first = [&](int e) { return static_cast<int>(static_cast<int64_t>(start(e)) * per / BM + e); };
    const int e = last_not_beyond(a.groups, index, first);
    const int from = start(e), rows = (clamped(a.group_starts[e + 1], from, a.entries) - from) * per, block = index - first(e);
    if (block < 0 || block > rows / BM || block * BM >= rows) return {-1, 0, 0, 0};
    return {e, block * BM, rows, from};
}
// Keys of a part of n: whole tiles, a.parts parts at most
__device__ __forceinline__ int part_keys(const CacheArgs &a, int n) { return max(1, ((n + a.parts - 1) / a.parts + TK - 1) / TK) * TK; }

// Block `index` of all blocks of BM rows.  Up to 64 entries, one to a lane: those that walk the most tiles of keys first, since a long sequence's last blocks, started last, would keep a few CUs
// busy after all others are done; the number of blocks that walk c tiles or more is a sum over the lanes, and c is searched for (64 chunks of 64 tokens
// behind 300 keys: 66 us, in the entries' order 80).  More entries: in their order, since the search would take longer than it gains (200 prompts of 82 tokens: 140 us, with four entries to a lane 170).
// index: uniform.  entry < 0: no such block.
struct TileItem { int entry, row0; TokenRun tokens; int base, keys; }; // base: of packed keys
template <int BM> __device__ __forceinline__ TileItem tile_item(const CacheArgs &a, int index) {
    const int lane = threadIdx.x % WAVE;
    int entry = -1, block = 0, from = 0, n = 0, base = 0, keys = 0;
    if (a.entries > WAVE) {
        auto first = [&](int e) { return static_cast<int>(static_cast<int64_t>(clamped(a.cu_q[e], 0, a.total_q)) * a.each / BM + e); };
        entry = last_not_beyond(a.entries, index, first);
        block = index - first(entry);
        const TokenRun t = tokens_of(a, entry);
        const KeyRun k = keys_of(a, entry);
        from = t.from;
        n = t.n;
        base = static_cast<int>(k.base);
        keys = k.n;
    } else {
        TokenRun my_tokens{0, 0};
        int my_base = 0, my_keys = 0, my_blocks = 0;
        if (lane < a.entries) {
            my_tokens = tokens_of(a, lane);
            const KeyRun k = keys_of(a, lane);
            my_base = static_cast<int>(k.base);
            my_keys = k.n;
            my_blocks = (my_tokens.n * a.each + BM - 1) / BM;
        }
        auto with = [&](int c) { // blocks of this lane's entry that walk c tiles or more
            const int token = a.causal ? TK * (c - 1) - (my_keys - my_tokens.n) : TK * (c - 1) < my_keys ? 0 : my_tokens.n; // the first one that sees so far
            return c <= 0 || token <= 0 ? my_blocks : token >= my_tokens.n ? 0 : my_blocks - token * a.each / BM;
        };
        auto all_with = [&](int c) { return __builtin_amdgcn_readfirstlane(static_cast<int>(wave_sum(static_cast<float>(with(c))))); }; // (below 2^24: exact)
        // all_with(lo) > index >= all_with(hi)
        int lo = 0, hi = 1 + __builtin_amdgcn_readfirstlane(static_cast<int>(wave_max(my_blocks > 0 ? static_cast<float>((my_keys + TK - 1) / TK) : 0.0f)));
        if (index >= all_with(0)) return {-1, 0, {0, 0}, 0, 0};
        while (hi - lo > 1) {
            const int mid = (lo + hi) / 2;
            if (all_with(mid) > index) lo = mid;
            else hi = mid;
        }
        const int longer = with(lo + 1), mine = with(lo) - longer; // `lo` tiles exactly
        int upto = mine;
#pragma unroll
        for (int d = 1; d < WAVE; d *= 2) {
            const int other = __shfl_up(upto, d, WAVE);
            if (lane >= d) upto += other;
        }
        const int left = index - all_with(lo + 1);
        const uint64_t reached = __builtin_amdgcn_ballot_w64(upto > left);
        if (reached) {
            entry = __builtin_ctzll(reached);
            block = __builtin_amdgcn_readlane(my_blocks - longer - upto, entry) + left;
            from = __builtin_amdgcn_readlane(my_tokens.from, entry);
            n = __builtin_amdgcn_readlane(my_tokens.n, entry);
            base = __builtin_amdgcn_readlane(my_base, entry);
            keys = __builtin_amdgcn_readlane(my_keys, entry);
        }
    }
    auto uniform = [](int v) { return __builtin_amdgcn_readfirstlane(v); };
    if (block < 0 || block > n * a.each / BM || block * BM >= n * a.each) entry = -1;
    return {uniform(entry), uniform(block * BM), {uniform(from), uniform(n)}, uniform(base), uniform(keys)};
}

} // namespace axhip
