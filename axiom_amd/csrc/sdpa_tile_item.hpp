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

// Block `index` of all blocks of BM rows, those that walk the most tiles of keys first: a long sequence's last blocks, started last, would keep a few CUs busy
// after all others are done.  Up to 256 entries: the number of blocks that walk c tiles or more is a sum over the entries, four to a lane, and c is searched for.
// More: in the order of the entries.  index: uniform.  entry < 0: no such block.
struct TileItem { int entry, block; };
template <int BM> __device__ __forceinline__ TileItem tile_item(const CacheArgs &a, int index) {
    const int lane = threadIdx.x % WAVE;
    if (a.entries > 256) {
        auto first = [&](int e) { return static_cast<int>(static_cast<int64_t>(clamped(a.cu_q[e], 0, a.total_q)) * a.each / BM + e); };
        const int e = last_not_beyond(a.entries, index, first);
        return {e, index - first(e)};
    }
    int blocks[4], past[4], last[4], tiles[4]; // of this lane's entries: blocks, keys in front of the first token, last token, tiles of keys
    float most = 0.0f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int e = lane + WAVE * i;
        blocks[i] = past[i] = last[i] = tiles[i] = 0;
        if (WAVE * i < a.entries && e < a.entries) {
            const TokenRun t = tokens_of(a, e);
            const int keys = keys_of(a, e).n;
            blocks[i] = (t.n * a.each + BM - 1) / BM;
            past[i] = keys - t.n;
            last[i] = t.n - 1;
            tiles[i] = (keys + TK - 1) / TK;
            if (blocks[i] > 0) most = fmaxf(most, static_cast<float>(tiles[i]));
        }
    }
    auto with = [&](int i, int c) { // blocks of entry i that walk c tiles or more
        if (c <= 0) return blocks[i];
        if (tiles[i] < c) return 0;
        if (!a.causal) return blocks[i];
        const int token = TK * (c - 1) - past[i]; // the first one that sees so far
        if (token <= 0) return blocks[i];
        return token > last[i] ? 0 : blocks[i] - token * a.each / BM;
    };
    auto all_with = [&](int c) {
        float n = 0.0f; // (below 2^24: exact)
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (WAVE * i < a.entries) n += static_cast<float>(with(i, c));
        return static_cast<int>(wave_sum(n));
    };
    int lo = 0, hi = static_cast<int>(wave_max(most)) + 1; // all_with(lo) > index >= all_with(hi)
    if (index >= all_with(0)) return {-1, 0};
    while (hi - lo > 1) {
        const int mid = (lo + hi) / 2;
        if (all_with(mid) > index) lo = mid;
        else hi = mid;
    }
    int left = index - all_with(lo + 1); // among those that walk `lo` tiles exactly
    TileItem item{-1, 0};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if (WAVE * i >= a.entries || item.entry >= 0) continue;
        const int mine = with(i, lo) - with(i, lo + 1);
        int upto = mine;
#pragma unroll
        for (int d = 1; d < WAVE; d *= 2) {
            const int other = __shfl_up(upto, d, WAVE);
            if (lane >= d) upto += other;
        }
        const uint64_t reached = __builtin_amdgcn_ballot_w64(upto > left);
        if (reached) {
            const int at = __builtin_ctzll(reached);
            item.entry = at + WAVE * i;
            item.block = __builtin_amdgcn_readlane(blocks[i] - with(i, lo) + left - (upto - mine), at);
        } else {
            left -= __builtin_amdgcn_readlane(upto, WAVE - 1);
        }
    }
    return item;
}

} // namespace axhip
