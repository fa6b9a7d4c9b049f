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
struct TileItem { int entry, row0; TokenRun tokens; int base, keys; }; // base: of packed keys
template <int BM> __device__ __forceinline__ TileItem tile_item(const CacheArgs &a, int index) {
    const int lane = threadIdx.x % WAVE;
    int entry = -1, block = 0, from = 0, n = 0, base = 0, keys = 0;
    if (a.entries > 256) {
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
        TokenRun tokens[4]; // of this lane's entries
        int bases[4], most_keys[4], blocks[4];
        float most = 0.0f;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int e = lane + WAVE * i;
            tokens[i] = {0, 0};
            bases[i] = most_keys[i] = blocks[i] = 0;
            if (WAVE * i < a.entries && e < a.entries) {
                tokens[i] = tokens_of(a, e);
                const KeyRun k = keys_of(a, e);
                bases[i] = static_cast<int>(k.base);
                most_keys[i] = k.n;
                blocks[i] = (tokens[i].n * a.each + BM - 1) / BM;
                if (blocks[i] > 0) most = fmaxf(most, static_cast<float>((k.n + TK - 1) / TK));
            }
        }
        auto with = [&](int i, int c) { // blocks of entry i that walk c tiles or more
            if (c <= 0) return blocks[i];
            if (most_keys[i] <= TK * (c - 1)) return 0;
            if (!a.causal) return blocks[i];
            const int token = TK * (c - 1) - (most_keys[i] - tokens[i].n); // the first one that sees so far
            if (token <= 0) return blocks[i];
            return token >= tokens[i].n ? 0 : blocks[i] - token * a.each / BM;
        };
        auto all_with = [&](int c) {
            float sum = 0.0f; // (below 2^24: exact)
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (WAVE * i < a.entries) sum += static_cast<float>(with(i, c));
            return __builtin_amdgcn_readfirstlane(static_cast<int>(wave_sum(sum)));
        };
        int lo = 0, hi = __builtin_amdgcn_readfirstlane(static_cast<int>(wave_max(most))) + 1; // all_with(lo) > index >= all_with(hi)
        if (index >= all_with(0)) return {-1, 0, {0, 0}, 0, 0};
        while (hi - lo > 1) {
            const int mid = (lo + hi) / 2;
            if (all_with(mid) > index) lo = mid;
            else hi = mid;
        }
        int left = index - all_with(lo + 1); // among those that walk `lo` tiles exactly
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if (WAVE * i >= a.entries || entry >= 0) continue;
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
                entry = at + WAVE * i;
                block = __builtin_amdgcn_readlane(blocks[i] - with(i, lo) + left - (upto - mine), at);
                from = __builtin_amdgcn_readlane(tokens[i].from, at);
                n = __builtin_amdgcn_readlane(tokens[i].n, at);
                base = __builtin_amdgcn_readlane(bases[i], at);
                keys = __builtin_amdgcn_readlane(most_keys[i], at);
            } else {
                left -= __builtin_amdgcn_readlane(upto, WAVE - 1);
            }
        }
    }
    auto uniform = [](int v) { return __builtin_amdgcn_readfirstlane(v); };
    if (block < 0 || block > n * a.each / BM || block * BM >= n * a.each) entry = -1;
    return {uniform(entry), uniform(block * BM), {uniform(from), uniform(n)}, uniform(base), uniform(keys)};
}

} // namespace axhip
