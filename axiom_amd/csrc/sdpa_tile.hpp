// Ragged attention on the matrix cores, 16 bits: the kernel of whole prompts, of chunks of them, and of prefixes that many sequences share.
//
// A work-group owns 32 * NW rows of one entry and key head and walks its keys in tiles of 64.  It computes S^T = K Q^T on v_mfma_f32_32x32x16, so that a
// lane owns one query and its softmax needs one exchange with lane ^ 32, and the exponentiated scores are the B operand of O^T += V^T P^T as they lie.  K and V go
// from memory straight into swizzled LDS, K a tile ahead of V; the MFMAs of a step -- the output of tile j, the scores of tile j + 1 -- are issued back to back in
// alternation, the softmax follows.  With eight waves the upper four (one of each SIMD's two) do that in the other order, so that one of the two is
// in its matrix phase while the other one is in its vector phase.
//
// Bound by the vector work between the matrix phases (32 exponentials and 80 other instructions a lane and tile, 930 cycles beside 1024 of MFMAs), which runs beside them for a small part only: 12
// prompts of 16384 tokens, 32 heads on 8 of 128 dims, 400 - 415 us, 0.96 - 0.99 PFLOP/s of the causal half, matrix pipe and vector instructions busy 47 % of the cycles each, at 1.9 GHz.
//
// What the ragged form asks for:
//  * rows are tokens times the heads that share a key head: one tile of keys serves them all, and a short sequence fills the work-group.
//  * a piece of a tile that one load instruction fetches (2 to 8 rows) lies in one page, so that its address is wave-uniform: the pages' numbers are asked for a step ahead, one to a lane, and
//    the addresses formed there.  Only the piece with the last key has lanes to aim elsewhere (at that key: what lies behind it is not read).
//  * work-groups find their rows in the lengths on the device, longest walks first (see tile_item).
//  * scores are scaled in fp32, in the FMA that subtracts the maximum: q rounded after its scaling, which would save nothing here, adds as much error as the output's rounding does.
#pragma once

#include "sdpa_tile_item.hpp"

#include <type_traits>

namespace axhip {

typedef int tile_int4_t __attribute__((ext_vector_type(4)));

template <bool BF16> __device__ __forceinline__ float16_t tile_mfma(uint4_t a, uint4_t b, float16_t c) {
    if constexpr (BF16) return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8_t, a), __builtin_bit_cast(bf16x8_t, b), c, 0, 0, 0);
    else return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(half8_t, a), __builtin_bit_cast(half8_t, b), c, 0, 0, 0);
}
// 4 consecutive keys of one dim out of [key][dim] rows: within a group of 16 lanes, lane i receives element i & 3 of the 8-byte pieces that lanes (i >> 2) + 4 j address
__device__ __forceinline__ uint2_t tile_transposed(const unsigned char *p) {
    typedef short short4_t __attribute__((ext_vector_type(4)));
    typedef __attribute__((address_space(3))) short4_t lds_short4_t;
    return __builtin_bit_cast(uint2_t, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_short4_t *)(p)));
}
// 16 bytes a lane from base + offset straight into LDS: lane i's land at lds_base + 16 i; a lane that is switched off leaves its place as it is.  (Five states between a vector instruction that
// writes the base's registers, such as the reading of a lane, and the load that reads them, which the compiler does not see to here; one behind M0.)
__device__ __forceinline__ void tile_fetch(uint64_t base_uniform, uint32_t offset, uint32_t lds_base_uniform) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 3\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(lds_base_uniform), "v"(offset), "s"(base_uniform) : "memory");
}
// XOR of the 16-byte chunk's place in a row, so that neither 16 rows of one chunk nor the 4 rows of a transposing read meet on a bank
template <int D> __device__ __forceinline__ int tile_swizzle_k(int row) { return D >= 128 ? (((row & 3) << 2) | ((row >> 2) & 3)) : ((row >> 1) & 7); }
template <int D> __device__ __forceinline__ int tile_swizzle_v(int row) { return D >= 128 ? (((row & 3) << 2) | ((row >> 2) & 3)) : (((row >> 1) & 1) << 2); }

__device__ __forceinline__ uint64_t uniform64(uint64_t v) {
    return (static_cast<uint64_t>(__builtin_amdgcn_readfirstlane(static_cast<int>(v >> 32))) << 32) | static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(static_cast<int>(v)));
}

// D: the LDS row in dims; DE: the dims that are computed; the head size in memory, a multiple of 8, may be less (zeros in its place)
// PREFIX: the rows of a group of sequences against a part of their prefix (decoding): fp32 results and the base-2 logarithm of their denominators, for sdpa_join_kernel
enum TileKeys { TILE_PACKED = 0, TILE_PAGED = 1, TILE_PREFIX = 2 };
template <bool BF16, int D, int DE, int NW, int KEYS>
__device__ __forceinline__ void tile_body(const CacheArgs &a, int index_of_all) {
    static_assert(DE % 32 == 0 && DE <= D, "dims");
    constexpr int PF = 3, RING = PF + 1; // LDS reads run this many MFMAs ahead
    constexpr int KT = DE / 16, DT = DE / 32, BM = 32 * NW, ROWB = 2 * D, CHUNKS = ROWB / 16, RPL = WAVE / CHUNKS;
    constexpr int NLOAD = TK / (RPL * NW), TILEB = TK * ROWB, NM = DE / 4;
    constexpr int NV = RPL * NW < 16 ? 2 : 1; // (the swizzles see row & 15)
    static_assert(NLOAD >= 1, "every wave fetches");
    extern __shared__ __attribute__((aligned(1024))) unsigned char tile_lds[]; // K0 K1 V0 V1

    const int tid = threadIdx.x, lane = tid % WAVE, wave = __builtin_amdgcn_readfirstlane(tid / WAVE);
    const int ql = lane % 32, g = lane / 32;
    const bool second = NW == 8 && wave >= 4;
    const int kvh = index_of_all % a.kv_heads;
    // entry, its rows from row0 on; its keys: n_all, of which [begin, nk) are this work-group's
    int rest = index_of_all / a.kv_heads, part = 0, entry, rows, row0, n_all, from;
    if (a.parts > 1) {
        part = rest % a.parts;
        rest /= a.parts;
    }
    KeyRun run;
    if constexpr (KEYS == TILE_PREFIX) {
        const GroupItem item = group_item<BM>(a, rest);
        entry = __builtin_amdgcn_readfirstlane(item.group);
        if (entry < 0) return;
        rows = __builtin_amdgcn_readfirstlane(item.rows);
        row0 = __builtin_amdgcn_readfirstlane(item.row0);
        from = item.first;
        run = prefix_of(a, entry);
    } else {
        const TileItem item = tile_item<BM>(a, rest);
        entry = item.entry;
        if (entry < 0) return;
        run = KeyRun{a.table ? a.table + entry * a.table_ld : nullptr, item.base, item.keys};
        rows = item.tokens.n * a.each;
        row0 = item.row0;
        from = item.tokens.from;
    }
    n_all = __builtin_amdgcn_readfirstlane(run.n);
    constexpr bool PAGED = KEYS != TILE_PACKED;
    const bool causal = KEYS != TILE_PREFIX && a.causal;
    const int dv = a.D;
    const int past = n_all - static_cast<int>(a.by_each.of(rows)); // keys in front of the first token
    auto sees = [&](int r) { return causal ? past + static_cast<int>(a.by_each.of(min(r, rows - 1))) : n_all - 1; }; // the last key that a row sees
    int begin = 0, nk = max(0, __builtin_amdgcn_readfirstlane(sees(row0 + BM - 1) + 1));
    if (a.parts > 1) {
        const int chunk = part_keys(a, nk);
        begin = part * chunk;
        nk = min(nk, begin + chunk);
        if (KEYS == TILE_PREFIX && begin >= nk) return; // (as many parts as that are there for the join)
    }

    // this lane's query, and the last key that it sees; rows behind the last one see what that one does and are not stored
    const int row = row0 + 32 * wave + ql;
    const bool row_ok = row < rows;
    const int token = static_cast<int>(a.by_each.of(min(row, rows - 1))), head = kvh * a.each + min(row, rows - 1) - token * a.each;
    const int limit = min(causal ? past + token : n_all - 1, nk - 1);
    const int wave_row = row0 + 32 * wave;
    const int least = __builtin_amdgcn_readfirstlane(min(sees(wave_row), nk - 1)), farthest = __builtin_amdgcn_readfirstlane(wave_row < rows ? min(sees(wave_row + 31), nk - 1) : -1);
    const int ntiles = (nk - begin + TK - 1) / TK; // (0 or less: none)
    int64_t at_q;
    if constexpr (KEYS == TILE_PREFIX) at_q = (from + token / a.new_tokens) * a.qs[0] + token % a.new_tokens * a.qs[1] + head * a.qs[2];
    else at_q = (from + token) * a.qs[1] + head * a.qs[2];

    uint4_t qf[KT];
    {
        const uint16_t *q = static_cast<const uint16_t *>(a.q) + at_q;
#pragma unroll
        for (int t = 0; t < KT; ++t) {
            qf[t] = uint4_t{0, 0, 0, 0};
            if (row_ok && 16 * t + 8 * g < dv) qf[t] = *reinterpret_cast<const uint4_t *>(q + 16 * t + 8 * g);
        }
    }

    // ---- memory -> LDS
    const uint64_t k_base = uniform64(reinterpret_cast<uint64_t>(a.k) + static_cast<uint64_t>(kvh * a.ks[2]) * 2), v_base = uniform64(reinterpret_cast<uint64_t>(a.v) + static_cast<uint64_t>(kvh * a.vs[2]) * 2);
    const uint32_t k_row = static_cast<uint32_t>(a.ks[1]) * 2, v_row = static_cast<uint32_t>(a.vs[1]) * 2;
    const int my = lane / CHUNKS; // row of a piece
    uint32_t k_off[NV], v_off[NV];
    int k_chunk[NV], v_chunk[NV];
#pragma unroll
    for (int o = 0; o < NV; ++o) {
        const int r = RPL * wave + my + 8 * o;
        k_chunk[o] = (lane % CHUNKS) ^ tile_swizzle_k<D>(r);
        v_chunk[o] = (lane % CHUNKS) ^ tile_swizzle_v<D>(r);
        k_off[o] = my * k_row + k_chunk[o] * 16;
        v_off[o] = my * v_row + v_chunk[o] * 16;
    }
    const uint32_t lds_base = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(tile_lds));
    const uint32_t lds_wave = __builtin_amdgcn_readfirstlane(lds_base + RPL * wave * ROWB);
    const int last_piece = (nk - 1) / RPL * RPL;
    bool bad = false;
    // lane n (modulo NLOAD) has the page of this wave's piece n, and forms its address; the wave takes them from there.  (One scalar instruction after the other for each piece, 20 of them, took a
    // third of a tile's time with four waves.)
    const int my_piece = RPL * wave + RPL * NW * (lane % NLOAD);
    auto page_at = [&](int tile) { return PAGED ? run.table[min(begin + tile * TK + my_piece, last_piece) >> a.page_shift] : 0; };
    auto fetch = [&](uint64_t base, int64_t page_elements, uint32_t row_bytes, const uint32_t (&off)[NV], const int (&chunk)[NV], int tile, int page, uint32_t to) __attribute__((always_inline)) {
        uint64_t mine = 0;
        if constexpr (PAGED) {
            uint32_t id = static_cast<uint32_t>(page);
            if (id >= static_cast<uint32_t>(a.n_pages)) {
                bad = true;
                id = 0;
            }
            const uint32_t row_in = static_cast<uint32_t>(min(begin + tile * TK + my_piece, last_piece) & ((1 << a.page_shift) - 1));
            mine = base + static_cast<uint64_t>(id) * static_cast<uint32_t>(page_elements * 2) + static_cast<uint64_t>(row_in) * row_bytes;
        }
        const uint64_t first = PAGED ? 0 : uniform64(base + static_cast<uint64_t>((run.base + begin + tile * TK + RPL * wave) * static_cast<int64_t>(row_bytes)));
        auto pieces = [&](auto all_rows) __attribute__((always_inline)) {
#pragma unroll
            for (int n = 0; n < NLOAD; ++n) {
                const int piece = all_rows ? begin + tile * TK + RPL * NW * n + RPL * wave : min(begin + tile * TK + RPL * NW * n + RPL * wave, last_piece);
                uint64_t at;
                if constexpr (PAGED) at = (static_cast<uint64_t>(static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(mine >> 32), n))) << 32) | static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(mine), n));
                else at = first + static_cast<uint64_t>(static_cast<int64_t>(piece - (begin + tile * TK + RPL * wave)) * row_bytes);
                uint32_t offset = off[n % NV];
                if (!all_rows && piece == last_piece) offset -= (my - min(my, nk - 1 - last_piece)) * row_bytes;
                if (chunk[n % NV] * 8 < dv) tile_fetch(at, offset, to + n * RPL * NW * ROWB);
            }
        };
        if (begin + tile * TK + TK <= last_piece) pieces(std::true_type{});
        else pieces(std::false_type{});
    };
    auto load_k = [&](int tile, int buf, int page) __attribute__((always_inline)) { fetch(k_base, a.ks[0], k_row, k_off, k_chunk, tile, page, lds_wave + buf * TILEB); };
    auto load_v = [&](int tile, int buf, int page) __attribute__((always_inline)) { fetch(v_base, a.vs[0], v_row, v_off, v_chunk, tile, page, lds_wave + (2 + buf) * TILEB); };

    // ---- LDS fragments (bytes)
    int k_at[KT]; // row ql (+ 32), chunk 2 t + g
#pragma unroll
    for (int t = 0; t < KT; ++t) k_at[t] = ql * ROWB + (((2 * t + g) ^ tile_swizzle_k<D>(ql)) * 16);
    int v_at[2][DT]; // rows 4 g + s (+ 8), dims 32 dt + lane % 32
    {
        const int s = (lane & 15) >> 2, c = ((lane >> 4) & 1) * 2 + ((lane & 3) >> 1), part = lane & 1;
#pragma unroll
        for (int hi = 0; hi < 2; ++hi)
#pragma unroll
            for (int dt = 0; dt < DT; ++dt) {
                const int r = 4 * g + s + 8 * hi;
                v_at[hi][dt] = r * ROWB + (((dt * 4 + c) ^ tile_swizzle_v<D>(r)) * 16) + part * 8;
            }
    }
    auto barrier = [] { asm volatile("s_barrier" ::: "memory"); };
    auto landed = [] { __builtin_amdgcn_s_waitcnt(0x0F70); }; // vmcnt(0)

    if (dv < DE) { // the dims that no load fills: zeros, whatever K and V hold there
        for (int i = tid; i < 4 * TILEB / 16; i += 64 * NW) reinterpret_cast<uint4_t *>(tile_lds)[i] = uint4_t{0, 0, 0, 0};
        __syncthreads();
    }

    float16_t oacc[DT], s[2];
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
        for (int i = 0; i < 16; ++i) oacc[dt][i] = 0.0f;
    float m_run = NEG_INF_F, l0 = 0.0f, l1 = 0.0f; // the reference that exponentials are taken against (base 2, scaled), may lag the maximum
    uint32_t w[16];
    auto larger = [](float x, float y) { return __builtin_elementwise_maximum(x, y); }; // (needs no canonical input; hands a NaN on)

    auto softmax_phase = [&](int j) __attribute__((always_inline)) {
        if (begin + j * TK + TK - 1 > least) {
#pragma unroll
            for (int kt = 0; kt < 2; ++kt)
#pragma unroll
                for (int i = 0; i < 16; ++i)
                    if (begin + j * TK + kt * 32 + (i / 4) * 8 + g * 4 + i % 4 > limit) s[kt][i] = NEG_INF_F;
        }
        float m[4];
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            m[c] = larger(s[c / 2][8 * (c % 2)], s[c / 2][8 * (c % 2) + 1]);
#pragma unroll
            for (int i = 2; i < 8; i += 2) m[c] = larger(larger(m[c], s[c / 2][8 * (c % 2) + i]), s[c / 2][8 * (c % 2) + i + 1]);
        }
        float top = larger(larger(m[0], m[1]), larger(m[2], m[3]));
        top = across32(top, [&](float x, float y) { return larger(x, y); });
        const float m_new = larger(m_run, top * a.scale_log2e);
        if (__builtin_amdgcn_ballot_w64(m_new - m_run > RESCALE_THRESHOLD) != 0) { // (rare; -inf - -inf compares false)
            const float alpha = m_new == NEG_INF_F ? 1.0f : __builtin_amdgcn_exp2f(m_run - m_new);
            m_run = m_new;
            l0 *= alpha;
            l1 *= alpha;
#pragma unroll
            for (int dt = 0; dt < DT; ++dt)
#pragma unroll
                for (int i = 0; i < 16; ++i) oacc[dt][i] *= alpha;
        }
        const float minus = m_run == NEG_INF_F ? 0.0f : -m_run;
#pragma unroll
        for (int pr = 0; pr < 16; ++pr) {
            const int kt = pr / 8, i = (pr % 8) * 2;
            const float p0 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[kt][i], a.scale_log2e, minus));
            const float p1 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[kt][i + 1], a.scale_log2e, minus));
            w[pr] = pack2<BF16>(p0, p1);
            l0 += p0; // (sums of pairs by the dot instruction wait for the matrix pipe)
            l1 += p1;
        }
    };
    // O^T += V^T P^T of tile j and S^T = K Q^T of tile j + 1 in turn, so that neighbours never share an accumulator
    auto matrix_phase = [&](const unsigned char *Kn, const unsigned char *Vb) __attribute__((always_inline)) {
        __builtin_amdgcn_s_setprio(1); // (the other wave's vector work goes in between; 12 prompts 418 -> 413 us)
        uint4_t fr[RING];
        auto read = [&](int m) __attribute__((always_inline)) {
            const int i = m / 2;
            if (m % 2 == 0) {
                fr[m % RING] = *reinterpret_cast<const uint4_t *>(Kn + (i & 1) * 32 * ROWB + k_at[i >> 1]);
            } else {
                const uint2_t lo = tile_transposed(Vb + (i / DT) * 16 * ROWB + v_at[0][i % DT]), hi = tile_transposed(Vb + (i / DT) * 16 * ROWB + v_at[1][i % DT]);
                fr[m % RING] = uint4_t{lo.x, lo.y, hi.x, hi.y};
            }
        };
#pragma unroll
        for (int m = 0; m < PF; ++m) read(m);
#pragma unroll
        for (int m = 0; m < NM; ++m) {
            if (m + PF < NM) read(m + PF);
            const int i = m / 2;
            if (m % 2 == 0) {
                const float16_t zero{};
                s[i & 1] = tile_mfma<BF16>(fr[m % RING], qf[i >> 1], i < 2 ? zero : s[i & 1]);
            } else {
                const uint4_t p = {w[4 * (i / DT)], w[4 * (i / DT) + 1], w[4 * (i / DT) + 2], w[4 * (i / DT) + 3]};
                oacc[i % DT] = tile_mfma<BF16>(fr[m % RING], p, oacc[i % DT]);
            }
            __builtin_amdgcn_sched_barrier(0);
        }
        __builtin_amdgcn_s_setprio(0);
    };

    if (ntiles > 0) {
        int here = page_at(0), next = page_at(1); // of the tile that V is fetched of next, of the one that K is
        load_k(0, 0, here);
        load_v(0, 0, here);
        if (ntiles > 1) load_k(1, 1, next);
        here = next;
        next = page_at(2);
        landed();
        barrier();
#pragma unroll
        for (int kt = 0; kt < 2; ++kt) {
#pragma unroll
            for (int t = 0; t < KT; ++t) {
                const float16_t zero{};
                s[kt] = tile_mfma<BF16>(*reinterpret_cast<const uint4_t *>(tile_lds + kt * 32 * ROWB + k_at[t]), qf[t], t == 0 ? zero : s[kt]);
            }
        }
        __builtin_amdgcn_s_waitcnt(0xC07F); // lgkmcnt(0): K buffer 0 is read
        auto active = [&](int j) { return begin + j * TK <= farthest; };
        // one barrier a tile: behind it tile j + 1 of K and j of V have landed, and every wave is done with the buffers that K(j + 2) and V(j + 1) go to
        auto step = [&](int j, auto parity) __attribute__((always_inline)) {
            constexpr int PAR = decltype(parity)::value;
            landed();
            barrier();
            if (j + 2 < ntiles) load_k(j + 2, PAR, next);
            if (j + 1 < ntiles) load_v(j + 1, 1 - PAR, here);
            here = next;
            next = page_at(j + 3);
            if (second && active(j)) softmax_phase(j);
            if (active(j)) matrix_phase(tile_lds + (1 - PAR) * TILEB, tile_lds + (2 + PAR) * TILEB);
            if (!second && j + 1 < ntiles && active(j + 1)) softmax_phase(j + 1);
        };
        if (!second && active(0)) softmax_phase(0);
        for (int j = 0; j < ntiles; j += 2) {
            step(j, std::integral_constant<int, 0>{});
            if (j + 1 < ntiles) step(j + 1, std::integral_constant<int, 1>{});
        }
    }

    float l = across32(l0 + l1, lanes_add);
    if constexpr (PAGED) { // a page that does not exist, seen by any wave
        __syncthreads();
        uint32_t *flags = reinterpret_cast<uint32_t *>(tile_lds);
        const bool wave_bad = __builtin_amdgcn_ballot_w64(bad) != 0;
        if (lane == 0) flags[wave] = wave_bad;
        __syncthreads();
        uint32_t any = 0;
#pragma unroll
        for (int i = 0; i < NW; ++i) any |= flags[i];
        if (any) l = __builtin_nanf("");
    }
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    if (KEYS == TILE_PREFIX || a.parts > 1) {
        if (!row_ok) return;
        int64_t place;
        if constexpr (KEYS == TILE_PREFIX) { // sequence, key head, token, head of the key head
            const int64_t per = static_cast<int64_t>(a.new_tokens) * a.each, of = from * per + row;
            place = (of / per * a.kv_heads + kvh) * per + of % per;
        } else { // token, head
            place = static_cast<int64_t>(from + token) * a.heads + head;
        }
        place = place * a.parts + part;
        if (ntiles > 0) {
#pragma unroll
            for (int dt = 0; dt < DT; ++dt)
#pragma unroll
                for (int i = 0; i < 16; i += 4) {
                    const int d = dt * 32 + i * 2 + 4 * g;
                    if (d < dv) *reinterpret_cast<float4_t *>(a.part_out + place * dv + d) = float4_t{oacc[dt][i] * inv, oacc[dt][i + 1] * inv, oacc[dt][i + 2] * inv, oacc[dt][i + 3] * inv};
                }
        }
        // (what is no number makes the joined row none: +inf minus itself)
        if (g == 0) a.part_lse[place] = l == 0.0f ? NEG_INF_F : l == l ? m_run + __builtin_amdgcn_logf(l) : -NEG_INF_F;
        return;
    }
    uint16_t *const orow = static_cast<uint16_t *>(a.o) + (from + token) * a.os[1] + head * a.os[2];
    // a lane holds 4 consecutive dims of each group of 8; the halves trade every second group: 16 bytes a store
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
        for (int ip = 0; ip < 2; ++ip) {
            const int ia = 8 * ip, ib = 8 * ip + 4;
            const uint32_t x0 = pack2<BF16>(oacc[dt][ia] * inv, oacc[dt][ia + 1] * inv), x1 = pack2<BF16>(oacc[dt][ia + 2] * inv, oacc[dt][ia + 3] * inv);
            const uint32_t y0 = pack2<BF16>(oacc[dt][ib] * inv, oacc[dt][ib + 1] * inv), y1 = pack2<BF16>(oacc[dt][ib + 2] * inv, oacc[dt][ib + 3] * inv);
            const auto r0 = __builtin_amdgcn_permlane32_swap(x0, y0, false, false);
            const auto r1 = __builtin_amdgcn_permlane32_swap(x1, y1, false, false);
            const int d = dt * 32 + (2 * ip + g) * 8;
            if (row_ok && d < dv) *reinterpret_cast<uint4_t *>(orow + d) = uint4_t{r0[0], r1[0], r0[1], r1[1]};
        }
}

template <bool BF16, int D, int DE, int NW, int KEYS>
__global__ __launch_bounds__(64 * NW, NW == 8 || D > 128 ? 1 : 2) void sdpa_tile_kernel(const CacheArgs a) {
    tile_body<BF16, D, DE, NW, KEYS>(a, blockIdx.x);
}

template <bool BF16, int D, int DE, int NW, int KEYS> int launch_tile_as(const CacheArgs &a, hipStream_t s) {
    constexpr int lds = 4 * TK * 2 * D, BM = 32 * NW;
    if constexpr (lds > 65536) {
        static const hipError_t attr = hipFuncSetAttribute(reinterpret_cast<const void *>(&sdpa_tile_kernel<BF16, D, DE, NW, KEYS>), hipFuncAttributeMaxDynamicSharedMemorySize, lds);
        AXHIP_CHECK_HIP(attr);
    }
    const int64_t blocks = (a.total_q * a.each / BM + a.entries) * a.kv_heads * a.parts; // at most
    AXHIP_REQUIRE(launch_fits(blocks, 64 * NW), AXHIP_ERR_UNSUPPORTED, "attention of ragged sequences: grid too large");
    hipLaunchKernelGGL((sdpa_tile_kernel<BF16, D, DE, NW, KEYS>), dim3(static_cast<unsigned>(blocks)), dim3(64 * NW), lds, s, a);
    AXHIP_CHECK_HIP(hipGetLastError());
    return AXHIP_OK;
}
template <bool BF16, int KEYS> int launch_tile_keys(const CacheArgs &a, int waves, hipStream_t s) {
    if (a.D > 128) return launch_tile_as<BF16, 256, 256, 4, KEYS>(a, s);
    if (a.D > 96) return waves == 8 ? launch_tile_as<BF16, 128, 128, 8, KEYS>(a, s) : launch_tile_as<BF16, 128, 128, 4, KEYS>(a, s);
    if (a.D > 64) return launch_tile_as<BF16, 128, 96, 4, KEYS>(a, s);
    return launch_tile_as<BF16, 64, 64, 4, KEYS>(a, s);
}
template <bool BF16> int launch_tile(const CacheArgs &a, int waves, hipStream_t s) { return a.table ? launch_tile_keys<BF16, TILE_PAGED>(a, waves, s) : launch_tile_keys<BF16, TILE_PACKED>(a, waves, s); }

} // namespace axhip
