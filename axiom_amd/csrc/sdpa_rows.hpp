// Ragged attention of few rows against many keys, and of fp32: 16 rows of one entry and key head, four waves that take 16 or 32 keys in turn and meet once, at the end, through LDS.
//
// Nothing is shared before that: K and V go from memory straight into the operands of the matrix instructions.  In what order keys and dims run through an MFMA is free as
// long as both operands agree, so:
//   S^T = K Q^T    leaves lane (l16, g) with row l16 and keys 4 g + i of a 16-key sub-tile;
//   O^T = V^T P^T  takes those keys as its k-slots (the probabilities are its B operand as they stand), and the lane needs, of V, rows of its own keys: in 16 bits 16-byte runs
//                  whose transpose is byte permutes between its registers, in fp32 the elements as they come.
// Bound by one read of K and V (decoding): a step's 16 loads are requested a step ahead, the page numbers they need a step earlier.  64 sequences of 2000 keys, 8 key heads of 128: 97 us and the join's
// 5 for 524 MB, 5.1 TB/s in all; one of 8000 keys: 11 and 4.7, which are latencies.  fp32 prompts are bound by v_mfma_f32_16x16x4 and by a work-group's start and end.
//
// A decoding step deals all its own keys out to its work-groups in equal shares, found from the lengths on the device, so that every CU has as much to do whatever they are: own_share
// below.  A share may be a part of one sequence or several whole ones.  A sequence within one share and without a prefix is finished there; the others leave fp32 results and the
// base-2 logarithm of their denominators for sdpa_join_kernel.
#pragma once

#include "sdpa_cache.hpp"
#include "sdpa_tile_item.hpp"

#include <type_traits>

namespace axhip {

typedef float rows_f32x4 __attribute__((ext_vector_type(4)));
template <int DT> __device__ __forceinline__ rows_f32x4 rows_mfma(uint4_t a, uint4_t b, rows_f32x4 c) {
    if constexpr (DT == AXHIP_DTYPE_BF16) return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, a), __builtin_bit_cast(bf16x8_t, b), c, 0, 0, 0);
    else return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(half8_t, a), __builtin_bit_cast(half8_t, b), c, 0, 0, 0);
}

constexpr int ROWS_WAVES = 4, ROWS = 16;
template <int D> constexpr int rows_lds_bytes() { return ROWS_WAVES * ROWS * (D + 4 + 2) * 4; }

// Keys are dealt out in units of UNIT; a sequence has one at least, so that somebody writes its rows.  With U units in all and W <= U shares, share i begins at unit i U / W, and unit u
// lies in share ((u + 1) W - 1) / U.  What a share leaves of a sequence that others have parts of goes to slot 2 i where the sequence began at the share's first unit or in front of it, else
// (it is the share's last one then) to slot 2 i + 1; of a whole sequence s that has a prefix, to slot 2 W + s.
constexpr int UNIT = 128;
__device__ __forceinline__ int units_of(int keys) { return max(1, (keys + UNIT - 1) / UNIT); }
struct Share { int units, shares, from, to, entry, entry_at; }; // of all; how many shares; this one's units; the sequence that the first one lies in, and its first unit
// By a wavefront; up to 256 sequences four to a lane, more in runs, one to a lane.
__device__ inline Share own_share(const CacheArgs &a, int index) {
    const int lane = threadIdx.x % WAVE, n = a.entries;
    auto scan = [&](int v, int count) { // over the first `count` lanes: as many trips as they need
#pragma unroll
        for (int d = 1; d < WAVE; d *= 2) {
            if (d >= count) break;
            const int other = __shfl_up(v, d, WAVE);
            if (lane >= d) v += other;
        }
        return v;
    };
    const bool few = n <= 4 * WAVE;
    const int run = (n + WAVE - 1) / WAVE, run_from = min(lane * run, n), run_to = min(run_from + run, n);
    int u[4] = {0, 0, 0, 0}, upto[4], total = 0;
    if (few) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (WAVE * i < n && lane + WAVE * i < n) u[i] = units_of(keys_of(a, lane + WAVE * i).n);
    } else {
        for (int e = run_from; e < run_to; ++e) u[0] += units_of(keys_of(a, e).n);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        upto[i] = 0;
        if (i > 0 && (!few || WAVE * i >= n)) continue;
        const int count = few ? min(n - WAVE * i, WAVE) : WAVE;
        upto[i] = total + scan(u[i], count);
        total = __builtin_amdgcn_readlane(upto[i], count - 1);
    }
    Share s;
    s.units = total;
    s.shares = min(a.shares, total); // (none is empty)
    s.from = s.to = s.entry = s.entry_at = 0;
    if (index >= s.shares) return s;
    if (total < (1 << 20) && s.shares < (1 << 11)) { // (a division of 64 bits is a hundred instructions)
        s.from = static_cast<int>(static_cast<uint32_t>(index * total) / static_cast<uint32_t>(s.shares));
        s.to = static_cast<int>(static_cast<uint32_t>((index + 1) * total) / static_cast<uint32_t>(s.shares));
    } else {
        s.from = static_cast<int>(static_cast<int64_t>(index) * total / s.shares);
        s.to = static_cast<int>(static_cast<int64_t>(index + 1) * total / s.shares);
    }
    bool found = false;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if (found || (i > 0 && (!few || WAVE * i >= n))) continue;
        const uint64_t beyond = __builtin_amdgcn_ballot_w64(upto[i] > s.from);
        if (beyond) {
            const int at = __builtin_ctzll(beyond);
            s.entry = at + WAVE * i;
            s.entry_at = __builtin_amdgcn_readlane(upto[i] - u[i], at);
            found = true;
        }
    }
    if (!few) { // within that lane's run
        int e = s.entry * run;
        for (; e < n - 1; ++e) {
            const int more = units_of(keys_of(a, e).n);
            if (s.entry_at + more > s.from) break;
            s.entry_at += more;
        }
        s.entry = e;
    }
    return s;
}

// What a work-group does: OWN, a share of all own keys (decoding); PACKED, 16 rows of a sequence by cu_q, or a part of their keys (prompts of fp32, and of few rows each); PREFIX, a part of a group's prefix for 16 of its
// rows (fp32); WHOLE, all keys of 16 rows, prefix and own (decoding, not divided).  Its four waves take the keys in turn and meet at the end.  APART: as PACKED, 64 rows, 16 to a wave, each of which
// walks all keys: where there are blocks enough, a quarter of the work-groups, whose start and end cost as much as 250 keys, and nothing to meet for.
enum RowsMode { ROWS_OWN = 0, ROWS_PACKED = 1, ROWS_PREFIX = 2, ROWS_WHOLE = 3, ROWS_APART = 4 };

// The rows of a work-group: ROWS from row0 on of `rows`, of a sequence or a group; and the keys [begin, end) of one run of keys that it takes next.
struct RowTile { int kvh, row0, rows; };
struct Segment {
    KeyRun run;
    int entry, begin, end, tokens, q_from; // tokens: of the entry, the last of which sees the last key (0: every row sees every key); q_from: its first token, or a group's first sequence
    bool more;                             // the segment behind it is of the same rows: nothing is finished yet
    int64_t slot;                          // where the results go for the join: own parts: their place; else the part's number; below 0: they are finished here
};

// Segments come from next(segment), one behind the other, until it answers false.  Their steps are one stream: while a wave works on a step, the next one's K and V are on their way and
// the page numbers of the one behind that, whether or not they are of the same segment.
template <int DT, int D, bool PAD, int OF, class Next> __device__ __forceinline__ void rows_stream(const CacheArgs &a, const RowTile &tile, Next next) {
    constexpr bool APART = OF == ROWS_APART;
    constexpr int MODE = APART ? ROWS_PACKED : OF;
    constexpr bool F32 = DT == AXHIP_DTYPE_F32;
    constexpr int ES = F32 ? 4 : 2;
    constexpr int SUB = F32 && D > 64 ? 1 : 2, KEYS = 16 * SUB, STRIDE = APART ? KEYS : KEYS * ROWS_WAVES;
    constexpr int KJ = F32 ? D / 16 : D / 32; // 16-byte pieces of a K row that a lane holds
    constexpr int NT = D / 16;                // 16 bits: output tiles, and elements of V that a lane holds of a key
    constexpr int VH = F32 ? D / 64 : (NT * 2 + 15) / 16; // 16-byte pieces of a V row that a lane holds (D = 64 in 16 bits: half of one)
    constexpr int VW = F32 ? 4 * VH : NT / 2;             // 32-bit words of that
    static_assert(!F32 || D <= 128, "fp32 head sizes");
    static_assert(!APART || F32, "the results lie as 32-bit ones do");
    // Large fp32 heads: a step's K takes the place of the one whose scores are done, its V of the one whose output is (two of each, and the registers do not suffice); those products take long
    // enough for the loads
    constexpr bool LEAN = F32 && D > 64;
    extern __shared__ __attribute__((aligned(1024))) unsigned char tile_lds[];
    float *const rows_lds = reinterpret_cast<float *>(tile_lds);
    const int tid = threadIdx.x, lane = tid % WAVE, wave = __builtin_amdgcn_readfirstlane(tid / WAVE), l16 = lane % 16, g = lane / 16;
    const int dv = a.D, kvh = tile.kvh, row0 = tile.row0, rows = tile.rows;

    // ---- this lane's row
    const int row = min(row0 + l16, rows - 1);
    const bool row_ok = row0 + l16 < rows;
    const int row_token = static_cast<int>(a.by_each.of(row)), first_token = static_cast<int>(a.by_each.of(row0));
    auto place_of = [&](const Segment &seg, int r) { // of the element strides
        const int token = static_cast<int>(a.by_each.of(r)), head = kvh * a.each + r - token * a.each;
        struct { int64_t q, o; } at;
        if constexpr (MODE == ROWS_PACKED) {
            at.q = (seg.q_from + token) * a.qs[1] + head * a.qs[2];
            at.o = (seg.q_from + token) * a.os[1] + head * a.os[2];
        } else {
            constexpr bool OF_GROUP = MODE == ROWS_PREFIX;
            const int seq = OF_GROUP ? seg.q_from + token / a.new_tokens : seg.entry, t = OF_GROUP ? token % a.new_tokens : token;
            at.q = seq * a.qs[0] + t * a.qs[1] + head * a.qs[2];
            at.o = seq * a.os[0] + t * a.os[1] + head * a.os[2];
        }
        return at;
    };
    struct Queries { uint4_t f[KJ]; };
    auto queries_of = [&](const Segment &seg) __attribute__((always_inline)) {
        Queries q;
        const unsigned char *from = static_cast<const unsigned char *>(a.q) + place_of(seg, row).q * ES;
#pragma unroll
        for (int j = 0; j < KJ; ++j) {
            const int d = F32 ? 16 * j + 4 * g : 32 * j + 8 * g;
            q.f[j] = row_ok && d < dv ? *reinterpret_cast<const uint4_t *>(from + d * ES) : uint4_t{0, 0, 0, 0};
        }
        return q;
    };

    // ---- K and V from memory.  Rows behind the last key are that key again; dims behind the head size: of K zeros, of V the first ones again, whose results nobody stores.
    const unsigned char *kb = static_cast<const unsigned char *>(a.k) + kvh * a.ks[2] * ES, *vb = static_cast<const unsigned char *>(a.v) + kvh * a.vs[2] * ES;
    const int64_t k_page = a.ks[0] * ES, v_page = a.vs[0] * ES, k_row = a.ks[1] * ES, v_row = a.vs[1] * ES;
    int k_dim[KJ], v_dim[VH]; // bytes into a row
    bool k_in[KJ];
#pragma unroll
    for (int j = 0; j < KJ; ++j) {
        const int d = F32 ? 16 * j + 4 * g : 32 * j + 8 * g;
        k_in[j] = d < dv;
        k_dim[j] = (PAD && d >= dv ? 0 : d) * ES;
    }
#pragma unroll
    for (int h = 0; h < VH; ++h) {
        const int d = F32 ? 64 * h + 4 * l16 : NT * l16 + 8 * h;
        v_dim[h] = (PAD && d >= dv ? 0 : d) * ES;
    }
    struct Ids { int k[SUB], v[SUB]; };
    const int mask = (1 << a.page_shift) - 1;
    bool bad = false, bad_next = false; // a page that does not exist, of the segment at hand and of the next one
    uint4_t kf[SUB][KJ];
    uint32_t vf[SUB][4][VW];
    auto ids_at = [&](const KeyRun &run, int at) __attribute__((always_inline)) {
        Ids p;
#pragma unroll
        for (int u = 0; u < SUB; ++u) {
            p.k[u] = run.table ? run.table[min(at + 16 * u + l16, run.n - 1) >> a.page_shift] : 0;
            p.v[u] = run.table ? run.table[min(at + 16 * u + 4 * g, run.n - 1) >> a.page_shift] : 0;
        }
        return p;
    };
    auto load = [&](const KeyRun &run, int at, Ids p, auto with_k, auto with_v) __attribute__((always_inline)) { // whether all pages exist
        constexpr bool K = decltype(with_k)::value, V = decltype(with_v)::value;
        bool exist = true;
#pragma unroll
        for (int u = 0; u < SUB; ++u) {
            const int key = min(at + 16 * u + l16, run.n - 1), vkey = min(at + 16 * u + 4 * g, run.n - 1);
            const unsigned char *k = kb, *v = vb;
            if (run.table) {
                if (static_cast<uint32_t>(p.k[u]) >= static_cast<uint32_t>(a.n_pages) || static_cast<uint32_t>(p.v[u]) >= static_cast<uint32_t>(a.n_pages)) {
                    exist = false;
                    p.k[u] = p.v[u] = 0;
                }
                k += p.k[u] * k_page + (key & mask) * k_row;
                v += p.v[u] * v_page + (vkey & mask) * v_row;
            } else {
                k += (run.base + key) * k_row;
                v += (run.base + vkey) * v_row;
            }
#pragma unroll
            for (int j = 0; K && j < KJ; ++j) kf[u][j] = *reinterpret_cast<const uint4_t *>(k + k_dim[j]);
#pragma unroll
            for (int i = 0; V && i < 4; ++i) {
                const unsigned char *vi = v + min(i, run.n - 1 - vkey) * v_row;
                if constexpr (!F32 && D == 64) {
                    const uint2_t t = *reinterpret_cast<const uint2_t *>(vi + v_dim[0]);
                    vf[u][i][0] = t.x;
                    vf[u][i][1] = t.y;
                } else {
#pragma unroll
                    for (int h = 0; h < VH; ++h) {
                        const uint4_t t = *reinterpret_cast<const uint4_t *>(vi + v_dim[h]);
#pragma unroll
                        for (int c = 0; c < 4; ++c) vf[u][i][4 * h + c] = t[c];
                    }
                }
            }
        }
        return exist;
    };

    constexpr int NACC = F32 ? 4 * VH : NT; // fp32: tile 4 h + c holds dims 64 h + 4 (4 g + i) + c; 16 bits: tile t dims (4 g + i) NT + t
    rows_f32x4 oacc[NACC];
    float m_run, l_run;
    auto fresh = [&]() __attribute__((always_inline)) {
#pragma unroll
        for (int t = 0; t < NACC; ++t) oacc[t] = rows_f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        m_run = NEG_INF_F;
        l_run = 0.0f;
    };
    fresh();

    // The wave's steps: one in registers (loaded), one whose page numbers are on their way (wanted); below 0: none.  *_next: of the segment behind the one at hand.
    Segment cur{}, nxt{};
    if (!next(cur)) return;
    bool has_next = next(nxt);
    int loaded, wanted;
    bool loaded_next = false, wanted_next = false;
    auto first_of = [&](const Segment &seg) { const int at = seg.begin + (APART ? 0 : KEYS * wave); return at < seg.end ? at : -1; };
    auto behind = [&](int at, bool of_next) { // the step behind one: into `wanted`
        wanted_next = of_next;
        wanted = at + STRIDE < (of_next ? nxt.end : cur.end) ? at + STRIDE : -1;
        if (wanted < 0 && !of_next) {
            wanted_next = true;
            wanted = has_next ? first_of(nxt) : -1;
        }
    };
    Ids ids{};
    auto want_ids = [&]() __attribute__((always_inline)) { if (wanted >= 0) ids = ids_at(wanted_next ? nxt.run : cur.run, wanted); };
    constexpr std::true_type yes{};
    constexpr std::false_type no{};
    auto load_wanted_k = [&]() __attribute__((always_inline)) { if (wanted >= 0) load(wanted_next ? nxt.run : cur.run, wanted, ids, yes, no); };
    auto load_wanted = [&](auto with_k) __attribute__((always_inline)) { // .. and on to the next one
        loaded = wanted;
        loaded_next = wanted_next;
        if (wanted < 0) return;
        const bool exist = load(wanted_next ? nxt.run : cur.run, wanted, ids, with_k, yes);
        if (wanted_next) bad_next = bad_next || !exist;
        else bad = bad || !exist;
        behind(loaded, loaded_next);
        want_ids();
    };
    auto start = [&]() __attribute__((always_inline)) { // nothing is loaded: from the first step of this segment, or of the next one
        wanted = first_of(cur);
        wanted_next = wanted < 0;
        if (wanted_next) wanted = has_next ? first_of(nxt) : -1;
        want_ids();
        load_wanted(yes);
    };
    Queries q = queries_of(cur), q_next{};
    start();
    if (MODE == ROWS_OWN && has_next) q_next = queries_of(nxt);

    for (;;) {
    const int limit = cur.tokens ? min(cur.end - 1, cur.run.n - cur.tokens + row_token) : cur.end - 1;   // last key that this row sees
    const int least = cur.tokens ? min(cur.end - 1, cur.run.n - cur.tokens + first_token) : cur.end - 1; // .. that every row of the tile sees
    while (loaded >= 0 && !loaded_next) {
        uint4_t kc[SUB][KJ];
        uint32_t vc[SUB][4][VW];
#pragma unroll
        for (int u = 0; u < SUB; ++u) {
#pragma unroll
            for (int j = 0; j < KJ; ++j) kc[u][j] = PAD && !k_in[j] ? uint4_t{0, 0, 0, 0} : kf[u][j];
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int c = 0; c < VW; ++c) vc[u][i][c] = vf[u][i][c];
        }
        const int now = loaded;
        if constexpr (!LEAN) load_wanted(yes);

        rows_f32x4 s[SUB];
#pragma unroll
        for (int u = 0; u < SUB; ++u) s[u] = rows_f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int j = 0; j < KJ; ++j)
#pragma unroll
            for (int u = 0; u < SUB; ++u) {
                if constexpr (F32) {
#pragma unroll
                    for (int c = 0; c < 4; ++c) s[u] = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(kc[u][j][c]), __uint_as_float(q.f[j][c]), s[u], 0, 0, 0);
                } else {
                    s[u] = rows_mfma<DT>(kc[u][j], q.f[j], s[u]);
                }
            }
        if constexpr (LEAN) {
            __builtin_amdgcn_sched_barrier(0);
            load_wanted_k();
            __builtin_amdgcn_sched_barrier(0);
        }
        if (now + KEYS - 1 > least) {
#pragma unroll
            for (int u = 0; u < SUB; ++u)
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (now + 16 * u + 4 * g + i > limit) s[u][i] = NEG_INF_F;
        }
        float top = NEG_INF_F;
#pragma unroll
        for (int u = 0; u < SUB; ++u)
#pragma unroll
            for (int i = 0; i < 4; ++i) top = fmaxf(top, s[u][i]);
        top = across32(across16(top, lanes_max), lanes_max);
        const float m_new = fmaxf(m_run, top * a.scale_log2e);
        if (__builtin_amdgcn_ballot_w64(m_new - m_run > RESCALE_THRESHOLD) != 0) {
            const float alpha = m_new == NEG_INF_F ? 1.0f : __builtin_amdgcn_exp2f(m_run - m_new);
            m_run = m_new;
            l_run *= alpha;
#pragma unroll
            for (int t = 0; t < NACC; ++t) oacc[t] *= alpha;
        }
        const float minus = m_run == NEG_INF_F ? 0.0f : -m_run;
        float p[SUB][4];
#pragma unroll
        for (int u = 0; u < SUB; ++u)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                p[u][i] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[u][i], a.scale_log2e, minus));
                l_run += p[u][i];
            }
        if constexpr (F32) {
#pragma unroll
            for (int u = 0; u < SUB; ++u)
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int t = 0; t < NACC; ++t) oacc[t] = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(vc[u][i][t]), p[u][i], oacc[t], 0, 0, 0);
            if constexpr (LEAN) {
                __builtin_amdgcn_sched_barrier(0);
                load_wanted(no);
            }
        } else {
            uint4_t pf; // slot 8 g + e of the second product is key 4 g + e % 4 of sub-tile e / 4
#pragma unroll
            for (int e = 0; e < 4; ++e) pf[e] = pack2<DT == AXHIP_DTYPE_BF16>(p[e / 2][2 * (e % 2)], p[e / 2][2 * (e % 2) + 1]);
#pragma unroll
            for (int t = 0; t < NACC; ++t) {
                uint4_t vt;
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    vt[e] = __builtin_amdgcn_perm(vc[e / 2][2 * (e % 2) + 1][t / 2], vc[e / 2][2 * (e % 2)][t / 2], t % 2 ? 0x07060302u : 0x05040100u);
                oacc[t] = rows_mfma<DT>(vt, pf, oacc[t]);
            }
        }
    }

    if constexpr (APART) {
        // ---- a lane holds 4 dims of its row in a place
        float den = across32(across16(l_run, lanes_add), lanes_add);
        if (__builtin_amdgcn_ballot_w64(bad)) den = __builtin_nanf("");
        if (!row_ok) return; // (one segment)
        const float inv = den == 0.0f ? 0.0f : 1.0f / den;
        float *const to = static_cast<float *>(a.o) + place_of(cur, row0 + l16).o;
#pragma unroll
        for (int h = 0; h < VH; ++h)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int d = 64 * h + 16 * g + 4 * i;
                if (d < dv) *reinterpret_cast<rows_f32x4 *>(to + d) = rows_f32x4{oacc[4 * h][i], oacc[4 * h + 1][i], oacc[4 * h + 2][i], oacc[4 * h + 3][i]} * inv;
            }
        return;
    }
    if (!cur.more) {
    // ---- the four waves' states meet: [wave][row][D + 4], then maxima and denominators
    const float l_tot = across32(across16(l_run, lanes_add), lanes_add);
    float *const tops = rows_lds + ROWS_WAVES * ROWS * (D + 4), *const dens = tops + ROWS_WAVES * ROWS;
    {
        float *mine = rows_lds + (wave * ROWS + l16) * (D + 4);
        if constexpr (F32) {
#pragma unroll
            for (int h = 0; h < VH; ++h)
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    *reinterpret_cast<rows_f32x4 *>(mine + 64 * h + 16 * g + 4 * i) = rows_f32x4{oacc[4 * h][i], oacc[4 * h + 1][i], oacc[4 * h + 2][i], oacc[4 * h + 3][i]};
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int t = 0; t < NT; t += 4)
                    *reinterpret_cast<rows_f32x4 *>(mine + (4 * g + i) * NT + t) = rows_f32x4{oacc[t][i], oacc[t + 1][i], oacc[t + 2][i], oacc[t + 3][i]};
        }
        if (g == 0) {
            tops[wave * ROWS + l16] = m_run;
            dens[wave * ROWS + l16] = l_tot;
        }
    }
    const int any_bad = __syncthreads_or(bad);

    const bool leave = cur.slot >= 0;
    for (int item = tid; item < ROWS * (D / 4); item += 64 * ROWS_WAVES) {
        const int r = item / (D / 4), d = item % (D / 4) * 4;
        if (row0 + r >= rows || d >= dv) continue;
        float top = NEG_INF_F, den = 0.0f;
        rows_f32x4 o = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int w = 0; w < ROWS_WAVES; ++w) top = fmaxf(top, tops[w * ROWS + r]);
        if (top != NEG_INF_F) {
#pragma unroll
            for (int w = 0; w < ROWS_WAVES; ++w) {
                const float scale = __builtin_amdgcn_exp2f(tops[w * ROWS + r] - top);
                o += scale * *reinterpret_cast<const rows_f32x4 *>(rows_lds + (w * ROWS + r) * (D + 4) + d);
                den += scale * dens[w * ROWS + r];
            }
        } else { // no key of this row, or no number among its scores
#pragma unroll
            for (int w = 0; w < ROWS_WAVES; ++w) den += dens[w * ROWS + r];
        }
        if (any_bad) den = __builtin_nanf("");
        o *= den == 0.0f ? 0.0f : 1.0f / den;
        if (leave) {
            float *outs = a.part_out, *lses = a.part_lse;
            int64_t place;
            if constexpr (MODE == ROWS_PREFIX) {
                const int64_t of = static_cast<int64_t>(cur.q_from) * a.new_tokens * a.each + row0 + r; // sequence, token, head of the key head
                const int64_t per = static_cast<int64_t>(a.new_tokens) * a.each;
                place = ((of / per * a.kv_heads + kvh) * per + of % per) * a.parts + cur.slot;
            } else if constexpr (MODE == ROWS_PACKED) {
                place = (static_cast<int64_t>(cur.q_from + (row0 + r) / a.each) * a.heads + kvh * a.each + (row0 + r) % a.each) * a.parts + cur.slot;
            } else {
                place = (cur.slot * a.kv_heads + kvh) * rows + row0 + r;
                outs = a.own_out;
                lses = a.own_lse;
            }
            *reinterpret_cast<rows_f32x4 *>(outs + place * dv + d) = o;
            // (what is no number makes the joined row none: +inf minus itself)
            if (d == 0) lses[place] = den == 0.0f ? NEG_INF_F : den == den ? top + __builtin_amdgcn_logf(den) : -NEG_INF_F;
        } else {
            unsigned char *out = static_cast<unsigned char *>(a.o) + (place_of(cur, row0 + r).o + d) * ES;
            if constexpr (F32) *reinterpret_cast<rows_f32x4 *>(out) = o;
            else *reinterpret_cast<uint2_t *>(out) = uint2_t{pack2<DT == AXHIP_DTYPE_BF16>(o[0], o[1]), pack2<DT == AXHIP_DTYPE_BF16>(o[2], o[3])};
        }
    }
    }
    // ---- on to the next segment
    if (!has_next) return;
    if (!cur.more) {
        fresh();
        bad = false;
        __syncthreads(); // (the states in LDS are read)
    }
    bad = bad || bad_next;
    bad_next = false;
    cur = nxt;
    if constexpr (MODE == ROWS_OWN) q = q_next;
    has_next = next(nxt);
    if (MODE == ROWS_OWN && has_next) q_next = queries_of(nxt);
    loaded_next = false;
    wanted_next = false;
    if (loaded < 0) {
        start();
    } else if (wanted < 0) {
        behind(loaded, false);
        want_ids();
    }
    }
}

template <int DT, int D, bool PAD, int MODE> __device__ __forceinline__ void rows_body(const CacheArgs &a, int index_of_all) {
    RowTile tile{index_of_all % a.kv_heads, 0, 0};
    int rest = index_of_all / a.kv_heads;
    if constexpr (MODE == ROWS_OWN) {
        tile.rows = a.new_tokens * a.each;
        const int tiles = (tile.rows + ROWS - 1) / ROWS, share = rest / tiles;
        tile.row0 = rest % tiles * ROWS;
        const Share s = own_share(a, share);
        const int from = __builtin_amdgcn_readfirstlane(s.from), to = __builtin_amdgcn_readfirstlane(s.to);
        int entry = __builtin_amdgcn_readfirstlane(s.entry), entry_at = __builtin_amdgcn_readfirstlane(s.entry_at), at = from;
        KeyRun ahead = at < to ? keys_of(a, entry) : KeyRun{}; // (a segment before it is needed)
        rows_stream<DT, D, PAD, MODE>(a, tile, [&](Segment &seg) {
            if (at >= to) return false;
            const int n = __builtin_amdgcn_readfirstlane(ahead.n), entry_to = entry_at + units_of(n);
            seg.run = ahead;
            seg.run.n = n;
            seg.entry = entry;
            seg.tokens = a.new_tokens;
            seg.begin = (at - entry_at) * UNIT;
            seg.end = min(n, (min(to, entry_to) - entry_at) * UNIT);
            const bool whole = entry_at >= from && entry_to <= to;
            seg.slot = 2 * share + (entry_at <= from ? 0 : 1);
            if (whole) {
                const int group = a.groups > 0 ? group_of(a, entry) : -1;
                seg.slot = group >= 0 && prefix_of(a, group).n > 0 ? 2 * a.shares + entry : -1;
            }
            if (entry_at >= from && tile.kvh == 0 && tile.row0 == 0 && threadIdx.x == 0) {
                const int last = static_cast<int>((static_cast<int64_t>(entry_to) * s.shares - 1) / s.units);
                a.parts_of[entry] = int2_t{static_cast<int>(seg.slot), seg.slot < 0 ? 0 : last - share + 1};
            }
            at = entry_at = entry_to;
            ++entry;
            if (at < to) ahead = keys_of(a, entry);
            return true;
        });
    } else if constexpr (MODE == ROWS_WHOLE) {
        tile.rows = a.new_tokens * a.each;
        const int tiles = (tile.rows + ROWS - 1) / ROWS, entry = rest / tiles;
        tile.row0 = rest % tiles * ROWS;
        KeyRun own = keys_of(a, entry), prefix{};
        const int group = a.groups > 0 ? group_of(a, entry) : -1;
        if (group >= 0) prefix = prefix_of(a, group);
        own.n = __builtin_amdgcn_readfirstlane(own.n);
        prefix.n = __builtin_amdgcn_readfirstlane(prefix.n);
        int count = prefix.n > 0 ? 0 : 1; // the prefix, which every row sees, then the sequence's own keys
        rows_stream<DT, D, PAD, MODE>(a, tile, [&](Segment &seg) {
            if (count > 1) return false;
            const KeyRun &run = count == 0 ? prefix : own;
            seg = Segment{run, entry, 0, run.n, count == 0 ? 0 : a.new_tokens, 0, count == 0, -1};
            ++count;
            return true;
        });
    } else {
        constexpr bool APART = MODE == ROWS_APART;
        constexpr int BM = APART ? ROWS * ROWS_WAVES : ROWS;
        const int to_row = APART ? __builtin_amdgcn_readfirstlane(threadIdx.x / WAVE) * ROWS : 0; // (a wave without rows has nothing to wait for)
        Segment only{};
        only.slot = -1;
        if constexpr (MODE == ROWS_PACKED || MODE == ROWS_APART) {
            int part = 0;
            if (a.parts > 1) {
                part = rest % a.parts;
                rest /= a.parts;
            }
            const TileItem item = tile_item<BM>(a, rest);
            if (item.entry < 0 || item.row0 + to_row >= item.tokens.n * a.each) return;
            only.entry = item.entry;
            only.tokens = a.causal ? item.tokens.n : 0;
            only.q_from = item.tokens.from;
            tile.rows = item.tokens.n * a.each;
            tile.row0 = item.row0 + to_row;
            only.run = KeyRun{a.table ? a.table + item.entry * a.table_ld : nullptr, item.base, item.keys};
            only.end = a.causal ? item.keys - item.tokens.n + static_cast<int>(a.by_each.of(min(tile.row0 + ROWS, tile.rows) - 1)) + 1 : item.keys;
            if (a.parts > 1) {
                const int chunk = part_keys(a, max(0, only.end));
                only.begin = part * chunk;
                only.end = min(only.end, only.begin + chunk);
                only.slot = part;
            }
        } else {
            const int part = rest % a.parts;
            const GroupItem item = group_item<ROWS>(a, rest / a.parts);
            only.entry = __builtin_amdgcn_readfirstlane(item.group);
            if (only.entry < 0) return;
            tile.rows = item.rows;
            tile.row0 = item.row0;
            only.q_from = item.first;
            only.run = prefix_of(a, only.entry);
            only.run.n = __builtin_amdgcn_readfirstlane(only.run.n);
            const int chunk = part_keys(a, only.run.n);
            only.begin = part * chunk;
            only.end = min(only.run.n, only.begin + chunk);
            if (only.begin >= only.run.n) return; // (as many parts as that are there for the join)
            only.slot = part;
        }
        bool first = true;
        rows_stream<DT, D, PAD, MODE>(a, tile, [&](Segment &seg) {
            if (!first) return false;
            seg = only;
            first = false;
            return true;
        });
    }
}
template <int DT, int D, bool PAD, int MODE>
__global__ __launch_bounds__(64 * ROWS_WAVES, D > 128 ? 1 : 2) void sdpa_rows_kernel(const CacheArgs a) {
    rows_body<DT, D, PAD, MODE>(a, blockIdx.x);
}

// out = sum_s 2^(lse_s - max lse) O_s / sum_s 2^(lse_s - max lse) over a row's prefix parts and own parts, in that order.  WAVES wavefronts to a row take them in turn, D / 4 lanes a
// result, and everything that fits the first trip to memory is requested before the weights are known.
// PACKED: of prompts, whose rows are token and head and which have a.parts each; rows that no sequence owns are left as they are.
template <int DT, int D, int WAVES, bool PACKED>
__global__ __launch_bounds__(256) void sdpa_join_kernel(const CacheArgs a) {
    constexpr int LANES = D / 4, TAKE = WAVE / LANES * WAVES, AHEAD = 8;
    __shared__ __attribute__((aligned(16))) float sums[4][D + 4];
    const int lane = threadIdx.x % WAVE, wave = threadIdx.x / WAVE, d = lane % LANES * 4, first = wave % WAVES * (WAVE / LANES) + lane / LANES;
    const int64_t id = static_cast<int64_t>(blockIdx.x) * (4 / WAVES) + wave / WAVES; // sequence, token, head
    int64_t pre, at;
    int prefix = 0, n, kvh = 0, row = 0, rows = 0;
    int2_t own = {0, 0};
    if constexpr (PACKED) {
        if (id >= a.total_q * a.heads) return; // (whole work-groups with WAVES = 4)
        const int token = static_cast<int>(id / a.heads), head = static_cast<int>(id % a.heads);
        const int e = last_not_beyond(a.entries, token, [&](int i) { return a.cu_q[i]; });
        if (a.cu_q[e] > token || a.cu_q[e + 1] <= token) return;
        prefix = n = a.parts;
        pre = id * a.parts;
        at = token * a.os[1] + head * a.os[2] + d;
    } else {
        const int per = a.new_tokens * a.heads;
        if (id >= static_cast<int64_t>(a.entries) * per) return;
        const int seq = static_cast<int>(id / per), token = static_cast<int>(id % per) / a.heads, head = static_cast<int>(id % per) % a.heads;
        kvh = head / a.each;
        row = token * a.each + head % a.each;
        rows = a.new_tokens * a.each;
        own = a.parts_of[seq];
        if (own.y == 0) return; // finished already
        if (a.groups > 0) {
            const int group = group_of(a, seq);
            if (group >= 0) {
                const int keys = prefix_of(a, group).n, chunk = part_keys(a, keys);
                prefix = (keys + chunk - 1) / chunk;
            }
        }
        n = prefix + own.y;
        pre = ((static_cast<int64_t>(seq) * a.kv_heads + kvh) * rows + row) * a.parts;
        at = seq * a.os[0] + token * a.os[1] + head * a.os[2] + d;
    }
    // (own parts: the first share's slot, then the first slots of the shares behind it)
    auto place = [&](int i) { return PACKED || i < prefix ? pre + i : (static_cast<int64_t>(i == prefix ? own.x : own.x / 2 * 2 + 2 * (i - prefix)) * a.kv_heads + kvh) * rows + row; };
    auto lse = [&](int i) { return (PACKED || i < prefix ? a.part_lse : a.own_lse)[place(i)]; };
    rows_f32x4 o[AHEAD];
    float w[AHEAD];
    auto fetch = [&](int i0) __attribute__((always_inline)) {
#pragma unroll
        for (int k = 0; k < AHEAD; ++k) {
            const int i = min(i0 + TAKE * k, n - 1);
            w[k] = i0 + TAKE * k < n ? lse(i) : NEG_INF_F;
            o[k] = *reinterpret_cast<const rows_f32x4 *>((PACKED || i < prefix ? a.part_out : a.own_out) + place(i) * a.D + (d < a.D ? d : 0));
        }
    };
    float top = NEG_INF_F;
    for (int i = lane; i < n; i += WAVE) top = fmaxf(top, lse(i));
    fetch(first);
    __builtin_amdgcn_sched_barrier(0);
    top = wave_max(top);
    float den = 0.0f;
    rows_f32x4 acc = {0.0f, 0.0f, 0.0f, 0.0f};
    if (top != NEG_INF_F) {
        for (int i0 = first;;) {
#pragma unroll
            for (int k = 0; k < AHEAD; ++k) {
                const float e = w[k] == NEG_INF_F ? 0.0f : __builtin_amdgcn_exp2f(w[k] - top);
                den += e;
                acc += e == 0.0f ? rows_f32x4{0.0f, 0.0f, 0.0f, 0.0f} : e * o[k];
            }
            i0 += TAKE * AHEAD;
            if (i0 >= n) break;
            fetch(i0);
        }
    }
#pragma unroll
    for (int x = LANES; x < WAVE; x *= 2) {
        den += __shfl_xor(den, x, WAVE);
#pragma unroll
        for (int c = 0; c < 4; ++c) acc[c] += __shfl_xor(acc[c], x, WAVE);
    }
    if constexpr (WAVES == 4) {
        if (lane < LANES) *reinterpret_cast<rows_f32x4 *>(&sums[wave][d]) = acc;
        if (lane == 0) sums[wave][D] = den;
        __syncthreads();
        if (wave != 0) return;
        acc = *reinterpret_cast<const rows_f32x4 *>(&sums[0][d]);
        den = sums[0][D];
#pragma unroll
        for (int i = 1; i < 4; ++i) {
            acc += *reinterpret_cast<const rows_f32x4 *>(&sums[i][d]);
            den += sums[i][D];
        }
    }
    if (lane >= LANES || d >= a.D) return;
    acc *= den == 0.0f ? 0.0f : 1.0f / den;
    if constexpr (DT == AXHIP_DTYPE_F32) *reinterpret_cast<rows_f32x4 *>(static_cast<float *>(a.o) + at) = acc;
    else *reinterpret_cast<uint2_t *>(static_cast<uint16_t *>(a.o) + at) = uint2_t{pack2<DT == AXHIP_DTYPE_BF16>(acc[0], acc[1]), pack2<DT == AXHIP_DTYPE_BF16>(acc[2], acc[3])};
}

template <int DT, int D, bool PAD, int MODE> int launch_rows_as(const CacheArgs &a, int64_t blocks, hipStream_t s) {
    constexpr int lds = rows_lds_bytes<D>();
    if constexpr (lds > 65536) {
        static const hipError_t attr = hipFuncSetAttribute(reinterpret_cast<const void *>(&sdpa_rows_kernel<DT, D, PAD, MODE>), hipFuncAttributeMaxDynamicSharedMemorySize, lds);
        AXHIP_CHECK_HIP(attr);
    }
    AXHIP_REQUIRE(launch_fits(blocks, 64 * ROWS_WAVES), AXHIP_ERR_UNSUPPORTED, "attention over pages: grid too large");
    hipLaunchKernelGGL((sdpa_rows_kernel<DT, D, PAD, MODE>), dim3(static_cast<unsigned>(blocks)), dim3(64 * ROWS_WAVES), lds, s, a);
    AXHIP_CHECK_HIP(hipGetLastError());
    return AXHIP_OK;
}
template <int DT, int MODE> int launch_rows_mode(const CacheArgs &a, int64_t blocks, hipStream_t s) {
    if (a.D == 64) return launch_rows_as<DT, 64, false, MODE>(a, blocks, s);
    if (a.D == 128) return launch_rows_as<DT, 128, false, MODE>(a, blocks, s);
    if (a.D < 64) return launch_rows_as<DT, 64, true, MODE>(a, blocks, s);
    if (a.D < 128) return launch_rows_as<DT, 128, true, MODE>(a, blocks, s);
    if constexpr (DT != AXHIP_DTYPE_F32) return launch_rows_as<DT, 256, true, MODE>(a, blocks, s);
    return AXHIP_ERR_UNSUPPORTED;
}
// the shares of a decoding step's own keys
template <int DT> int launch_rows_own(const CacheArgs &a, hipStream_t s) { return launch_rows_mode<DT, ROWS_OWN>(a, own_blocks(a), s); }
template <int DT> int launch_rows_whole(const CacheArgs &a, hipStream_t s) { return launch_rows_mode<DT, ROWS_WHOLE>(a, (static_cast<int64_t>(a.new_tokens) * a.each + ROWS - 1) / ROWS * a.kv_heads * a.entries, s); }
// rows by cu_q, at most one block more than they need for each entry
template <int DT> int launch_rows_packed(const CacheArgs &a, hipStream_t s) { return launch_rows_mode<DT, ROWS_PACKED>(a, (a.total_q * a.each / ROWS + a.entries) * a.kv_heads * a.parts, s); }
template <int DT, int D, bool PACKED> void launch_join_as(const CacheArgs &a, int64_t rows, hipStream_t s) {
    // a work-group to a row where those are few (up to 128 results in the first trip), else a wavefront
    if (rows <= 1024) hipLaunchKernelGGL((sdpa_join_kernel<DT, D, 4, PACKED>), dim3(static_cast<unsigned>(rows)), dim3(256), 0, s, a);
    else hipLaunchKernelGGL((sdpa_join_kernel<DT, D, 1, PACKED>), dim3(static_cast<unsigned>((rows + 3) / 4)), dim3(256), 0, s, a);
}
template <int DT, bool PACKED> int launch_join_of(const CacheArgs &a, hipStream_t s) {
    const int64_t rows = PACKED ? a.total_q * a.heads : static_cast<int64_t>(a.entries) * a.new_tokens * a.heads;
    AXHIP_REQUIRE(launch_fits((rows + 3) / 4, 256), AXHIP_ERR_UNSUPPORTED, "attention of ragged sequences: grid too large");
    if (a.D <= 64) launch_join_as<DT, 64, PACKED>(a, rows, s);
    else if (a.D <= 128) launch_join_as<DT, 128, PACKED>(a, rows, s);
    else launch_join_as<DT, 256, PACKED>(a, rows, s);
    AXHIP_CHECK_HIP(hipGetLastError());
    return AXHIP_OK;
}
template <int DT> int launch_join(const CacheArgs &a, hipStream_t s) { return a.new_tokens ? launch_join_of<DT, false>(a, s) : launch_join_of<DT, true>(a, s); }

} // namespace axhip
