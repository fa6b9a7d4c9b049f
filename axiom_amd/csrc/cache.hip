// Rotary positions, new tokens into the pages of a cache, and pages copied: axhip_rope, axhip_kv_append, axhip_kv_copy_pages.
//
// All three move every element once and compute next to nothing: the bound is HBM, and for a decoding step the launch.
#include "divisor.hpp"

#include <cmath>
#include <initializer_list>

namespace axhip {
namespace {

// The angle position * turns modulo 2^64 as (cos, sin): the nearest quarter turn is taken off, which leaves |r| <= pi / 4 for the series of
// both; the first term left out is r^11 / 11! < 1.8e-9 and r^12 / 12! < 1.2e-10.  (An angle formed in 32 bits is 0.004 radians off at
// position 100000; here the fraction of a turn is rounded to 32 bits, 7e-10 radians.)
struct CosSin { float c, s; };
__device__ __forceinline__ CosSin turned(int64_t position, uint64_t turns, float amplitude) {
    const uint32_t at = static_cast<uint32_t>((static_cast<uint64_t>(position) * turns + 0x80000000u) >> 32);
    const uint32_t quarter = (at + 0x20000000u) >> 30;
    const float r = static_cast<float>(static_cast<int32_t>(at - (quarter << 30))) * 1.46291807926715968e-9f; // 2 pi / 2^32
    const float z = r * r;
    float s = __builtin_fmaf(z, 2.75573192e-6f, -1.98412698e-4f);
    s = __builtin_fmaf(s, z, 8.33333333e-3f);
    s = __builtin_fmaf(s, z, -1.66666667e-1f);
    s = __builtin_fmaf(s * z, r, r);
    float c = __builtin_fmaf(z, -2.75573192e-7f, 2.48015873e-5f);
    c = __builtin_fmaf(c, z, -1.38888889e-3f);
    c = __builtin_fmaf(c, z, 4.16666667e-2f);
    c = __builtin_fmaf(c, z, -0.5f);
    c = __builtin_fmaf(c, z, 1.0f);
    const float x = quarter & 1 ? s : c, y = quarter & 1 ? c : s; // a quarter turn: (c, s) -> (-s, c)
    return {(quarter + 1) & 2 ? -x * amplitude : x * amplitude, quarter & 2 ? -y * amplitude : y * amplitude};
}

// V consecutive elements (V * element size: 16 bytes, aligned to as much, or less)
template <int DT, int V> struct Pack;
template <int V> struct alignas(4 * V > 16 ? 16 : 4 * V) Pack<AXHIP_DTYPE_F32, V> { uint32_t w[V]; };
template <int V> struct alignas(2 * V > 16 ? 16 : 2 * V) Pack<AXHIP_DTYPE_F16, V> { uint16_t w[V]; };
template <int V> struct alignas(2 * V > 16 ? 16 : 2 * V) Pack<AXHIP_DTYPE_BF16, V> { uint16_t w[V]; };
template <int DT, int V> __device__ __forceinline__ float get(const Pack<DT, V> &p, int i) {
    if constexpr (DT == AXHIP_DTYPE_F32) return __uint_as_float(p.w[i]);
    else if constexpr (DT == AXHIP_DTYPE_F16) return f16_bits_to_f32(p.w[i]);
    else return bf16_bits_to_f32(p.w[i]);
}
template <int DT, int V> __device__ __forceinline__ void put(Pack<DT, V> &p, int i, float v) {
    if constexpr (DT == AXHIP_DTYPE_F32) p.w[i] = __float_as_uint(v);
    else if constexpr (DT == AXHIP_DTYPE_F16) p.w[i] = static_cast<uint16_t>(f32_to_f16_bits(v));
    else p.w[i] = static_cast<uint16_t>(pack_bf16x2(v, v));
}

// STREAM: past the caches.  Outputs of 64 MiB and more (STREAMING_OUTPUT_BYTES) are gone from them before anyone reads them, and stores that take a line in there first cost a third of the
// rate: 8192 tokens of 48 heads of 128, 100 MB each way, 51.2 -> 35.2 us; 300 pages of 32 KiB in 8 layers, 157 MB each way, 85 -> 62.
template <bool STREAM, class T> __device__ __forceinline__ void put_down(void *to, const T &v) {
    if constexpr (STREAM && sizeof(T) == 16) __builtin_nontemporal_store(__builtin_bit_cast(uint4_t, v), static_cast<uint4_t *>(to));
    else *static_cast<T *>(to) = v;
}

// Heads of a token in this order: those of q, of k, of v.  A unit is V elements of a head, whole pairs with PAIRS, else two such groups
// `apart` (rot / 2 dims; 1 where pairs lie side by side but are not aligned to two elements); a thread takes one unit of `per` heads of a token, so that an angle's sine is formed once for all of them.
struct MoveArgs {
    const void *q, *k, *v;
    void *q_out, *k_pages, *v_pages;
    const void *positions;
    const uint64_t *turns;
    const int64_t *slots; // NULL: only q
    int64_t qs[2], ks[2], vs[2], os[2], kp[3], vp[3], slots_end;
    Divisor units, groups; // units of a head; groups of heads that threads take in turn
    uint32_t total;        // threads with work
    int heads, kv_heads, rot, position_bytes, page_shift;
    int turning, step, apart; // how many units turn; from one of them to the next; from a group of dims to the one it turns with
    float amplitude, direction;
};

template <int DT, int V, bool PAIRS, int PER, bool STREAM>
__global__ __launch_bounds__(256) void move_heads_kernel(const MoveArgs a) {
    using E = typename Elem<DT>::type;
    const uint32_t id = blockIdx.x * 256u + threadIdx.x;
    if (id >= a.total) return;
    const uint32_t rest = a.units.of(id), unit = id - rest * a.units.d;
    const uint32_t token = a.groups.of(rest), group = rest - token * a.groups.d;
    const bool turns = static_cast<int>(unit) < a.turning;
    // where the unit lies in a head: of halves, V dims and those rot / 2 behind; else V dims
    const int d0 = turns ? static_cast<int>(unit) * a.step : a.rot + (static_cast<int>(unit) - a.turning) * V;
    const bool two = !PAIRS && turns;
    int64_t page = -1, row = 0;
    if (a.slots) {
        const int64_t slot = a.slots[token];
        if (slot >= 0 && slot < a.slots_end) {
            page = slot >> a.page_shift;
            row = slot & ((int64_t(1) << a.page_shift) - 1);
        }
    }
    const int all = a.heads + 2 * a.kv_heads;
    Pack<DT, V> x[PER], y[PER];
    E *to[PER];
    // (every load of the thread is on its way before the angles are formed; a thread's head behind the last one is the last one again, and not stored)
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        const int wanted = static_cast<int>(group + i * a.groups.d), head = min(wanted, all - 1);
        const E *from;
        if (head < a.heads) {
            from = static_cast<const E *>(a.q) + token * a.qs[0] + head * a.qs[1];
            to[i] = static_cast<E *>(a.q_out) + token * a.os[0] + head * a.os[1];
        } else {
            int h = head - a.heads;
            const bool is_k = h < a.kv_heads;
            if (!is_k) h -= a.kv_heads;
            from = is_k ? static_cast<const E *>(a.k) + token * a.ks[0] + h * a.ks[1] : static_cast<const E *>(a.v) + token * a.vs[0] + h * a.vs[1];
            to[i] = is_k ? static_cast<E *>(a.k_pages) + page * a.kp[0] + row * a.kp[1] + h * a.kp[2] : static_cast<E *>(a.v_pages) + page * a.vp[0] + row * a.vp[1] + h * a.vp[2];
            if (page < 0) to[i] = nullptr;
        }
        if (wanted >= all) to[i] = nullptr;
        x[i] = *reinterpret_cast<const Pack<DT, V> *>(from + d0);
        if (two) y[i] = *reinterpret_cast<const Pack<DT, V> *>(from + d0 + a.apart);
    }
    __builtin_amdgcn_sched_barrier(0);
    constexpr int ANGLES = PAIRS ? V / 2 : V;
    CosSin t[ANGLES];
    if (turns) {
        const int64_t position = a.position_bytes == 8 ? static_cast<const int64_t *>(a.positions)[token] : static_cast<const int32_t *>(a.positions)[token];
#pragma unroll
        for (int i = 0; i < ANGLES; ++i) {
            t[i] = turned(position, a.turns[static_cast<int>(unit) * ANGLES + i], a.amplitude);
            t[i].s *= a.direction;
        }
    }
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        if (!to[i]) continue;
        // (Which of two products keeps all its bits is written down: left to the compiler, it was not the same one in every variant of the kernel, and a token's result could depend on the batch.)
        if (turns && static_cast<int>(group + i * a.groups.d) < a.heads + a.kv_heads) {
            if constexpr (PAIRS) {
#pragma unroll
                for (int j = 0; j < V / 2; ++j) {
                    const float p = get<DT, V>(x[i], 2 * j), r = get<DT, V>(x[i], 2 * j + 1);
                    put<DT, V>(x[i], 2 * j, __builtin_fmaf(p, t[j].c, -(r * t[j].s)));
                    put<DT, V>(x[i], 2 * j + 1, __builtin_fmaf(r, t[j].c, p * t[j].s));
                }
            } else {
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    const float p = get<DT, V>(x[i], j), r = get<DT, V>(y[i], j);
                    put<DT, V>(x[i], j, __builtin_fmaf(p, t[j].c, -(r * t[j].s)));
                    put<DT, V>(y[i], j, __builtin_fmaf(r, t[j].c, p * t[j].s));
                }
            }
        }
        put_down<STREAM>(to[i] + d0, x[i]);
        if (two) put_down<STREAM>(to[i] + d0 + a.apart, y[i]);
    }
}

// Pages.  `vectors` pieces of V bytes a page and tensor; the row of piece v, by which a pair's count of rows leaves it in or out, is
// v / row_div, modulo the page where heads lie outside.  DENSE: piece v lies V * v bytes into the page.
struct CopyArgs {
    unsigned char *pool[2];
    int64_t page_bytes[2], row_bytes[2], head_bytes[2], layer_bytes[2];
    const int32_t *src, *dst, *rows;
    int64_t n_pages;
    Divisor slices, layers, row_div, dim_div, head_div;
    uint32_t vectors;
    int page_size;
};
constexpr int COPY_DEEP = 8; // pieces of a thread, all requested before the first is stored

template <int V, bool DENSE, bool STREAM>
__global__ __launch_bounds__(256) void copy_pages_kernel(const CopyArgs a) {
    struct alignas(V) Piece { unsigned char b[V]; };
    const uint32_t rest = a.slices.of(blockIdx.x), slice = blockIdx.x - rest * a.slices.d;
    const uint32_t both = a.layers.of(rest), layer = rest - both * a.layers.d, pair = both >> 1, which = both & 1;
    const int32_t src = a.src[pair], dst = a.dst[pair];
    if (src < 0 || dst < 0 || src >= a.n_pages || dst >= a.n_pages || src == dst) return;
    const int rows = a.rows ? min(max(a.rows[pair], 0), a.page_size) : a.page_size;
    unsigned char *base = a.pool[which] + layer * a.layer_bytes[which];
    const unsigned char *from = base + src * a.page_bytes[which];
    unsigned char *to = base + dst * a.page_bytes[which];
    Piece p[COPY_DEEP];
    const uint32_t v0 = slice * (COPY_DEEP * 256u) + threadIdx.x;
    if (DENSE && rows == a.page_size && (slice + 1) * (COPY_DEEP * 256u) <= a.vectors) { // nothing to leave out
#pragma unroll
        for (int i = 0; i < COPY_DEEP; ++i) {
            const unsigned char *at = from + static_cast<int64_t>(v0 + i * 256u) * V;
            if constexpr (STREAM && V == 16) p[i] = __builtin_bit_cast(Piece, __builtin_nontemporal_load(reinterpret_cast<const uint4_t *>(at)));
            else p[i] = *reinterpret_cast<const Piece *>(at);
        }
#pragma unroll
        for (int i = 0; i < COPY_DEEP; ++i) put_down<STREAM>(to + static_cast<int64_t>(v0 + i * 256u) * V, p[i]);
        return;
    }
    int64_t at[COPY_DEEP];
#pragma unroll
    for (int i = 0; i < COPY_DEEP; ++i) {
        const uint32_t v = v0 + i * 256u;
        at[i] = -1;
        if (v >= a.vectors) continue;
        if constexpr (DENSE) {
            if (static_cast<int>(a.row_div.of(v) & static_cast<uint32_t>(a.page_size - 1)) < rows) at[i] = static_cast<int64_t>(v) * V;
        } else { // piece of a head, head, row
            const uint32_t line = a.dim_div.of(v), r = a.head_div.of(line);
            const int row = static_cast<int>(r);
            if (row < rows) at[i] = row * a.row_bytes[which] + static_cast<int64_t>(line - r * a.head_div.d) * a.head_bytes[which] + static_cast<int64_t>(v - line * a.dim_div.d) * V;
        }
        if (at[i] >= 0) p[i] = *reinterpret_cast<const Piece *>(from + at[i]);
    }
#pragma unroll
    for (int i = 0; i < COPY_DEEP; ++i)
        if (at[i] >= 0) put_down<STREAM>(to + at[i], p[i]);
}

// ------------------------------------------------------------------ host side
int shift_of(int power) { return __builtin_ctz(static_cast<unsigned>(power)); }

int launch_moves(MoveArgs &a, int dtype, bool pairs, int dim, int64_t tokens, int v, hipStream_t s, const char *who) {
    // (a head's units: of halves rot / 2 / v pairs of groups, else groups of v; then what is only copied)
    const bool loose = pairs && v == 1; // pairs one by one
    pairs = pairs && !loose;
    a.turning = pairs ? a.rot / v : a.rot / 2 / v;
    a.step = loose ? 2 : v;
    a.apart = loose ? 1 : a.rot / 2;
    const int units = a.turning + (dim - a.rot) / v;
    const int all = a.heads + 2 * a.kv_heads;
    // Heads of a thread: two share an angle's sines, one where that would leave the chip's 1024 SIMDs without two wavefronts each.  (8192 tokens of 48 heads of 128: two 35.2 us, four 36.4;
    // stores through the caches: one 48.7, two 48.2, four 51.2, eight 52.1.)
    const double work = static_cast<double>(tokens) * all * units;
    const bool many = all >= 2 && work >= 2.0 * 2 * 64 * 1024;
    const bool stream = many && static_cast<double>(tokens) * all * dim * static_cast<double>(dtype_size(dtype)) >= STREAMING_OUTPUT_BYTES;
    const int per = many ? 2 : 1, groups = (all + per - 1) / per;
    AXHIP_REQUIRE(static_cast<double>(tokens) * groups * units < 2147483648.0, AXHIP_ERR_UNSUPPORTED, "%s: %lld tokens of %d heads are too many for one launch", who, static_cast<long long>(tokens), all);
    const int64_t total = tokens * groups * units;
    a.units = Divisor(static_cast<uint32_t>(units));
    a.groups = Divisor(static_cast<uint32_t>(groups));
    a.total = static_cast<uint32_t>(total);
    const dim3 grid(static_cast<unsigned>((total + 255) / 256)), block(256);
#define AXHIP_MOVE_AS(DT, V, PAIRS)                                                                                             \
    do {                                                                                                                        \
        if (stream) hipLaunchKernelGGL((move_heads_kernel<DT, V, PAIRS, 2, true>), grid, block, 0, s, a);                       \
        else if (many) hipLaunchKernelGGL((move_heads_kernel<DT, V, PAIRS, 2, false>), grid, block, 0, s, a);                   \
        else hipLaunchKernelGGL((move_heads_kernel<DT, V, PAIRS, 1, false>), grid, block, 0, s, a);                             \
    } while (0)
#define AXHIP_MOVE(DT, V)                                      \
    do {                                                       \
        if (pairs) AXHIP_MOVE_AS(DT, ((V) < 2 ? 2 : (V)), true); \
        else AXHIP_MOVE_AS(DT, V, false);                      \
    } while (0)
#define AXHIP_MOVE16(DT)                   \
    do {                                   \
        if (v == 8) AXHIP_MOVE(DT, 8);     \
        else if (v == 4) AXHIP_MOVE(DT, 4); \
        else if (v == 2) AXHIP_MOVE(DT, 2); \
        else AXHIP_MOVE(DT, 1);            \
    } while (0)
    if (dtype == AXHIP_DTYPE_BF16) AXHIP_MOVE16(AXHIP_DTYPE_BF16);
    else if (dtype == AXHIP_DTYPE_F16) AXHIP_MOVE16(AXHIP_DTYPE_F16);
    else if (v == 4) AXHIP_MOVE(AXHIP_DTYPE_F32, 4);
    else if (v == 2) AXHIP_MOVE(AXHIP_DTYPE_F32, 2);
    else AXHIP_MOVE(AXHIP_DTYPE_F32, 1);
#undef AXHIP_MOVE16
#undef AXHIP_MOVE
#undef AXHIP_MOVE_AS
    AXHIP_CHECK_HIP(hipGetLastError());
    return AXHIP_OK;
}

bool sane(int64_t stride) { return stride >= 0 && stride < (int64_t(1) << 40); }
bool sane(const int64_t *strides, int n) {
    for (int i = 0; i < n; ++i)
        if (!sane(strides[i])) return false;
    return true;
}
// Rows of `dim` elements that are written: no two of them may share any, so far as two neighbours along one dimension tell
bool apart(const int64_t *strides, std::initializer_list<int64_t> counts, int dim) {
    for (int64_t n : counts)
        if (*strides++ < dim && n > 1) return false;
    return true;
}
bool elements_aligned(const void *p, int dtype) { return (reinterpret_cast<uintptr_t>(p) & (dtype_size(dtype) - 1)) == 0; }

bool pages_apart(const AxhipKvPages &g) { return apart(g.k_strides, {g.n_pages, g.page_size, g.heads}, g.head_dim) && apart(g.v_strides, {g.n_pages, g.page_size, g.heads}, g.head_dim); }

// The widest groups of elements (16 bytes at most) that every address and number given keeps whole.
struct Width {
    int dtype;
    uint64_t seen = 0; // bits of everything that has to be a multiple, in bytes
    void address(const void *p) { seen |= reinterpret_cast<uintptr_t>(p); }
    void elements(int64_t n) { seen |= static_cast<uint64_t>(n) * dtype_size(dtype); }
    void strides(const int64_t *s, int n) { for (int i = 0; i < n; ++i) elements(s[i]); }
    int bytes() const {
        int b = 16;
        while (seen & static_cast<uint64_t>(b - 1)) b /= 2;
        return b;
    }
    int width() const { return bytes() / static_cast<int>(dtype_size(dtype)); }
};

int check_rotation(const char *who, int rot, int dim, int interleaved, float amplitude, int position_bytes, const void *positions, const uint64_t *turns) {
    AXHIP_REQUIRE(rot >= 0 && rot % 2 == 0 && rot <= dim, AXHIP_ERR_INVALID_ARG, "%s: rot_dim %d is not an even number up to head_dim %d", who, rot, dim);
    AXHIP_REQUIRE(interleaved == 0 || interleaved == 1, AXHIP_ERR_INVALID_ARG, "%s: interleaved is %d, neither 0 nor 1", who, interleaved);
    AXHIP_REQUIRE(std::isfinite(amplitude), AXHIP_ERR_INVALID_ARG, "%s: amplitude must be a finite number", who);
    if (rot == 0) return AXHIP_OK;
    AXHIP_REQUIRE(position_bytes == 4 || position_bytes == 8, AXHIP_ERR_INVALID_ARG, "%s: position_bytes is %d, neither 4 nor 8", who, position_bytes);
    AXHIP_REQUIRE(positions && turns, AXHIP_ERR_INVALID_ARG, "%s: NULL positions or turns", who);
    AXHIP_REQUIRE((reinterpret_cast<uintptr_t>(positions) & static_cast<uintptr_t>(position_bytes - 1)) == 0 && (reinterpret_cast<uintptr_t>(turns) & 7u) == 0, AXHIP_ERR_INVALID_ARG,
                  "%s: positions or turns are not aligned to their elements", who);
    return AXHIP_OK;
}
} // namespace

int check_pages(const char *who, const AxhipKvPages &p) {
    AXHIP_REQUIRE(valid_dtype(p.dtype), AXHIP_ERR_INVALID_ARG, "%s: bad dtype %d of the pages", who, p.dtype);
    AXHIP_REQUIRE(p.page_size > 0 && p.page_size <= 65536 && (p.page_size & (p.page_size - 1)) == 0, AXHIP_ERR_INVALID_ARG, "%s: page_size %d is not a power of two up to 65536", who, p.page_size);
    AXHIP_REQUIRE(p.heads > 0 && p.heads < (1 << 20) && p.head_dim > 0 && p.head_dim < (1 << 20), AXHIP_ERR_INVALID_ARG, "%s: pages of %d heads of %d", who, p.heads, p.head_dim);
    AXHIP_REQUIRE(p.n_pages >= 0 && p.n_pages < (int64_t(1) << 31), AXHIP_ERR_INVALID_ARG, "%s: bad number of pages", who);
    AXHIP_REQUIRE(sane(p.k_strides, 3) && sane(p.v_strides, 3), AXHIP_ERR_INVALID_ARG, "%s: bad stride of the pages", who);
    AXHIP_REQUIRE(p.n_pages == 0 || (p.k && p.v), AXHIP_ERR_INVALID_ARG, "%s: NULL pages", who);
    AXHIP_REQUIRE(elements_aligned(p.k, p.dtype) && elements_aligned(p.v, p.dtype), AXHIP_ERR_INVALID_ARG, "%s: the pages are not aligned to their elements", who);
    return AXHIP_OK;
}
} // namespace axhip
using namespace axhip;

extern "C" {

int axhip_rope_turns(const AxhipRopeScaling *scaling, uint64_t *turns) {
    AXHIP_REQUIRE(scaling && turns, AXHIP_ERR_INVALID_ARG, "axhip_rope_turns: NULL argument");
    const AxhipRopeScaling &c = *scaling;
    AXHIP_REQUIRE(c.rot_dim >= 2 && c.rot_dim <= 1024 && c.rot_dim % 2 == 0, AXHIP_ERR_INVALID_ARG, "axhip_rope_turns: rot_dim %d is not an even number from 2 to 1024", c.rot_dim);
    AXHIP_REQUIRE(c.kind >= AXHIP_ROPE_PLAIN && c.kind <= AXHIP_ROPE_BANDS, AXHIP_ERR_INVALID_ARG, "axhip_rope_turns: bad kind %d", c.kind);
    AXHIP_REQUIRE(c.theta >= 1.0 && std::isfinite(c.theta), AXHIP_ERR_INVALID_ARG, "axhip_rope_turns: theta must be a finite number, 1 or more");
    AXHIP_REQUIRE(c.kind == AXHIP_ROPE_PLAIN || (c.factor > 0.0 && std::isfinite(c.factor)), AXHIP_ERR_INVALID_ARG, "axhip_rope_turns: factor must be a finite number above 0");
    AXHIP_REQUIRE(c.kind != AXHIP_ROPE_BANDS || (c.low >= 0.0 && c.high > c.low && std::isfinite(c.high) && c.length > 0.0 && std::isfinite(c.length)), AXHIP_ERR_INVALID_ARG,
                  "axhip_rope_turns: 0 <= low < high and length > 0 are needed");
    // (80-bit numbers: a turn is 2^64, of which 64 bits of the fraction are kept)
    const long double two_pi = 6.283185307179586476925286766559005768L;
    const long double r = c.rot_dim, f = c.factor;
    long double theta = c.theta;
    if (c.kind == AXHIP_ROPE_BASE && c.rot_dim > 2) theta *= powl(f, r / (r - 2.0L));
    AXHIP_REQUIRE(std::isfinite(theta) && theta > 0.0L, AXHIP_ERR_INVALID_ARG, "axhip_rope_turns: theta and factor are out of range");
    for (int i = 0; i < c.rot_dim / 2; ++i) {
        long double w = powl(theta, -2.0L * i / r);
        if (c.kind == AXHIP_ROPE_LINEAR) w /= f;
        if (c.kind == AXHIP_ROPE_BANDS) {
            const long double t = static_cast<long double>(c.length) * w / two_pi;
            long double keep = (t - static_cast<long double>(c.low)) / (static_cast<long double>(c.high) - static_cast<long double>(c.low));
            keep = keep < 0.0L ? 0.0L : keep > 1.0L ? 1.0L : keep;
            w = w * keep + w / f * (1.0L - keep);
        }
        const long double part = fmodl(w / two_pi, 1.0L) * 18446744073709551616.0L; // [0, 2^64]
        turns[i] = part >= 18446744073709551615.0L ? 0 : static_cast<uint64_t>(part + 0.5L);
    }
    return AXHIP_OK;
}

int axhip_rope(const void *x, void *y, const AxhipRopeParams *params, void *stream) {
    AXHIP_REQUIRE(params != nullptr, AXHIP_ERR_INVALID_ARG, "axhip_rope: params is NULL");
    const AxhipRopeParams &p = *params;
    AXHIP_REQUIRE(valid_dtype(p.dtype), AXHIP_ERR_INVALID_ARG, "axhip_rope: bad dtype %d", p.dtype);
    AXHIP_REQUIRE(p.tokens >= 0 && p.heads >= 0 && p.heads < (1 << 20) && p.head_dim >= 2 && p.head_dim < (1 << 20), AXHIP_ERR_INVALID_ARG, "axhip_rope: bad extent");
    AXHIP_REQUIRE(p.rot_dim >= 2, AXHIP_ERR_INVALID_ARG, "axhip_rope: rot_dim %d is not an even number from 2 to head_dim %d", p.rot_dim, p.head_dim);
    AXHIP_REQUIRE(p.inverse == 0 || p.inverse == 1, AXHIP_ERR_INVALID_ARG, "axhip_rope: inverse is %d, neither 0 nor 1", p.inverse);
    AXHIP_REQUIRE(sane(p.x_strides, 2) && sane(p.y_strides, 2), AXHIP_ERR_INVALID_ARG, "axhip_rope: bad stride");
    if (p.tokens == 0 || p.heads == 0) return AXHIP_OK;
    int rc = check_rotation("axhip_rope", p.rot_dim, p.head_dim, p.interleaved, p.amplitude, p.position_bytes, p.positions, p.turns);
    if (rc) return rc;
    AXHIP_REQUIRE(x && y, AXHIP_ERR_INVALID_ARG, "axhip_rope: NULL tensor");
    AXHIP_REQUIRE(elements_aligned(x, p.dtype) && elements_aligned(y, p.dtype), AXHIP_ERR_INVALID_ARG, "axhip_rope: a tensor is not aligned to its elements");
    AXHIP_REQUIRE(apart(p.y_strides, {p.tokens, p.heads}, p.head_dim), AXHIP_ERR_INVALID_ARG, "axhip_rope: rows of y overlap");
    AXHIP_REQUIRE(x != y || ((p.tokens == 1 || p.x_strides[0] == p.y_strides[0]) && (p.heads == 1 || p.x_strides[1] == p.y_strides[1])), AXHIP_ERR_INVALID_ARG,
                  "axhip_rope: in place with other strides");
    rc = ensure_init();
    if (rc) return rc;
    MoveArgs a{};
    a.q = x; a.q_out = y;
    a.positions = p.positions; a.turns = p.turns;
    a.heads = p.heads; a.rot = p.rot_dim; a.position_bytes = p.position_bytes;
    a.amplitude = p.amplitude == 0.0f ? 1.0f : p.amplitude;
    a.direction = p.inverse ? -1.0f : 1.0f;
    Width w{p.dtype};
    w.address(x); w.address(y);
    for (int i = 0; i < 2; ++i) { a.qs[i] = p.x_strides[i]; a.os[i] = p.y_strides[i]; }
    w.strides(a.qs, 2); w.strides(a.os, 2);
    w.elements(p.head_dim); w.elements(p.rot_dim);
    if (!p.interleaved) w.elements(p.rot_dim / 2);
    return launch_moves(a, p.dtype, p.interleaved != 0, p.head_dim, p.tokens, w.width(), resolve_stream(stream), "axhip_rope");
}

int axhip_kv_append(const void *q, const void *k, const void *v, void *q_out, const AxhipKvAppendParams *params, void *stream) {
    const char *who = "axhip_kv_append";
    AXHIP_REQUIRE(params != nullptr, AXHIP_ERR_INVALID_ARG, "axhip_kv_append: params is NULL");
    const AxhipKvAppendParams &p = *params;
    const AxhipKvPages &g = p.pages;
    int rc = check_pages(who, g);
    if (rc) return rc;
    AXHIP_REQUIRE(p.tokens >= 0 && p.heads >= 0 && p.heads < (1 << 20), AXHIP_ERR_INVALID_ARG, "axhip_kv_append: bad extent");
    AXHIP_REQUIRE(sane(p.q_strides, 2) && sane(p.k_strides, 2) && sane(p.v_strides, 2) && sane(p.q_out_strides, 2), AXHIP_ERR_INVALID_ARG, "axhip_kv_append: bad stride");
    if (p.tokens == 0) return AXHIP_OK;
    rc = check_rotation(who, p.rot_dim, g.head_dim, p.interleaved, p.amplitude, p.position_bytes, p.positions, p.turns);
    if (rc) return rc;
    AXHIP_REQUIRE(k && v && p.slots && (p.heads == 0 || (q && q_out)), AXHIP_ERR_INVALID_ARG, "axhip_kv_append: NULL tensor");
    AXHIP_REQUIRE(elements_aligned(k, g.dtype) && elements_aligned(v, g.dtype) && (p.heads == 0 || (elements_aligned(q, g.dtype) && elements_aligned(q_out, g.dtype))) &&
                      (reinterpret_cast<uintptr_t>(p.slots) & 7u) == 0,
                  AXHIP_ERR_INVALID_ARG, "axhip_kv_append: a tensor is not aligned to its elements");
    if (p.heads > 0) {
        AXHIP_REQUIRE(apart(p.q_out_strides, {p.tokens, p.heads}, g.head_dim), AXHIP_ERR_INVALID_ARG, "axhip_kv_append: rows of q_out overlap");
        AXHIP_REQUIRE(q != q_out || ((p.tokens == 1 || p.q_strides[0] == p.q_out_strides[0]) && (p.heads == 1 || p.q_strides[1] == p.q_out_strides[1])), AXHIP_ERR_INVALID_ARG,
                      "axhip_kv_append: in place with other strides");
    }
    AXHIP_REQUIRE(pages_apart(g), AXHIP_ERR_INVALID_ARG, "axhip_kv_append: rows of the pages overlap");
    rc = ensure_init();
    if (rc) return rc;
    MoveArgs a{};
    a.q = q; a.k = k; a.v = v; a.q_out = q_out;
    a.k_pages = g.k; a.v_pages = g.v;
    a.positions = p.positions; a.turns = p.turns; a.slots = p.slots;
    a.heads = p.heads; a.kv_heads = g.heads; a.rot = p.rot_dim; a.position_bytes = p.position_bytes;
    a.page_shift = shift_of(g.page_size);
    a.slots_end = g.n_pages * g.page_size;
    a.amplitude = p.amplitude == 0.0f ? 1.0f : p.amplitude;
    a.direction = 1.0f;
    Width w{g.dtype};
    w.address(k); w.address(v); w.address(g.k); w.address(g.v);
    for (int i = 0; i < 2; ++i) { a.qs[i] = p.q_strides[i]; a.ks[i] = p.k_strides[i]; a.vs[i] = p.v_strides[i]; a.os[i] = p.q_out_strides[i]; }
    for (int i = 0; i < 3; ++i) { a.kp[i] = g.k_strides[i]; a.vp[i] = g.v_strides[i]; }
    if (p.heads > 0) { w.address(q); w.address(q_out); w.strides(a.qs, 2); w.strides(a.os, 2); }
    w.strides(a.ks, 2); w.strides(a.vs, 2); w.strides(a.kp, 3); w.strides(a.vp, 3);
    w.elements(g.head_dim); w.elements(p.rot_dim);
    if (!p.interleaved) w.elements(p.rot_dim / 2);
    const bool pairs = p.interleaved && p.rot_dim > 0;
    return launch_moves(a, g.dtype, pairs, g.head_dim, p.tokens, w.width(), resolve_stream(stream), who);
}

int axhip_kv_copy_pages(const AxhipKvCopyParams *params, void *stream) {
    const char *who = "axhip_kv_copy_pages";
    AXHIP_REQUIRE(params != nullptr, AXHIP_ERR_INVALID_ARG, "axhip_kv_copy_pages: params is NULL");
    const AxhipKvCopyParams &p = *params;
    const AxhipKvPages &g = p.pages;
    int rc = check_pages(who, g);
    if (rc) return rc;
    AXHIP_REQUIRE(p.pairs >= 0 && p.layers >= 0 && p.layers < (1 << 20), AXHIP_ERR_INVALID_ARG, "axhip_kv_copy_pages: bad extent");
    AXHIP_REQUIRE(sane(p.k_layer_stride) && sane(p.v_layer_stride), AXHIP_ERR_INVALID_ARG, "axhip_kv_copy_pages: bad stride");
    if (p.pairs == 0 || p.layers == 0 || g.n_pages == 0) return AXHIP_OK;
    AXHIP_REQUIRE(p.src && p.dst, AXHIP_ERR_INVALID_ARG, "axhip_kv_copy_pages: NULL src or dst");
    AXHIP_REQUIRE(((reinterpret_cast<uintptr_t>(p.src) | reinterpret_cast<uintptr_t>(p.dst) | reinterpret_cast<uintptr_t>(p.rows)) & 3u) == 0, AXHIP_ERR_INVALID_ARG,
                  "axhip_kv_copy_pages: src, dst or rows are not aligned to their elements");
    AXHIP_REQUIRE(pages_apart(g) && (p.layers == 1 || (p.k_layer_stride >= g.head_dim && p.v_layer_stride >= g.head_dim)), AXHIP_ERR_INVALID_ARG, "axhip_kv_copy_pages: rows of the pages overlap");
    rc = ensure_init();
    if (rc) return rc;
    CopyArgs a{};
    const int es = static_cast<int>(dtype_size(g.dtype));
    a.pool[0] = static_cast<unsigned char *>(g.k);
    a.pool[1] = static_cast<unsigned char *>(g.v);
    Width w{g.dtype};
    w.address(g.k); w.address(g.v);
    w.elements(g.head_dim);
    w.elements(p.k_layer_stride); w.elements(p.v_layer_stride);
    bool row_major = true, head_major = true; // the pages are whole pieces of memory, rows or heads outside
    const int64_t dim = g.head_dim, line = dim * g.heads, head = dim * g.page_size;
    for (int t = 0; t < 2; ++t) {
        const int64_t *s = t ? g.v_strides : g.k_strides;
        w.strides(s, 3);
        a.page_bytes[t] = s[0] * es; a.row_bytes[t] = s[1] * es; a.head_bytes[t] = s[2] * es;
        a.layer_bytes[t] = (t ? p.v_layer_stride : p.k_layer_stride) * es;
        row_major = row_major && (g.page_size == 1 || s[1] == line) && (g.heads == 1 || s[2] == dim);
        head_major = head_major && (g.page_size == 1 || s[1] == dim) && (g.heads == 1 || s[2] == head);
    }
    a.src = p.src; a.dst = p.dst; a.rows = p.rows;
    a.n_pages = g.n_pages;
    a.page_size = g.page_size;
    const int v = w.bytes(), per = static_cast<int>(dim) * es / v; // pieces of a head
    const int64_t vectors = static_cast<int64_t>(per) * g.heads * g.page_size;
    const int64_t slices = (vectors + 256 * COPY_DEEP - 1) / (256 * COPY_DEEP);
    AXHIP_REQUIRE(vectors < (int64_t(1) << 31) && slices * p.layers < (int64_t(1) << 31) && p.pairs < (1 << 30) && launch_fits(slices * p.layers * 2 * p.pairs, 256), AXHIP_ERR_UNSUPPORTED,
                  "axhip_kv_copy_pages: %d pairs of %d layers are too many for one launch", p.pairs, p.layers);
    const int64_t blocks = slices * p.layers * 2 * p.pairs;
    a.vectors = static_cast<uint32_t>(vectors);
    a.slices = Divisor(static_cast<uint32_t>(slices));
    a.layers = Divisor(static_cast<uint32_t>(p.layers));
    a.dim_div = Divisor(static_cast<uint32_t>(per));
    a.head_div = Divisor(static_cast<uint32_t>(g.heads));
    a.row_div = Divisor(static_cast<uint32_t>(row_major ? per * g.heads : per));
    const bool dense = row_major || head_major;
    const dim3 grid(static_cast<unsigned>(blocks)), block(256);
    hipStream_t s = resolve_stream(stream);
    const bool past_caches = static_cast<double>(vectors) * v * p.layers * 2 * p.pairs >= STREAMING_OUTPUT_BYTES;
#define AXHIP_COPY(V)                                                                                              \
    do {                                                                                                           \
        if (dense && past_caches) hipLaunchKernelGGL((copy_pages_kernel<V, true, true>), grid, block, 0, s, a);         \
        else if (dense) hipLaunchKernelGGL((copy_pages_kernel<V, true, false>), grid, block, 0, s, a);             \
        else hipLaunchKernelGGL((copy_pages_kernel<V, false, false>), grid, block, 0, s, a);                       \
    } while (0)
    if (v == 16) AXHIP_COPY(16);
    else if (v == 8) AXHIP_COPY(8);
    else if (v == 4) AXHIP_COPY(4);
    else AXHIP_COPY(2);
#undef AXHIP_COPY
    AXHIP_CHECK_HIP(hipGetLastError());
    return AXHIP_OK;
}

} // extern "C"
