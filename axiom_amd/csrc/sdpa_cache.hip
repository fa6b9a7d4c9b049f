// Attention of sequences of different lengths, packed or over the pages of a cache: axhip_sdpa_packed, axhip_sdpa_paged.
#include "sdpa_cache.hpp"

#include <algorithm>
#include <cmath>
#include <cstdlib>

namespace axhip {

// ------------------------------------------------------------- generic kernel
// Every type, head size up to 256, stride and alignment, in fp32: 16 rows of 16 lanes, keys 32 at a time through LDS.  Lane c of a row
// computes the scores of keys c and c + 16 and the dims c, c + 16, ...
constexpr int CM = 16, CN = 32, CMAXD = 256;

__global__ __launch_bounds__(256) void sdpa_cache_generic_kernel(const CacheArgs a) {
    extern __shared__ float smem[];
    const int D = a.D, ksd = D + 1;
    float *Qs = smem;           // [CM][D]
    float *Ksm = Qs + CM * D;   // [CN][D + 1]
    float *Vs = Ksm + CN * ksd; // [CN][D]
    float *Ps = Vs + CN * D;    // [CM][CN]
    __shared__ int bad_page;
    const int tid = threadIdx.x, r = tid / 16, c = tid % 16;
    const int kvh = blockIdx.x % a.kv_heads;
    int64_t block = blockIdx.x / a.kv_heads;
    // which entry: with cu_q entry s gets the blocks from cu_q[s] * each / CM + s on, one more than it needs at most
    int s;
    if (a.new_tokens) {
        const int per = (a.new_tokens * a.each + CM - 1) / CM;
        s = static_cast<int>(block / per);
        block %= per;
    } else {
        auto first = [&](int e) { return static_cast<int64_t>(clamped(a.cu_q[e], 0, a.total_q)) * a.each / CM + e; };
        int lo = 0, hi = a.entries - 1; // first(lo) <= block
        while (lo < hi) {
            const int mid = (lo + hi + 1) / 2;
            if (first(mid) <= block) lo = mid;
            else hi = mid - 1;
        }
        s = lo;
        block -= first(s);
    }
    const TokenRun t = tokens_of(a, s);
    const int64_t rows = static_cast<int64_t>(t.n) * a.each, row0 = block * CM;
    if (block < 0 || row0 >= rows) return;
    const int64_t row = row0 + r;
    const bool row_ok = row < rows;
    const int token = static_cast<int>(row / a.each), head = kvh * a.each + static_cast<int>(row % a.each);
    auto q_at = [&](int64_t rr) {
        const int64_t tok = rr / a.each, h = kvh * a.each + rr % a.each;
        return s * a.qs[0] + (t.from + tok) * a.qs[1] + h * a.qs[2];
    };
    for (int i = tid; i < CM * D; i += 256) {
        const int rr = i / D, d = i % D;
        Qs[i] = row0 + rr < rows ? load_any(a.q, a.dtype, q_at(row0 + rr) + d) : 0.0f;
    }
    if (tid == 0) bad_page = 0;

    float acc[CMAXD / 16];
#pragma unroll
    for (int i = 0; i < CMAXD / 16; ++i) acc[i] = 0.0f;
    float m_run = NEG_INF_F, l_run = 0.0f;

    auto walk = [&](const KeyRun &run, bool causal) {
        const int limit = causal ? run.n - t.n + token : run.n - 1; // last key that this row sees
        const int last_token = static_cast<int>(min(row0 + CM - 1, rows - 1) / a.each);
        const int end = causal ? min(run.n, run.n - t.n + last_token + 1) : run.n;
        for (int kv0 = 0; kv0 < end; kv0 += CN) {
            __syncthreads();
            for (int i = tid; i < CN * D; i += 256) {
                const int rr = i / D, d = i % D, key = kv0 + rr;
                float kx = 0.0f, vx = 0.0f;
                if (key < run.n) {
                    int64_t page = 0, in_page = run.base + key;
                    if (run.table) {
                        page = run.table[key >> a.page_shift];
                        in_page = key & ((1 << a.page_shift) - 1);
                        if (page < 0 || page >= a.n_pages) {
                            bad_page = 1;
                            page = -1;
                        }
                    }
                    if (page >= 0) {
                        kx = load_any(a.k, a.dtype, page * a.ks[0] + in_page * a.ks[1] + kvh * a.ks[2] + d);
                        vx = load_any(a.v, a.dtype, page * a.vs[0] + in_page * a.vs[1] + kvh * a.vs[2] + d);
                    }
                }
                Ksm[rr * ksd + d] = kx;
                Vs[rr * D + d] = vx;
            }
            __syncthreads();
            float sc[CN / 16];
#pragma unroll
            for (int jj = 0; jj < CN / 16; ++jj) {
                const int j = c + 16 * jj;
                float dot = 0.0f;
                for (int d = 0; d < D; ++d) dot = __builtin_fmaf(Qs[r * D + d], Ksm[j * ksd + d], dot);
                sc[jj] = kv0 + j > limit || kv0 + j >= run.n ? NEG_INF_F : dot * a.scale_log2e;
            }
            float mloc = fmaxf(sc[0], sc[1]);
#pragma unroll
            for (int o = 8; o > 0; o >>= 1) mloc = fmaxf(mloc, __shfl_xor(mloc, o, WAVE));
            const float m_new = fmaxf(m_run, mloc), m_use = m_new == NEG_INF_F ? 0.0f : m_new;
            const float alpha = exp2f(m_run - m_use);
            m_run = m_new;
            float lsum = 0.0f;
#pragma unroll
            for (int jj = 0; jj < CN / 16; ++jj) {
                const float p = exp2f(sc[jj] - m_use);
                Ps[r * CN + c + 16 * jj] = p;
                lsum += p;
            }
#pragma unroll
            for (int o = 8; o > 0; o >>= 1) lsum += __shfl_xor(lsum, o, WAVE);
            l_run = l_run * alpha + lsum;
            __syncthreads();
#pragma unroll
            for (int dd = 0; dd < CMAXD / 16; ++dd) {
                const int d = c + 16 * dd;
                if (d < D) {
                    float x = acc[dd] * alpha;
                    for (int j = 0; j < CN; ++j) x = __builtin_fmaf(Ps[r * CN + j], Vs[j * D + d], x);
                    acc[dd] = x;
                }
            }
        }
    };
    if (a.groups > 0) {
        const int g = group_of(a, s);
        if (g >= 0) walk(prefix_of(a, g), false);
    }
    walk(keys_of(a, s), a.causal != 0);
    __syncthreads();
    const float inv = bad_page ? __builtin_nanf("") : l_run > 0.0f ? 1.0f / l_run : 0.0f;
    if (row_ok) {
        const int64_t at = s * a.os[0] + (t.from + token) * a.os[1] + head * a.os[2];
#pragma unroll
        for (int dd = 0; dd < CMAXD / 16; ++dd) {
            const int d = c + 16 * dd;
            if (d < D) store_any(a.o, a.dtype, at + d, acc[dd] * inv);
        }
    }
}

// ------------------------------------------------------------------ host side
namespace {

thread_local const char *last_kernel = "none";

bool sane(const int64_t *s, int n) {
    for (int i = 0; i < n; ++i)
        if (s[i] < 0 || s[i] >= (int64_t(1) << 40)) return false;
    return true;
}
bool int_aligned(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 3u) == 0; }

int launch_generic(const CacheArgs &a, hipStream_t s, const char *who) {
    const int64_t blocks = (a.new_tokens ? (static_cast<int64_t>(a.new_tokens) * a.each + CM - 1) / CM * a.entries : a.total_q * a.each / CM + a.entries) * a.kv_heads;
    AXHIP_REQUIRE(launch_fits(blocks, 256), AXHIP_ERR_UNSUPPORTED, "%s: grid too large", who);
    const size_t lds = sizeof(float) * (static_cast<size_t>(CM) * a.D + static_cast<size_t>(CN) * (a.D + 1) + static_cast<size_t>(CN) * a.D + CM * CN);
    static const hipError_t attr = hipFuncSetAttribute(reinterpret_cast<const void *>(sdpa_cache_generic_kernel), hipFuncAttributeMaxDynamicSharedMemorySize, 96 * 1024);
    AXHIP_CHECK_HIP(attr);
    last_kernel = "generic";
    hipLaunchKernelGGL(sdpa_cache_generic_kernel, dim3(static_cast<unsigned>(blocks)), dim3(256), lds, s, a);
    AXHIP_CHECK_HIP(hipGetLastError());
    return AXHIP_OK;
}

// What both entry points check alike, and the arguments that follow from it.
int common_args(const char *who, CacheArgs &a, int dtype, int heads, int kv_heads, int head_dim, float scale) {
    AXHIP_REQUIRE(valid_dtype(dtype), AXHIP_ERR_INVALID_ARG, "%s: bad dtype %d", who, dtype);
    AXHIP_REQUIRE(heads > 0 && kv_heads > 0 && heads < (1 << 20) && heads % kv_heads == 0, AXHIP_ERR_INVALID_ARG, "%s: %d heads over %d key heads", who, heads, kv_heads);
    AXHIP_REQUIRE(head_dim > 0, AXHIP_ERR_INVALID_ARG, "%s: head_dim %d", who, head_dim);
    AXHIP_REQUIRE(head_dim <= CMAXD, AXHIP_ERR_UNSUPPORTED, "%s: head_dim %d > %d is not supported", who, head_dim, CMAXD);
    AXHIP_REQUIRE(!std::isnan(scale) && !std::isinf(scale), AXHIP_ERR_INVALID_ARG, "%s: scale must be a finite number", who);
    a.dtype = dtype;
    a.heads = heads;
    a.kv_heads = kv_heads;
    a.each = heads / kv_heads;
    a.by_each = Divisor(static_cast<uint32_t>(a.each));
    a.D = head_dim;
    a.scale_log2e = static_cast<float>((scale > 0.0f ? static_cast<double>(scale) : 1.0 / std::sqrt(static_cast<double>(head_dim))) * 1.44269504088896340736);
    return AXHIP_OK;
}
int page_args(const char *who, CacheArgs &a, const AxhipKvPages &g, const int32_t *table, int64_t table_ld, const int32_t *lengths) {
    const int rc = check_pages(who, g);
    if (rc) return rc;
    AXHIP_REQUIRE(table_ld > 0 && table_ld < (int64_t(1) << 31), AXHIP_ERR_INVALID_ARG, "%s: bad table_ld", who);
    AXHIP_REQUIRE(table && lengths && int_aligned(table) && int_aligned(lengths), AXHIP_ERR_INVALID_ARG, "%s: NULL or unaligned page_table or kv_lengths", who);
    a.k = g.k;
    a.v = g.v;
    a.table = table;
    a.lengths = lengths;
    a.table_ld = table_ld;
    a.n_pages = g.n_pages;
    a.page_shift = __builtin_ctz(static_cast<unsigned>(g.page_size));
    for (int i = 0; i < 3; ++i) {
        a.ks[i] = g.k_strides[i];
        a.vs[i] = g.v_strides[i];
    }
    return AXHIP_OK;
}

int packed_args(CacheArgs &a, const AxhipSdpaPackedParams *params) {
    const char *who = "axhip_sdpa_packed";
    AXHIP_REQUIRE(params != nullptr, AXHIP_ERR_INVALID_ARG, "axhip_sdpa_packed: params is NULL");
    const AxhipSdpaPackedParams &p = *params;
    int rc = common_args(who, a, p.dtype, p.heads, p.kv_heads, p.head_dim, p.scale);
    if (rc) return rc;
    AXHIP_REQUIRE(p.n_seqs >= 0 && p.n_seqs < (1 << 24) && p.total_q >= 0 && p.total_q < MOST_KEYS, AXHIP_ERR_INVALID_ARG, "axhip_sdpa_packed: bad extent");
    AXHIP_REQUIRE(p.is_causal == 0 || p.is_causal == 1, AXHIP_ERR_INVALID_ARG, "axhip_sdpa_packed: is_causal is %d, neither 0 nor 1", p.is_causal);
    AXHIP_REQUIRE(sane(p.q_strides, 2) && sane(p.o_strides, 2), AXHIP_ERR_INVALID_ARG, "axhip_sdpa_packed: bad stride");
    a.entries = p.n_seqs;
    a.causal = p.is_causal;
    a.total_q = p.total_q;
    a.cu_q = p.cu_q;
    for (int i = 0; i < 2; ++i) {
        a.qs[i + 1] = p.q_strides[i];
        a.os[i + 1] = p.o_strides[i];
    }
    if (p.n_seqs == 0 || p.total_q == 0) return AXHIP_OK;
    AXHIP_REQUIRE((p.total_q == 1 || p.o_strides[0] >= p.head_dim) && (p.heads == 1 || p.o_strides[1] >= p.head_dim), AXHIP_ERR_INVALID_ARG, "axhip_sdpa_packed: rows of o overlap");
    AXHIP_REQUIRE(p.cu_q && int_aligned(p.cu_q), AXHIP_ERR_INVALID_ARG, "axhip_sdpa_packed: NULL or unaligned cu_q");
    if (p.page_table) {
        rc = page_args(who, a, p.pages, p.page_table, p.table_ld, p.kv_lengths);
        if (rc) return rc;
        AXHIP_REQUIRE(p.pages.dtype == p.dtype && p.pages.heads == p.kv_heads && p.pages.head_dim == p.head_dim, AXHIP_ERR_INVALID_ARG,
                      "axhip_sdpa_packed: pages of another type, other heads or another head_dim");
        return AXHIP_OK;
    }
    AXHIP_REQUIRE(p.total_kv >= 0 && p.total_kv < MOST_KEYS, AXHIP_ERR_INVALID_ARG, "axhip_sdpa_packed: bad extent");
    AXHIP_REQUIRE(sane(p.k_strides, 2) && sane(p.v_strides, 2), AXHIP_ERR_INVALID_ARG, "axhip_sdpa_packed: bad stride");
    AXHIP_REQUIRE(p.cu_kv && int_aligned(p.cu_kv), AXHIP_ERR_INVALID_ARG, "axhip_sdpa_packed: NULL or unaligned cu_kv");
    a.cu_kv = p.cu_kv;
    a.total_kv = p.total_kv;
    for (int i = 0; i < 2; ++i) {
        a.ks[i + 1] = p.k_strides[i];
        a.vs[i + 1] = p.v_strides[i];
    }
    return AXHIP_OK;
}

int paged_args(CacheArgs &a, const AxhipSdpaPagedParams *params) {
    const char *who = "axhip_sdpa_paged";
    AXHIP_REQUIRE(params != nullptr, AXHIP_ERR_INVALID_ARG, "axhip_sdpa_paged: params is NULL");
    const AxhipSdpaPagedParams &p = *params;
    int rc = common_args(who, a, p.pages.dtype, p.heads, p.pages.heads, p.pages.head_dim, p.scale);
    if (rc) return rc;
    AXHIP_REQUIRE(p.n_seqs >= 0 && p.n_seqs < (1 << 24) && p.new_tokens > 0 && p.new_tokens < (1 << 20) && static_cast<int64_t>(p.new_tokens) * p.heads < (1 << 30), AXHIP_ERR_INVALID_ARG, "axhip_sdpa_paged: %d sequences of %d new tokens", p.n_seqs,
                  p.new_tokens);
    AXHIP_REQUIRE(p.n_groups >= 0 && p.n_groups < (1 << 24) && p.reserved == 0, AXHIP_ERR_INVALID_ARG, "axhip_sdpa_paged: bad number of groups, or reserved is not 0");
    AXHIP_REQUIRE(sane(p.q_strides, 3) && sane(p.o_strides, 3), AXHIP_ERR_INVALID_ARG, "axhip_sdpa_paged: bad stride");
    a.entries = p.n_seqs;
    a.causal = 1;
    a.new_tokens = p.new_tokens;
    for (int i = 0; i < 3; ++i) {
        a.qs[i] = p.q_strides[i];
        a.os[i] = p.o_strides[i];
    }
    if (p.n_seqs == 0) return AXHIP_OK;
    const int64_t dim = p.pages.head_dim;
    AXHIP_REQUIRE((p.n_seqs == 1 || p.o_strides[0] >= dim) && (p.new_tokens == 1 || p.o_strides[1] >= dim) && (p.heads == 1 || p.o_strides[2] >= dim), AXHIP_ERR_INVALID_ARG,
                  "axhip_sdpa_paged: rows of o overlap");
    rc = page_args(who, a, p.pages, p.page_table, p.table_ld, p.kv_lengths);
    if (rc) return rc;
    if (p.n_groups > 0) {
        AXHIP_REQUIRE(p.prefix_ld > 0 && p.prefix_ld < (int64_t(1) << 31), AXHIP_ERR_INVALID_ARG, "axhip_sdpa_paged: bad prefix_ld");
        AXHIP_REQUIRE(p.group_starts && p.prefix_table && p.prefix_lengths && int_aligned(p.group_starts) && int_aligned(p.prefix_table) && int_aligned(p.prefix_lengths),
                      AXHIP_ERR_INVALID_ARG, "axhip_sdpa_paged: NULL or unaligned group_starts, prefix_table or prefix_lengths");
        a.groups = p.n_groups;
        a.group_starts = p.group_starts;
        a.prefix_table = p.prefix_table;
        a.prefix_lengths = p.prefix_lengths;
        a.prefix_ld = p.prefix_ld;
    }
    return AXHIP_OK;
}
// Whether the matrix-core kernels take the head size and the numbers of rows
bool form_for_matrix_cores(const CacheArgs &a) {
    const int es = static_cast<int>(dtype_size(a.dtype)), v = 16 / es;
    if (a.D % v != 0 || a.D > (es == 2 ? 256 : 128) || (a.table && a.page_shift < 3)) return false;
    // (numbers of rows with one more block for each entry are 32-bit ones; numbers of blocks are added up as floats, exactly below 2^24)
    const int64_t rows = (a.new_tokens ? static_cast<int64_t>(a.entries) * a.new_tokens : a.total_q) * a.each;
    return rows + int64_t(256) * a.entries < (int64_t(1) << (es == 4 ? 27 : 30));
}
// .. and rows can be moved 16 bytes at a time (and offsets inside a piece of 8 rows are 32-bit ones, and from one page to the next)
bool for_matrix_cores(const CacheArgs &a) {
    const int es = static_cast<int>(dtype_size(a.dtype));
    uint64_t seen = reinterpret_cast<uintptr_t>(a.q) | reinterpret_cast<uintptr_t>(a.k) | reinterpret_cast<uintptr_t>(a.v) | reinterpret_cast<uintptr_t>(a.o);
    for (int i = 0; i < 3; ++i) seen |= static_cast<uint64_t>(a.qs[i] | a.ks[i] | a.vs[i] | a.os[i]) * es;
    // (page 0 is read in the place of pages that do not exist)
    return form_for_matrix_cores(a) && (!a.table || a.n_pages > 0) && (seen & 15) == 0 && a.ks[1] < (1 << 26) && a.vs[1] < (1 << 26) && std::max(a.ks[0], a.vs[0]) * es < (int64_t(1) << 32);
}
// AXHIP_SDPA_TILE_WAVES=4|8: waves of a work-group of the tile kernel (measurements only)
const int tile_waves = [] {
    const char *e = getenv("AXHIP_SDPA_TILE_WAVES");
    return e ? atoi(e) : 0;
}();

// AXHIP_SDPA_F32_ROWS=16|64: rows of a work-group of the fp32 kernel of prompts (measurements only)
const int f32_rows = [] {
    const char *e = getenv("AXHIP_SDPA_F32_ROWS");
    return e ? atoi(e) : 0;
}();

// AXHIP_SDPA_FEW_ROWS=16|128: rows of a work-group of the 16-bit kernels of prompts (measurements only)
const int few_rows = [] {
    const char *e = getenv("AXHIP_SDPA_FEW_ROWS");
    return e ? atoi(e) : 0;
}();

// How a call is divided, and its temporary memory: what the parts leave for the join.  By the numbers in the arguments and the hints alone: nothing of it depends on addresses or on what the
// device holds.
struct CachePlan {
    int shares, parts;
    bool whole;                                         // decoding: one launch, nothing is divided
    bool apart;                                         // fp32 prompts: 64 rows to a work-group, not 16
    bool few;                                           // 16-bit prompts: 16 rows to a work-group, not 128
    size_t own_out, own_lse, part_out, part_lse, bytes; // places; all of it
};
void place_parts(CachePlan &p, const CacheArgs &a, size_t rows) {
    auto place = [&](size_t floats) { const size_t here = p.bytes; p.bytes = CallScratch::rounded(p.bytes + floats * sizeof(float)); return here; };
    p.part_out = place(rows * p.parts * a.D);
    p.part_lse = place(rows * p.parts);
}
// AXHIP_SDPA_STEP_GROUPS: work-groups of a step's own keys (measurements only)
const int step_groups = [] {
    const char *e = getenv("AXHIP_SDPA_STEP_GROUPS");
    return e ? atoi(e) : 0;
}();
CachePlan step_plan(const CacheArgs &a, int max_kv, int max_prefix) {
    CachePlan p{};
    p.parts = 1;
    const int64_t rows = static_cast<int64_t>(a.new_tokens) * a.each, tiles = (rows + 15) / 16, most = std::min(a.table_ld << a.page_shift, MOST_KEYS);
    const int64_t most_prefix = a.groups > 0 ? std::min(a.prefix_ld << a.page_shift, MOST_KEYS) : 0;
    // Short sequences stay whole: the join is a launch, 4 - 5 us, and a work-group walks 128 keys in 1.1 us.  (One sequence or eight, 32 heads of 128: of 640 keys 11.5 whole, 12.3 - 13.6 in shares; of
    // 1000 15.5 - 16.1, 12.4 - 13.5.  60 keys behind 400 of a prefix: 4 sequences 11.0 and 13.1, 256 49 and 52, the prefix being read by each.)
    const int64_t walk = std::min<int64_t>(std::max(max_kv, 0), most) + std::min<int64_t>(std::max(max_prefix, 0), most_prefix);
    p.whole = walk <= 640 && (a.groups == 0 || a.entries * tiles * a.kv_heads * walk <= 3 * 512 * 640);
    if (p.whole) return p;
    // parts of a prefix: one work-group for each CU, of 128 rows, in 32 bits two
    const bool f32 = a.dtype == AXHIP_DTYPE_F32;
    const int64_t per = f32 ? 16 : 128, blocks = (a.entries * rows + per - 1) / per * a.kv_heads;
    const int64_t prefix = std::min<int64_t>(std::max(max_prefix, 1), most_prefix);
    int64_t places = (f32 ? 512 : 256) / blocks;
    // .. half as many, of up to 1024 keys, beside own keys that would take more than 15 us if every sequence had as many as the hint says (lengths apart count for more than they are).  64
    // sequences behind 8192, all places and half of them: of 100 keys 31.4 us and 37.6, of 200 38.9 and 40.4, of 300 45.2 and 44.4 (lengths around that, the longest eight times as long, 46.4 and
    // 44.9), of 1000 83.9 and 76.0
    const double own_us = static_cast<double>(a.entries) * static_cast<double>(std::min<int64_t>(std::max(max_kv, 0), most)) * a.kv_heads * a.D * 4 / 5.2e6;
    if (!f32 && own_us > 15) places = std::min(places, std::max(128 / blocks, (prefix + 1023) / 1024));
    p.parts = a.groups == 0 ? 0 : static_cast<int>(std::max<int64_t>(1, std::min<int64_t>({64, places, (prefix + 63) / 64})));
    // shares of the own keys: two work-groups of four waves on each CU (64 sequences of 2000: 256 work-groups 105 us, 512 103, 1024 105), less what prefixes take of them in the same launch
    const int64_t groups = step_groups ? step_groups : f32 ? 512 : std::max<int64_t>(256, 512 - blocks * p.parts);
    p.shares = static_cast<int>(std::min<int64_t>(std::max<int64_t>(1, groups / (a.kv_heads * tiles)), (most + 127) / 128 * a.entries));
    const size_t own = (static_cast<size_t>(2 * p.shares) + (a.groups > 0 ? a.entries : 0)) * a.kv_heads * rows;
    p.bytes = CallScratch::rounded(sizeof(int2_t) * a.entries);
    auto place = [&](size_t floats) { const size_t here = p.bytes; p.bytes = CallScratch::rounded(p.bytes + floats * sizeof(float)); return here; };
    p.own_out = place(own * a.D);
    p.own_lse = place(own);
    place_parts(p, a, static_cast<size_t>(a.entries) * a.kv_heads * rows);
    return p;
}
// Prompts: the keys of a block of rows in parts where there are few blocks for the chip, or a few that are long.  In tiles of 64 keys at 1.5 us (16 rows of 16 bits: 0.55, of fp32: 0.9), the time is
// that of the longest walk or of all walks over the 512 work-groups that the chip holds, and with parts the join's: a launch and one write and one read of the partial results.  (Three of 333 tokens
// behind 1500 keys, 16 heads on 4: undivided 45.8 us, in two parts 44.6, in three 39.2, in four 49.7.)
CachePlan prompt_plan(const CacheArgs &a, int max_kv) {
    CachePlan p{};
    p.parts = 1;
    const int64_t most = std::min(a.table ? a.table_ld << a.page_shift : a.total_kv, MOST_KEYS), longest = std::min<int64_t>(std::max(max_kv, 1), std::max<int64_t>(most, 1));
    // 16 bits: 16 rows to a work-group, whose waves share the keys, where those fit the chip's 512 places and no walk is long (or no entry has more than those 16 rows, on average); else tiles of 128
    // rows.  (128 -> 16 rows: 31 prompts of 14 tokens behind 448 keys, 4 heads on 2, 18.8 -> 12.6 us; one of 1000, 8 heads of 64, 20.1 -> 13.4; 16 of 4 behind 2000, 32 heads on 8, 47.0 -> 40.2.
    // Beyond: 60 of 5 behind 600, 32 heads on 8, 34.7 -> 46.8; one of 2000, 4 heads of 64, 21.1 -> 27.6.)
    const bool fit = (a.total_q * a.each / 16 + (a.entries + 1) / 2) * a.kv_heads <= 512, short_ones = longest <= 1280 || a.total_q * a.each <= int64_t(16) * a.entries;
    p.few = a.dtype != AXHIP_DTYPE_F32 && (few_rows ? few_rows == 16 : fit && short_ones);
    const int rows = a.dtype == AXHIP_DTYPE_F32 || p.few ? 16 : 128;
    const double blocks = static_cast<double>(a.total_q * a.each / rows + (a.entries + 1) / 2) * a.kv_heads, tile = a.dtype == AXHIP_DTYPE_F32 ? 0.9 : p.few ? 0.55 : 1.5;
    const double tokens = static_cast<double>(std::min<int64_t>(longest, a.total_q / std::max(a.entries, 1))), average = a.causal ? static_cast<double>(longest) - tokens / 2 : static_cast<double>(longest);
    const double traffic = static_cast<double>(a.total_q) * a.heads * a.D * 8 / 4e6;
    double best = 0;
    for (int parts = 1; parts <= 32 && (parts == 1 || longest >= 128 * parts); ++parts) {
        const double time = tile / 64 * std::max(static_cast<double>(longest) / parts, blocks * average / 512) + (parts > 1 ? 4.5 + traffic * parts : 0.0);
        if (parts == 1 || time < 0.93 * best) {
            best = time;
            p.parts = parts;
        }
    }
    // fp32, nothing divided: work-groups of 16 rows whose waves take a step's keys in turn, or of 64 rows whose waves take 16 each, a quarter of the keys a step.  A work-group takes 6 us beside its
    // steps, of 2.8 us or 3.8 with others on the CU, and the chip holds 512.  16 -> 64 rows: 64 prompts of 62 tokens, 16 heads of 64, 49 -> 25 us, 8 of 500 89 -> 67; one of 2048, 32 heads of 128, stays:
    // 435, 494
    if (a.dtype == AXHIP_DTYPE_F32 && p.parts == 1) {
        auto time = [&](double count, double step_keys, double step) {
            return 6 * std::max(1.0, count / 512) + step * std::max(std::max(1.0, longest / step_keys), count / 512 * std::max(1.0, average / step_keys));
        };
        const double keys = a.D <= 64 ? 128 : 64, wide = static_cast<double>(a.total_q * a.each / 64 + (a.entries + 1) / 2) * a.kv_heads;
        p.apart = f32_rows ? f32_rows == 64 : time(wide, keys / 4, 3.8) < time(blocks, keys, 2.8);
    }
    if (p.parts > 1) place_parts(p, a, static_cast<size_t>(a.total_q) * a.heads);
    return p;
}
// The plan's places in temporary memory
int take_parts(const char *who, CacheArgs &a, const CachePlan &plan, CallScratch &scratch) {
    a.shares = plan.shares;
    a.parts = plan.parts;
    if (plan.bytes == 0) return AXHIP_OK;
    void *at = nullptr;
    const int rc = scratch.take(&at, plan.bytes, who);
    if (rc) return rc;
    char *p = static_cast<char *>(at);
    a.parts_of = reinterpret_cast<int2_t *>(p);
    a.own_out = reinterpret_cast<float *>(p + plan.own_out);
    a.own_lse = reinterpret_cast<float *>(p + plan.own_lse);
    a.part_out = reinterpret_cast<float *>(p + plan.part_out);
    a.part_lse = reinterpret_cast<float *>(p + plan.part_lse);
    return AXHIP_OK;
}
// (units of 128 keys are counted in 32 bits)
bool step_fits(const CacheArgs &a) { return (std::min(a.table_ld << a.page_shift, MOST_KEYS) / 128 + 1) * a.entries < (int64_t(1) << 31); }
bool tensor_ok(const void *p, int dtype) { return p && (reinterpret_cast<uintptr_t>(p) & (dtype_size(dtype) - 1)) == 0; }

} // namespace
} // namespace axhip
using namespace axhip;

extern "C" {

const char *axhip_sdpa_cache_last_kernel(void) { return last_kernel; }

// (asked for by form: a call whose addresses or strides send it to the generic kernel leaves it alone)
size_t axhip_sdpa_packed_workspace_bytes(const AxhipSdpaPackedParams *params) {
    CacheArgs a{};
    if (packed_args(a, params) != AXHIP_OK || a.entries == 0 || a.total_q == 0 || !form_for_matrix_cores(a)) return 0;
    return prompt_plan(a, params->max_kv).bytes;
}

int axhip_sdpa_packed(const void *q, const void *k, const void *v, void *o, const AxhipSdpaPackedParams *params, void *stream) {
    return axhip_sdpa_packed_ws(q, k, v, o, params, nullptr, 0, stream);
}

int axhip_sdpa_packed_ws(const void *q, const void *k, const void *v, void *o, const AxhipSdpaPackedParams *params, void *workspace, size_t workspace_bytes, void *stream) {
    CacheArgs a{};
    int rc = packed_args(a, params);
    if (rc) return rc;
    last_kernel = "empty";
    if (a.entries == 0 || a.total_q == 0) return AXHIP_OK;
    AXHIP_REQUIRE(tensor_ok(q, a.dtype) && tensor_ok(o, a.dtype), AXHIP_ERR_INVALID_ARG, "axhip_sdpa_packed: q or o is NULL or not aligned to its elements");
    if (a.table) {
        AXHIP_REQUIRE(!k && !v, AXHIP_ERR_INVALID_ARG, "axhip_sdpa_packed: k or v beside a page_table");
    } else {
        AXHIP_REQUIRE(a.total_kv == 0 || (tensor_ok(k, a.dtype) && tensor_ok(v, a.dtype)), AXHIP_ERR_INVALID_ARG, "axhip_sdpa_packed: k or v is NULL or not aligned to its elements");
        a.k = k;
        a.v = v;
    }
    a.q = q;
    a.o = o;
    rc = ensure_init();
    if (rc) return rc;
    hipStream_t s = resolve_stream(stream);
    if (!for_matrix_cores(a)) return launch_generic(a, s, "axhip_sdpa_packed");
    const CachePlan plan = prompt_plan(a, params->max_kv);
    CallScratch scratch(workspace, workspace_bytes, s);
    rc = take_parts("axhip_sdpa_packed", a, plan, scratch);
    if (rc) return rc;
    const bool f32 = a.dtype == AXHIP_DTYPE_F32, bf16 = a.dtype == AXHIP_DTYPE_BF16;
    if (f32) {
        last_kernel = plan.parts > 1 ? "f32, parts" : plan.apart ? "f32, apart" : "f32";
        rc = launch_rows_packed_f32(a, plan.apart, s);
    } else {
        const int64_t blocks = (a.total_q * a.each + 255) / 256 * a.kv_heads;
        // Two work-groups of four waves on a CU start and end beside each other's walk; eight waves of one go in pairs of opposite phases, which long walks of 97 .. 128 dims gain by: 32 heads of
        // 128, one prompt of 4096 136.6 -> 133.0 us, four of 512 behind 4000 keys 148.5 -> 144.8, 12 of 300 .. 5000 407 -> 399; 12 of 1365 238 either way, 64 of 256 112 -> 129; of 64 dims
        // 12 of 1365 134 -> 165, of 96 199 -> 207.
        const int waves = a.D <= 96 || a.D > 128 ? 4 : tile_waves ? tile_waves : blocks >= 256 && params->max_kv > 2048 && plan.parts == 1 ? 8 : 4;
        last_kernel = plan.few ? plan.parts > 1 ? "few, parts" : "few" : plan.parts > 1 ? "tile, parts" : waves == 8 ? "tile, eight waves" : "tile";
        if (plan.few) rc = bf16 ? launch_rows_packed_bf16(a, s) : launch_rows_packed_f16(a, s);
        else rc = bf16 ? launch_tile_bf16(a, waves, s) : launch_tile_f16(a, waves, s);
    }
    if (!rc && plan.parts > 1) rc = f32 ? launch_join_f32(a, s) : bf16 ? launch_join_bf16(a, s) : launch_join_f16(a, s);
    return rc ? rc : scratch.release();
}

size_t axhip_sdpa_paged_workspace_bytes(const AxhipSdpaPagedParams *params) {
    CacheArgs a{};
    if (paged_args(a, params) != AXHIP_OK || a.entries == 0 || !form_for_matrix_cores(a) || !step_fits(a)) return 0;
    return step_plan(a, params->max_kv, params->max_prefix).bytes;
}

int axhip_sdpa_paged(const void *q, void *o, const AxhipSdpaPagedParams *params, void *stream) { return axhip_sdpa_paged_ws(q, o, params, nullptr, 0, stream); }

int axhip_sdpa_paged_ws(const void *q, void *o, const AxhipSdpaPagedParams *params, void *workspace, size_t workspace_bytes, void *stream) {
    CacheArgs a{};
    int rc = paged_args(a, params);
    if (rc) return rc;
    last_kernel = "empty";
    if (a.entries == 0) return AXHIP_OK;
    AXHIP_REQUIRE(tensor_ok(q, a.dtype) && tensor_ok(o, a.dtype), AXHIP_ERR_INVALID_ARG, "axhip_sdpa_paged: q or o is NULL or not aligned to its elements");
    a.q = q;
    a.o = o;
    rc = ensure_init();
    if (rc) return rc;
    hipStream_t s = resolve_stream(stream);
    if (!for_matrix_cores(a) || !step_fits(a)) return launch_generic(a, s, "axhip_sdpa_paged");
    const CachePlan plan = step_plan(a, params->max_kv, params->max_prefix);
    CallScratch scratch(workspace, workspace_bytes, s);
    rc = take_parts("axhip_sdpa_paged", a, plan, scratch);
    if (rc) return rc;
    const bool f32 = a.dtype == AXHIP_DTYPE_F32, bf16 = a.dtype == AXHIP_DTYPE_BF16;
    if (plan.whole) {
        last_kernel = "whole";
        return f32 ? launch_rows_whole_f32(a, s) : bf16 ? launch_rows_whole_bf16(a, s) : launch_rows_whole_f16(a, s);
    }
    last_kernel = a.groups > 0 ? "shares, prefix" : "shares";
    if (a.groups > 0 && !f32) {
        rc = bf16 ? launch_step_bf16(a, s) : launch_step_f16(a, s);
    } else {
        if (a.groups > 0) {
            rc = launch_prefix_f32(a, s);
            if (rc) return rc;
        }
        rc = f32 ? launch_rows_own_f32(a, s) : bf16 ? launch_rows_own_bf16(a, s) : launch_rows_own_f16(a, s);
    }
    if (!rc) rc = f32 ? launch_join_f32(a, s) : bf16 ? launch_join_bf16(a, s) : launch_join_f16(a, s);
    return rc ? rc : scratch.release();
}

} // extern "C"
