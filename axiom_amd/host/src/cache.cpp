// Rotary positions, packed attention and a paged cache over the C ABI.
#include "axiom/cache.hpp"

#include <algorithm>
#include <atomic>
#include <cstdint>
#include <functional>
#include <string>

#include "axiom/operations.hpp"
#include "hip_call.hpp"

namespace axiom {
namespace {
void need_gpu(const char *who, const Tensor &t) {
    if (t.empty()) throw ValueError(std::string(who) + ": an empty tensor");
    if (t.device() != Device::GPU) throw RuntimeError(std::string(who) + " on CPU tensors: this library is the gfx950 GPU backend only; move the operands with .gpu()");
}
void need_floating(const char *who, const Tensor &t) {
    if (t.dtype() != DType::Float32 && t.dtype() != DType::Float16 && t.dtype() != DType::BFloat16) throw TypeError(std::string(who) + ": Float32, Float16 or BFloat16; got " + dtype_name(t.dtype()));
}
void need_type(const char *who, const char *what, const Tensor &t, DType want) {
    if (t.dtype() != want) throw TypeError(std::string(who) + ": " + what + " must be " + dtype_name(want) + ", got " + dtype_name(t.dtype()));
}
// contiguous, materialised
Tensor settled(const Tensor &t) {
    Tensor c = t.ascontiguousarray();
    c.sync();
    return c.ascontiguousarray();
}
// materialised, dims of a head side by side: views of a product's output stay views
Tensor rows_settled(const Tensor &t) {
    Tensor c = t;
    c.sync();
    const int64_t e = static_cast<int64_t>(c.itemsize());
    if (c.strides().back() != e && c.shape().back() > 1) return settled(c);
    for (int64_t s : c.strides())
        if (s < 0 || s % e != 0) return settled(c);
    return c;
}
const char *at(const Tensor &t) { return t.empty() ? nullptr : static_cast<const char *>(t.storage()->raw()) + t.offset(); }
char *out_at(const Tensor &t) { return static_cast<char *>(t.storage()->raw()) + t.offset(); }
template <class T> const T *as(const Tensor &t) { return reinterpret_cast<const T *>(at(t)); }
template <size_t N> void strides_into(int64_t (&to)[N], const Tensor &t) { // of the leading N dims, in elements
    for (size_t i = 0; i < N; ++i) to[i] = t.strides()[i] / static_cast<int64_t>(t.itemsize());
}
Tensor on_device(const std::vector<int32_t> &v, Shape shape) { return Tensor::from_data(v.data(), shape, Device::GPU); }
Tensor on_device(const std::vector<int64_t> &v, Shape shape) { return Tensor::from_data(v.data(), shape, Device::GPU); }
Tensor workspace_of(size_t bytes) { return bytes ? Tensor(Shape{bytes}, DType::UInt8, Device::GPU) : Tensor(); }
void *workspace_at(const Tensor &t) { return t.empty() ? nullptr : out_at(t); }

// q, k or v of a call: (tokens, heads, head_dim)
void need_heads(const char *who, const char *what, const Tensor &t, DType dtype, size_t head_dim) {
    need_gpu(who, t);
    if (t.ndim() != 3 || t.shape()[2] != head_dim) throw ShapeError(std::string(who) + ": " + what + " must be (tokens, heads, " + std::to_string(head_dim) + ")");
    need_type(who, what, t, dtype);
}
} // namespace

namespace ops {

Tensor rotary_turns(size_t rot_dim, double theta, const RotaryScaling &scaling) {
    if (rot_dim < 2 || rot_dim > 1024 || rot_dim % 2 != 0) throw ValueError("rotary_turns: rot_dim must be an even number from 2 to 1024, got " + std::to_string(rot_dim));
    AxhipRopeScaling s{};
    s.rot_dim = static_cast<int32_t>(rot_dim);
    s.kind = static_cast<int32_t>(scaling.kind);
    s.theta = theta;
    s.factor = scaling.factor;
    s.low = scaling.low;
    s.high = scaling.high;
    s.length = scaling.length;
    std::vector<uint64_t> turns(rot_dim / 2);
    if (axhip_rope_turns(&s, turns.data()) != 0) throw ValueError(axhip_last_error());
    return on_device(std::vector<int64_t>(turns.begin(), turns.end()), Shape{rot_dim / 2});
}

Tensor rotary(const Tensor &x, const Tensor &positions, const Tensor &turns, bool interleaved, bool inverse, float amplitude) {
    const char *who = "rotary";
    need_gpu(who, x);
    need_floating(who, x);
    need_gpu(who, positions);
    need_gpu(who, turns);
    need_type(who, "turns", turns, DType::Int64);
    if (positions.dtype() != DType::Int32 && positions.dtype() != DType::Int64) throw TypeError("rotary: positions must be Int32 or Int64, got " + dtype_name(positions.dtype()));
    if (x.ndim() < 2) throw ShapeError("rotary: (..., heads, head_dim)");
    const size_t dim = x.shape().back(), heads = x.shape()[x.ndim() - 2], tokens = dim != 0 && heads != 0 ? x.size() / (dim * heads) : 0;
    if (2 * turns.size() > dim || turns.size() == 0) throw ShapeError("rotary: " + std::to_string(turns.size()) + " angles for heads of " + std::to_string(dim));
    if (positions.size() != tokens) throw ShapeError("rotary: a position for each of " + std::to_string(tokens) + " rows of heads, got " + std::to_string(positions.size()));
    const Tensor src = settled(x), pos = settled(positions), table = settled(turns);
    Tensor out(x.shape(), x.dtype(), Device::GPU);
    AxhipRopeParams p{};
    p.dtype = ::axiom::detail::to_axhip_dtype(x.dtype());
    p.heads = static_cast<int32_t>(heads);
    p.head_dim = static_cast<int32_t>(dim);
    p.rot_dim = static_cast<int32_t>(2 * turns.size());
    p.interleaved = interleaved;
    p.inverse = inverse;
    p.amplitude = amplitude;
    p.position_bytes = static_cast<int32_t>(positions.itemsize());
    p.tokens = static_cast<int64_t>(tokens);
    for (int64_t(*s)[2] : {&p.x_strides, &p.y_strides}) {
        (*s)[0] = static_cast<int64_t>(heads * dim);
        (*s)[1] = static_cast<int64_t>(dim);
    }
    p.positions = at(pos);
    p.turns = as<uint64_t>(table);
    AXHIP_CALL(axhip_rope(at(src), out_at(out), &p, nullptr));
    return out; // asynchronous; .cpu() / item() synchronise
}

Tensor packed_attention(const Tensor &q, const Tensor &k, const Tensor &v, const Tensor &starts_q, const Tensor &starts_kv, bool is_causal, float scale, size_t longest_keys) {
    const char *who = "packed_attention";
    need_gpu(who, q);
    need_floating(who, q);
    if (q.ndim() != 3) throw ShapeError("packed_attention: q must be (tokens, heads, head_dim)");
    need_heads(who, "k", k, q.dtype(), q.shape()[2]);
    need_heads(who, "v", v, q.dtype(), q.shape()[2]);
    if (k.shape() != v.shape()) throw ShapeError("packed_attention: k and v must have one shape");
    if (k.shape()[1] == 0 || q.shape()[1] % k.shape()[1] != 0)
        throw ShapeError("packed_attention: " + std::to_string(q.shape()[1]) + " heads are no multiple of " + std::to_string(k.shape()[1]) + " key heads");
    for (const Tensor *t : {&starts_q, &starts_kv}) {
        need_gpu(who, *t);
        need_type(who, "starts", *t, DType::Int32);
        if (t->ndim() != 1 || t->size() == 0 || t->size() != starts_q.size()) throw ShapeError("packed_attention: starts of n sequences have n + 1 numbers");
    }
    const Tensor qs = rows_settled(q), ks = rows_settled(k), vs = rows_settled(v), cq = settled(starts_q), ck = settled(starts_kv);
    Tensor out = Tensor::zeros(q.shape(), q.dtype(), Device::GPU);
    AxhipSdpaPackedParams p{};
    p.dtype = ::axiom::detail::to_axhip_dtype(q.dtype());
    p.heads = static_cast<int32_t>(q.shape()[1]);
    p.kv_heads = static_cast<int32_t>(k.shape()[1]);
    p.head_dim = static_cast<int32_t>(q.shape()[2]);
    p.n_seqs = static_cast<int32_t>(starts_q.size() - 1);
    p.is_causal = is_causal;
    p.scale = scale;
    p.total_q = static_cast<int64_t>(q.shape()[0]);
    p.total_kv = static_cast<int64_t>(k.shape()[0]);
    // (What the starts hold is on the device: a sequence is taken to have up to twice the average. As many as all together have, 20 prompts of 60 tokens would be computed in three parts and joined.)
    const size_t total = k.shape()[0], n = starts_q.size() - 1;
    p.max_kv = static_cast<int32_t>(std::min<size_t>(longest_keys ? longest_keys : n == 0 ? total : std::min(total, 2 * ((total + n - 1) / n)), 1u << 30));
    strides_into(p.q_strides, qs);
    strides_into(p.k_strides, ks);
    strides_into(p.v_strides, vs);
    strides_into(p.o_strides, out);
    p.cu_q = as<int32_t>(cq);
    p.cu_kv = as<int32_t>(ck);
    const size_t need = axhip_sdpa_packed_workspace_bytes(&p);
    const Tensor ws = workspace_of(need);
    AXHIP_CALL(axhip_sdpa_packed_ws(at(qs), at(ks), at(vs), out_at(out), &p, workspace_at(ws), need, nullptr));
    return out;
}

} // namespace ops

namespace nn {

PageBook::PageBook(size_t pages, size_t page_size) : page_size_(page_size), users_(pages, 0) {
    if (page_size == 0 || page_size > 65536 || (page_size & (page_size - 1)) != 0) throw ValueError("PageBook: a page has a power of two of rows, up to 65536; got " + std::to_string(page_size));
    if (pages >= (size_t(1) << 31)) throw ValueError("PageBook: too many pages");
    for (size_t i = pages; i > 0; --i) free_.push_back(static_cast<int32_t>(i - 1));
}

PageBook::Sequence &PageBook::at(int sequence) {
    if (sequence < 0 || static_cast<size_t>(sequence) >= sequences_.size() || !sequences_[sequence].live) throw IndexError("PageBook: no sequence " + std::to_string(sequence));
    return sequences_[sequence];
}
int PageBook::place() {
    for (size_t i = 0; i < sequences_.size(); ++i)
        if (!sequences_[i].live) return static_cast<int>(i);
    sequences_.emplace_back();
    return static_cast<int>(sequences_.size() - 1);
}
int32_t PageBook::take() {
    const int32_t page = free_.back();
    free_.pop_back();
    users_[page] = 1;
    return page;
}
void PageBook::drop(int32_t page) {
    if (--users_[page] > 0) return;
    // (the lowest free page is taken first, which keeps the pool's end empty)
    free_.insert(std::upper_bound(free_.begin(), free_.end(), page, std::greater<int32_t>()), page);
}

int PageBook::add() {
    const int s = place();
    sequences_[s] = Sequence{true, 0, {}};
    return s;
}
int PageBook::fork(int sequence) {
    at(sequence);
    const int s = place();
    sequences_[s] = sequences_[sequence];
    for (int32_t page : sequences_[s].pages) ++users_[page];
    return s;
}
void PageBook::release(int sequence) {
    Sequence &s = at(sequence);
    for (int32_t page : s.pages) drop(page);
    s = Sequence{};
}
void PageBook::truncate(int sequence, size_t length) {
    Sequence &s = at(sequence);
    if (length > s.length) throw ValueError("PageBook: a sequence of " + std::to_string(s.length) + " tokens has no first " + std::to_string(length));
    const size_t keep = (length + page_size_ - 1) / page_size_;
    while (s.pages.size() > keep) {
        drop(s.pages.back());
        s.pages.pop_back();
    }
    s.length = length;
}

void PageBook::extend(const std::vector<int> &sequences, const std::vector<size_t> &new_tokens, std::vector<Copy> &copies) {
    if (sequences.size() != new_tokens.size()) throw ValueError("PageBook: a number of new tokens for each sequence");
    std::vector<char> named(sequences_.size(), 0);
    // What it takes, before anything is changed.  A shared last page is copied for each sequence that writes to it but the last one that lists it.
    size_t need = 0;
    std::vector<std::pair<int32_t, int32_t>> left; // pages whose users go down
    auto users_left = [&](int32_t page) -> int32_t & {
        for (auto &p : left)
            if (p.first == page) return p.second;
        left.emplace_back(page, users_[page]);
        return left.back().second;
    };
    for (size_t i = 0; i < sequences.size(); ++i) {
        const Sequence &s = at(sequences[i]);
        if (named[sequences[i]]++) throw ValueError("PageBook: sequence " + std::to_string(sequences[i]) + " is named twice");
        if (new_tokens[i] == 0) continue;
        if (s.length + new_tokens[i] > (size_t(1) << 30)) throw ValueError("PageBook: a sequence has up to 2^30 tokens");
        need += (s.length + new_tokens[i] + page_size_ - 1) / page_size_ - s.pages.size();
        if (s.length % page_size_ != 0) {
            int32_t &users = users_left(s.pages.back());
            if (users > 1) {
                --users;
                ++need;
            }
        }
    }
    if (need > free_.size()) throw RuntimeError("PageBook: " + std::to_string(need) + " pages are needed, " + std::to_string(free_.size()) + " are free");
    for (size_t i = 0; i < sequences.size(); ++i) {
        Sequence &s = at(sequences[i]);
        if (new_tokens[i] == 0) continue;
        if (s.length % page_size_ != 0 && users_[s.pages.back()] > 1) {
            const int32_t old = s.pages.back();
            s.pages.back() = take();
            drop(old);
            copies.push_back(Copy{old, s.pages.back(), static_cast<int32_t>(s.length % page_size_)});
        }
        s.length += new_tokens[i];
        while (s.pages.size() * page_size_ < s.length) s.pages.push_back(take());
    }
}

void PageBook::take_back(const std::vector<int> &sequences, const std::vector<size_t> &new_tokens, const std::vector<Copy> &copies) {
    size_t copied = copies.size(); // (in the sequences' order)
    for (size_t i = sequences.size(); i-- > 0;) {
        if (new_tokens[i] == 0) continue;
        Sequence &s = at(sequences[i]);
        s.length -= new_tokens[i];
        while (s.pages.size() > (s.length + page_size_ - 1) / page_size_) {
            drop(s.pages.back());
            s.pages.pop_back();
        }
        if (s.length % page_size_ != 0 && copied > 0 && copies[copied - 1].dst == s.pages.back()) {
            drop(s.pages.back());
            s.pages.back() = copies[--copied].src;
            ++users_[s.pages.back()];
        }
    }
}

std::vector<PageBook::Copy> PageBook::compact() {
    const size_t used = users_.size() - free_.size();
    std::vector<int32_t> to(users_.size(), -1); // where a page moves
    std::vector<Copy> copies;
    for (size_t page = used; page < users_.size(); ++page) {
        if (users_[page] == 0) continue;
        const int32_t dst = free_.back(); // the lowest free one: below `used`, as many as there are pages in use behind it
        free_.pop_back();
        to[page] = dst;
        users_[dst] = users_[page];
        users_[page] = 0;
        copies.push_back(Copy{static_cast<int32_t>(page), dst, static_cast<int32_t>(page_size_)});
    }
    free_.clear();
    for (size_t i = users_.size(); i > used; --i) free_.push_back(static_cast<int32_t>(i - 1));
    for (Sequence &s : sequences_)
        for (int32_t &page : s.pages)
            if (to[page] >= 0) page = to[page];
    return copies;
}

std::vector<PageBook::Group> PageBook::groups(const std::vector<int> &sequences, const std::vector<size_t> &new_tokens) const {
    if (sequences.size() != new_tokens.size()) throw ValueError("PageBook: a number of new tokens for each sequence");
    const size_t n = sequences.size();
    // What neighbours have in common; that of a run is the least of its neighbours'
    std::vector<size_t> common(n, 0);
    for (size_t i = 0; i < n; ++i) {
        const Sequence &s = at(sequences[i]);
        if (new_tokens[i] > s.length) throw ValueError("PageBook: a sequence of " + std::to_string(s.length) + " tokens has no last " + std::to_string(new_tokens[i]));
        if (i == 0) continue;
        const Sequence &before = at(sequences[i - 1]);
        const size_t most = std::min(s.length - new_tokens[i], before.length - new_tokens[i - 1]) / page_size_;
        while (common[i] < most && s.pages[common[i]] == before.pages[common[i]]) ++common[i];
    }
    // Runs may begin in front of any sequence, but where several neighbours in turn have as much in common, only the first and the last of them need be tried: a border between those moves to
    // one side without loss, since no run counts them for more than they have in common.
    std::vector<size_t> borders{0};
    for (size_t i = 1; i < n; ++i)
        if (i == 1 || i == n - 1 || common[i] != common[i - 1] || common[i] != common[i + 1]) borders.push_back(i);
    if (n > 0) borders.push_back(n);
    // A run of m sequences saves m - 1 readings of its common pages: saved[j] is the most that those in front of border j can, from[j] the border where their last run begins.  (Pairs of
    // borders: 256 sequences behind one prefix 5 us, 127 where no two neighbours in turn have as much in common.)
    std::vector<size_t> saved(borders.size(), 0), from(borders.size(), 0), pages(borders.size(), 0);
    for (size_t j = 1; j < borders.size(); ++j) {
        size_t shared = SIZE_MAX;
        for (size_t i = j; i-- > 0;) {
            if (i + 1 < j) shared = std::min(shared, common[borders[i + 1]]);
            if (borders[i] + 1 < borders[i + 1]) shared = std::min(shared, common[borders[i] + 1]);
            const size_t more = borders[j] - borders[i] - 1, with = saved[i] + (more ? more * shared : 0);
            if (i + 1 == j || with > saved[j]) {
                saved[j] = with;
                from[j] = i;
                pages[j] = more ? shared : 0;
            }
            if (shared == 0) break;
        }
    }
    std::vector<Group> found; // the last one first
    for (size_t j = borders.size() - 1; n > 0 && j > 0; j = from[j]) {
        if (pages[j] > 0) {
            found.push_back(Group{borders[j], pages[j]});
        } else {
            for (size_t end = borders[j]; end > borders[from[j]]; --end) found.push_back(Group{end, 0});
        }
    }
    std::reverse(found.begin(), found.end());
    return found;
}

int64_t PageBook::slot(int sequence, size_t position) const {
    const Sequence &s = at(sequence);
    if (position >= s.length) throw IndexError("PageBook: no token " + std::to_string(position) + " of " + std::to_string(s.length));
    return static_cast<int64_t>(s.pages[position / page_size_]) * static_cast<int64_t>(page_size_) + static_cast<int64_t>(position % page_size_);
}

PagedCache::PagedCache(size_t layers, size_t pages, size_t page_size, size_t kv_heads, size_t head_dim, DType dtype)
    : book_(pages, page_size), layers_(layers), kv_heads_(kv_heads), head_dim_(head_dim) {
    if (dtype != DType::Float32 && dtype != DType::Float16 && dtype != DType::BFloat16) throw TypeError("PagedCache: Float32, Float16 or BFloat16; got " + dtype_name(dtype));
    if (layers == 0 || pages == 0 || kv_heads == 0 || head_dim == 0) throw ValueError("PagedCache: no layers, pages, heads or dims");
    k_ = Tensor(Shape{layers, pages, page_size, kv_heads, head_dim}, dtype, Device::GPU);
    v_ = Tensor(Shape{layers, pages, page_size, kv_heads, head_dim}, dtype, Device::GPU);
    changed();
}
void PagedCache::changed() {
    static std::atomic<uint64_t> versions{0};
    version_ = ++versions;
}
void PagedCache::need_current(const CacheStep &step) const {
    if (step.version != version_) throw ValueError("PagedCache: the step is of another cache, or of sequences that have changed since");
}

namespace {
AxhipKvPages pages_of(const Tensor &k, const Tensor &v, size_t layer) {
    AxhipKvPages g{};
    const Shape &s = k.shape();
    const size_t bytes = layer * s[1] * s[2] * s[3] * s[4] * k.itemsize();
    g.k = out_at(k) + bytes;
    g.v = out_at(v) + bytes;
    g.dtype = ::axiom::detail::to_axhip_dtype(k.dtype());
    g.n_pages = static_cast<int64_t>(s[1]);
    g.page_size = static_cast<int32_t>(s[2]);
    g.heads = static_cast<int32_t>(s[3]);
    g.head_dim = static_cast<int32_t>(s[4]);
    const int64_t strides[3] = {static_cast<int64_t>(s[2] * s[3] * s[4]), static_cast<int64_t>(s[3] * s[4]), static_cast<int64_t>(s[4])};
    std::copy(strides, strides + 3, g.k_strides);
    std::copy(strides, strides + 3, g.v_strides);
    return g;
}
} // namespace

void PagedCache::copy(const std::vector<PageBook::Copy> &copies) {
    if (copies.empty()) return;
    std::vector<int32_t> src, dst, rows;
    for (const PageBook::Copy &c : copies) {
        src.push_back(c.src);
        dst.push_back(c.dst);
        rows.push_back(c.rows);
    }
    const Shape n{copies.size()};
    const Tensor s = on_device(src, n), d = on_device(dst, n), r = on_device(rows, n);
    AxhipKvCopyParams p{};
    p.pages = pages_of(k_, v_, 0);
    p.layers = static_cast<int32_t>(layers_);
    p.pairs = static_cast<int32_t>(copies.size());
    p.k_layer_stride = p.v_layer_stride = p.pages.k_strides[0] * p.pages.n_pages;
    p.src = as<int32_t>(s);
    p.dst = as<int32_t>(d);
    p.rows = as<int32_t>(r);
    AXHIP_CALL(axhip_kv_copy_pages(&p, nullptr));
}

// (Pages are copied to pages that are free by the old book: until the new one holds, nobody minds what lies there.)
size_t PagedCache::compact() {
    PageBook compacted = book_;
    const std::vector<PageBook::Copy> copies = compacted.compact();
    copy(copies);
    book_ = std::move(compacted);
    changed();
    return copies.size();
}

CacheStep PagedCache::extend(const std::vector<int> &sequences, const std::vector<size_t> &new_tokens) {
    if (sequences.empty()) throw ValueError("PagedCache: a step of no sequences");
    for (size_t n : new_tokens)
        if (n == 0) throw ValueError("PagedCache: a step has a token at least of each of its sequences");
    std::vector<PageBook::Copy> copies;
    book_.extend(sequences, new_tokens, copies);
    CacheStep step;
    try {
        copy(copies);
        step = step_of(sequences, new_tokens);
    } catch (...) { // (memory, a launch that is refused)
        book_.take_back(sequences, new_tokens, copies);
        throw;
    }
    changed();
    step.version = version_;
    return step;
}

CacheStep PagedCache::step_of(const std::vector<int> &sequences, const std::vector<size_t> &new_tokens) const {
    const size_t n = sequences.size(), page = book_.page_size();
    CacheStep step;
    step.sequences = sequences;
    step.new_tokens = new_tokens;
    step.each = new_tokens[0];
    std::vector<int64_t> positions, slots;
    std::vector<int32_t> starts{0};
    for (size_t i = 0; i < n; ++i) {
        if (new_tokens[i] != step.each) step.each = 0;
        const size_t length = book_.length(sequences[i]);
        for (size_t t = length - new_tokens[i]; t < length; ++t) {
            positions.push_back(static_cast<int64_t>(t));
            slots.push_back(book_.slot(sequences[i], t));
        }
        starts.push_back(static_cast<int32_t>(positions.size()));
    }
    step.tokens = positions.size();
    // Sequences behind common pages.  More than 16 new tokens of each are prompts, whose attention reads every sequence's pages by itself.
    std::vector<int32_t> groups{0}, prefixes;
    std::vector<size_t> skipped(n, 0);
    bool shared = false;
    if (step.each && step.each <= 16) {
        for (const PageBook::Group &g : book_.groups(sequences, new_tokens)) {
            for (size_t j = static_cast<size_t>(groups.back()); j < g.end; ++j) skipped[j] = g.pages;
            prefixes.push_back(static_cast<int32_t>(g.pages * page));
            groups.push_back(static_cast<int32_t>(g.end));
            shared = shared || g.pages > 0;
        }
    }
    size_t columns = 1;
    for (size_t i = 0; i < n; ++i) columns = std::max(columns, book_.pages(sequences[i]).size() - skipped[i]);
    std::vector<int32_t> table(n * columns, -1), lengths;
    for (size_t i = 0; i < n; ++i) {
        const std::vector<int32_t> &own = book_.pages(sequences[i]);
        std::copy(own.begin() + static_cast<ptrdiff_t>(skipped[i]), own.end(), table.begin() + static_cast<ptrdiff_t>(i * columns));
        lengths.push_back(static_cast<int32_t>(book_.length(sequences[i]) - skipped[i] * page));
        step.longest = std::max(step.longest, static_cast<size_t>(lengths.back()));
    }
    step.positions = on_device(positions, Shape{step.tokens});
    step.slots = on_device(slots, Shape{step.tokens});
    step.starts = on_device(starts, Shape{n + 1});
    step.page_table = on_device(table, Shape{n, columns});
    step.lengths = on_device(lengths, Shape{n});
    if (shared) {
        size_t prefix_columns = 1;
        for (int32_t p : prefixes) prefix_columns = std::max(prefix_columns, static_cast<size_t>(p) / page);
        std::vector<int32_t> prefix_table(prefixes.size() * prefix_columns, -1);
        for (size_t g = 0; g < prefixes.size(); ++g) {
            const std::vector<int32_t> &own = book_.pages(sequences[groups[g]]);
            std::copy(own.begin(), own.begin() + static_cast<ptrdiff_t>(static_cast<size_t>(prefixes[g]) / page), prefix_table.begin() + static_cast<ptrdiff_t>(g * prefix_columns));
            step.longest_prefix = std::max(step.longest_prefix, static_cast<size_t>(prefixes[g]));
        }
        step.group_starts = on_device(groups, Shape{groups.size()});
        step.prefix_table = on_device(prefix_table, Shape{prefixes.size(), prefix_columns});
        step.prefix_lengths = on_device(prefixes, Shape{prefixes.size()});
    }
    return step;
}

Tensor PagedCache::append(size_t layer, const CacheStep &step, const Tensor &q, const Tensor &k, const Tensor &v, const Tensor &turns, bool interleaved, float amplitude) {
    const char *who = "PagedCache::append";
    if (layer >= layers_) throw IndexError("PagedCache: no layer " + std::to_string(layer));
    need_current(step);
    need_heads(who, "q", q, k_.dtype(), head_dim_);
    for (const Tensor *t : {&k, &v}) {
        need_heads(who, t == &k ? "k" : "v", *t, k_.dtype(), head_dim_);
        if (t->shape()[1] != kv_heads_) throw ShapeError("PagedCache: " + std::to_string(kv_heads_) + " key heads, got " + std::to_string(t->shape()[1]));
    }
    for (const Tensor *t : {&q, &k, &v})
        if (t->shape()[0] != step.tokens) throw ShapeError("PagedCache: the step has " + std::to_string(step.tokens) + " tokens, got " + std::to_string(t->shape()[0]));
    Tensor table;
    if (!turns.empty()) {
        need_gpu(who, turns);
        need_type(who, "turns", turns, DType::Int64);
        if (turns.size() == 0 || 2 * turns.size() > head_dim_) throw ShapeError("PagedCache: " + std::to_string(turns.size()) + " angles for heads of " + std::to_string(head_dim_));
        table = settled(turns);
    }
    const Tensor qs = rows_settled(q), ks = rows_settled(k), vs = rows_settled(v);
    Tensor out(q.shape(), q.dtype(), Device::GPU);
    AxhipKvAppendParams p{};
    p.pages = pages_of(k_, v_, layer);
    p.heads = static_cast<int32_t>(q.shape()[1]);
    p.rot_dim = turns.empty() ? 0 : static_cast<int32_t>(2 * turns.size());
    p.interleaved = interleaved;
    p.amplitude = amplitude;
    p.position_bytes = 8;
    p.tokens = static_cast<int64_t>(step.tokens);
    strides_into(p.q_strides, qs);
    strides_into(p.k_strides, ks);
    strides_into(p.v_strides, vs);
    strides_into(p.q_out_strides, out);
    p.positions = at(step.positions);
    p.turns = as<uint64_t>(table);
    p.slots = as<int64_t>(step.slots);
    AXHIP_CALL(axhip_kv_append(at(qs), at(ks), at(vs), out_at(out), &p, nullptr));
    return out;
}

Tensor PagedCache::attend(size_t layer, const CacheStep &step, const Tensor &q, float scale) const {
    const char *who = "PagedCache::attend";
    if (layer >= layers_) throw IndexError("PagedCache: no layer " + std::to_string(layer));
    need_current(step);
    need_heads(who, "q", q, k_.dtype(), head_dim_);
    const size_t heads = q.shape()[1];
    if (q.shape()[0] != step.tokens) throw ShapeError("PagedCache: the step has " + std::to_string(step.tokens) + " tokens, got " + std::to_string(q.shape()[0]));
    if (heads == 0 || heads % kv_heads_ != 0) throw ShapeError("PagedCache: " + std::to_string(heads) + " heads are no multiple of " + std::to_string(kv_heads_) + " key heads");
    const Tensor qs = rows_settled(q);
    Tensor out(q.shape(), q.dtype(), Device::GPU);
    // A few tokens of each sequence are a decoding step; more of them, or different numbers, prompts
    if (step.each && step.each <= 16) {
        AxhipSdpaPagedParams p{};
        p.pages = pages_of(k_, v_, layer);
        p.heads = static_cast<int32_t>(heads);
        p.n_seqs = static_cast<int32_t>(step.sequences.size());
        p.new_tokens = static_cast<int32_t>(step.each);
        p.max_kv = static_cast<int32_t>(step.longest);
        p.max_prefix = static_cast<int32_t>(step.longest_prefix);
        p.scale = scale;
        int64_t s[2];
        strides_into(s, qs);
        const int64_t q_strides[3] = {s[0] * p.new_tokens, s[0], s[1]};
        std::copy(q_strides, q_strides + 3, p.q_strides);
        strides_into(s, out);
        const int64_t o_strides[3] = {s[0] * p.new_tokens, s[0], s[1]};
        std::copy(o_strides, o_strides + 3, p.o_strides);
        p.page_table = as<int32_t>(step.page_table);
        p.table_ld = static_cast<int64_t>(step.page_table.shape()[1]);
        p.kv_lengths = as<int32_t>(step.lengths);
        if (!step.group_starts.empty()) {
            p.n_groups = static_cast<int32_t>(step.prefix_lengths.size());
            p.group_starts = as<int32_t>(step.group_starts);
            p.prefix_table = as<int32_t>(step.prefix_table);
            p.prefix_ld = static_cast<int64_t>(step.prefix_table.shape()[1]);
            p.prefix_lengths = as<int32_t>(step.prefix_lengths);
        }
        const size_t need = axhip_sdpa_paged_workspace_bytes(&p);
        const Tensor ws = workspace_of(need);
        AXHIP_CALL(axhip_sdpa_paged_ws(at(qs), out_at(out), &p, workspace_at(ws), need, nullptr));
        return out;
    }
    AxhipSdpaPackedParams p{};
    p.pages = pages_of(k_, v_, layer);
    p.dtype = p.pages.dtype;
    p.heads = static_cast<int32_t>(heads);
    p.kv_heads = static_cast<int32_t>(kv_heads_);
    p.head_dim = static_cast<int32_t>(head_dim_);
    p.n_seqs = static_cast<int32_t>(step.sequences.size());
    p.is_causal = 1;
    p.scale = scale;
    p.max_kv = static_cast<int32_t>(step.longest);
    p.total_q = static_cast<int64_t>(step.tokens);
    strides_into(p.q_strides, qs);
    strides_into(p.o_strides, out);
    p.cu_q = as<int32_t>(step.starts);
    p.page_table = as<int32_t>(step.page_table);
    p.table_ld = static_cast<int64_t>(step.page_table.shape()[1]);
    p.kv_lengths = as<int32_t>(step.lengths);
    const size_t need = axhip_sdpa_packed_workspace_bytes(&p);
    const Tensor ws = workspace_of(need);
    AXHIP_CALL(axhip_sdpa_packed_ws(at(qs), nullptr, nullptr, out_at(out), &p, workspace_at(ws), need, nullptr));
    return out;
}

} // namespace nn
} // namespace axiom
