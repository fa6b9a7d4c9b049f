// A decoder's positions and its cache: rotary positions, attention of packed prompts, and keys and values in pages that sequences share, fork and give back.  None of it has a
// counterpart in Axiom; names and checks follow ops:: and nn::.  Everything runs when called, on the materialised inputs, and needs Device::GPU (PageBook alone needs no device).
#pragma once

#include <cstdint>
#include <utility>
#include <vector>

#include "axiom/tensor.hpp"

namespace axiom {
namespace ops {

// Contexts longer than the trained `length` (see axhip_rope_turns for the formulas)
struct RotaryScaling {
    enum Kind { Plain = 0, Linear = 1, Base = 2, Bands = 3 };
    Kind kind = Plain;
    double factor = 1.0, low = 1.0, high = 4.0, length = 8192.0;
};
// The angles of rotary positions, made once: Int64 (rot_dim / 2) on the GPU, fractions of a turn a position in units of 2^-64.
Tensor rotary_turns(size_t rot_dim, double theta = 10000.0, const RotaryScaling &scaling = {});
// x (..., heads, head_dim) with the first 2 * turns.size() dims of each head rotated by its row's position: positions Int32 or Int64, one for each (...) row.
// inverse: rotated back, the gradient of the call without it.
Tensor rotary(const Tensor &x, const Tensor &positions, const Tensor &turns, bool interleaved = false, bool inverse = false, float amplitude = 1.0f);

// Attention of sequences side by side: q (tokens, heads, head_dim), k and v (tokens', kv_heads, head_dim), starts Int32 (n + 1) on the GPU: sequence i owns rows starts[i] ..
// starts[i + 1] - 1.  Causal: the last query of a sequence sees every key of it.  longest_keys: about how many keys the longest sequence has (for the division of
// the work alone), 0: not known, and taken to be up to twice the average.  Rows of the result that no sequence owns are zeros.
Tensor packed_attention(const Tensor &q, const Tensor &k, const Tensor &v, const Tensor &starts_q, const Tensor &starts_kv, bool is_causal = true, float scale = -1.0f, size_t longest_keys = 0);

} // namespace ops

namespace nn {

// Which pages hold what: the bookkeeping of a cache, on the host.  Sequences are numbers; a page belongs to every sequence that lists it, and is free when none does.
class PageBook {
  public:
    PageBook(size_t pages, size_t page_size);
    // page src's first `rows` rows are to be copied to page dst
    struct Copy {
        int32_t src, dst, rows;
    };
    int add();                               // an empty sequence
    int fork(int sequence);                  // one with the same tokens, in the same pages
    void release(int sequence);              // its pages are given back
    void truncate(int sequence, size_t length); // the first tokens stay
    // Room for so many new tokens behind each sequence: the copies that have to be made first (a page that a sequence is to write to and shares) are added to `copies`.  Either all of
    // them get room, or RuntimeError and nothing changes.  A sequence may be named once.
    void extend(const std::vector<int> &sequences, const std::vector<size_t> &new_tokens, std::vector<Copy> &copies);
    // .. undone, where nothing has changed since; `copies` are those of that extension alone, and what they would have written to is free again
    void take_back(const std::vector<int> &sequences, const std::vector<size_t> &new_tokens, const std::vector<Copy> &copies);
    // Pages in use move to the front of the pool, the others' places behind them: the copies that do so, which have been entered already
    std::vector<Copy> compact();

    // Neighbours that begin with the same pages, counting whole ones in front of their last new_tokens: the sequences from the group before it up to `end` have the first `pages` pages in
    // common (0 for one by itself).  Of all divisions, one that leaves the fewest pages to read where each group's common ones are read once.
    struct Group {
        size_t end, pages;
    };
    std::vector<Group> groups(const std::vector<int> &sequences, const std::vector<size_t> &new_tokens) const;

    size_t length(int sequence) const { return at(sequence).length; }
    const std::vector<int32_t> &pages(int sequence) const { return at(sequence).pages; }
    int64_t slot(int sequence, size_t position) const; // page * page_size + row
    size_t free_pages() const { return free_.size(); }
    size_t page_size() const { return page_size_; }
    size_t page_count() const { return users_.size(); }

  private:
    struct Sequence {
        bool live = false;
        size_t length = 0;
        std::vector<int32_t> pages;
    };
    Sequence &at(int sequence);
    const Sequence &at(int sequence) const { return const_cast<PageBook *>(this)->at(sequence); }
    int place();
    int32_t take();
    void drop(int32_t page);

    size_t page_size_;
    std::vector<int32_t> users_; // of each page
    std::vector<int32_t> free_;  // the lowest last
    std::vector<Sequence> sequences_;
};

// New tokens of a batch of sequences: what a pass through a decoder's layers needs of them, on the GPU.  It is good until the cache is extended, truncated or compacted again or
// a sequence is released; append and attend refuse it then, and a step of another cache.
struct CacheStep {
    uint64_t version = 0;
    std::vector<int> sequences;
    std::vector<size_t> new_tokens;
    size_t tokens = 0;                             // all of them, sequence by sequence
    Tensor positions, slots;                       // Int64 (tokens)
    Tensor starts;                                 // Int32 (n + 1): each sequence's first token
    Tensor page_table, lengths;                    // Int32 (n, ..) and (n): the pages and keys of each sequence, without a prefix below
    Tensor group_starts, prefix_table, prefix_lengths; // Int32; empty where no neighbours share their first pages
    size_t longest = 0, longest_prefix = 0, each = 0; // each: as many new tokens as every sequence has, 0 where they differ
};

// Keys and values of the layers of a decoder, in pages: pools (layers, pages, page_size, kv_heads, head_dim) on the GPU.
class PagedCache {
  public:
    PagedCache(size_t layers, size_t pages, size_t page_size, size_t kv_heads, size_t head_dim, DType dtype);
    PagedCache(const PagedCache &) = delete; // (two books of the same pages)
    PagedCache &operator=(const PagedCache &) = delete;
    int add() { return book_.add(); }
    int fork(int sequence) { return book_.fork(sequence); }
    void release(int sequence) {
        book_.release(sequence);
        changed();
    }
    void truncate(int sequence, size_t length) {
        book_.truncate(sequence, length);
        changed();
    }
    size_t length(int sequence) const { return book_.length(sequence); }
    // Where one of the following fails, on the device too, nothing has changed: sequences, pages and steps are as they were.
    size_t compact(); // how many pages moved
    // Room for new tokens behind each sequence (pages that have to be copied for it are).  Neighbours whose first pages are the same, as forks have them, are read as one prefix
    // when every sequence gets as many tokens, 16 at most: by PageBook::groups.
    CacheStep extend(const std::vector<int> &sequences, const std::vector<size_t> &new_tokens);
    // Keys and values (tokens, kv_heads, head_dim) of a step into a layer, keys rotated by `turns` (empty: not rotated); the answer is q (tokens, heads, head_dim) rotated alike.
    Tensor append(size_t layer, const CacheStep &step, const Tensor &q, const Tensor &k, const Tensor &v, const Tensor &turns = Tensor(), bool interleaved = false, float amplitude = 1.0f);
    // Causal attention of the step's queries (tokens, heads, head_dim) to everything that the cache holds of their sequences
    Tensor attend(size_t layer, const CacheStep &step, const Tensor &q, float scale = -1.0f) const;

    const PageBook &book() const { return book_; }
    const Tensor &keys() const { return k_; }
    const Tensor &values() const { return v_; }

  private:
    void copy(const std::vector<PageBook::Copy> &copies);
    CacheStep step_of(const std::vector<int> &sequences, const std::vector<size_t> &new_tokens) const;
    void changed();
    void need_current(const CacheStep &step) const;

    PageBook book_;
    size_t layers_, kv_heads_, head_dim_;
    uint64_t version_ = 0; // unlike any other's
    Tensor k_, v_;
};

} // namespace nn
} // namespace axiom
