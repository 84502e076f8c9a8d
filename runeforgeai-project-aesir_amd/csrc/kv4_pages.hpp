// Which pages of a paged cache belong to which sequence: reference counts, the free pages, and the moves
// that sharing, copying and compaction ask for. Host only; the caller validates ids and counts.
#pragma once

#include <cstdint>
#include <functional>
#include <queue>
#include <vector>

namespace aesir {

struct PageMove {
    int32_t src, dst;
};

class PageBook {
  public:
    PageBook(int64_t num_pages, int64_t page_size, int64_t max_seqs)
        : page_size_(page_size), seqs_((size_t)max_seqs), refs_((size_t)num_pages, 0) {
        for (int64_t p = 0; p < num_pages; p++) free_.push((int32_t)p);
    }

    struct Seq {
        int64_t length = 0;
        std::vector<int32_t> pages;
        int64_t synced = 0;  // leading entries the device's table already holds
    };

    const Seq &seq(int64_t s) const { return seqs_[(size_t)s]; }
    int64_t max_seqs() const { return (int64_t)seqs_.size(); }
    int64_t free_pages() const { return (int64_t)free_.size(); }
    int64_t pages_for(int64_t positions) const { return (positions + page_size_ - 1) / page_size_; }
    void mark_synced(int64_t s) { seqs_[(size_t)s].synced = (int64_t)seqs_[(size_t)s].pages.size(); }
    void mark_unsynced(int64_t s) { seqs_[(size_t)s].synced = 0; }

    // Pages that `rows` new positions of every listed sequence take: new ones, and one per shared last page
    // that would be written to (of k sequences on one page the last keeps it, if no other sequence has it).
    int64_t pages_needed(const int64_t *seqs, const int64_t *rows, int64_t n) {
        int64_t need = 0;
        std::vector<int32_t> left;  // shared last pages whose count this walk has lowered
        left.reserve((size_t)n);
        for (int64_t i = 0; i < n; i++) {
            const Seq &s = seqs_[(size_t)seqs[i]];
            need += pages_for(s.length + rows[i]) - (int64_t)s.pages.size();
            if (writes_shared(s, rows[i])) {
                need++;
                refs_[(size_t)s.pages.back()]--;
                left.push_back(s.pages.back());
            }
        }
        for (int32_t p : left) refs_[(size_t)p]++;
        return need;
    }

    // Room in the vectors that grow, copy and fork fill, taken before anything changes.
    void reserve(int64_t id, int64_t length) { seqs_[(size_t)id].pages.reserve((size_t)pages_for(length)); }

    // Grows a sequence (enough pages are free, reserve() was called); a shared last page that the new rows write to is replaced by
    // a copy of its own, appended to `copies`.
    void grow(int64_t id, int64_t rows, std::vector<PageMove> &copies) {
        Seq &s = seqs_[(size_t)id];
        if (writes_shared(s, rows)) {
            const int32_t old = s.pages.back(), own = take();
            refs_[(size_t)old]--;
            s.pages.back() = own;
            touch(s, (int64_t)s.pages.size() - 1);
            copies.push_back({old, own});
        }
        s.length += rows;
        while ((int64_t)s.pages.size() < pages_for(s.length)) s.pages.push_back(take());
    }

    // Takes back what grow(id, rows, copies) did, in reverse order of several; copies loses the sequence's own.
    void shrink(int64_t id, int64_t rows, std::vector<PageMove> &copies) {
        Seq &s = seqs_[(size_t)id];
        truncate(id, s.length - rows);
        if (!copies.empty() && !s.pages.empty() && s.pages.back() == copies.back().dst) {
            s.pages.back() = copies.back().src;
            refs_[(size_t)copies.back().src]++;
            refs_[(size_t)copies.back().dst] = 0;
            free_.push(copies.back().dst);
            touch(s, (int64_t)s.pages.size() - 1);
            copies.pop_back();
        }
    }

    void fork(int64_t src, int64_t dst) {
        Seq &d = seqs_[(size_t)dst];  // (the assignment may throw; nothing has changed then)
        d.pages = seqs_[(size_t)src].pages;
        for (int32_t p : d.pages) refs_[(size_t)p]++;
        d.length = seqs_[(size_t)src].length;
        d.synced = 0;
    }

    void copy(int64_t src, int64_t dst, std::vector<PageMove> &copies) {
        Seq &d = seqs_[(size_t)dst];
        const Seq &s = seqs_[(size_t)src];
        reserve(dst, s.length);
        copies.reserve(s.pages.size());
        for (int32_t p : s.pages) {
            const int32_t own = take();
            d.pages.push_back(own);
            copies.push_back({p, own});
        }
        d.length = s.length;
        d.synced = 0;
    }

    void truncate(int64_t id, int64_t length) {
        Seq &s = seqs_[(size_t)id];
        s.length = length;
        const int64_t keep = pages_for(length);
        while ((int64_t)s.pages.size() > keep) {
            const int32_t p = s.pages.back();
            s.pages.pop_back();
            if (--refs_[(size_t)p] == 0) free_.push(p);
        }
        touch(s, keep);
    }

    // The moves of every used page above the used count into a free one below it, both in ascending order: no move's
    // destination is another's source. Returns the used count.
    int64_t compaction(std::vector<PageMove> &moves) const {
        const int64_t total = (int64_t)refs_.size(), used = total - free_pages();
        int64_t dst = 0;
        for (int64_t p = used; p < total; p++) {
            if (refs_[(size_t)p] == 0) continue;
            while (refs_[(size_t)dst] > 0) dst++;  // below `used` while sources are left
            moves.push_back({(int32_t)p, (int32_t)dst++});
        }
        return used;
    }

    // Makes these moves; afterwards pages [0, used) are the used ones.
    void compact(const std::vector<PageMove> &moves) {
        if (moves.empty()) return;
        const int64_t total = (int64_t)refs_.size(), used = total - free_pages();
        std::vector<int32_t> to((size_t)total, -1), rest;  // (what can throw comes before what changes)
        rest.reserve((size_t)total);
        for (int64_t p = used; p < total; p++) rest.push_back((int32_t)p);
        for (const PageMove &m : moves) {
            to[(size_t)m.src] = m.dst;
            refs_[(size_t)m.dst] = refs_[(size_t)m.src];
            refs_[(size_t)m.src] = 0;
        }
        for (Seq &s : seqs_)
            for (size_t i = 0; i < s.pages.size(); i++)
                if (const int32_t dst = to[(size_t)s.pages[i]]; dst >= 0) {
                    s.pages[i] = dst;
                    touch(s, (int64_t)i);
                }
        free_ = Free(std::greater<int32_t>(), std::move(rest));
    }

  private:
    using Free = std::priority_queue<int32_t, std::vector<int32_t>, std::greater<int32_t>>;  // lowest page first

    bool writes_shared(const Seq &s, int64_t rows) const {
        return rows > 0 && s.length % page_size_ != 0 && refs_[(size_t)s.pages.back()] > 1;
    }
    int32_t take() {
        const int32_t p = free_.top();
        free_.pop();
        refs_[(size_t)p] = 1;
        return p;
    }
    static void touch(Seq &s, int64_t entry) {
        if (s.synced > entry) s.synced = entry;
    }

    int64_t page_size_;
    std::vector<Seq> seqs_;
    std::vector<int32_t> refs_;  // sequences that hold each page
    Free free_;  // (holds all pages at first, and compact() gives it as much room again: pushes take no memory)
};

}  // namespace aesir
