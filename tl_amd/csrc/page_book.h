// Host-side book of a paged KV cache: which pages each sequence holds, how many sequences share
// a page, and which page moves the device copies have to follow.  No device work and no HIP
// types here (unit-tested on the CPU); the caller carries the moves out with
// tl_hip_launch_kv_copy_pages and uploads the rows of the page table.
//
// Pages are shared by forked sequences and never written while shared: a sequence that grows
// into a shared tail page first gets a page of its own (copy on write).  Every choice of a page
// takes the lowest free one, so the same calls give the same book.
#pragma once
#include <cstdint>
#include <map>
#include <set>
#include <utility>
#include <vector>

namespace tlhip {

class PageBook {
public:
    enum Result { OK, NO_SEQUENCE, NO_PAGES, NO_ROOM };
    using Pair = std::pair<int32_t, int32_t>;  // (source page, destination page)

    PageBook(int32_t n_pages, int32_t page_size) : page_size_(page_size), users_(n_pages, 0) {}

    int32_t n_pages() const { return (int32_t)users_.size(); }
    int32_t page_size() const { return page_size_; }
    int64_t n_free() const { return (int64_t)returned_.size() + (n_pages() - fresh_); }

    int64_t open() {
        seqs_.emplace(next_, Seq{});
        return next_++;
    }
    // A sequence with the same positions on the same pages; -1 for one that is not open.
    int64_t fork(int64_t id) {
        auto it = seqs_.find(id);
        if (it == seqs_.end()) return -1;
        Seq copy = it->second;
        seqs_.emplace(next_, std::move(copy));
        for (int32_t p : it->second.pages) users_[p]++;
        return next_++;
    }
    Result close(int64_t id) {
        auto it = seqs_.find(id);
        if (it == seqs_.end()) return NO_SEQUENCE;
        for (int32_t p : it->second.pages) drop(p);
        seqs_.erase(it);
        return OK;
    }
    // Room for `tokens` more positions.  At most one move is added: of the tail page, where it is
    // shared and the first new position falls into it.  Without enough free pages nothing changes.
    Result grow(int64_t id, int64_t tokens, std::vector<Pair>* moves) {
        auto it = seqs_.find(id);
        if (it == seqs_.end()) return NO_SEQUENCE;
        Seq& s = it->second;
        if (tokens == 0) return OK;
        if (tokens > (int64_t)n_pages() * page_size_ - s.length) return NO_PAGES;
        const int64_t want = (s.length + tokens + page_size_ - 1) / page_size_;
        const bool own = s.length % page_size_ != 0 && users_[s.pages.back()] > 1;
        if (want - (int64_t)s.pages.size() + (own ? 1 : 0) > n_free()) return NO_PAGES;
        s.pages.reserve(want);
        if (own) {
            const int32_t from = s.pages.back(), to = take();
            moves->emplace_back(from, to);
            drop(from);
            s.pages.back() = to;
        }
        while ((int64_t)s.pages.size() < want) s.pages.push_back(take());
        s.length += tokens;
        return OK;
    }
    // Forgets the last positions, down to `length`; whole pages go back.
    Result cut(int64_t id, int64_t length) {
        auto it = seqs_.find(id);
        if (it == seqs_.end()) return NO_SEQUENCE;
        Seq& s = it->second;
        if (length < 0 || length > s.length) return NO_ROOM;
        const int64_t want = (length + page_size_ - 1) / page_size_;
        while ((int64_t)s.pages.size() > want) {
            drop(s.pages.back());
            s.pages.pop_back();
        }
        s.length = length;
        return OK;
    }
    // Moves that compact() would make.
    int64_t to_move() const {
        int64_t n = 0;
        for (int64_t p = n_pages() - n_free(); p < fresh_; p++) n += users_[p] != 0;
        return n;
    }
    // The used pages brought down to pages 0 .. used - 1: the highest used pages move to the
    // lowest free ones.  Sources and destinations are distinct and no page is both.
    void compact(std::vector<Pair>* moves) {
        const int32_t used = (int32_t)(n_pages() - n_free());
        std::map<int32_t, int32_t> to;
        moves->reserve(moves->size() + to_move());
        int32_t hole = 0;
        for (int32_t p = used; p < fresh_; p++) {
            if (!users_[p]) continue;
            while (users_[hole]) hole++;
            to[p] = hole;
            moves->emplace_back(p, hole);
            hole++;
        }
        for (const auto& m : to) {
            users_[m.second] = users_[m.first];
            users_[m.first] = 0;
        }
        for (auto& s : seqs_)
            for (int32_t& p : s.second.pages) {
                auto it = to.find(p);
                if (it != to.end()) p = it->second;
            }
        returned_.clear();
        fresh_ = used;
    }
    // Positions and pages of a sequence; nullptr for one that is not open.
    const std::vector<int32_t>* pages(int64_t id) const {
        auto it = seqs_.find(id);
        return it == seqs_.end() ? nullptr : &it->second.pages;
    }
    int64_t length(int64_t id) const {
        auto it = seqs_.find(id);
        return it == seqs_.end() ? -1 : it->second.length;
    }

private:
    struct Seq {
        std::vector<int32_t> pages;
        int64_t length = 0;
    };
    int32_t take() {
        int32_t p;
        if (!returned_.empty()) {
            p = *returned_.begin();
            returned_.erase(returned_.begin());
        } else {
            p = fresh_++;
        }
        users_[p] = 1;
        return p;
    }
    void drop(int32_t p) {
        if (--users_[p] == 0) returned_.insert(p);
    }

    int32_t page_size_;
    std::vector<int32_t> users_;   // sequences that hold each page
    std::set<int32_t> returned_;   // free pages below fresh_
    int32_t fresh_ = 0;            // pages from here on were never used: counted, not listed
    std::map<int64_t, Seq> seqs_;
    int64_t next_ = 0;
};

}  // namespace tlhip
