// Host bookkeeping of the paged key/value cache: which pages each sequence
// holds.  Plain C++ with no device code, so that it can be checked without a
// GPU.  Pages are handed out lowest number first; a page that several
// sequences hold (after a fork) is copied before one of them grows in it.
// Every operation either happens whole or returns an error and changes
// nothing; std::bad_alloc can leave it only before the first change.
#pragma once

#include <cstdint>
#include <vector>

namespace exq {

// Copy the first `used` tokens of page src to page dst, in every layer.
struct KvMove {
    int src, dst, used;
};

enum class KvStatus { ok, bad_seq, repeated, bad_count, no_pages, no_seqs };

class KvTables {
  public:
    struct Seq {
        bool live = false;
        int len = 0;
        std::vector<int> pages;
    };

    KvTables(int page_tokens, int n_pages, int max_seqs)
        : page_(page_tokens), free_(n_pages), refs_(n_pages, 0), bits_((n_pages + 63) / 64, ~0ull), seqs_(max_seqs),
          mark_(max_seqs, 0) {
        if (n_pages % 64 != 0) bits_.back() = (1ull << (n_pages % 64)) - 1;
    }

    int page_tokens() const { return page_; }
    int free_pages() const { return free_; }
    int n_pages() const { return (int)refs_.size(); }
    // Changes whenever a sequence's length or pages, or a page's holders, do.
    uint64_t epoch() const { return epoch_; }
    bool valid(int s) const { return s >= 0 && s < (int)seqs_.size() && seqs_[s].live; }
    const Seq &seq(int s) const { return seqs_[s]; }
    int holders(int page) const { return refs_[page]; }

    int new_seq() {
        const int s = lowest_seq(0);
        if (s >= 0) seqs_[s].live = true;
        return s;
    }

    KvStatus fork(int n, const int *parents, bool copy, int *children, std::vector<KvMove> &moves) {
        long long need = 0;
        for (int i = 0; i < n; ++i) {
            if (!valid(parents[i])) return KvStatus::bad_seq;
            need += (long long)seqs_[parents[i]].pages.size();
        }
        std::vector<int> made(n);
        for (int i = 0, at = -1; i < n; ++i) {
            at = lowest_seq(at + 1);
            if (at < 0) return KvStatus::no_seqs;
            made[i] = at;
        }
        if (copy && need > free_) return KvStatus::no_pages;
        std::vector<std::vector<int>> pages(n);
        for (int i = 0; i < n; ++i) pages[i] = seqs_[parents[i]].pages;
        if (copy) moves.reserve(moves.size() + (size_t)need);
        for (int i = 0; i < n; ++i) {
            Seq &c = seqs_[made[i]];
            const Seq &p = seqs_[parents[i]];
            c.live = true;
            c.len = p.len;
            c.pages.swap(pages[i]);
            for (size_t j = 0; j < c.pages.size(); ++j) {
                if (!copy) {
                    refs_[c.pages[j]]++;
                    continue;
                }
                const int left = c.len - (int)j * page_;
                const int dst = take();
                moves.push_back({c.pages[j], dst, left < page_ ? left : page_});
                c.pages[j] = dst;
            }
            children[i] = made[i];
        }
        ++epoch_;
        return KvStatus::ok;
    }

    KvStatus extend(int n, const int *seqs, const int *n_new, std::vector<KvMove> &moves) {
        const KvStatus st = distinct(n, seqs);
        if (st != KvStatus::ok) return st;
        for (int i = 0; i < n; ++i)
            if (n_new[i] < 0) return KvStatus::bad_count;
        std::vector<int> copied;  // sequences whose last page is shared and must be theirs alone
        copied.reserve(n);
        moves.reserve(moves.size() + n);
        long long need = 0;
        for (int i = 0; i < n; ++i) {
            const Seq &s = seqs_[seqs[i]];
            if (n_new[i] > 0 && s.len % page_ != 0 && refs_[s.pages.back()] > 1) {
                refs_[s.pages.back()]--;
                copied.push_back(i);
                ++need;
            }
            need += ((long long)s.len + n_new[i] + page_ - 1) / page_ - (long long)s.pages.size();
        }
        bool fits = need <= free_;
        try {
            if (fits)
                for (int i = 0; i < n; ++i) {
                    Seq &s = seqs_[seqs[i]];
                    s.pages.reserve((size_t)(((long long)s.len + n_new[i] + page_ - 1) / page_));
                }
        } catch (...) {
            for (int i : copied) refs_[seqs_[seqs[i]].pages.back()]++;
            throw;
        }
        if (!fits) {
            for (int i : copied) refs_[seqs_[seqs[i]].pages.back()]++;
            return KvStatus::no_pages;
        }
        size_t c = 0;
        for (int i = 0; i < n; ++i) {
            Seq &s = seqs_[seqs[i]];
            if (c < copied.size() && copied[c] == i) {
                ++c;
                const int old = s.pages.back();
                s.pages.back() = take();
                moves.push_back({old, s.pages.back(), s.len % page_});
            }
            s.len += n_new[i];
            while ((long long)s.pages.size() * page_ < s.len) s.pages.push_back(take());
        }
        ++epoch_;
        return KvStatus::ok;
    }

    KvStatus truncate(int s, int len) {
        if (!valid(s)) return KvStatus::bad_seq;
        Seq &q = seqs_[s];
        if (len < 0 || len > q.len) return KvStatus::bad_count;
        q.len = len;
        while ((long long)q.pages.size() * page_ >= (long long)len + page_) {
            drop(q.pages.back());
            q.pages.pop_back();
        }
        ++epoch_;
        return KvStatus::ok;
    }

    KvStatus release(int n, const int *seqs) {
        const KvStatus st = distinct(n, seqs);
        if (st != KvStatus::ok) return st;
        for (int i = 0; i < n; ++i) {
            Seq &q = seqs_[seqs[i]];
            for (int p : q.pages) drop(p);
            q.pages.clear();
            q.live = false;
            q.len = 0;
        }
        ++epoch_;
        return KvStatus::ok;
    }

    // Pages from the count in use on move to the free ones below it.
    int compact(std::vector<KvMove> &moves) {
        const int used = n_pages() - free_;
        std::vector<int> to(n_pages());
        moves.reserve(moves.size() + (size_t)(used < free_ ? used : free_));
        for (int src = used, dst = 0; src < n_pages(); ++src) {
            if (refs_[src] == 0) continue;
            while (refs_[dst] != 0) ++dst;
            refs_[dst] = refs_[src];
            refs_[src] = 0;
            set_free(dst, false);
            set_free(src, true);
            to[src] = dst;
            moves.push_back({src, dst, page_});
        }
        for (Seq &s : seqs_)
            for (int &p : s.pages)
                if (p >= used) p = to[p];
        low_ = (size_t)used / 64;
        ++epoch_;
        return used;
    }

    // ok when every number is in use and none comes twice.
    KvStatus distinct(int n, const int *seqs) {
        ++stamp_;
        for (int i = 0; i < n; ++i) {
            if (!valid(seqs[i])) return KvStatus::bad_seq;
            if (mark_[seqs[i]] == stamp_) return KvStatus::repeated;
            mark_[seqs[i]] = stamp_;
        }
        return KvStatus::ok;
    }

  private:
    int lowest_seq(int from) const {
        for (int s = from; s < (int)seqs_.size(); ++s)
            if (!seqs_[s].live) return s;
        return -1;
    }
    void set_free(int p, bool is_free) {
        if (is_free) bits_[(size_t)p / 64] |= 1ull << (p % 64);
        else bits_[(size_t)p / 64] &= ~(1ull << (p % 64));
    }
    int take() {  // (the caller has seen that one is free)
        while (bits_[low_] == 0) ++low_;
        const int p = (int)(low_ * 64) + __builtin_ctzll(bits_[low_]);
        set_free(p, false);
        refs_[p] = 1;
        --free_;
        return p;
    }
    void drop(int p) {
        if (--refs_[p] > 0) return;
        set_free(p, true);
        ++free_;
        if ((size_t)p / 64 < low_) low_ = (size_t)p / 64;
    }

    int page_, free_;
    size_t low_ = 0;  // no free page in the words below
    std::vector<int> refs_;
    std::vector<uint64_t> bits_;  // a set bit: the page is free
    std::vector<Seq> seqs_;
    std::vector<uint64_t> mark_;
    uint64_t stamp_ = 0, epoch_ = 0;
};

}  // namespace exq
