// Which pages of a paged KV cache belong to which sequences: host bookkeeping with reference counts,
// so that forked sequences share pages. Nothing here touches the device; a call that cannot be done
// throws and leaves the map as it was.
#pragma once
#include <map>
#include <stdexcept>
#include <string>
#include <utility>
#include <vector>

namespace cb {
namespace kv4 {

class PageMap {
public:
    PageMap(int num_pages, int page_size, int max_seqs, int max_pages)
        : page_(page_size), max_pages_(max_pages), refs_(num_pages, 0), seqs_(max_seqs) {
        free_.reserve(num_pages);
        for (int p = num_pages - 1; p >= 0; --p) free_.push_back(p);
    }

    int length(int s) const { return seqs_[check(s)].len; }
    const std::vector<int>& pages(int s) const { return seqs_[check(s)].pages; }
    int free_pages() const { return (int)free_.size(); }
    int refs(int page) const { return refs_.at(page); }
    int max_seqs() const { return (int)seqs_.size(); }

    // Makes room for `counts[i]` more rows at the end of sequence seqs[i]. A last page that is partly
    // filled and shared is replaced: (old, new) pairs to be copied before anything is written.
    std::vector<std::pair<int, int>> grow(const std::vector<int>& seqs, const std::vector<int>& counts) {
        distinct(seqs);
        long long need = 0;
        std::map<int, int> left;  // references to a shared last page after those already replaced
        for (size_t i = 0; i < seqs.size(); ++i) {
            const Seq& q = seqs_[check(seqs[i])];
            if (counts[i] < 0) throw std::invalid_argument("a negative number of rows");
            const long long total = (long long)q.len + counts[i], n = (total + page_ - 1) / page_;
            if (n > max_pages_) throw std::length_error("sequence " + std::to_string(seqs[i]) + " would pass its longest context");
            need += n - (long long)q.pages.size();
            if (counts[i] > 0 && q.len % page_ && refs_[q.pages.back()] > 1) {
                int& r = left.emplace(q.pages.back(), refs_[q.pages.back()]).first->second;
                if (r > 1) {
                    --r;
                    ++need;
                }
            }
        }
        if (need > (long long)free_.size())
            throw std::length_error("out of pages: " + std::to_string(need) + " needed, " + std::to_string(free_.size()) + " free");
        std::vector<std::pair<int, int>> copies;
        for (size_t i = 0; i < seqs.size(); ++i) {
            Seq& q = seqs_[seqs[i]];
            if (counts[i] > 0 && q.len % page_ && refs_[q.pages.back()] > 1) {
                const int fresh = take();
                copies.emplace_back(q.pages.back(), fresh);
                --refs_[q.pages.back()];
                q.pages.back() = fresh;
            }
            q.len += counts[i];
            while ((long long)q.pages.size() * page_ < q.len) q.pages.push_back(take());
        }
        return copies;
    }

    // Sequence dst[i] becomes what src[i] was before the call, sharing its pages; what dst[i] had is
    // released. Any reordering is possible in one call.
    void fork(const std::vector<int>& src, const std::vector<int>& dst) {
        distinct(dst);
        std::vector<Seq> now;
        for (int s : src) now.push_back(seqs_[check(s)]);
        for (const Seq& q : now)
            for (int p : q.pages) ++refs_[p];
        for (size_t i = 0; i < dst.size(); ++i) {
            release(seqs_[dst[i]].pages, 0);
            seqs_[dst[i]] = std::move(now[i]);
        }
    }

    // Keeps the first `len` rows.
    void truncate(int s, int len) {
        Seq& q = seqs_[check(s)];
        if (len < 0 || len > q.len) throw std::invalid_argument("a length that the sequence does not have");
        q.len = len;
        release(q.pages, (len + page_ - 1) / page_);
    }

    // Gives each sequence new pages for counts[i] rows and returns its old ones, which are released:
    // the rows to keep are moved before anything else is written.
    std::vector<std::vector<int>> renew(const std::vector<int>& seqs, const std::vector<int>& counts) {
        distinct(seqs);
        long long need = 0;
        for (size_t i = 0; i < seqs.size(); ++i) {
            if (counts[i] < 0 || counts[i] > (long long)max_pages_ * page_) throw std::invalid_argument("a bad number of rows");
            check(seqs[i]);
            need += (counts[i] + page_ - 1) / page_;
        }
        if (need > (long long)free_.size())
            throw std::length_error("out of pages: " + std::to_string(need) + " needed, " + std::to_string(free_.size()) + " free");
        std::vector<std::vector<int>> old;
        for (size_t i = 0; i < seqs.size(); ++i) {  // all new pages first: none of them is an old one
            Seq fresh;
            fresh.len = counts[i];
            while ((long long)fresh.pages.size() * page_ < fresh.len) fresh.pages.push_back(take());
            old.push_back(seqs_[seqs[i]].pages);
            std::swap(seqs_[seqs[i]], fresh);
        }
        for (auto pages : old) release(pages, 0);
        return old;
    }

private:
    struct Seq {
        int len = 0;
        std::vector<int> pages;
    };

    int check(int s) const {
        if (s < 0 || s >= (int)seqs_.size()) throw std::out_of_range("no sequence " + std::to_string(s));
        return s;
    }
    void distinct(const std::vector<int>& seqs) const {
        std::vector<char> seen(seqs_.size(), 0);
        for (int s : seqs)
            if (seen[check(s)]++) throw std::invalid_argument("sequence " + std::to_string(s) + " named twice");
    }
    int take() {
        const int p = free_.back();
        free_.pop_back();
        refs_[p] = 1;
        return p;
    }
    void release(std::vector<int>& pages, size_t keep) {  // the last pages first: they are taken again first
        while (pages.size() > keep) {
            if (--refs_[pages.back()] == 0) free_.push_back(pages.back());
            pages.pop_back();
        }
    }

    int page_, max_pages_;
    std::vector<int> refs_, free_;
    std::vector<Seq> seqs_;
};

}  // namespace kv4
}  // namespace cb
