// The page bookkeeping of the 4-bit KV cache (csrc/kv4/page_map.h) against a plain model: rows are
// numbers, a write goes to the page that the map names, and every sequence must read what was written
// to it, whatever was forked, cut, freed or compacted in between. Prints "ok" and returns 0.
#include <cstdio>
#include <cstdlib>
#include <random>

#include "kv4/page_map.h"

using cb::kv4::PageMap;

#define CHECK(x)                                                  \
    do {                                                          \
        if (!(x)) {                                               \
            std::printf("line %d: %s\n", __LINE__, #x);           \
            return 1;                                             \
        }                                                         \
    } while (0)

template <typename E, typename F>
bool throws(F f) {
    try {
        f();
    } catch (const E&) {
        return true;
    }
    return false;
}

struct Model {
    int page;
    PageMap map;
    std::vector<std::vector<long>> store;           // [page][row]: what the device would hold
    std::vector<std::vector<long>> rows;            // [sequence]: what it should read
    long next = 1;
    Model(int pages, int page_size, int seqs, int max_pages)
        : page(page_size), map(pages, page_size, seqs, max_pages), store(pages, std::vector<long>(page_size, 0)), rows(seqs) {}
    void grow(const std::vector<int>& s, const std::vector<int>& n) {
        for (auto c : map.grow(s, n)) store[c.second] = store[c.first];
        for (size_t i = 0; i < s.size(); ++i)
            for (int k = 0; k < n[i]; ++k) {
                const int r = (int)rows[s[i]].size();
                store[map.pages(s[i])[r / page]][r % page] = next;
                rows[s[i]].push_back(next++);
            }
    }
    bool good() const {
        std::vector<int> refs(store.size(), 0);
        for (size_t s = 0; s < rows.size(); ++s) {
            if (map.length((int)s) != (int)rows[s].size()) return false;
            const auto& p = map.pages((int)s);
            if (p.size() != (rows[s].size() + page - 1) / page) return false;
            for (int x : p) ++refs[x];
            for (size_t r = 0; r < rows[s].size(); ++r)
                if (store[p[r / page]][r % page] != rows[s][r]) return false;
        }
        int used = 0;
        for (size_t x = 0; x < refs.size(); ++x) {
            if (refs[x] != map.refs((int)x)) return false;
            used += refs[x] > 0;
        }
        return used + map.free_pages() == (int)store.size();
    }
};

int main() {
    {  // sharing: a fork takes no page, the first write to a shared last page takes one
        Model m(8, 4, 4, 8);
        m.grow({0}, {6});
        m.map.fork({0, 0}, {1, 2});
        m.rows[1] = m.rows[2] = m.rows[0];
        CHECK(m.good() && m.map.free_pages() == 6);
        m.grow({0, 1, 2}, {1, 1, 0});  // 0 and 1 get their own last page; 2 keeps the old one alone
        CHECK(m.good() && m.map.free_pages() == 4 && m.map.refs(m.map.pages(2).back()) == 1);
        m.grow({2}, {1});
        CHECK(m.good() && m.map.free_pages() == 4);
        m.grow({0}, {1});  // fills the page; the next row needs a new one
        m.grow({0}, {1});
        CHECK(m.good() && m.map.free_pages() == 3);
    }
    {  // all three write at once: the last one may write in place
        Model m(5, 4, 3, 8);
        m.grow({0}, {5});
        m.map.fork({0, 0}, {1, 2});
        m.rows[1] = m.rows[2] = m.rows[0];
        m.grow({0, 1, 2}, {1, 1, 1});
        CHECK(m.good() && m.map.free_pages() == 1);
    }
    {  // refusals change nothing
        Model m(4, 4, 3, 3);
        m.grow({0, 1}, {6, 4});
        CHECK(throws<std::length_error>([&] { m.map.grow({1, 2}, {4, 4}); }));      // out of pages
        CHECK(throws<std::length_error>([&] { m.map.grow({0}, {7}); }));            // past the longest context
        CHECK(throws<std::invalid_argument>([&] { m.map.grow({0, 0}, {1, 1}); }));  // twice
        CHECK(throws<std::invalid_argument>([&] { m.map.grow({0}, {-1}); }));
        CHECK(throws<std::out_of_range>([&] { m.map.grow({3}, {1}); }));
        CHECK(throws<std::out_of_range>([&] { m.map.fork({0}, {-1}); }));
        CHECK(throws<std::invalid_argument>([&] { m.map.fork({0, 1}, {2, 2}); }));
        CHECK(throws<std::invalid_argument>([&] { m.map.truncate(0, 7); }));
        CHECK(throws<std::length_error>([&] { m.map.renew({0}, {6}); }));           // needs new pages beside the old
        CHECK(m.good());
    }
    for (int seed = 0; seed < 200; ++seed) {  // random programs
        std::mt19937 g(seed);
        auto pick = [&](int n) { return (int)(g() % (unsigned)n); };
        const int page = 1 << (1 + pick(4)), seqs = 1 + pick(6);
        Model m(10 + pick(40), page, seqs, 2 + pick(12));
        for (int step = 0; step < 300; ++step) {
            const int s = pick(seqs);
            switch (pick(5)) {
                case 0: case 1: {
                    std::vector<int> ids, n;
                    for (int i = 0; i < seqs; ++i)
                        if (pick(2)) {
                            ids.push_back(i);
                            n.push_back(pick(3) ? pick(3) : pick(2 * page));
                        }
                    try {
                        m.grow(ids, n);
                    } catch (const std::length_error&) {
                    }
                    break;
                }
                case 2: {  // a reordering: every sequence takes another's place
                    std::vector<int> src, dst;
                    std::vector<std::vector<long>> now(seqs);
                    for (int i = 0; i < seqs; ++i) {
                        src.push_back(pick(seqs));
                        dst.push_back(i);
                        now[i] = m.rows[src.back()];
                    }
                    m.map.fork(src, dst);
                    m.rows = now;
                    break;
                }
                case 3: {
                    const int n = pick((int)m.rows[s].size() + 1);
                    m.map.truncate(s, n);
                    m.rows[s].resize(n);
                    break;
                }
                default: {  // compaction: some rows stay
                    std::vector<int> kept;
                    for (int r = 0; r < (int)m.rows[s].size(); ++r)
                        if (pick(3)) kept.push_back(r);
                    try {
                        const auto old = m.map.renew({s}, {(int)kept.size()});
                        std::vector<long> now;
                        const auto before = m.store;
                        for (size_t j = 0; j < kept.size(); ++j) {
                            now.push_back(m.rows[s][kept[j]]);
                            m.store[m.map.pages(s)[j / page]][j % page] = before[old[0][kept[j] / page]][kept[j] % page];
                        }
                        m.rows[s] = now;
                    } catch (const std::length_error&) {
                    }
                }
            }
            CHECK(m.good());
        }
    }
    std::printf("ok\n");
    return 0;
}
