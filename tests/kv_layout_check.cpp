// Host check of the 4-bit K/V cache's index arithmetic (csrc/kv.cuh): every
// word and scale of a group is addressed exactly once, groups of different
// (page, head, position) do not overlap and lie in the layer, and entries
// outside the cache, its reserved positions or the buffers have no rows.
#include <cstdio>
#include <set>
#include <vector>

#include "kv.cuh"

using namespace brew;

static int fails = 0;
#define EXPECT(c) do { if (!(c)) { printf("line %d: %s\n", __LINE__, #c); ++fails; } } while (0)

template <int R>
void layout() {
    std::set<int> words, kscales, vscales;
    for (int u = 0; u < 2; ++u)
        for (int b = 0; b < R; ++b)
            for (int lane = 0; lane < 32; ++lane) words.insert(kv_word(R, u, b, lane));
    EXPECT((int)words.size() == 64 * R && *words.begin() == 0 && *words.rbegin() == 64 * R - 1);
    for (int p = 0; p < 16; ++p)
        for (int b = 0; b < R; ++b) {
            kscales.insert(kv_kscale(R, p, b));
            vscales.insert(kv_vscale(R, p, b));
        }
    for (const std::set<int>& s : {kscales, vscales})
        EXPECT((int)s.size() == 16 * R && *s.begin() == 0 && *s.rbegin() == 16 * R - 1);
    EXPECT(kv_group_bytes(R) == 2 * 256 * R + 2 * 32 * R && kv_group_bytes(R) % 16 == 0);
    for (int shift = 4; shift <= 7; ++shift) {
        const int n_pages = 7, n_kv = 3, max_pages = 3, page = 1 << shift;
        const int32_t table[2 * 3] = {6, 0, 3, 1, 5, 2};
        KvView kv = {};
        kv.table = table;
        kv.max_pages = max_pages;
        kv.page_shift = shift;
        kv.n_kv = n_kv;
        std::set<int64_t> at;
        for (int seq = 0; seq < 2; ++seq)
            for (int pos = 0; pos < 3 * page; ++pos)
                for (int hk = 0; hk < n_kv; ++hk) {
                    const int64_t o = kv_group_at<R>(kv, seq, pos, hk);
                    EXPECT(o >= 0 && o % kv_group_bytes(R) == 0 &&
                           o + kv_group_bytes(R) <= (int64_t)n_pages * n_kv * page / 16 * kv_group_bytes(R));
                    at.insert(o);
                }
        EXPECT((int)at.size() == 2 * 3 * page / 16 * n_kv);
    }
}

static KvEntry entry(int seq, int pos, int r0, int r1, int n_rows = 8, int max_rows = 4) {
    static const int32_t reserved[2] = {64, 0};
    const int32_t starts[2] = {r0, r1};
    KvView kv = {};
    kv.reserved = reserved;
    kv.max_seqs = 2;
    KvRowsDev r = {&seq, &pos, starts, 1, n_rows, max_rows};
    return kv_check_entry(kv, r, 0);
}

int main() {
    layout<1>(); layout<2>(); layout<3>(); layout<4>(); layout<8>();
    EXPECT(entry(0, 0, 0, 4).rows == 4 && !entry(0, 0, 0, 4).bad);
    EXPECT(entry(0, 60, 4, 8).rows == 4);
    EXPECT(entry(0, 61, 4, 8).rows == 0 && entry(0, 61, 4, 8).bad);      // past the reserved positions
    EXPECT(entry(0, 2147483646, 0, 2).bad && entry(0, -1, 0, 1).bad);
    EXPECT(entry(1, 0, 0, 1).bad);                                       // nothing reserved
    EXPECT(entry(2, 0, 0, 1).bad && entry(-1, 0, 0, 1).bad);             // no such sequence
    EXPECT(entry(0, 0, 0, 5).bad);                                       // more than max_rows
    EXPECT(entry(0, 0, 6, 9).bad && entry(0, 0, -1, 1).bad && entry(0, 0, 3, 2).bad);
    EXPECT(entry(0, 0, -2147483647, 2147483647).bad);
    EXPECT(entry(0, 0, 3, 3).rows == 0 && !entry(0, 0, 3, 3).bad);       // no rows: nothing is looked up
    EXPECT(!entry(-5, -5, 8, 8).bad);
    printf(fails ? "%d failures\n" : "ok\n", fails);
    return fails != 0;
}
