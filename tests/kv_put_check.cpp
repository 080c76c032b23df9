// Host check of a reservation's launches (csrc/kv.cuh): every page id is
// handed over once and in order, and the reserved length moves with the last
// of them alone, so that launches which fail midway leave the old one.
#include <cstdio>

#include "kv.cuh"

using namespace brew;

int main() {
    int fails = 0;
    for (int first = 0; first < 300; first += 7)
        for (int end = first; end < first + 700; ++end) {
            int at = first, reserved = -7, launches = 0;   // -7: the length before
            do {
                if (reserved != -7) ++fails;               // it moved before this launch
                const KvPut p = kv_put(at, end, 16 * end);
                if (p.first != at || p.n < 0 || p.n > KV_PUT_PAGES || at + p.n > end || (p.n == 0 && at < end)) ++fails;
                if (p.tokens >= 0) reserved = p.tokens;
                at += p.n;
                ++launches;
            } while (at < end && launches < 100);
            if (at != end || reserved != 16 * end) ++fails;
        }
    const KvPut none = kv_put(0, 0, 0);                    // a release: no page, length 0
    if (none.n != 0 || none.tokens != 0) ++fails;
    printf(fails ? "%d failures\n" : "ok\n", fails);
    return fails != 0;
}
