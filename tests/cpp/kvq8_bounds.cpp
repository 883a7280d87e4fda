// Host check of hipgpt_amd/csrc/kvq8.h: the byte layout of a page is a
// bijection inside the page, and no sequence, page index or row that the
// kernels derive from device-side arrays leaves its range, whatever those
// arrays hold.  Prints the number of cases and exits 0, or names the failure.
#include <cstdio>
#include <cstdlib>
#include <vector>

#include "../../hipgpt_amd/csrc/kvq8.h"

using namespace hipgpt::kvq8;

#define CHECK(x)                                              \
    do {                                                      \
        if (!(x)) {                                           \
            fprintf(stderr, "line %d: %s\n", __LINE__, #x);   \
            exit(1);                                          \
        }                                                     \
    } while (0)

int main() {
    long cases = 0;
    for (int D : {32, 64, 128, 256})
        for (int ps : {32, 64, 128}) {
            std::vector<char> k(ps * D), v(ps * D);
            for (int t = 0; t < ps; ++t)
                for (int d = 0; d < D; ++d) {
                    const int a = k_byte(t, d, D), b = v_byte(t, d, D);
                    CHECK(a >= 0 && a < ps * D && !k[a]++);
                    CHECK(b >= 0 && b < ps * D && !v[b]++);
                    // the kernels read 16 bytes a lane: tokens of a lane quarter, two head dims
                    CHECK(v_byte(t & ~3, d, D) + (t & 3) == b);
                    if (d % 32 < 16) CHECK(v_byte(t, d + 16, D) == b + 8);
                    ++cases;
                }
        }
    const int huge = 0x7fffffff;
    for (int n0 : {-huge - 1, -5, 0, 1, 3, 7, huge})
        for (int n1 : {-huge - 1, -1, 0, 1, 4, 7, 9, huge})
            for (int len : {-huge - 1, -1, 0, 1, 4, 63, 64, 128, 129, huge})
                for (int max_new : {1, 4, 7})
                    for (int pg : {-huge - 1, -1, 0, 4, 5, huge}) {
                        const int cu[2] = {n0, n1};
                        const int table[2] = {pg, pg};
                        Cache c{};
                        c.num_pages = 5;
                        c.lps = 6;
                        c.table = table;
                        c.t_stride = 2;
                        c.max_pages = 2;
                        c.lens = &len;
                        c.cu = cu;
                        c.B = 1;
                        c.T = 7;
                        c.max_new = max_new;
                        const Seq s = sequence(c, 0);
                        CHECK(s.n >= 0 && s.n <= max_new);
                        if (s.n > 0) CHECK(s.row0 >= 0 && s.row0 + s.n <= c.T);
                        if (!s.bad) CHECK(s.len >= s.n && s.len <= 2 * 64);
                        if (n0 == 0 && n1 == 4 && max_new == 4) CHECK(s.n == 4 && s.bad == (len < 4 || len > 128));
                        if (n0 == 0 && n1 == 4 && max_new == 1) CHECK(s.n == 1 && s.bad);  // more rows than promised
                        const int p = page_of(c, 0, 70);
                        CHECK(p == (pg >= 0 && pg < 5 ? pg : -1));
                        ++cases;
                    }
    printf("%ld cases\n", cases);
    return 0;
}
