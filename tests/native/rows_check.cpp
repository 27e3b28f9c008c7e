// Whose rows a call's rows are (kv_seq): each row of at most one sequence for the
// row starts that the GPU tests use, whatever they hold, and none outside the call.
#include <algorithm>
#include <cstdio>
#include <random>
#include <vector>

#include "../../modgrad_amd/csrc/kv_device.hpp"

static int fails = 0;
#define EXPECT(c, ...)                        \
    do {                                      \
        if (!(c)) {                           \
            std::printf("FAIL %s: ", #c);     \
            std::printf(__VA_ARGS__);         \
            std::printf("\n");                \
            ++fails;                          \
        }                                     \
    } while (0)

static mgq::KvView view(const std::vector<int> &len, const std::vector<int> &cu, int n_tokens, int max_new) {
    mgq::KvView c = {};
    c.len = len.data();
    c.cu = cu.empty() ? nullptr : cu.data();
    c.n_seqs = (int)len.size();
    c.max_pages = 5;
    c.page_shift = 4;
    c.n_tokens = n_tokens;
    c.max_new = max_new;
    return c;
}

// The sequence of each row, -1 of none.
static std::vector<int> owners(const mgq::KvView &c, const char *what) {
    std::vector<int> own(c.n_tokens, -1);
    for (int b = 0; b < c.n_seqs; ++b) {
        const mgq::SeqInfo s = mgq::kv_seq(c, b);
        EXPECT(s.n >= 0 && s.n <= c.max_new, "%s: sequence %d has %d rows", what, b, s.n);
        EXPECT(s.n == 0 || (s.t0 >= 0 && s.t0 <= c.n_tokens - s.n), "%s: sequence %d rows %d + %d", what, b, s.t0, s.n);
        EXPECT(s.pos0 >= -(1 << 30) && s.pos0 <= 1 << 30 && s.len >= 0 && s.len <= c.max_pages << c.page_shift,
               "%s: sequence %d position %d length %d", what, b, s.pos0, s.len);
        for (int i = 0; i < s.n && s.t0 >= 0 && s.t0 + i < c.n_tokens; ++i) {
            EXPECT(own[s.t0 + i] < 0, "%s: row %d is of sequences %d and %d", what, s.t0 + i, own[s.t0 + i], b);
            own[s.t0 + i] = b;
        }
    }
    return own;
}

int main() {
    const int big = 0x7FFFFFFF;
    // sequence 0 has rows 0 .., sequence 5 rows new .., the others none
    for (int n : {1, 4, 60}) {
        const std::vector<std::vector<int>> lens = {{75, 3, -5, big, -big, 80}, {75, 0, 1, -big, big, 80}, {75, 0, 2, 5, -1, 80}};
        const std::vector<std::vector<int>> starts = {
            {0, n, n, n, n, n, 2 * n}, {0, n, -big, big, -1, n, 2 * n}, {0, n, 2 * n + 9, -3, big, n, 2 * n}};
        for (size_t i = 0; i < starts.size(); ++i) {
            const std::vector<int> own = owners(view(lens[i], starts[i], 2 * n, n), "wild row starts");
            for (int r = 0; r < 2 * n; ++r) EXPECT(own[r] == (r < n ? 0 : 5), "new %d, list %zu: row %d is of %d", n, i, r, own[r]);
        }
    }
    // one row each
    const std::vector<int> own = owners(view({7, 0, 9}, {}, 3, 1), "one each");
    for (int r = 0; r < 3; ++r) EXPECT(own[r] == r, "row %d is of %d", r, own[r]);
    // row starts that rise: every row its sequence's, up to max_new of them
    std::mt19937 rng(1);
    for (int k = 0; k < 2000; ++k) {
        const int seqs = 1 + (int)(rng() % 8), rows = 1 + (int)(rng() % 40), most = 1 + (int)(rng() % 12);
        std::vector<int> cu(seqs + 1), len(seqs, 50);
        for (int &x : cu) x = (int)(rng() % (rows + 1));
        std::sort(cu.begin(), cu.end());
        const std::vector<int> o = owners(view(len, cu, rows, most), "rising");
        for (int b = 0; b < seqs; ++b)
            for (int r = cu[b]; r < cu[b + 1]; ++r)
                EXPECT(o[r] == (r - cu[b] < most ? b : -1), "rising: row %d is of %d", r, o[r]);
        // and with one of them anything
        std::vector<int> wild = cu;
        wild[rng() % wild.size()] = (int)rng();
        const mgq::KvView c = view(len, wild, rows, most);
        for (int b = 0; b < seqs; ++b) {
            const mgq::SeqInfo s = mgq::kv_seq(c, b);
            const bool in = wild[b] >= 0 && wild[b] <= wild[b + 1] && wild[b + 1] <= rows;
            EXPECT(s.n == (in ? std::min(most, wild[b + 1] - wild[b]) : 0), "sequence %d of %d .. %d has %d rows", b, wild[b],
                   wild[b + 1], s.n);
        }
    }
    std::printf(fails ? "%d failures\n" : "ok\n", fails);
    return fails != 0;
}
