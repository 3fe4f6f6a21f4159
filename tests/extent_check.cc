// Which strided buffers vs::meet takes to overlap, against their bytes one by one.
#include "../dart-pytorch_amd/csrc/vs_host.h"

#include <cstdio>
#include <random>
#include <set>

namespace vs {
int report(int code, const char *, ...) { return code; }
int report_hip(hipError_t, const char *) { return VS_ERR_OOM; }
hipError_t device_alloc(void **, size_t) { return hipErrorOutOfMemory; }
}  // namespace vs

struct Rows {
    int64_t at, row, head, nrows, heads, dim;
    vs::Extent extent() const {
        return vs::Extent((const char *)0x100000 + at * 2, row, head, nrows, heads, dim, 2);
    }
    std::set<int64_t> elements() const {
        std::set<int64_t> s;
        for (int64_t i = 0; i < nrows; ++i)
            for (int64_t h = 0; h < heads; ++h)
                for (int64_t x = 0; x < dim; ++x) s.insert(at + i * row + h * head + x);
        return s;
    }
};

static bool share(const Rows &a, const Rows &b) {
    const auto s = a.elements();
    for (int64_t x : b.elements())
        if (s.count(x)) return true;
    return false;
}

int main() {
    int bad = 0;
    auto check = [&](const char *what, const Rows &a, const Rows &b) {
        if (share(a, b) != vs::meet(a.extent(), b.extent()) || share(b, a) != vs::meet(b.extent(), a.extent()))
            std::printf("%s\n", what), bad = 1;
    };
    const int64_t D = 8, R = 7, H = 4;
    // [rows, H + 2 G, D]: queries, keys and values side by side
    check("parts of a row", {0, 8 * D, D, R, H, D}, {H * D, 8 * D, D, R, 2, D});
    check("the last part", {H * D, 8 * D, D, R, 2, D}, {(H + 2) * D, 8 * D, D, R, 2, D});
    // [rows, H, 3, D]: side by side per head
    for (int64_t nrows : {(int64_t)1, R})
        for (int i = 0; i < 3; ++i)
            for (int j = 0; j < 3; ++j)
                check("parts of a head", {i * D, 3 * H * D, 3 * D, nrows, H, D}, {j * D, 3 * H * D, 3 * D, nrows, H, D});
    // padded rows of it
    check("parts of a head, padded", {0, 3 * H * D + 3, 3 * D, R, H, D}, {D, 3 * H * D + 3, 3 * D, R, H, D});
    // [H, 3, rows, D], [H, rows, 3, D], [3, H, rows, D]
    check("a head's rows", {0, D, 3 * R * D, R, H, D}, {R * D, D, 3 * R * D, R, H, D});
    check("parts of a head's rows", {0, 3 * D, 3 * R * D, R, H, D}, {2 * D, 3 * D, 3 * R * D, R, H, D});
    check("whole parts", {0, D, R * D, R, H, D}, {R * H * D, D, R * D, R, H, D});
    // keys of the second half of a head, fewer heads than the queries
    check("fewer heads", {0, 2 * H * D, 2 * D, R, H, D}, {D, 2 * H * D, 4 * D, R, 2, D});
    // upside down
    check("backwards", {(R - 1) * 3 * H * D, -3 * H * D, 3 * D, R, H, D}, {D, 3 * H * D, 3 * D, R, H, D});
    check("backwards, shifted", {(R - 1) * 3 * H * D + 1, -3 * H * D, 3 * D, R, H, D}, {D, 3 * H * D, 3 * D, R, H, D});
    check("an element too far", {1, 3 * H * D, 3 * D, R, H, D}, {D, 3 * H * D, 3 * D, R, H, D});
    check("one for all", {0, 0, D, R, H, D}, {H * D - 1, H * D, D, R, H, D});
    // whatever they are: what does share an element is never missed
    std::mt19937 rng(1);
    auto in = [&](int lo, int hi) { return (int64_t)(lo + (int)(rng() % (unsigned)(hi - lo + 1))); };
    int apart = 0;
    for (int i = 0; i < 200000; ++i) {
        Rows x[2];
        const int64_t row = in(-40, 40), head = in(-20, 20);
        for (auto &r : x)
            r = {in(0, 60), in(0, 2) ? row : in(-40, 40), in(0, 2) ? head : in(-20, 20), in(1, 4), in(1, 4), in(1, 5)};
        const bool met = vs::meet(x[0].extent(), x[1].extent());
        apart += !met;
        if (!met && share(x[0], x[1])) return std::printf("an overlap is missed\n"), 1;
    }
    if (apart < 1000) std::printf("%d\n", apart), bad = 1;
    return bad;
}
