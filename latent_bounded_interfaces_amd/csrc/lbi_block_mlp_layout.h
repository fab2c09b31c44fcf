// Which tile each product of the gated MLP takes, and where sums are cut into parts: arithmetic on sizes, with no device code, so that a host
// program can ask it too.
#pragma once

#include <stddef.h>
#include <stdint.h>

namespace lbi {
namespace block_mlp {

constexpr int STEP = 64;  // terms of a step
constexpr int FEW = 4;    // rows that a kernel of their own takes
constexpr int64_t FEW_TERMS = 4 << 20;  // there, of a weight, from three rows on

// What becomes of the sums.
enum Finish {
    PLAIN,   // out = C + bias
    GATED,   // C is up and gate of one column: activation, and z where it is kept
    UNGATED  // C is the activation's cotangent: that of z
};

// How a product is laid out: the tile, and into how many parts the sums of those tiles are cut that do not fill the chip once more.
constexpr int NONE = -1, FORMS = 7, FEW_ROWS = FORMS;
// A tile's fragments, the steps of its ring, how many workgroups of it LDS lets share a CU, and what it takes there, in us (see layout_of).  Where
// there is one workgroup a CU a ring of three is the better one (8192 x 768 x 4096 in tiles of 128 x 192: 64 -> 51 us).
struct Form {
    int fm, fn, deep, a_cu;
    double step[3], alone[3], start;
};
constexpr Form forms[FORMS] = {
    {4, 4, 2, 1, {1.33, 1.33, 1.56}, {1.32, 1.28, 1.82}, 2.8}, {3, 2, 2, 2, {1.10, 1.11, 1.11}, {0.59, 0.64, 0.62}, 1.9},
    {3, 2, 3, 1, {0.60, 0.64, 0.57}, {0.49, 0.54, 0.51}, 2.2}, {2, 3, 3, 1, {0.60, 0.69, 0.64}, {0.52, 0.54, 0.57}, 2.2},
    {2, 2, 2, 2, {0.86, 0.89, 0.93}, {0.49, 0.48, 0.62}, 2.0}, {2, 2, 3, 1, {0.48, 0.44, 0.39}, {0.42, 0.36, 0.47}, 2.2},
    {1, 2, 3, 2, {0.55, 0.59, 0.54}, {0.31, 0.27, 0.32}, 2.8}};
struct Layout {
    int form;
    int tiles, whole, parts, part_steps;
    double us;
    size_t bytes() const {
        return parts > 1 ? (size_t)(tiles - whole) * parts * (64 * forms[form].fm) * (64 * forms[form].fn) * sizeof(float) : 0;
    }
};

// By what a call takes, in us: for each round of workgroups over the chip its steps, its start and the results on their way out (20 GB/s a CU, all
// finishing together; less of it shows where two share a CU); for parts a second launch and their sums out and back (of the gated product's two
// sums a column one; the fit counted both).  The constants were fitted to 438 products of 73 blocks (1 ... 16384 rows, widths 128 ... 11264), each in
// up to 60 layouts, the weights' gradients one by one; what is chosen of them took 1.013 times the best on average, 1.36 at most (540 rows,
// 1920 -> 2 x 640, gated).  A step of 256 x 256 takes 1.3 ... 1.6 us; of 192 x 128 two on a CU 1.1, one 0.6; of 128 x 128 0.9 and 0.4 ... 0.5;
// of 64 x 128 0.55 and 0.3.
// cus: compute units; by_rows: operands whose terms are their rows.  M2, N2: of a second product that is laid out together with the first.
inline Layout layout_of(int cus, int64_t M, int64_t N, int64_t K, Finish finish, int by_rows, int64_t M2 = 0, int64_t N2 = 0) {
    constexpr double out[3][2] = {{2.2, 1.7}, {4.4, 3.5}, {5.6, 2.6}};  // bytes of a result that show
    const int steps = (int)((K + STEP - 1) / STEP);
    Layout best{NONE, 0, 0, 1, 0, 0.0};
    if (by_rows == 0 && M <= FEW && (M <= 2 || N * K <= FEW_TERMS)) return {FEW_ROWS, 0, 0, 1, 0, 0.0};
    for (int f = 0; f < FORMS; ++f) {
        const Form& form = forms[f];
        if (finish == GATED && form.fn % 2) continue;  // up and gate are half of a wave's columns each
        const int rows = 64 * form.fm, wide = 64 * form.fn, columns = finish == GATED ? wide / 2 : wide, slots = cus * form.a_cu;
        const auto tiles_of = [&](int64_t m, int64_t n) { return (m + rows - 1) / rows * ((n + columns - 1) / columns); };
        const int64_t tiles = tiles_of(M, N) + tiles_of(M2, N2);
        if (tiles >= 1 << 24) continue;
        const double full = form.step[by_rows], alone = form.alone[by_rows];
        const double fixed = form.start + out[finish][form.a_cu - 1] * rows * columns * form.a_cu / 20e3;
        const auto rounds = [&](int64_t items, int of) {
            const int deep = (int)((items % slots + cus - 1) / cus);  // workgroups that share a CU in the last round
            return (double)(items / slots) * (of * full + fixed) + (deep ? of * (deep == 1 ? alone : full) + fixed : 0.0);
        };
        for (int s : {1, 2, 3, 4, 5, 6, 8, 12, 16}) {
            const int part_steps = (steps + s - 1) / s, parts = (steps + part_steps - 1) / part_steps;
            if (parts != s) continue;
            const int64_t whole = s == 1 ? tiles : tiles / slots * slots, rest = tiles - whole;
            if (s > 1 && (rest == 0 || part_steps < 2 || rest * s > 2 * slots)) break;  // parts for two rounds at most
            double us = rounds(whole, steps);
            if (rest) us += rounds(rest * s, part_steps) + 4.2 + (double)rest * s * rows * columns * 8.0 / 6.5e6;
            if (best.form == NONE || us < best.us) best = {f, (int)tiles, (int)whole, s, part_steps, us};
        }
    }
    return best;
}

}  // namespace block_mlp
}  // namespace lbi
