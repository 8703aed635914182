// Walks every address that the few-row form of the linear cross entropy reads of w, for small matrices of every shape.
#include <algorithm>
#include <cstdio>

#include "rg_lce_plan.h"

static int check(int D, int V) {
    const long long total = (long long)D * V;
    for (int warp = 0; warp < 8; warp++) {
        const int shift = lce_few_shift(V, warp), last = lce_few_last(V, shift), safe = lce_few_safe(D, V, warp);
        const int rows = warp < D ? (D - warp + 7) / 8 : 0;
        if (safe < 0 || safe > rows) return printf("D %d V %d warp %d: %d rows of %d\n", D, V, warp, safe, rows), 1;
        // at most the rows whose last group may leave the matrix are guarded: those that start within 3 + V values of its end
        for (int k = safe; k < rows; k++)
            if ((long long)(warp + 8 * k) * V + last + 4 <= total) return printf("D %d V %d warp %d: row %d is guarded for nothing\n", D, V, warp, warp + 8 * k), 1;
        for (int k = 0; k < safe; k++)
            for (int c0 = 0; c0 < V; c0 += 124)
                for (int lane = 0; lane < 32; lane++) {
                    const long long at = (long long)(warp + 8 * k) * V + std::min(c0 - shift + 4 * lane, last);
                    if (at < 0 || at % 4 || at + 4 > total)
                        return printf("D %d V %d warp %d row %d lane %d: %lld..%lld of %lld\n", D, V, warp, warp + 8 * k, lane, at, at + 3, total), 1;
                }
    }
    return 0;
}

int main() {
    for (int D = 1; D <= 70; D++)
        for (int V = 1; V <= 40; V++)
            if (check(D, V)) return 1;
    const int shapes[][2] = {{2, 125}, {9, 257}, {768, 97}, {1026, 1}, {1026, 2}, {1026, 3}, {33, 1025}};
    for (const auto& s : shapes)
        if (check(s[0], s[1])) return 1;
    // the largest matrix of the op: no overflow on the way
    if (lce_few_safe(1 << 20, 1 << 24, 7) != (1 << 20) / 8) return printf("largest: %d\n", lce_few_safe(1 << 20, 1 << 24, 7)), 1;
    puts("OK");
}
