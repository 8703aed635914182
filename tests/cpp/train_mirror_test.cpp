// Exercises the training ops of the C++ host mirror (include/rg_b200.hpp) on cuda:0 with values that can be worked out by
// hand.  Prints "OK" and returns 0.
#include <cmath>
#include <cstdio>

#include "rg_b200.hpp"

#define EXPECT(c)                                                     \
    do {                                                              \
        if (!(c)) {                                                   \
            std::printf("FAILED %s:%d: %s\n", __FILE__, __LINE__, #c); \
            return 1;                                                 \
        }                                                             \
    } while (0)

static bool near(float a, double b, double tol = 1e-5) { return std::fabs(a - b) <= tol * (1 + std::fabs(b)); }

int main() {
    for (int own = 0; own < 2; own++) {
        rg::B200Backend be = own ? rg::B200Backend(0) : rg::B200Backend(0, nullptr);
        // a row [1, 3]: mean 2, variance 1; dy = [1, 0], gamma = 1: a sums cancel, dx = 0
        auto x = be.from_slice({1, 3}, {1, 2}), one = be.ones({2}), zero = be.zeros({2});
        auto ln = be.layer_norm_fwd(x, one, zero, 0.f);
        EXPECT(near(be.to_vec(ln.y)[0], -1) && near(be.to_vec(ln.y)[1], 1) && near(be.to_vec(ln.mean)[0], 2) && near(be.to_vec(ln.rstd)[0], 1));
        auto lg = be.layer_norm_bwd(be.from_slice({1, 0}, {1, 2}), x, one, ln.mean, ln.rstd);
        EXPECT(near(be.to_vec(lg.dgamma)[0], -1) && near(be.to_vec(lg.dbeta)[0], 1) && near(be.to_vec(lg.dx)[0], 0) && near(be.to_vec(lg.dx)[1], 0));
        // logits [0, log 3] for two rows, the second without a target: p = [1/4, 3/4], loss = log 4
        auto h = be.from_slice({1, 1}, {2, 1}), w = be.from_slice({0, std::log(3.f)}, {1, 2}), b = be.zeros({2});
        auto t = be.from_slice({0, -100}, {2});
        auto ce = be.linear_cross_entropy(h, w, &b, t);
        EXPECT(near(be.to_vec(ce.loss)[0], std::log(4.0)) && near(be.to_vec(ce.lse)[1], std::log(4.0)));
        auto g = be.linear_cross_entropy_bwd(h, w, &b, t, ce.lse);
        auto dw = be.to_vec(g.dw), db = be.to_vec(g.dbias), dx = be.to_vec(g.dx);
        EXPECT(near(dw[0], -0.75) && near(dw[1], 0.75) && near(db[0], -0.75) && near(db[1], 0.75));
        EXPECT(near(dx[0], 0.75 * std::log(3.0)) && dx[1] == 0);
        EXPECT(be.linear_cross_entropy_bwd(h, w, nullptr, t, ce.lse).dbias.get() == nullptr);
        auto clip = be.clip_grad_norm({be.from_slice({3}, {1}), be.cast(be.from_slice({4}, {1}), RG_DTYPE_BF16)}, 1.f);
        EXPECT(near(be.to_vec(clip.second)[0], 5) && near(be.to_vec(clip.first[0])[0], 0.6) && near(be.to_vec(clip.first[1])[0], 0.8, 4e-3));
        EXPECT(clip.first[1].is_bf16() && !clip.first[0].is_bf16());
        bool threw = false;
        try {
            be.linear_cross_entropy(h, w, &b, be.from_slice({0, 2}, {2}));
        } catch (const rg::ShapeError&) {
            threw = true;
        }
        EXPECT(threw);
        threw = false;
        try {
            be.clip_grad_norm({h}, -1.f);
        } catch (const rg::InvalidInput&) {
            threw = true;
        }
        EXPECT(threw);
    }
    std::printf("OK\n");
    return 0;
}
