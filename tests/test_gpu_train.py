"""GPU parity of the training ops (LayerNorm with statistics and gradient, linear cross entropy with gradient, clipping
by the global norm) against their formulas in 64 bits.

Tolerances are worst-case bounds of the arithmetic, worked out per element beside each check: U is half a step of the
output type (relative), E32 = 2^-23 one step of f32."""
import numpy as np
import pytest

import rustygradients_b200 as rg

pytestmark = pytest.mark.gpu

E32 = 2.0 ** -23
U = {"f32": 2.0 ** -24, "bf16": 2.0 ** -8}
EPS = 1e-5


def rounded(a, dtype):
    """The f32 array whose values are exactly representable in dtype."""
    a = np.ascontiguousarray(a, np.float32)
    if dtype == "f32":
        return a
    b = a.view(np.uint32).astype(np.uint64)
    b = ((b + 0x7FFF + ((b >> 16) & 1)) & 0xFFFF0000).astype(np.uint32)
    return b.view(np.float32).reshape(a.shape)


def put(be, a, dtype="f32"):
    st = be.from_slice(a, list(a.shape))
    return st if dtype == "f32" else be.cast(st, dtype)


def get(be, st):
    return be.to_array(st).astype(np.float64)


def within(got, want, tol, what=""):
    assert got.shape == want.shape, (what, got.shape, want.shape)
    bad = ~(np.abs(got - want) <= tol)
    assert not bad.any(), (what, int(bad.sum()), float(np.nanmax(np.abs(got - want) / tol)), np.argwhere(bad)[:3].tolist())


# ---------------------------------------------------------------------------------------------------------------------
# storages: types and other owners' memory
# ---------------------------------------------------------------------------------------------------------------------
def test_cast_and_dtype(backend):
    be = backend
    x = np.array([0.0, -0.0, 1.0, 1.00390625, 1.01171875, 3.4e38, np.inf, -np.inf, 1e-40], np.float32)   # ties both ways
    s = be.from_slice(x, [9])
    h = be.cast(s, "bf16")
    assert (s.dtype, h.dtype) == ("f32", "bf16") and h.shape == [9] and len(h) == 9
    assert np.array_equal(be.to_vec(h), rounded(x, "bf16"))
    assert np.isnan(be.to_vec(be.cast(be.from_slice([np.nan], [1]), "bf16")))[0]
    assert np.array_equal(be.to_vec(be.cast(h, "f32")), be.to_vec(h))
    assert be.cast(h, "bf16").dtype == "bf16" and be.reshape(h, [3, 3]).dtype == "bf16"
    for op in (lambda: be.add(h, h), lambda: be.relu(h), lambda: be.softmax(h), lambda: be.sum(h), lambda: be.sum_axis(h, 0),
               lambda: be.transpose(be.reshape(h, [3, 3]), 0, 1), lambda: be.matmul(be.reshape(h, [3, 3]), be.reshape(h, [3, 3])),
               lambda: be.layer_norm(h, s, s, EPS), lambda: be.embedding(s, be.reshape(h, [3, 3])),
               lambda: be.sparse_cross_entropy(be.reshape(h, [3, 3]), be.zeros([3]))):
        with pytest.raises(rg.Unsupported):
            op()
    with pytest.raises(rg.Unsupported):
        be.cast(s, "f16")


def test_arrays_of_another_owner():
    import torch
    torch.cuda.set_device(0)
    side = torch.cuda.Stream()
    for stream in (torch.cuda.current_stream(), side):
        with torch.cuda.stream(stream):
            be = rg.B200Backend(0, stream=stream.cuda_stream)
            t = torch.arange(24, dtype=torch.float32, device="cuda").reshape(4, 6)
            s = be.from_device(t)
            assert s.shape == [4, 6] and np.array_equal(be.to_array(s), t.cpu().numpy())
            back = torch.from_dlpack(be.add(s, s))
            assert torch.equal(back, 2 * t) and back.is_cuda
            # a slice that starts off a 16-byte boundary is copied: later writes to the tensor are not seen
            odd = be.from_device(t.reshape(-1)[1:])
            t.add_(1)
            assert np.array_equal(be.to_vec(odd), np.arange(1, 24, dtype=np.float32))
            assert np.array_equal(be.to_vec(s), t.reshape(-1).cpu().numpy())
            t16 = torch.randn(5, 7, device="cuda").bfloat16()
            h = be.from_device(t16)
            assert h.dtype == "bf16" and torch.equal(torch.from_dlpack(be.cast(h, "f32")), t16.float())
            assert torch.equal(torch.utils.dlpack.from_dlpack(be.cast(be.from_device(t16.float()), "bf16").to_dlpack()), t16)
            # views keep the borrowed tensor alive
            view = be.reshape(be.from_device(torch.full((8,), 3.0, device="cuda")), [2, 4])
            torch.full((8,), 5.0, device="cuda")
            assert np.all(be.to_vec(view) == 3)
            assert be.from_device(torch.empty(0, 3, device="cuda")).shape == [0, 3]
            # capsules nobody takes, and tensors that outlive their storage and the backend object
            be.ones([1 << 20]).to_dlpack()
            keep = torch.from_dlpack(be.ones([3]))
            with pytest.raises(BufferError):
                be.ones([1]).__dlpack__(stream=12345)
            with pytest.raises(rg.Unsupported):
                s.to_dlpack()
            for bad, err in ((t.t(), rg.InvalidInput), (t.cpu(), rg.InvalidInput), (t.double(), rg.Unsupported),
                             (np.ones(3, np.float32), rg.InvalidInput), (t.reshape((1,) * 7 + (4, 6)), rg.DimensionError)):
                with pytest.raises(err):
                    be.from_device(bad)
            with pytest.raises(rg.Unsupported):
                rg.GPTModel(be, rg.GptConfig(16, 30, 1, 2, 64))
            stream.synchronize()
            be.close()
            assert keep.sum().item() == 3


def test_a_context_refuses_storages_of_another(backend):
    other = rg.B200Backend(0)
    x, g = other.ones([2, 4]), backend.ones([4])
    for call in (lambda: backend.layer_norm_fwd(x, g, g, EPS), lambda: backend.clip_grad_norm([x], 1.0), lambda: backend.cast(x, "bf16"),
                 lambda: backend.linear_cross_entropy(x, backend.ones([4, 3]), None, backend.zeros([2]))):
        with pytest.raises(rg.InvalidInput):
            call()


def test_calls_inside_a_capture_are_refused():
    import torch
    torch.cuda.set_device(0)
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        be = rg.B200Backend(0, stream=stream.cuda_stream)
        x, g, w, t = be.ones([2, 4]), be.ones([4]), be.ones([4, 3]), be.zeros([2])
        y, m, r = be.layer_norm_fwd(x, g, g, EPS)
        dead = be.ones([5])
        graph = torch.cuda.CUDAGraph()
        a = torch.zeros(4, device="cuda")
        stream.synchronize()
        with torch.cuda.graph(graph, stream=stream):
            a.add_(1)
            for call in (lambda: be.layer_norm_fwd(x, g, g, EPS), lambda: be.layer_norm_bwd(y, x, g, m, r),
                         lambda: be.linear_cross_entropy(x, w, None, t), lambda: be.linear_cross_entropy_bwd(x, w, None, t, t),
                         lambda: be.clip_grad_norm([x], 1.0), lambda: be.add(x, x), lambda: be.cast(x, "bf16"), lambda: be.ones([3])):
                with pytest.raises(rg.Unsupported):
                    call()
            del dead      # its memory is given back after the capture
        graph.replay()
        stream.synchronize()
        assert a.sum().item() == 4
        assert np.allclose(be.to_vec(be.layer_norm_fwd(x, g, g, EPS)[0]), be.to_vec(y))


# ---------------------------------------------------------------------------------------------------------------------
# LayerNorm
# ---------------------------------------------------------------------------------------------------------------------
def ln_inputs(rows, n, dtype, seed=0):
    rng = np.random.default_rng(seed + 31 * rows + n)
    x = rounded(rng.standard_normal((rows, n)) * rng.uniform(0.3, 4, (rows, 1)) + rng.uniform(-5, 5, (rows, 1)), dtype)
    dy = rounded(rng.standard_normal((rows, n)), dtype)
    g = (1 + 0.3 * rng.standard_normal((1, n))).astype(np.float32)
    b = (0.5 * rng.standard_normal((1, n))).astype(np.float32)
    return x, dy, g, b


def ln_exact(x, g, b):
    x = x.astype(np.float64)
    mean = x.mean(-1, keepdims=True)
    rstd = 1 / np.sqrt(((x - mean) ** 2).mean(-1, keepdims=True) + np.float64(np.float32(EPS)))
    return (x - mean) * rstd * g + b, mean, rstd


LN_SHAPES = [(1, 1), (3, 1), (1, 768), (2, 2), (5, 7), (64, 8), (33, 192), (9, 255), (17, 256), (4, 257), (6, 514), (300, 768),
             (37, 1023), (8, 1024), (3, 1026), (650, 1600), (5, 2050), (3, 4097), (2, 4104), (2, 8192), (3, 8200), (2, 12001),
             (2, 16384), (3, 16386), (70, 20001)]


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("rows,n", LN_SHAPES)
def test_layer_norm_forward_and_gradient(backend, rows, n, dtype):
    be = backend
    x, dy, g, b = ln_inputs(rows, n, dtype)
    X, DY, G, B = put(be, x, dtype), put(be, dy, dtype), put(be, g), put(be, b)
    y, mean, rstd = be.layer_norm_fwd(X, G, B, EPS)
    assert (y.dtype, mean.dtype, y.shape, mean.shape, rstd.shape) == (dtype, "f32", [rows, n], [rows], [rows])
    wy, wm, wr = ln_exact(x, g, b)
    # a sum of n terms: per-thread chains of at most 40 terms (n <= 20001 over 512 threads), then <= 10 levels
    chain = 52 * 2.0 ** -24
    tm = chain * np.abs(x).mean(-1, keepdims=True) + 2 * E32 * np.abs(wm)
    within(get(be, mean), wm[:, 0], tm[:, 0] + 1e-45, "mean")
    # variance: relative chain error, 3 roundings a term, and the mean's error squared; half of it in rstd
    dev = np.abs(x - wm).max(-1, keepdims=True) + tm
    tr = wr * ((chain + 4 * E32) + 0.5 * wr ** 2 * (tm ** 2 + 2 * E32 * dev ** 2) + 2 * E32)
    within(get(be, rstd), wr[:, 0], tr[:, 0], "rstd")
    xh = np.abs((x - wm) * wr)
    ty = np.abs(g) * (tm * wr + xh * (tr / wr) + 4 * E32 * (xh + np.abs(x) * wr)) + E32 * (np.abs(wy) + np.abs(b))
    within(get(be, y), wy, ty + U[dtype] * (np.abs(wy) + ty), "y")
    if n == 1 or rows * n < 3:
        assert np.all(np.isfinite(get(be, y)))
    # gradient, from exact statistics rounded to f32
    m32, r32 = wm[:, 0].astype(np.float32), wr[:, 0].astype(np.float32)
    dx, dg, db = be.layer_norm_bwd(DY, X, G, put(be, m32), put(be, r32))
    assert (dx.dtype, dg.dtype, dx.shape, dg.shape, db.shape) == (dtype, "f32", [rows, n], [1, n], [1, n])
    x6, d6, m6, r6 = x.astype(np.float64), dy.astype(np.float64), m32[:, None].astype(np.float64), r32[:, None].astype(np.float64)
    h = (x6 - m6) * r6
    a = d6 * g
    wdx = r6 * (a - a.mean(-1, keepdims=True) - h * (a * h).mean(-1, keepdims=True))
    th = 2 * E32 * (np.abs(h) + np.abs(x6) * 0)                 # one subtraction (exact to half a step of x - m) and one product
    mag = np.abs(a) + np.abs(a).mean(-1, keepdims=True) + np.abs(h) * np.abs(a * h).mean(-1, keepdims=True)
    tdx = np.abs(r6) * mag * (2 * chain + 8 * E32)
    within(get(be, dx), wdx, tdx + U[dtype] * (np.abs(wdx) + tdx), "dx")
    # columns: a chain of at most rows / partial rows terms, then the partial rows (32 slices)
    steps = (rows + 40) * 2.0 ** -24
    within(get(be, dg), (d6 * h).sum(0, keepdims=True), (steps + 4 * E32) * np.abs(d6 * h).sum(0, keepdims=True) +
           (np.abs(d6) * th).sum(0, keepdims=True) + 1e-45, "dgamma")
    within(get(be, db), d6.sum(0, keepdims=True), steps * np.abs(d6).sum(0, keepdims=True) + 1e-45, "dbeta")


def test_layer_norm_gradient_against_differences(backend):
    be = backend
    x, dy, g, b = ln_inputs(4, 96, "f32", 5)
    y, mean, rstd = be.layer_norm_fwd(put(be, x), put(be, g), put(be, b), EPS)
    dx, dg, db = (get(be, s) for s in be.layer_norm_bwd(put(be, dy), put(be, x), put(be, g), mean, rstd))
    rng = np.random.default_rng(3)

    def f(x_, g_, b_):
        return float((ln_exact(x_, g_, b_)[0] * dy).sum())

    for k in range(3):
        vx, vg, vb = rng.standard_normal(x.shape), rng.standard_normal(g.shape), rng.standard_normal(b.shape)
        e = 1e-5
        num = (f(x + e * vx, g + e * vg, b + e * vb) - f(x - e * vx, g - e * vg, b - e * vb)) / (2 * e)
        ana = (dx * vx).sum() + (dg * vg).sum() + (db * vb).sum()
        # differences: O(e^2) third derivatives ~ 1e-10 of scale 1e3, cancellation 2^-52 * 1e3 / e ~ 2e-8; f32 gradient 1e-5
        assert abs(num - ana) <= 2e-4 * (1 + np.abs(dx * vx).sum())


def test_layer_norm_far_from_zero_and_not_finite(backend):
    """Rows whose mean is far from zero keep their variance; a row with a NaN or infinity leaves the other rows alone."""
    be = backend
    x = np.random.default_rng(9).standard_normal((4, 768)).astype(np.float32) + np.array([[1e4], [0], [0], [-3e3]], np.float32)
    x[1, 5], x[2, 700] = np.nan, np.inf
    g, b = np.ones((1, 768), np.float32), np.zeros((1, 768), np.float32)
    y, mean, rstd = (get(be, s) for s in be.layer_norm_fwd(put(be, x), put(be, g), put(be, b), EPS))
    for r in (0, 3):
        wy, wm, wr = ln_exact(x[r:r + 1], g, b)
        # the mean is off by its chain (16 terms a thread, 6 levels) relative to 1e4; the deviations from it are exact
        tm = 24 * 2.0 ** -24 * np.abs(x[r]).mean() + E32 * abs(float(wm[0, 0]))
        assert abs(mean[r] - wm[0, 0]) <= tm and abs(rstd[r] / wr[0, 0] - 1) <= 1e-5 + tm ** 2
        assert np.abs(y[r] - wy[0]).max() <= 2 * tm + 1e-4
    assert np.isnan(y[1]).all() and np.isnan(mean[1])
    assert np.isnan(y[2]).any() and not np.isfinite(mean[2])


def test_layer_norm_ranks_empty_and_refusals(backend):
    be = backend
    x, dy, g, b = ln_inputs(6, 10, "f32")
    G, B = put(be, g), put(be, b)
    y3, m3, r3 = be.layer_norm_fwd(be.from_slice(x, [2, 3, 10]), G, B, EPS)
    y2, m2, r2 = be.layer_norm_fwd(put(be, x), G, B, EPS)
    assert y3.shape == [2, 3, 10] and m3.shape == [2, 3] and np.array_equal(be.to_vec(y3), be.to_vec(y2))
    y1, m1, r1 = be.layer_norm_fwd(be.from_slice(x[0], [10]), G, B, EPS)
    assert m1.shape == [] and np.array_equal(be.to_vec(y1), be.to_vec(y2)[:10])
    dx, dg, db = be.layer_norm_bwd(be.from_slice(dy[0], [10]), be.from_slice(x[0], [10]), G, m1, r1)
    assert dx.shape == [10] and dg.shape == [1, 10]
    y0, m0, r0 = be.layer_norm_fwd(be.zeros([0, 10]), G, B, EPS)
    assert y0.shape == [0, 10] and m0.shape == [0]
    dx, dg, db = be.layer_norm_bwd(be.zeros([0, 10]), be.zeros([0, 10]), G, m0, r0)
    assert dx.shape == [0, 10] and not be.to_vec(dg).any() and not be.to_vec(db).any()
    X, M, R = put(be, x), m2, r2
    H = be.cast(X, "bf16")
    for call, err in ((lambda: be.layer_norm_fwd(X, be.ones([9]), B, EPS), rg.ShapeError),
                      (lambda: be.layer_norm_fwd(X, G, be.ones([11]), EPS), rg.ShapeError),
                      (lambda: be.layer_norm_fwd(be.zeros([3, 0]), be.zeros([0]), be.zeros([0]), EPS), rg.ShapeError),
                      (lambda: be.layer_norm_fwd(be.from_slice([1.0], []), G, B, EPS), rg.DimensionError),
                      (lambda: be.layer_norm_fwd(X, be.cast(G, "bf16"), B, EPS), rg.Unsupported),
                      (lambda: be.layer_norm_bwd(H, X, G, M, R), rg.Unsupported),
                      (lambda: be.layer_norm_bwd(be.zeros([10, 6]), X, G, M, R), rg.ShapeError),
                      (lambda: be.layer_norm_bwd(X, X, G, be.zeros([5]), R), rg.ShapeError),
                      (lambda: be.layer_norm_bwd(X, X, G, M, be.zeros([7])), rg.ShapeError)):
        with pytest.raises(err):
            call()


def test_layer_norm_gives_the_same_bits_again(backend):
    be = backend
    x, dy, g, b = ln_inputs(4000, 768, "f32")
    X, DY, G, B = put(be, x), put(be, dy), put(be, g), put(be, b)
    y, m, r = be.layer_norm_fwd(X, G, B, EPS)
    first = [be.to_vec(s) for s in be.layer_norm_bwd(DY, X, G, m, r)]
    for _ in range(3):
        again = [be.to_vec(s) for s in be.layer_norm_bwd(DY, X, G, m, r)]
        assert all(np.array_equal(p, q) for p, q in zip(first, again))


# ---------------------------------------------------------------------------------------------------------------------
# linear cross entropy
# ---------------------------------------------------------------------------------------------------------------------
IGNORE = -100


def ce_inputs(R, D, V, dtype, bias=True, ignored=0.2, seed=0, scale=2.5):
    rng = np.random.default_rng(seed + R * 7 + D * 3 + V)
    x = rounded(rng.standard_normal((R, D)), dtype)
    w = rounded(rng.standard_normal((D, V)) * scale / np.sqrt(D), dtype)
    b = (0.5 * rng.standard_normal(V)).astype(np.float32) if bias else None
    t = rng.integers(0, V, R).astype(np.float32)
    t[rng.random(R) < ignored] = IGNORE
    return x, w, b, t


def ce_exact(x, w, b, t, dloss=1.0, ignore=IGNORE):
    x, w = x.astype(np.float64), w.astype(np.float64)
    z = x @ w + (0 if b is None else b.astype(np.float64))
    m = z.max(-1, keepdims=True)
    lse = (m + np.log(np.exp(z - m).sum(-1, keepdims=True)))[:, 0]
    live = t != ignore
    at = np.where(live, t, 0).astype(int)
    n = max(1, int(live.sum()))
    loss = float(np.where(live, lse - z[np.arange(len(t)), at], 0).sum() / n)
    p = np.exp(z - lse[:, None])
    dz = p.copy()
    dz[np.arange(len(t)), at] -= 1
    scale = dloss / n if live.any() else 0.0
    dz *= live[:, None]
    return {"z": z, "lse": lse, "loss": loss, "p": p, "dz": dz, "scale": scale, "dx": scale * dz @ w.T, "dw": scale * x.T @ dz,
            "db": scale * dz.sum(0)}


def ce_bounds(x, w, b, dtype, ex, live):
    """Worst cases.  A logit: one chain of additions that truncate (D / 16 steps of a step each, doubled for the additions
    inside a step) in bf16; in f32 chains of 16 steps, the products left out (2^-21 of the magnitudes) and the additions of the
    pieces; relative to the sum of magnitudes.  exp: 2 steps and the rounding of its argument."""
    ax, aw = np.abs(x).astype(np.float64), np.abs(w).astype(np.float64)
    D = x.shape[1]
    steps = (2 * (D / 16 + 2) if dtype == "bf16" else 2 * 18 + 4 + D / 256)
    steps = max(steps, D / 8 + 8)           # the form for few rows: 8 chains of D / 8 terms
    ez = steps * E32 * (ax @ aw) + E32 * (np.abs(ex["z"]) + (0 if b is None else np.abs(b)))
    ez_row = ez.max(-1)
    elsum = 300 * 2.0 ** -24                # chains of at most 128 terms, then partial sums over slices of the vocabulary
    elogs = E32 * (np.abs(ex["lse"]) + 1)
    tlse = ez_row + elsum + 2 * elogs + 2 * E32 * np.abs(ex["z"]).max(-1)
    tloss = float((tlse + ez_row)[live].mean() if live.any() else 0) + E32 * (abs(ex["loss"]) + 1)
    # gradient, from an lse that is given rounded to f32
    earg = ez + 2 * E32 * (np.abs(ex["z"]) + np.abs(ex["lse"])[:, None])
    edz = live[:, None] * (ex["p"] * (earg + 4 * E32) * 1.01 + E32 * np.abs(ex["dz"]))
    if dtype == "bf16":
        store = U["bf16"]                   # dz is multiplied as bf16
    else:
        store = 2.0 ** -21
    ez2 = edz + store * (np.abs(ex["dz"]) + edz)
    V, R, s = w.shape[1], x.shape[0], abs(ex["scale"])
    chain_v = 2 * (V / 16 + 2) if dtype == "bf16" else 2 * 18 + 4 + V / 256
    chain_r = 2 * (R / 16 + 2) if dtype == "bf16" else 2 * 18 + 4 + R / 256
    adz = np.abs(ex["dz"])
    tdx = s * (ez2 @ aw.T + max(chain_v, 60) * E32 * (adz @ aw.T)) + 3 * E32 * np.abs(ex["dx"])
    tdw = s * (ax.T @ ez2 + max(chain_r, 24) * E32 * (ax.T @ adz)) + 3 * E32 * np.abs(ex["dw"])
    tdb = s * (edz.sum(0) + (R / 32 + 40) * E32 * adz.sum(0))
    return tlse, tloss, tdx + U[dtype] * (np.abs(ex["dx"]) + tdx), tdw + U[dtype] * (np.abs(ex["dw"]) + tdw), tdb


def ce_check(be, R, D, V, dtype, bias=True, ignored=0.2, dloss=None, seed=0):
    x, w, b, t = ce_inputs(R, D, V, dtype, bias, ignored, seed)
    X, W, B, T = put(be, x, dtype), put(be, w, dtype), put(be, b) if bias else None, put(be, t)
    ex = ce_exact(x, w, b, t, 1.0 if dloss is None else dloss)
    live = t != IGNORE
    tlse, tloss, tdx, tdw, tdb = ce_bounds(x, w, b, dtype, ex, live)
    loss, lse = be.linear_cross_entropy(X, W, B, T)
    assert (loss.shape, lse.shape, loss.dtype, lse.dtype) == ([1], [R], "f32", "f32")
    within(get(be, lse), ex["lse"], tlse, "lse")
    within(get(be, loss), np.array([ex["loss"]]), tloss + 1e-45, "loss")
    L = put(be, ex["lse"].astype(np.float32))
    dx, dw, db = be.linear_cross_entropy_bwd(X, W, B, T, L, None if dloss is None else put(be, np.array([dloss], np.float32)))
    assert (dx.shape, dw.shape, dx.dtype, dw.dtype) == ([R, D], [D, V], dtype, dtype) and (db is None) == (not bias)
    within(get(be, dx), ex["dx"], tdx + 1e-45, "dx")
    within(get(be, dw), ex["dw"], tdw + 1e-45, "dw")
    if bias:
        assert db.shape == [V]
        within(get(be, db), ex["db"], tdb + 1e-45, "dbias")
    return ex


FEW = [(1, 1, 1), (1, 8, 2), (1, 64, 1000), (2, 13, 97), (3, 768, 257), (4, 32, 128), (5, 300, 1025), (8, 128, 129), (9, 31, 63),
       (16, 257, 2047), (13, 520, 333), (2, 70, 5000), (6, 129, 20011), (3, 9000, 65), (14, 9000, 65)]
MANY = [(17, 1, 1), (17, 8, 2), (33, 13, 97), (64, 64, 64), (64, 192, 97), (127, 65, 255), (128, 128, 256), (129, 72, 257), (200, 100, 1000),
        (300, 320, 513), (511, 257, 775), (640, 768, 1024), (1025, 40, 2049), (260, 520, 5003), (30, 700, 2000), (200, 768, 1500),
        (2500, 40, 300), (8000, 128, 97), (192, 130, 515), (193, 60, 131), (70, 130, 20011), (33, 257, 40001), (40, 9000, 65),
        (300, 9000, 72)]


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("R,D,V", FEW + MANY)
def test_linear_cross_entropy(backend, R, D, V, dtype):
    ce_check(backend, R, D, V, dtype, bias=(R + V) % 3 != 0, dloss=None if R % 2 else 0.25)


# ---------------------------------------------------------------------------------------------------------------------
# clipping by the global norm
# ---------------------------------------------------------------------------------------------------------------------
def clip_check(be, arrays, dtypes, max_norm):
    arrays = [rounded(a, t) for a, t in zip(arrays, dtypes)]
    out, norm = be.clip_grad_norm([put(be, a, t) for a, t in zip(arrays, dtypes)], max_norm)
    n = float(np.sqrt(sum(float((a.astype(np.float64) ** 2).sum()) for a in arrays)))
    c = min(1.0, float(np.float32(max_norm)) / n) if n else 1.0
    assert norm.shape == [1] and norm.dtype == "f32"
    if n > float(np.finfo(np.float32).max):                    # no f32 holds it (each of the gradients does)
        assert np.isinf(get(be, norm)[0])
    else:
        # at most 4 f32 roundings (2^-24 each) on the way of a square into the f64 sum, half of that in the root, one
        # rounding of the root: 3 * 2^-24
        within(get(be, norm), np.array([n]), 1.5 * E32 * n + 1e-45, "norm")
    for a, t, o in zip(arrays, dtypes, out):
        assert o.shape == list(a.shape) and o.dtype == t
        want = a.astype(np.float64) * c
        # the factor is off by 2 steps; 2^-149 / 2^-133: the smallest steps of f32 and bf16
        within(get(be, o), want, (2 * E32 + U[t]) * np.abs(want) + (1.5e-45 if t == "f32" else 9.2e-41), "gradient")
        if c == 1.0:
            assert np.array_equal(be.to_vec(o).reshape(a.shape), a)
    return n


@pytest.mark.parametrize("sizes", [[1], [7], [8191, 8192, 8193], [3, 0, 5, 65536 + 1], [20000] * 3 + [1] * 40, [33] * 600,
                                   [1000003]])
@pytest.mark.parametrize("kind", ["f32", "bf16", "mixed"])
def test_clip_grad_norm(backend, sizes, kind):
    rng = np.random.default_rng(len(sizes) + sizes[0])
    arrays = [rng.standard_normal(n).astype(np.float32) for n in sizes]
    dtypes = [kind if kind != "mixed" else ("f32", "bf16")[i % 2] for i in range(len(sizes))]
    n = clip_check(backend, arrays, dtypes, 0.5)
    clip_check(backend, arrays, dtypes, 2 * n)          # nothing to clip: the values themselves
    clip_check(backend, arrays, dtypes, float("inf"))


def test_clip_grad_norm_extremes(backend):
    be = backend
    # squares beyond the range of f32 both ways
    clip_check(be, [np.full(100, 1e30, np.float32), np.full(5, -3e38, np.float32)], ["f32", "f32"], 1.0)
    clip_check(be, [np.full(100, 1e-30, np.float32)], ["f32"], 1e-30)
    clip_check(be, [np.zeros(64, np.float32)], ["bf16"], 1.0)
    out, norm = be.clip_grad_norm([], 1.0)
    assert out == [] and be.to_vec(norm)[0] == 0
    for bad, where in ((np.nan, 3), (np.nan, 9)):
        a = np.ones(10, np.float32)
        a[where] = bad
        out, norm = be.clip_grad_norm([put(be, a), put(be, np.ones(4, np.float32), "bf16")], 1.0)
        assert np.isnan(be.to_vec(norm)[0]) and np.isnan(be.to_vec(out[0])).all() and np.isnan(be.to_vec(out[1])).all()
    a = np.ones(10, np.float32)
    a[2] = np.inf
    out, norm = be.clip_grad_norm([put(be, a)], 1.0)     # 1 / inf = 0
    v = be.to_vec(out[0])
    assert np.isinf(be.to_vec(norm)[0]) and np.isnan(v[2]) and not v[:2].any() and not v[3:].any()
    g = put(be, np.array([3.0, 4.0], np.float32))        # the same tensor twice is two tensors of the list
    out, norm = be.clip_grad_norm([g, g], 5.0)
    assert abs(be.to_vec(norm)[0] - np.sqrt(50.0)) < 1e-6 and np.array_equal(be.to_vec(g), [3, 4])
    for m in (0.0, -1.0, float("nan")):
        with pytest.raises(rg.InvalidInput):
            be.clip_grad_norm([g], m)


def test_linear_cross_entropy_scales_of_rows_and_columns(backend):
    """f32 rows and columns of very different magnitudes, large channels, columns of zeros: the result depends on the products."""
    be = backend
    R, D, V = 150, 200, 300
    x, w, b, t = ce_inputs(R, D, V, "f32", True, 0.1, 77)
    x *= 1e-15 * 2.0 ** np.random.default_rng(1).integers(-6, 7, (R, 1))
    x[:, 3] *= 1000
    w *= 1e15 * 2.0 ** np.random.default_rng(2).integers(-6, 1, (1, V))
    w[3] *= 1e-3
    w[:, 17], x[5] = 0, 0
    x, w = x.astype(np.float32), w.astype(np.float32)
    w *= np.float32(20 / np.abs(x.astype(np.float64) @ w).max())
    ex, live = ce_exact(x, w, b, t), t != IGNORE
    tlse, tloss, tdx, tdw, tdb = ce_bounds(x, w, b, "f32", ex, live)
    X, W, B, T = put(be, x), put(be, w), put(be, b), put(be, t)
    loss, lse = be.linear_cross_entropy(X, W, B, T)
    within(get(be, lse), ex["lse"], tlse, "lse")
    within(get(be, loss), np.array([ex["loss"]]), tloss, "loss")
    dx, dw, db = be.linear_cross_entropy_bwd(X, W, B, T, put(be, ex["lse"].astype(np.float32)))
    within(get(be, dx), ex["dx"], tdx + 1e-45, "dx")
    within(get(be, dw), ex["dw"], tdw + 1e-45, "dw")
    within(get(be, db), ex["db"], tdb, "dbias")


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("R", [5, 40])
def test_linear_cross_entropy_masked_and_empty_rows(backend, R, dtype):
    """Vocabulary entries masked by a bias of -inf or the lowest value, no row with a target, non-finite rows."""
    be = backend
    D, V = 48, 205
    x, w, b, t = ce_inputs(R, D, V, dtype, True, 0.0, 3)
    b[10:40], b[100:204] = -np.inf, np.finfo(np.float32).min
    t[:] = np.where((t >= 10) & (t < 40) | (t >= 100), 3, t)
    with np.errstate(all="ignore"):
        ex, live = ce_exact(x, w, b, t), t != IGNORE
    z = ex["z"].copy()
    keep = np.isfinite(b) & (b > -1e30)
    sub = ce_exact(x, w[:, keep], b[keep], np.searchsorted(np.flatnonzero(keep), t).astype(np.float32))
    tl, tloss, tdx, _, _ = ce_bounds(x, w[:, keep], b[keep], dtype, sub, live)
    X, W, B, T = put(be, x, dtype), put(be, w, dtype), put(be, b), put(be, t)
    loss, lse = be.linear_cross_entropy(X, W, B, T)
    within(get(be, lse), sub["lse"], tl, "lse")
    within(get(be, loss), np.array([sub["loss"]]), tloss, "loss")
    dx, dw, db = (get(be, s) for s in be.linear_cross_entropy_bwd(X, W, B, T, lse))
    within(dx, sub["dx"], tdx + 2e-5 * np.abs(sub["dx"]).max(), "dx")   # lse of the forward pass instead of the exact one
    assert not dw[:, 10:40].any() and not dw[:, 100:204].any() and not db[10:40].any() and np.isfinite(dw).all()
    # no row has a target: loss 0, all gradients 0
    T0 = put(be, np.full(R, IGNORE, np.float32))
    loss, lse0 = be.linear_cross_entropy(X, W, B, T0)
    assert be.to_vec(loss)[0] == 0 and np.array_equal(be.to_vec(lse0), be.to_vec(lse))
    assert not any(be.to_vec(s).any() for s in be.linear_cross_entropy_bwd(X, W, B, T0, lse0))
    # every entry masked: no distribution, the loss says so; the other rows of lse are untouched by a row of NaN
    allm = put(be, np.full(V, -np.inf, np.float32))
    loss, lsem = be.linear_cross_entropy(X, W, allm, T)
    assert np.isnan(be.to_vec(loss)[0]) and np.all(be.to_vec(lsem) == -np.inf)
    xn = x.copy()
    xn[1, 7] = np.nan
    tn = t.copy()
    tn[1] = IGNORE
    loss, lsen = be.linear_cross_entropy(put(be, xn, dtype), W, B, put(be, tn))
    got = be.to_vec(lsen)
    assert np.isnan(got[1]) and np.array_equal(np.delete(got, 1), np.delete(be.to_vec(lse), 1)) and np.isfinite(be.to_vec(loss)[0])
    dxn, _, _ = be.linear_cross_entropy_bwd(put(be, xn, dtype), W, B, put(be, tn), lsen)
    assert np.isfinite(np.delete(get(be, dxn), 1, 0)).all() and not get(be, dxn)[1].any()


@pytest.mark.parametrize("R", [6, 70])
def test_linear_cross_entropy_targets_and_refusals(backend, R):
    be = backend
    D, V = 24, 50
    x, w, b, t = ce_inputs(R, D, V, "f32", True, 0.0, 8)
    X, W, B, T = put(be, x), put(be, w), put(be, b), put(be, t)
    loss, lse = be.linear_cross_entropy(X, W, B, T)
    # an ignore_index that is a class, and ids that are not whole are truncated like other index inputs
    t0 = t.copy()
    t0[: R // 2] = 7
    ex = ce_exact(x, w, b, t0, ignore=7)
    assert abs(be.to_vec(be.linear_cross_entropy(X, W, B, put(be, t0), ignore_index=7)[0])[0] - ex["loss"]) < 1e-4
    assert np.array_equal(be.to_vec(be.linear_cross_entropy(X, W, B, put(be, t + 0.5))[0]), be.to_vec(loss))
    for bad in (-1.0, float(V), np.nan, np.inf, -np.inf, 1e30, -0.5):
        tb = t.copy()
        tb[R - 1] = bad
        TB = put(be, tb)
        with pytest.raises(rg.ShapeError):
            be.linear_cross_entropy(X, W, B, TB)
        with pytest.raises(rg.ShapeError):
            be.linear_cross_entropy_bwd(X, W, B, TB, lse)
    # the context works on
    assert np.array_equal(be.to_vec(be.linear_cross_entropy(X, W, B, T)[0]), be.to_vec(loss))
    # siblings agree: the loss over materialised logits
    z = be.add(be.matmul(X, W), be.reshape(B, [1, V]))
    assert abs(be.to_vec(be.sparse_cross_entropy(z, T))[0] - be.to_vec(loss)[0]) < 1e-4
    H = be.cast(X, "bf16")
    for call, err in ((lambda: be.linear_cross_entropy(H, W, B, T), rg.Unsupported),
                      (lambda: be.linear_cross_entropy(X, W, be.cast(B, "bf16"), T), rg.Unsupported),
                      (lambda: be.linear_cross_entropy(X, W, be.ones([V + 1]), T), rg.ShapeError),
                      (lambda: be.linear_cross_entropy(X, W, B, be.zeros([R + 1])), rg.ShapeError),
                      (lambda: be.linear_cross_entropy(X, be.zeros([D + 1, V]), B, T), rg.ShapeError),
                      (lambda: be.linear_cross_entropy(X, be.zeros([D, 0]), None, T), rg.ShapeError),
                      (lambda: be.linear_cross_entropy(be.zeros([2, 3, 4]), W, B, T), rg.DimensionError),
                      (lambda: be.linear_cross_entropy_bwd(X, W, B, T, be.zeros([R + 1])), rg.ShapeError),
                      (lambda: be.linear_cross_entropy_bwd(X, W, B, T, lse, be.zeros([2])), rg.ShapeError),
                      (lambda: be.linear_cross_entropy_bwd(X, W, B, T, be.cast(lse, "bf16")), rg.Unsupported)):
        with pytest.raises(err):
            call()
    loss0, lse0 = be.linear_cross_entropy(be.zeros([0, D]), W, B, be.zeros([0]))
    assert be.to_vec(loss0)[0] == 0 and lse0.shape == [0]
    dx, dw, db = be.linear_cross_entropy_bwd(be.zeros([0, D]), W, B, be.zeros([0]), lse0)
    assert dx.shape == [0, D] and not be.to_vec(dw).any() and not be.to_vec(db).any()


@pytest.mark.parametrize("R", [7, 33])
def test_linear_cross_entropy_gradient_against_differences(backend, R):
    be = backend
    D, V = 20, 31
    x, w, b, t = ce_inputs(R, D, V, "f32", True, 0.2, 21)
    X, W, B, T = put(be, x), put(be, w), put(be, b), put(be, t)
    _, lse = be.linear_cross_entropy(X, W, B, T)
    dx, dw, db = (get(be, s) for s in be.linear_cross_entropy_bwd(X, W, B, T, lse))
    rng = np.random.default_rng(2)
    for _ in range(3):
        vx, vw, vb = rng.standard_normal(x.shape), rng.standard_normal(w.shape), rng.standard_normal(b.shape)
        e = 1e-5
        num = (ce_exact(x + e * vx, w + e * vw, b + e * vb, t)["loss"] - ce_exact(x - e * vx, w - e * vw, b - e * vb, t)["loss"]) / (2 * e)
        ana = (dx * vx).sum() + (dw * vw).sum() + (db * vb).sum()
        # third derivatives O(1e2) e^2 = 1e-8, cancellation 2^-52 * 5 / e = 1e-10, f32 gradient relative 1e-5
        assert abs(num - ana) <= 1e-4 * (1 + abs(num))


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_linear_cross_entropy_over_pieces_of_the_vocabulary(backend, dtype):
    """Enough rows that the gradient goes over the vocabulary in pieces (512 MiB of dz): rows of zeros keep the oracle small."""
    be = backend
    D, V = 8, 2100
    R = 200000 if dtype == "bf16" else 70000
    live = 600
    x, w, b, t = ce_inputs(live, D, V, dtype, True, 0.1, 4)
    xf, tf = np.zeros((R, D), np.float32), np.full(R, IGNORE, np.float32)
    at = np.sort(np.random.default_rng(0).permutation(R)[:live])
    xf[at], tf[at] = x, t
    X, W, B, T = put(be, xf, dtype), put(be, w, dtype), put(be, b), put(be, tf)
    ex = ce_exact(x, w, b, t)
    tlse, tloss, tdx, tdw, tdb = ce_bounds(x, w, b, dtype, ex, t != IGNORE)
    loss, lse = be.linear_cross_entropy(X, W, B, T)
    within(get(be, lse)[at], ex["lse"], tlse, "lse")
    within(get(be, loss), np.array([ex["loss"]]), tloss, "loss")
    dx, dw, db = (get(be, s) for s in be.linear_cross_entropy_bwd(X, W, B, T, lse))
    slack = 1e-5          # lse of the forward pass instead of the exact one: |p| (tlse) <= 1e-5 of each term
    within(dx[at], ex["dx"], tdx + slack * ex["scale"] * (ex["p"] @ np.abs(w.astype(np.float64)).T), "dx")
    within(dw, ex["dw"], tdw + slack * ex["scale"] * (np.abs(x.astype(np.float64)).T @ ex["p"]), "dw")
    # 200000 rows: their dz is 0, the chains of the column sums are longer than the live rows' only by exact additions of 0
    within(db, ex["db"], tdb + slack * ex["scale"] * ex["p"].sum(0), "dbias")
    gone = np.ones(R, bool)
    gone[at] = False
    assert not dx[gone].any()


def test_linear_cross_entropy_of_few_rows_over_pieces_of_the_vocabulary(backend):
    """So wide a vocabulary that a few hundred rows go over it in pieces: dx is summed over both."""
    torch = pytest.importorskip("torch")
    be = backend
    R, D, V = 200, 256, 450000
    gen = torch.Generator(device="cuda").manual_seed(5)
    x = torch.randn(R, D, device="cuda", generator=gen)
    w = torch.randn(D, V, device="cuda", generator=gen) * 2.5 / D ** 0.5
    t = torch.randint(0, V, (R,), device="cuda", generator=gen).float()
    z = x.double() @ w.double()
    exact = torch.logsumexp(z, -1)
    p = torch.exp(z - exact[:, None])
    dz = p.clone()
    dz[torch.arange(R), t.long()] -= 1
    torch.cuda.synchronize()
    X, W, T = be.from_device(x), be.from_device(w), be.from_device(t)
    L = put(be, exact.cpu().numpy().astype(np.float32))
    dx, dw, _ = be.linear_cross_entropy_bwd(X, W, None, T, L)
    # as ce_bounds has it: a logit's error is max(D / 8 + 8, 2 * 18 + 4 + D / 256) half steps of the magnitudes, the chain over
    # the vocabulary 2 * 18 + 4 + V / 256
    mags = x.double().abs() @ w.double().abs()
    edz = p * ((41 * mags + 3 * (z.abs() + exact.abs()[:, None])) * E32 + 4 * E32) * 1.01 + E32 * dz.abs()
    ez = edz + 2.0 ** -21 * dz.abs()
    tdx = (ez + (40 + V / 256) * E32 * dz.abs()) @ w.double().abs().T / R
    ex = dz @ w.double().T / R
    got = torch.from_numpy(get(be, dx)).cuda()
    assert bool(((got - ex).abs() <= tdx + 4 * E32 * ex.abs() + 1e-45).all())
    tdw = x.double().abs().T @ (ez + 41 * E32 * dz.abs()) / R
    exw = x.double().T @ dz / R
    got = torch.from_numpy(be.to_vec(dw).reshape(D, V)).cuda().double()
    assert bool(((got - exw).abs() <= tdw + 4 * E32 * exw.abs() + 1e-45).all())


def test_linear_cross_entropy_gives_the_same_bits_again(backend):
    be = backend
    for R in (9, 500):
        x, w, b, t = ce_inputs(R, 100, 3001, "f32", True, 0.1)
        X, W, B, T = put(be, x), put(be, w), put(be, b), put(be, t)
        loss, lse = be.linear_cross_entropy(X, W, B, T)
        first = [be.to_vec(s) for s in (loss, lse, *be.linear_cross_entropy_bwd(X, W, B, T, lse))]
        for _ in range(3):
            loss, lse2 = be.linear_cross_entropy(X, W, B, T)
            again = [be.to_vec(s) for s in (loss, lse2, *be.linear_cross_entropy_bwd(X, W, B, T, lse))]
            assert all(np.array_equal(p, q) for p, q in zip(first, again))


# ---------------------------------------------------------------------------------------------------------------------
# together
# ---------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("rows", [12, 96])
def test_training_step_behind_the_last_block(backend, rows, dtype):
    """Final LayerNorm -> LM head with its loss -> gradients -> clipping of all of them, as WasmGptTrainer::train_step runs them,
    against the formulas in 64 bits, and against differences of the whole loss."""
    be = backend
    D, V, max_norm = 64, 333, 0.05
    h, _, g, b = ln_inputs(rows, D, dtype, 40)
    _, w, bias, t = ce_inputs(rows, D, V, dtype, True, 0.25, 41)
    H, W, G, B, BI, T = put(be, h, dtype), put(be, w, dtype), put(be, g), put(be, b), put(be, bias), put(be, t)
    y, mean, rstd = be.layer_norm_fwd(H, G, B, EPS)
    loss, lse = be.linear_cross_entropy(y, W, BI, T)
    dy, dw, dbias = be.linear_cross_entropy_bwd(y, W, BI, T, lse)
    dh, dg, db = be.layer_norm_bwd(dy, H, G, mean, rstd)
    clipped, norm = be.clip_grad_norm([dh, dg, db, dw, dbias], max_norm)

    def total(h_, g_, b_, w_, bi_):
        return ce_exact(ln_exact(h_, g_, b_)[0], w_, bi_, t)["loss"]

    wy, wm, wr = ln_exact(h, g, b)
    ex = ce_exact(wy, w, bias, t)
    xh = (h - wm) * wr
    a = ex["dx"] * g
    want = [wr * (a - a.mean(-1, keepdims=True) - xh * (a * xh).mean(-1, keepdims=True)), (ex["dx"] * xh).sum(0, keepdims=True),
            ex["dx"].sum(0, keepdims=True), ex["dw"], ex["db"]]
    # every step rounds its matrices to dtype: y, dz, dx, dw by half a step each, and each of them reaches the gradients once
    tol = 8 * U[dtype] + 2e-5
    assert abs(get(be, loss)[0] - ex["loss"]) <= tol * (1 + np.abs(ex["z"]).max())
    for got, exact, name in zip((dh, dg, db, dw, dbias), want, ("dh", "dgamma", "dbeta", "dw", "dbias")):
        e = np.linalg.norm(get(be, got).reshape(exact.shape) - exact) / np.linalg.norm(exact)
        assert e <= tol * (1 + np.abs(ex["z"]).max()), (name, e)
    n = np.sqrt(sum((e ** 2).sum() for e in want))
    assert n > max_norm and abs(get(be, norm)[0] / n - 1) <= tol * (1 + np.abs(ex["z"]).max())
    sq = sum((get(be, c) ** 2).sum() for c in clipped)
    assert abs(np.sqrt(sq) / max_norm - 1) <= 2 * U[dtype] + 1e-6
    rng = np.random.default_rng(5)
    v = [rng.standard_normal(p.shape) for p in (h, g, b, w, bias)]
    e = 1e-5
    num = (total(*[p + e * q for p, q in zip((h, g, b, w, bias), v)]) - total(*[p - e * q for p, q in zip((h, g, b, w, bias), v)])) / (2 * e)
    ana = sum((get(be, got).reshape(q.shape) * q).sum() for got, q in zip((dh, dg, db, dw, dbias), v))
    size = sum(np.abs(x * q).sum() for x, q in zip(want, v))
    assert abs(num - ana) <= tol * (1 + np.abs(ex["z"]).max()) * size / 10 + 1e-6


@pytest.mark.parametrize("shared", [True, False])
def test_calls_from_several_threads(backend, shared):
    """Three threads with the forms of all sizes, on one context (its calls take turns) and on one each (their kernels share
    the GPU): every result has the bits of the call alone."""
    import threading
    shapes = [(3, 130, 2001, "f32"), (40, 130, 2001, "f32"), (40, 130, 2001, "bf16"), (300, 130, 2001, "f32"), (300, 136, 2000, "bf16")]

    def run(be, order):
        out = {}
        for k in order:
            R, D, V, dtype = shapes[k]
            x, w, b, t = ce_inputs(R, D, V, dtype, True, 0.1, k)
            X, W, B, T = put(be, x, dtype), put(be, w, dtype), put(be, b), put(be, t)
            loss, lse = be.linear_cross_entropy(X, W, B, T)
            dx, dw, db = be.linear_cross_entropy_bwd(X, W, B, T, lse)
            y, m, r = be.layer_norm_fwd(dx, be.ones([D]), be.zeros([D]), EPS)
            clipped, norm = be.clip_grad_norm([dw, db, y], 1e-3)
            out[k] = [be.to_vec(s) for s in (loss, lse, dx, dw, db, y, m, r, norm, *clipped)]
        return out

    alone = run(backend, range(len(shapes)))
    got, backends = [None] * 3, [backend if shared else rg.B200Backend(0) for _ in range(3)]

    def work(i):
        got[i] = [run(backends[i], [(k + 2 * i) % len(shapes) for k in range(len(shapes))]) for _ in range(4)]

    threads = [threading.Thread(target=work, args=(i,)) for i in range(3)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for rounds in got:
        for out in rounds:
            for k, want in alone.items():
                assert all(np.array_equal(a, b, equal_nan=True) for a, b in zip(out[k], want)), shapes[k]


@pytest.mark.parametrize("R,dtype", [(3, "f32"), (20, "f32"), (200, "f32"), (3, "bf16"), (20, "bf16"), (200, "bf16")])
def test_linear_cross_entropy_beyond_32_bits(R, dtype):
    """A matrix of more than 2^31 values: the logits, dz and gradients of its last columns."""
    import torch
    torch.cuda.set_device(0)
    stream = torch.cuda.current_stream()
    be = rg.B200Backend(0, stream=stream.cuda_stream)
    D, V, step = 180, 12000001, 1 << 20
    assert D * V > 2 ** 31
    gen = torch.Generator(device="cuda").manual_seed(R)
    kind = torch.float32 if dtype == "f32" else torch.bfloat16
    w = torch.empty(D, V, device="cuda", dtype=kind)
    for v in range(0, V, step):
        w[:, v:v + step] = torch.randn(D, min(step, V - v), device="cuda", generator=gen) * (2.5 / D ** 0.5)
    x = torch.randn(R, D, device="cuda", generator=gen).to(kind)
    t = (V - 1 - torch.randint(0, 1000, (R,), device="cuda", generator=gen)).float()
    pieces, xd = [], x.double()
    mags = torch.zeros(R, device="cuda", dtype=torch.float64)
    for v in range(0, V, step):
        wd = w[:, v:v + step].double()
        pieces.append(torch.logsumexp(xd @ wd, -1))
        mags = torch.maximum(mags, (xd.abs() @ wd.abs()).amax(-1))
    exact = torch.logsumexp(torch.stack(pieces), 0)
    X, W, T = be.from_device(x), be.from_device(w), be.from_device(t)
    loss, lse = be.linear_cross_entropy(X, W, None, T)
    # as ce_bounds has it, with the partial sums of the slices (at least 64 columns) in 32 chains
    steps = max(2 * (D / 16 + 2) if dtype == "bf16" else 40 + D / 256, D / 8 + 8)
    tol = steps * E32 * mags + (300 + V / 64 / 32) * E32 + 4 * E32 * (exact.abs() + 1)
    got = torch.from_dlpack(lse).double()
    assert bool(((got - exact).abs() <= tol).all())
    wt = w[:, t.long()].double()
    assert abs(torch.from_dlpack(loss).item() - (exact - (xd * wt.T).sum(-1)).mean().item()) <= 2 * tol.max().item()
    dx, dw, _ = be.linear_cross_entropy_bwd(X, W, None, T, be.from_device(exact.float()))
    tail = 5000
    wd = w[:, V - tail:].double()
    z = xd @ wd
    p = torch.exp(z - exact[:, None])
    dz = p.clone()
    dz[torch.arange(R), (t.long() - (V - tail))] -= 1
    edz = p * (steps * E32 * (xd.abs() @ wd.abs()) + 3 * E32 * (z.abs() + exact.abs()[:, None]) + 4 * E32) * 1.01 + E32 * dz.abs()
    ez = edz + (2.0 ** -21 if dtype == "f32" else U["bf16"] * 1.01) * dz.abs()
    want = xd.T @ dz / R
    tol = xd.abs().T @ (ez + (40 + R / 8) * E32 * dz.abs()) / R
    got = torch.from_dlpack(dw)[:, V - tail:].double()
    assert bool(((got - want).abs() <= tol + (U[dtype] + 3 * E32) * (want.abs() + tol) + 1e-45).all())
    # dx: the targets' columns, all of them at the end, carry nearly all of it; the rest are 12 million tiny terms
    want, bound = dz @ wd.T, (ez + (40 + V / 16) * E32 * dz.abs()) @ wd.abs().T
    for v in range(0, V - tail, step):
        wd = w[:, v:min(v + step, V - tail)].double()
        p = torch.exp(xd @ wd - exact[:, None])
        e = (steps + 40 + V / 16) * E32 * p * (1 + mags[:, None] + exact.abs()[:, None]) + (2.0 ** -21 if dtype == "f32" else U["bf16"] * 1.01) * p
        want, bound = want + p @ wd.T, bound + e @ wd.abs().T
    got, want, bound = torch.from_dlpack(dx).double(), want / R, bound / R
    assert bool(((got - want).abs() <= bound + (U[dtype] + 3 * E32) * (want.abs() + bound) + 1e-45).all())
    # and the same call gives the first columns too: bf16 rounds dz and dw by 2^-8 each, the exponentials are off by less than 1 %
    z = xd @ w[:, :64].double()
    want = xd.T @ torch.exp(z - exact[:, None]) / R
    assert bool((torch.from_dlpack(dw)[:, :64].double() - want).abs().max() <= 0.02 * want.abs().max())


def test_rows_and_tensors_beyond_32_bits():
    import torch
    torch.cuda.set_device(0)
    be = rg.B200Backend(0, stream=torch.cuda.current_stream().cuda_stream)
    rows, n, last = 140000, 16000, 4
    assert rows * n > 2 ** 31
    x = torch.zeros(rows, n, device="cuda", dtype=torch.bfloat16)
    dy = torch.zeros(rows, n, device="cuda", dtype=torch.bfloat16)
    gen = torch.Generator(device="cuda").manual_seed(1)
    x[-last:] = torch.randn(last, n, device="cuda", generator=gen).bfloat16()
    dy[-last:] = torch.randn(last, n, device="cuda", generator=gen).bfloat16()
    g = torch.randn(n, device="cuda", generator=gen)
    G, B = be.from_device(g), be.from_device(torch.zeros(n, device="cuda"))

    def step(x, dy):
        X, DY = be.from_device(x), be.from_device(dy)
        y, m, r = be.layer_norm_fwd(X, G, B, EPS)
        return [torch.from_dlpack(s) for s in (y, m, r, *be.layer_norm_bwd(DY, X, G, m, r))]

    big, small = step(x, dy), step(x[-last:], dy[-last:])
    assert all(torch.equal(a[-last:], b) for a, b in zip(big[:4], small[:4]))
    # rows of zeros add nothing to the column sums; the order of the others' additions may differ
    assert all(torch.allclose(a, b, rtol=0, atol=8 * E32 * float(dy.abs().max() * 6 * last)) for a, b in zip(big[4:], small[4:]))
    clipped, norm = be.clip_grad_norm([be.from_device(x)], 1.0)
    exact = x[-last:].double().norm().item()
    assert abs(torch.from_dlpack(norm).item() / exact - 1) <= 2 * E32
    got, want = torch.from_dlpack(clipped[0]), x[-last:].double() / exact
    assert bool(((got[-last:].double() - want).abs() <= (U["bf16"] + 3 * E32) * want.abs() + 1e-40).all()) and not bool(got[:last].any())


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("R", [1, 3, 8])
@pytest.mark.parametrize("D,V", [(2, 1), (3, 1), (5, 1), (9, 1), (5, 2), (10, 3), (1026, 1), (1025, 2), (1, 3)])
def test_linear_cross_entropy_of_few_rows_and_classes(backend, R, D, V, dtype):
    """Vocabularies narrower than a read of w: several of the last rows end past the matrix."""
    ce_check(backend, R, D, V, dtype, bias=R != 3, dloss=0.5)


# Inputs that took a form for some rows when their tests were written, for the tiles of many rows too.
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("R", [200, 300])
def test_linear_cross_entropy_masked_and_empty_rows_of_many(backend, R, dtype):
    test_linear_cross_entropy_masked_and_empty_rows(backend, R, dtype)


@pytest.mark.parametrize("R", [200, 300])
def test_linear_cross_entropy_refusals_and_differences_of_many(backend, R):
    test_linear_cross_entropy_targets_and_refusals(backend, R)
    test_linear_cross_entropy_gradient_against_differences(backend, R)


def ce_one_large_value(be, R, D, V, dtype, kind, size):
    """One large weight whose products count for nothing: every other logit keeps its digits.  The oracle leaves out the class
    that has no probability (a bias of -inf, or a logit of -size: exp of it is 0 in 64 bits too)."""
    x, w, b, t = ce_inputs(R, D, V, dtype, True, 0.1, 9)
    d0, v0, r0 = 5, 31 % V, R // 2
    t[t == v0] = (v0 + 1) % V
    big = rounded(np.array([size], np.float32), dtype)[0]
    if kind == "dead channel":
        x[:, d0], w[d0, v0] = 0, big
    elif kind == "masked class":
        x[:, d0], w[d0, v0], b[v0] = 1, big, -np.inf
    elif kind == "class switched off":
        x[:, d0], w[d0, v0] = 1, -big
    else:
        assert kind == "dead row of w"
        x[r0, d0], w[d0] = big, 0
    keep = np.ones(V, bool)
    keep[v0] = kind not in ("masked class", "class switched off")
    sub = np.cumsum(keep) - 1
    ts = np.where(t == IGNORE, IGNORE, sub[np.where(t == IGNORE, 0, t).astype(int)]).astype(np.float32)
    wk, bk, live = w[:, keep], b[keep], t != IGNORE
    ex = ce_exact(x, wk, bk, ts)
    tlse, tloss, tdx, tdw, tdb = ce_bounds(x, wk, bk, dtype, ex, live)
    X, W, B, T = put(be, x, dtype), put(be, w, dtype), put(be, b), put(be, t)
    loss, lse = be.linear_cross_entropy(X, W, B, T)
    within(get(be, lse), ex["lse"], tlse, "lse")
    within(get(be, loss), np.array([ex["loss"]]), tloss, "loss")
    dx, dw, db = be.linear_cross_entropy_bwd(X, W, B, T, put(be, ex["lse"].astype(np.float32)))
    within(get(be, dx), ex["dx"], tdx + 1e-45, "dx")
    within(get(be, dw)[:, keep], ex["dw"], tdw + 1e-45, "dw")
    within(get(be, db)[keep], ex["db"], tdb + 1e-45, "dbias")
    if not keep.all():
        assert not get(be, dw)[:, ~keep].any() and not get(be, db)[~keep].any()


@pytest.mark.parametrize("kind", ["dead channel", "masked class", "class switched off", "dead row of w"])
@pytest.mark.parametrize("dtype,R", [("f32", 6), ("f32", 70), ("f32", 200), ("f32", 300), ("bf16", 300)])
@pytest.mark.parametrize("size", [1e4, 1e6, 1e8, 1e12, 1e30])
def test_linear_cross_entropy_with_one_large_value(backend, R, dtype, kind, size):
    ce_one_large_value(backend, R, 64, 1000, dtype, kind, size)


@pytest.mark.parametrize("R,D,V", [(193, 8, 5), (257, 100, 1000), (500, 64, 129), (1000, 40, 2049), (300, 700, 385)])
def test_linear_cross_entropy_on_both_sides_of_the_range_rule(backend, R, D, V):
    """Just below and just above D max|x| max|w| = 2^22, where the products of f32 change from pairs to triples."""
    be = backend
    x, w, b, t = ce_inputs(R, D, V, "f32", True, 0.1, 12)
    for factor in (0.98, 1.02):
        ce_one_large_value(be, R, D, V, "f32", "dead channel", factor * 2.0 ** 22 / D / np.abs(np.delete(x, 5, 1)).max())


def test_linear_cross_entropy_scales_of_many_rows_and_columns(backend):
    """As test_linear_cross_entropy_scales_of_rows_and_columns, at 300 rows, with rows and columns whose scales differ by 2^12, and
    by 2^40 where only one side of a product is far from 1."""
    be = backend
    R, D, V = 300, 200, 300
    for spread in (6, 20):
        x, w, b, t = ce_inputs(R, D, V, "f32", True, 0.1, 77)
        x *= 1e-15 * 2.0 ** np.random.default_rng(1).integers(-spread, spread + 1, (R, 1))
        x[:, 3] *= 1000
        w *= 1e15 * 2.0 ** np.random.default_rng(2).integers(-spread, 1, (1, V))
        w[3] *= 1e-3
        w[:, 17], x[5] = 0, 0
        x, w = x.astype(np.float32), w.astype(np.float32)
        w *= np.float32(20 / np.abs(x.astype(np.float64) @ w).max())
        ex, live = ce_exact(x, w, b, t), t != IGNORE
        tlse, tloss, tdx, tdw, tdb = ce_bounds(x, w, b, "f32", ex, live)
        # pairs add up to 2^-38 D max|x| max|w| to a logit
        off = 2.0 ** -38 * D * float(np.abs(x).max()) * float(np.abs(w).max())
        off = off if off <= 2.0 ** -16 else 0.0
        more = off * ex["scale"] * live[:, None] * ex["p"]
        X, W, B, T = put(be, x), put(be, w), put(be, b), put(be, t)
        loss, lse = be.linear_cross_entropy(X, W, B, T)
        within(get(be, lse), ex["lse"], tlse + off, "lse")
        within(get(be, loss), np.array([ex["loss"]]), tloss + 2 * off, "loss")
        dx, dw, db = be.linear_cross_entropy_bwd(X, W, B, T, put(be, ex["lse"].astype(np.float32)))
        within(get(be, dx), ex["dx"], tdx + 1.01 * more @ np.abs(w.astype(np.float64)).T + 1e-45, "dx")
        within(get(be, dw), ex["dw"], tdw + 1.01 * np.abs(x.astype(np.float64)).T @ more + 1e-45, "dw")
        within(get(be, db), ex["db"], tdb + 1.01 * more.sum(0), "dbias")


def test_linear_cross_entropy_with_one_large_value_over_pieces(backend):
    """The triples of f32 where the gradient goes over pieces of the vocabulary (512 MiB of dz)."""
    be = backend
    R, D, V = 70000, 8, 2100
    rng = np.random.default_rng(6)
    keep = np.sort(rng.permutation(R)[:300])
    x, w, b, t = ce_inputs(300, D, V, "f32", True, 0.1, 14)
    x[:, 5], w[5, [3, 1300, 2099]] = 0, 1e10
    xf, tf = np.zeros((R, D), np.float32), np.full(R, IGNORE, np.float32)
    xf[keep], tf[keep] = x, t
    ex = ce_exact(x, w, b, t)
    tlse, tloss, tdx, tdw, tdb = ce_bounds(x, w, b, "f32", ex, t != IGNORE)
    X, W, B, T = put(be, xf), put(be, w), put(be, b), put(be, tf)
    loss, lse = be.linear_cross_entropy(X, W, B, T)
    within(get(be, lse)[keep], ex["lse"], tlse, "lse")
    within(get(be, loss), np.array([ex["loss"]]), tloss, "loss")
    L = np.zeros(R, np.float32)
    L[keep] = ex["lse"]
    dx, dw, db = (get(be, s) for s in be.linear_cross_entropy_bwd(X, W, B, T, put(be, L)))
    within(dx[keep], ex["dx"], tdx + 1e-45, "dx")
    within(dw, ex["dw"], tdw + 1e-45, "dw")
    within(db, ex["db"], tdb + 1e-45, "dbias")
    assert not np.delete(dx, keep, 0).any()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_clip_grad_norm_only_measures_with_an_infinite_maximum(backend, dtype):
    """Overflowed gradients are measured, not destroyed; a NaN still shows everywhere."""
    be = backend
    a = rounded(np.random.default_rng(0).standard_normal(9000), dtype)
    b = rounded(np.array([1.0, -2.0, 3e38], np.float32), dtype)
    for bad in (np.inf, -np.inf, None):
        a[8500] = bad if bad is not None else 1
        out, norm = be.clip_grad_norm([put(be, a, dtype), put(be, b, dtype)], float("inf"))
        n = be.to_vec(norm)[0]
        assert np.isinf(n) if bad is not None else abs(n / np.sqrt((a.astype(np.float64) ** 2).sum() + (b.astype(np.float64) ** 2).sum()) - 1) < 2 * E32
        assert all(np.array_equal(be.to_vec(o), v) for o, v in zip(out, (a, b)))
    a[3] = np.nan
    out, norm = be.clip_grad_norm([put(be, a, dtype), put(be, b, dtype)], float("inf"))
    assert np.isnan(be.to_vec(norm)[0]) and np.isnan(be.to_vec(out[0])).all() and np.isnan(be.to_vec(out[1])).all()


def test_an_exported_tensor_is_never_an_unasked_alias():
    import torch
    torch.cuda.set_device(0)
    be = rg.B200Backend(0, stream=torch.cuda.current_stream().cuda_stream)
    st = be.ones([4])
    with pytest.raises(BufferError):
        torch.from_dlpack(st, copy=True)
    with pytest.raises(BufferError):
        st.__dlpack__(dl_device=(1, 0))
    try:
        there = torch.from_dlpack(st, device="cpu")      # a consumer may move the values itself
        assert there.device.type == "cpu" and there.tolist() == [1, 1, 1, 1]
    except BufferError:
        pass
    mine = torch.from_dlpack(st).clone()
    mine.add_(1)
    assert np.array_equal(be.to_vec(st), np.ones(4, np.float32)) and torch.equal(torch.from_dlpack(st, copy=False), mine - 1)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_linear_cross_entropy_gradient_scratch(backend, dtype):
    """No scratch grows with rows times vocabulary: beside 512 MiB of dz, only what grows with one of them.  dbias comes out of
    every piece."""
    rt, driver = pytest.importorskip("cuda.bindings.runtime"), pytest.importorskip("cuda.bindings.driver")
    be = backend
    R, D, V = 300000, 8, 20003
    x, w, b, t = ce_inputs(400, D, V, dtype, True, 0.1, 4)
    xf, tf = np.zeros((R, D), np.float32), np.full(R, IGNORE, np.float32)
    at = np.sort(np.random.default_rng(0).permutation(R)[:400])
    xf[at], tf[at] = x, t
    L, ex = np.zeros(R, np.float32), ce_exact(x, w, b, t)
    L[at] = ex["lse"]
    X, W, B, T, LS = put(be, xf, dtype), put(be, w, dtype), put(be, b), put(be, tf), put(be, L)
    be.synchronize()
    err, pool = rt.cudaDeviceGetDefaultMemPool(0)
    high, used = rt.cudaMemPoolAttr.cudaMemPoolAttrUsedMemHigh, rt.cudaMemPoolAttr.cudaMemPoolAttrUsedMemCurrent
    before = int(rt.cudaMemPoolGetAttribute(pool, used)[1])
    assert int(rt.cudaMemPoolSetAttribute(pool, high, driver.cuuint64_t(0))[0]) == 0
    _, dw, db = be.linear_cross_entropy_bwd(X, W, B, T, LS)
    be.synchronize()
    grown = int(rt.cudaMemPoolGetAttribute(pool, high)[1]) - before
    assert 256 << 20 <= grown <= (512 << 20) + R * D * 16 + D * V * 20 + (64 << 20), grown
    _, _, _, tdw, tdb = ce_bounds(x, w, b, dtype, ex, t != IGNORE)
    within(get(be, dw), ex["dw"], tdw + 1e-45, "dw")
    within(get(be, db), ex["db"], tdb + 1e-45, "dbias")


def test_one_step_on_two_streams_in_turn():
    """A backend per torch stream: every step is ordered with the inputs that its own stream made."""
    import torch
    torch.cuda.set_device(0)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    backends = [rg.B200Backend(0, stream=s.cuda_stream) for s in streams]
    g, b = torch.ones(1600, device="cuda"), torch.zeros(1600, device="cuda")
    torch.cuda.synchronize()
    got = []
    for k in range(8):
        s, be = streams[k % 2], backends[k % 2]
        with torch.cuda.stream(s):
            x = torch.zeros(4000, 1600, device="cuda")
            for _ in range(20):                            # the op must wait for these
                x.add_(torch.arange(1600, device="cuda") * (k + 1.0))
            y, mean, _ = be.layer_norm_fwd(be.from_device(x), be.from_device(g), be.from_device(b), EPS)
            got.append((k, torch.from_dlpack(mean) + 0, torch.from_dlpack(y)[-1] + 0))
    torch.cuda.synchronize()
    for k, mean, y in got:
        want = 20 * (k + 1.0) * 799.5                      # whole numbers: the sums are exact up to the last division
        assert bool(((mean - want).abs() <= 60 * 2.0 ** -24 * want).all()) and abs(y[-1].item() / (1599 - 799.5) * 461.8802 - 1) < 1e-3


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("R,D,V", [(3, 40, 300), (40, 40, 300), (300, 41, 300), (700, 768, 300)])
def test_linear_cross_entropy_overflowed_upstream_gradient(backend, R, D, V, dtype):
    """dloss of infinity or NaN: the rows without a target still have a gradient of 0, the others show it."""
    be = backend
    x, w, b, t = ce_inputs(R, D, V, dtype, True, 0.0, 2)
    t[::3] = IGNORE
    X, W, B, T = put(be, x, dtype), put(be, w, dtype), put(be, b), put(be, t)
    _, lse = be.linear_cross_entropy(X, W, B, T)
    for bad in (np.inf, -np.inf, np.nan):
        dx, dw, db = (be.to_array(s) for s in be.linear_cross_entropy_bwd(X, W, B, T, lse, put(be, np.array([bad], np.float32))))
        assert not dx[::3].any() and not np.isfinite(np.delete(dx, np.arange(0, R, 3), 0)).any()
        assert not np.isfinite(dw).all() and not np.isfinite(db).all()


def test_a_synchronise_waits_for_its_own_stream_only():
    import torch
    torch.cuda.set_device(0)
    side = torch.cuda.Stream()
    be = rg.B200Backend(0, stream=side.cuda_stream)
    be.to_vec(be.ones([3]))
    torch.cuda.synchronize()
    torch.cuda._sleep(2_000_000_000)            # about a second of the default stream
    assert np.array_equal(be.to_vec(be.ones([3])), np.ones(3, np.float32))
    be.synchronize()
    busy = not torch.cuda.default_stream().query()
    torch.cuda.synchronize()
    assert busy


def test_synchronising_calls_inside_a_capture_are_refused_and_leave_it_alone():
    import torch
    torch.cuda.set_device(0)
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        be = rg.B200Backend(0, stream=stream.cuda_stream)
        x = be.ones([5])
        a = torch.zeros(4, device="cuda")
        graph = torch.cuda.CUDAGraph()
        stream.synchronize()
        with torch.cuda.graph(graph, stream=stream):
            a.add_(1)
            for call in (be.synchronize, lambda: be.to_vec(x), be.close, lambda: be.from_slice([1.0], [1])):
                with pytest.raises(rg.Unsupported):
                    call()
            a.add_(1)
        graph.replay()
        stream.synchronize()
        assert a.tolist() == [2, 2, 2, 2] and np.array_equal(be.to_vec(x), np.ones(5, np.float32))
        del x
        be.close()
        be.close()


def test_a_wait_that_gave_up_is_reported_once():
    """The flag word of the bounded waits, raised as a wait that gave up would: the next synchronising call says so, once."""
    be = rg.B200Backend(0)
    x, w, b, t = ce_inputs(300, 40, 300, "f32", True, 0.1)
    args = [put(be, a) for a in (x, w, b, t)]
    want = be.to_vec(be.linear_cross_entropy(*args)[0])
    assert be._lib.rg_debug_hook(be._ctx, None, 1, 0) == 0
    loss, _ = be.linear_cross_entropy(*args)
    with pytest.raises(rg.DeviceTimeout):
        be.to_vec(loss)
    assert np.array_equal(be.to_vec(loss), want)
    be.synchronize()


def ce_norm_errors(be, R, D, V, dtype):
    x, w, b, t = ce_inputs(R, D, V, dtype, True, 0.1, 3)
    ex = ce_exact(x, w, b, t)
    X, W, B, T = put(be, x, dtype), put(be, w, dtype), put(be, b), put(be, t)
    _, lse = be.linear_cross_entropy(X, W, B, T)
    dx, dw, db = be.linear_cross_entropy_bwd(X, W, B, T, put(be, ex["lse"].astype(np.float32)))
    # dbias adds dz of both signs (p, and p - 1 in the target's row): an error relative to the terms is relative to the sum of
    # their magnitudes, which is larger than the sum
    terms = ex["scale"] * np.abs(ex["dz"]).sum(0)
    return {k: np.linalg.norm(get(be, g) - e) / np.linalg.norm(of) for k, g, e, of in
            (("lse", lse, ex["lse"], ex["lse"]), ("dx", dx, ex["dx"], ex["dx"]), ("dw", dw, ex["dw"], ex["dw"]), ("dbias", db, ex["db"], terms))}


@pytest.mark.parametrize("R,D,V", [(17, 8, 300), (64, 8, 300), (192, 8, 300), (64, 128, 300), (193, 128, 33), (600, 128, 300), (600, 1600, 33),
                                   (2500, 128, 33), (2500, 512, 300), (600, 128, 3000)])
def test_linear_cross_entropy_f32_keeps_f32(backend, R, D, V):
    """The norm of the error, which sums that are truncated in one direction would fill.  A probability has an argument z - lse
    of up to 16: lse rounded to f32, the difference, and its product with log2(e), each off by at most 2^-21 (2.8e-7 in the
    mean square, the last one times ln 2), and 2 steps of the exponential: 4.5e-7 together; the logit itself half of that.  Twice
    the sum of squares is 1e-6.  lse: the same over a logarithm of 4 to 9, an eighth."""
    e = ce_norm_errors(backend, R, D, V, "f32")
    assert e["dx"] <= 1e-6 and e["dw"] <= 1e-6 and e["dbias"] <= 1e-6 and e["lse"] <= 1.5e-7, e


@pytest.mark.parametrize("R,D,V", [(17, 768, 33), (17, 1600, 33), (64, 1600, 301), (300, 800, 72), (300, 9000, 33), (64, 9000, 301), (2500, 416, 96)])
def test_linear_cross_entropy_f32_results_of_bf16_inputs(backend, R, D, V):
    """lse and dbias are f32 whatever the matrices are, also for a wide D: accumulators of at most 768 (lse) and 384 of K (dbias), 48
    and 24 steps that truncate by half a step (2^-24) in the mean, of a partial sum that is half of the logit in the mean.  A
    logit of magnitude 2.5 is then off by 3.6e-6 and 1.8e-6: 1.4e-6 of lse, and 1.8e-6 of each term of dbias; 1e-6 for the
    arguments of the exponentials as in f32."""
    e = ce_norm_errors(backend, R, D, V, "bf16")
    assert e["lse"] <= 1.5e-6 and e["dbias"] <= 2.1e-6, e


# ---------------------------------------------------------------------------------------------------------------------
# memory that was something else before
# ---------------------------------------------------------------------------------------------------------------------
def poison(be):
    """What the context and the device's pool hand out next is full of NaN."""
    held = [be.from_slice(np.full(n, np.nan, np.float32), [n]) for size in range(9, 21) for n in [2 ** size // 4] for _ in range(24)]
    held += [be.from_slice(np.full(n << 18, np.nan, np.float32), [n << 18]) for n in (2, 3, 5, 8, 16, 32, 64) for _ in range(4)]
    be.synchronize()
    del held


def bits(be, storages):
    return [be.to_vec(s).copy() for s in storages if s is not None]


# (10, 8, 8548): the K axis of dx in 15 pieces where a vocabulary rounded up to whole tiles would have 16
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("R,D,V", [(10, 8, 8548), (23, 9, 8472), (12, 12, 12379), (16, 9, 8598), (300, 40, 5700), (3, 70, 5000), (5, 8, 2), (17, 8, 33), (64, 192, 97),
                                   (200, 100, 1000), (193, 60, 131), (511, 257, 775), (700, 768, 300), (1025, 40, 2049), (8000, 128, 97)])
def test_linear_cross_entropy_in_memory_of_nan(backend, R, D, V, dtype):
    """No result depends on what its scratch held before."""
    be = backend
    x, w, b, t = ce_inputs(R, D, V, dtype, True, 0.2, 1)
    ex = ce_exact(x, w, b, t)
    X, W, B, T, L = put(be, x, dtype), put(be, w, dtype), put(be, b), put(be, t), put(be, ex["lse"].astype(np.float32))
    _, _, tdx, tdw, tdb = ce_bounds(x, w, b, dtype, ex, t != IGNORE)
    for turn in range(2):
        poison(be)
        loss, lse = bits(be, be.linear_cross_entropy(X, W, B, T))
        poison(be)
        dx, dw, db = (get(be, s) for s in be.linear_cross_entropy_bwd(X, W, B, T, L))
        assert np.isfinite(loss).all() and np.isfinite(lse).all()
        within(dx, ex["dx"], tdx + 1e-45, "dx")
        within(dw, ex["dw"], tdw + 1e-45, "dw")
        within(db, ex["db"], tdb + 1e-45, "dbias")


def test_linear_cross_entropy_wide_values_in_memory_of_nan(backend):
    for R, D, V in ((200, 64, 1000), (300, 30, 8548), (193, 9, 8590)):
        poison(backend)
        ce_one_large_value(backend, R, D, V, "f32", "dead channel", 1e10)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_other_training_ops_in_memory_of_nan(backend, dtype):
    be = backend
    for rows, n in ((1, 1), (3, 7), (256, 192), (37, 1023), (650, 1600), (5, 4097), (2, 16386), (3000, 768)):
        x, dy, g, b = ln_inputs(rows, n, dtype)
        X, DY, G, B = put(be, x, dtype), put(be, dy, dtype), put(be, g), put(be, b)
        y, m, r = be.layer_norm_fwd(X, G, B, EPS)
        want = bits(be, (y, m, r, *be.layer_norm_bwd(DY, X, G, m, r), *be.clip_grad_norm([X, DY, G], 0.5)[0]))
        poison(be)
        y, m, r = be.layer_norm_fwd(X, G, B, EPS)
        poison(be)
        got = bits(be, (y, m, r, *be.layer_norm_bwd(DY, X, G, m, r), *be.clip_grad_norm([X, DY, G], 0.5)[0]))
        assert all(np.isfinite(a).all() and np.array_equal(a, b) for a, b in zip(got, want)), (rows, n)
    poison(be)
    assert np.array_equal(be.to_vec(be.cast(put(be, x, dtype), "f32")).reshape(x.shape), x)


def backlogged(call, room=[]):
    """`call` is enqueued behind work that lasts and empties the caches, so that all of its launches are there when the first one
    starts, and the first one has to fetch everything from memory."""
    import torch
    room[:] = room or [torch.empty(1 << 29, device="cuda")]
    for _ in range(3):
        room[0].fill_(0)
    return call()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("R,D,V", [(1, 64, 1000), (4, 64, 1000), (16, 96, 1003), (40, 64, 304), (150, 64, 301), (200, 64, 304), (300, 72, 304), (1390, 24, 152),
                                   (1243, 176, 232), (509, 480, 776), (476, 176, 184), (1500, 40, 1001)])
def test_linear_cross_entropy_enqueued_behind_other_work(R, D, V, dtype):
    """The launches of a call start behind one another early; none may read what the one before has not written.  In memory of NaN,
    with all launches waiting in the stream."""
    import torch
    torch.cuda.set_device(0)
    be = rg.B200Backend(0, stream=torch.cuda.current_stream().cuda_stream)
    x, w, b, t = ce_inputs(R, D, V, dtype, True, 0.2, 1)
    X, W, B, T = put(be, x, dtype), put(be, w, dtype), put(be, b), put(be, t)
    loss, lse = be.linear_cross_entropy(X, W, B, T)
    L = put(be, be.to_vec(lse))
    want = bits(be, (loss, lse)), bits(be, be.linear_cross_entropy_bwd(X, W, B, T, L))
    nan = torch.full((1 << 18,), float("nan"), device="cuda").bfloat16()
    N = {n: be.from_device(nan[:n]) for n in (128, 256, 512, 1024, 2048, 4096, 8192, 16384, 32768, 65536, 131072, 262144)}
    for turn in range(40):
        held = [be.cast(s, "f32") for s in N.values() for _ in range(8)]       # f32 NaN in buffers of every small size
        torch.cuda.synchronize()
        del held
        got = backlogged(lambda: be.linear_cross_entropy(X, W, B, T))
        assert all(np.array_equal(p, q) for p, q in zip(bits(be, got), want[0])), turn
        held = [be.cast(s, "f32") for s in N.values() for _ in range(8)]
        torch.cuda.synchronize()
        del held, got
        got = backlogged(lambda: be.linear_cross_entropy_bwd(X, W, B, T, L))
        assert all(np.array_equal(p, q) for p, q in zip(bits(be, got), want[1])), turn


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_other_training_ops_enqueued_behind_other_work(dtype):
    import torch
    torch.cuda.set_device(0)
    be = rg.B200Backend(0, stream=torch.cuda.current_stream().cuda_stream)
    nan = torch.full((1 << 18,), float("nan"), device="cuda").bfloat16()
    N = {n: be.from_device(nan[:n]) for n in (128, 256, 512, 1024, 2048, 4096, 8192, 16384, 32768, 65536, 131072, 262144)}
    for rows, n in ((1, 64), (256, 192), (40, 1023), (300, 1600), (5, 16400)):
        x, dy, g, b = ln_inputs(rows, n, dtype)
        X, DY, G, B = put(be, x, dtype), put(be, dy, dtype), put(be, g), put(be, b)
        y, m, r = be.layer_norm_fwd(X, G, B, EPS)

        def step():
            out = be.layer_norm_bwd(DY, X, G, m, r)
            clipped, norm = be.clip_grad_norm([X, DY, G, B], 0.5)
            return (*out, *clipped, norm)

        want = bits(be, step())
        for turn in range(20):
            held = [be.cast(s, "f32") for s in N.values() for _ in range(8)]
            torch.cuda.synchronize()
            del held
            assert all(np.array_equal(p, q) for p, q in zip(bits(be, backlogged(step)), want)), (rows, n, turn)
