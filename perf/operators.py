"""Cases for timing the training operators of the library beside their plain forms: LayerNorm forward with its saved
statistics and backward, the softmax cross entropy of a vocabulary projection without its logits (loss and gradients),
and clipping by the global gradient norm.  They are the steps of a GPT training step behind the last block: final
LayerNorm, LM head with its loss, their gradients, clipping of all gradients.

`run` takes device tensors and returns device tensors.  With `own` false it computes the operators with elementary torch
operations in 32 bits; with `own` true it calls the library through its Python mirror, on torch's current stream."""
import math

import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
IGNORE = -100
EPS = 1e-5


# ---------------------------------------------------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------------------------------------------------
def listed():
    return [
        # one sequence of 64 ids through the final LayerNorm: a call whose latency counts
        {"name": "ln_fwd 64x768 bf16", "op": "ln_fwd", "dtype": "bf16", "rows": 64, "dim": 768},
        # a training batch of 32 sequences of 1024 ids at the GPT-2-small width
        {"name": "ln_fwd 32768x768 f32", "op": "ln_fwd", "dtype": "f32", "rows": 32768, "dim": 768},
        # the crate's command-line model: width 192, 4 windows of 64 ids
        {"name": "ln_bwd 256x192 f32", "op": "ln_bwd", "dtype": "f32", "rows": 256, "dim": 192},
        # 16 sequences of 1024 ids at the GPT-2-XL width
        {"name": "ln_bwd 16384x1600 bf16", "op": "ln_bwd", "dtype": "bf16", "rows": 16384, "dim": 1600},
        # scoring one position of each of 8 sequences over the full vocabulary
        {"name": "ce 8x768x50257 f32", "op": "ce", "dtype": "f32", "rows": 8, "dim": 768, "vocab": 50257, "bias": True, "ignored": 0.0},
        # evaluation of 4 sequences of 1024 ids
        {"name": "ce 4096x768x50257 f32", "op": "ce", "dtype": "f32", "rows": 4096, "dim": 768, "vocab": 50257, "bias": True, "ignored": 0.0},
        # a padded evaluation batch in bf16, three rows of ten without a target
        {"name": "ce 8192x768x50257 bf16", "op": "ce", "dtype": "bf16", "rows": 8192, "dim": 768, "vocab": 50257, "bias": False, "ignored": 0.3},
        # training step of a character model (97 characters, width 192, one window of 64 ids)
        {"name": "ce_bwd 64x192x97 f32", "op": "ce_bwd", "dtype": "f32", "rows": 64, "dim": 192, "vocab": 97, "bias": True, "ignored": 0.0},
        # GPT-2-small shape, 2 sequences of 1024 ids, f32 weights
        {"name": "ce_bwd 2048x768x50257 f32", "op": "ce_bwd", "dtype": "f32", "rows": 2048, "dim": 768, "vocab": 50257, "bias": True, "ignored": 0.1},
        # GPT-2-XL shape, 4 sequences of 1024 ids, bf16 weights
        {"name": "ce_bwd 4096x1600x50257 bf16", "op": "ce_bwd", "dtype": "bf16", "rows": 4096, "dim": 1600, "vocab": 50257, "bias": False, "ignored": 0.0},
        # gradients of a character model of 3 blocks: 54 tensors, the largest of 148 thousand values
        {"name": "clip 54 tensors f32", "op": "clip", "dtype": "f32", "dim": 192, "vocab": 97, "layers": 3, "odd": 0, "scale": 1.0},
        # gradients of 2 blocks and both tables at the GPT-2-XL shape: 38 tensors, 223 million values, bf16 matrices
        {"name": "clip 38 tensors bf16", "op": "clip", "dtype": "bf16", "dim": 1600, "vocab": 50257, "layers": 2, "odd": 0, "scale": 0.001},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["ln_fwd", "ln_bwd", "ce", "ce_bwd", "ce", "ce_bwd", "clip"])
    dtype = rng.choice(["f32", "bf16"])
    if op in ("ln_fwd", "ln_bwd"):
        dim = rng.choice([_log(rng, 8, 12000), 128, 192, 768, 1600])
        return {"op": op, "dtype": dtype, "rows": min(_log(rng, 1, 32768), 25_000_000 // dim), "dim": dim}
    if op == "clip":
        # the parameter list of a GPT of any width; `odd` shifts sizes off the powers of two
        dim = _log(rng, 16, 900)
        return {"op": op, "dtype": dtype, "dim": dim, "vocab": _log(rng, 32, 50257), "layers": rng.choice([1, 2, 3]),
                "odd": rng.choice([0, 1, 3, 5]), "scale": rng.choice([1.0, 0.001, 1e-6])}
    dim = rng.choice([_log(rng, 8, 1600), 128, 192, 768])
    vocab = rng.choice([_log(rng, 2, 60000), 50257, 1024])
    rows = min(_log(rng, 1, 8192), int(1.2e11 / (dim * vocab)), int(4e8 / vocab))
    return {"op": op, "dtype": dtype, "rows": max(1, rows), "dim": dim, "vocab": vocab, "bias": rng.random() < 0.6,
            "ignored": rng.choice([0.0, 0.1, 0.5])}


def _clip_shapes(case):
    """The parameter shapes of a GPT in parameters() order; matrices carry the case's type, vectors f32."""
    d, v, o = case["dim"], case["vocab"], case["odd"]
    h = 4 * d
    block = [(d, d), (1, d)] * 4 + [(1, d), (1, d), (d, h + o), (1, h + o), (h, d + o), (1, d), (1, d), (1, d)]
    return [(v, d), (64, d)] + block * case["layers"] + [(1, d), (1, d), (d, v), (1, v)]


def work(case):
    e = 4 if case["dtype"] == "f32" else 2
    if case["op"] in ("ln_fwd", "ln_bwd"):
        r, d = case["rows"], case["dim"]
        if case["op"] == "ln_fwd":  # x, gamma, beta in; y and two statistics a row out
            return {"bytes": 2 * r * d * e + 8 * d + 8 * r, "flops": 8 * r * d}
        return {"bytes": 3 * r * d * e + 12 * d + 8 * r, "flops": 13 * r * d}
    if case["op"] == "clip":
        n = [(a * b, e if a > 1 else 4) for a, b in _clip_shapes(case)]
        return {"bytes": sum(2 * k * w for k, w in n) + 4, "flops": sum(3 * k for k, _ in n)}
    r, d, v = case["rows"], case["dim"], case["vocab"]
    b = 4 * v if case["bias"] else 0
    if case["op"] == "ce":  # one product, an exponential an element
        return {"bytes": (r * d + d * v) * e + b + 8 * r + 4, "flops": 2 * r * d * v + 4 * r * v}
    # the logits once more, and the products that give dx and dw
    return {"bytes": 2 * (r * d + d * v) * e + 2 * b + 8 * r + 4, "flops": 6 * r * d * v + 6 * r * v}


# ---------------------------------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------------------------------
def _residual(g, r, d):
    """Rows of a residual stream: a spread that differs from row to row, an offset, a few large channels."""
    x = torch.randn(r, d, generator=g, device="cuda") * (0.5 + torch.rand(r, 1, generator=g, device="cuda") * 3) + 0.3
    big = torch.randint(0, d, (max(1, d // 256),), generator=g, device="cuda")
    x[:, big] *= 8.0
    return x


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed * 7919 + 13)
    t = DTYPES[case["dtype"]]

    def normal(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    if case["op"] in ("ln_fwd", "ln_bwd"):
        r, d = case["rows"], case["dim"]
        s = {"x": _residual(g, r, d).to(t), "gamma": 1 + 0.2 * normal(1, d), "beta": 0.1 * normal(1, d)}
        if case["op"] == "ln_bwd":
            x = s["x"].double()
            s["mean"] = x.mean(-1).float()
            s["rstd"] = (1 / torch.sqrt(x.var(-1, unbiased=False) + EPS)).float()
            s["dy"] = (0.02 * normal(r, d)).to(t)
    elif case["op"] == "clip":
        s = {"grads": [(normal(a, b) * (case["scale"] * 10.0 ** (i % 3 - 1))).to(t if a > 1 else torch.float32)
                       for i, (a, b) in enumerate(_clip_shapes(case))], "max_norm": 1.0}
    else:
        r, d, v = case["rows"], case["dim"], case["vocab"]
        s = {"x": normal(r, d).to(t), "w": (normal(d, v) * (2.5 / math.sqrt(d))).to(t), "bias": 0.3 * normal(v) if case["bias"] else None}
        # ids of a text: small ids are frequent
        ids = ((torch.rand(r, generator=g, device="cuda") ** 3) * v).floor().clamp(0, v - 1)
        gone = torch.rand(r, generator=g, device="cuda") < case["ignored"]
        s["targets"] = torch.where(gone, torch.full_like(ids, IGNORE), ids)
        if case["op"] == "ce_bwd":
            s["lse"] = _row_lse(s["x"], s["w"], s["bias"])
            s["dloss"] = torch.full((1,), 0.25, device="cuda")  # four micro-batches share one step
    s["op"] = case["op"]
    return s


def _row_lse(x, w, bias):
    """What the forward pass saved: log of the sum of exponentials of each row of logits, from 64 bits, 512 rows at a time."""
    w, parts = w.double(), x.split(512)
    b = 0.0 if bias is None else bias.double()
    return torch.cat([torch.logsumexp(p.double() @ w + b, -1) for p in parts]).float()


# ---------------------------------------------------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------------------------------------------------
def run(state):
    if own:
        return _run_own(state)
    return {"ln_fwd": _ln_fwd, "ln_bwd": _ln_bwd, "ce": _ce, "ce_bwd": _ce_bwd, "clip": _clip}[state["op"]](state)


def _ln_fwd(s):
    x = s["x"].float()
    mean = x.mean(-1, keepdim=True)
    c = x - mean
    rstd = 1 / torch.sqrt((c * c).mean(-1, keepdim=True) + EPS)
    return {"y": (c * rstd * s["gamma"] + s["beta"]).to(s["x"].dtype), "mean": mean[:, 0], "rstd": rstd[:, 0]}


def _ln_bwd(s):
    x, dy = s["x"].float(), s["dy"].float()
    rstd = s["rstd"][:, None]
    xh = (x - s["mean"][:, None]) * rstd
    a = dy * s["gamma"]
    dx = rstd * (a - a.mean(-1, keepdim=True) - xh * (a * xh).mean(-1, keepdim=True))
    return {"dx": dx.to(s["x"].dtype), "dgamma": (dy * xh).sum(0, keepdim=True), "dbeta": dy.sum(0, keepdim=True)}


def _logits(s):
    z = s["x"].float() @ s["w"].float()
    return z if s["bias"] is None else z + s["bias"]


def _ce(s):
    z = _logits(s)
    m = z.amax(-1, keepdim=True)
    lse = (m + torch.log(torch.exp(z - m).sum(-1, keepdim=True)))[:, 0]
    live = s["targets"] != IGNORE
    at = torch.where(live, s["targets"], 0.0).long()
    rows = torch.where(live, lse - z.gather(1, at[:, None])[:, 0], 0.0)
    return {"loss": (rows.sum() / live.sum().clamp(min=1)).reshape(1), "lse": lse}


def _ce_bwd(s):
    live = s["targets"] != IGNORE
    at = torch.where(live, s["targets"], 0.0).long()
    p = torch.exp(_logits(s) - s["lse"][:, None])
    p.scatter_add_(1, at[:, None], torch.full_like(s["lse"], -1.0)[:, None])
    p *= (live * (s["dloss"] / live.sum().clamp(min=1)))[:, None]
    # a sum over the whole vocabulary is long for 32 bits: pieces of it are added in 64
    pieces = zip(p.split(4096, 1), s["w"].float().split(4096, 1))
    dx = torch.stack([a @ b.t() for a, b in pieces]).sum(0, dtype=torch.float64)
    out = {"dx": dx.to(s["x"].dtype), "dw": (s["x"].float().t() @ p).to(s["w"].dtype)}
    if s["bias"] is not None:
        out["dbias"] = p.sum(0)
    return out


def _clip(s):
    total = torch.stack([g.float().square().sum(dtype=torch.float64) for g in s["grads"]]).sum()
    norm = torch.sqrt(total).float()
    c = torch.clamp(s["max_norm"] / norm, max=1.0)
    return {"norm": norm.reshape(1), "grads": [(g.float() * c).to(g.dtype) for g in s["grads"]]}


# ---- the same through the library
_backends = {}  # one for each device and stream that was current in a call


def _run_own(s):
    where = torch.cuda.current_device(), torch.cuda.current_stream().cuda_stream
    if where not in _backends:
        import rustygradients_b200 as rg
        _backends[where] = rg.B200Backend(where[0], stream=where[1])
    be = _backends[where]

    def given(*names):
        return [None if s[n] is None else be.from_device(s[n]) for n in names]

    def tensor(st):
        return torch.utils.dlpack.from_dlpack(st.to_dlpack())

    if s["op"] == "ln_fwd":
        out = be.layer_norm_fwd(*given("x", "gamma", "beta"), EPS)
        return dict(zip(("y", "mean", "rstd"), map(tensor, out)))
    if s["op"] == "ln_bwd":
        out = be.layer_norm_bwd(*given("dy", "x", "gamma", "mean", "rstd"))
        return dict(zip(("dx", "dgamma", "dbeta"), map(tensor, out)))
    if s["op"] == "ce":
        out = be.linear_cross_entropy(*given("x", "w", "bias", "targets"), ignore_index=IGNORE)
        return dict(zip(("loss", "lse"), map(tensor, out)))
    if s["op"] == "ce_bwd":
        out = be.linear_cross_entropy_bwd(*given("x", "w", "bias", "targets", "lse", "dloss"), ignore_index=IGNORE)
        return {k: tensor(st) for k, st in zip(("dx", "dw", "dbias"), out) if st is not None}
    grads, norm = be.clip_grad_norm([be.from_device(g) for g in s["grads"]], s["max_norm"])
    return {"norm": tensor(norm), "grads": [tensor(g) for g in grads]}


# ---------------------------------------------------------------------------------------------------------------------
# 64 bits
# ---------------------------------------------------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    f = torch.nn.functional
    if case["op"] in ("ln_fwd", "ln_bwd"):
        x = s["x"].double().requires_grad_()
        gamma, beta = s["gamma"][0].double().requires_grad_(), s["beta"][0].double().requires_grad_()
        y = f.layer_norm(x, (case["dim"],), gamma, beta, EPS)
        if case["op"] == "ln_fwd":
            var, mean = torch.var_mean(x, -1, unbiased=False)
            return {"y": y.detach(), "mean": mean.detach(), "rstd": torch.rsqrt(var + EPS).detach()}
        dx, dg, db = torch.autograd.grad(y, (x, gamma, beta), s["dy"].double())
        return {"dx": dx, "dgamma": dg[None], "dbeta": db[None]}
    if case["op"] == "clip":
        flat = torch.cat([g.double().reshape(-1) for g in s["grads"]])
        norm = torch.linalg.vector_norm(flat)
        k = min(1.0, s["max_norm"] / float(norm))
        return {"norm": norm.reshape(1), "grads": [g.double() * k for g in s["grads"]]}
    x, w = s["x"].double().requires_grad_(), s["w"].double().requires_grad_()
    b = torch.zeros(case["vocab"], dtype=torch.float64, device="cuda") if s["bias"] is None else s["bias"].double()
    b.requires_grad_()
    z = torch.addmm(b, x, w)
    t = s["targets"].long()
    if case["op"] == "ce":
        loss = f.cross_entropy(z, t, ignore_index=IGNORE) if bool((t != IGNORE).any()) else z.sum() * 0
        return {"loss": loss.detach().reshape(1), "lse": torch.logsumexp(z, -1).detach()}
    loss = f.cross_entropy(z, t, ignore_index=IGNORE) if bool((t != IGNORE).any()) else z.sum() * 0
    grads = torch.autograd.grad(loss * s["dloss"].double()[0], (x, w, b))
    out = {"dx": grads[0], "dw": grads[1]}
    if s["bias"] is not None:
        out["dbias"] = grads[2]
    return out
