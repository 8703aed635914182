"""Host side of the training ops without a GPU: refusals of the C entries, and the number forms the tensor cores get."""
import ctypes as C
import os
import subprocess

import numpy as np
import pytest

from rustygradients_b200 import _lib, build

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
EXE = os.path.join(ROOT, "tests", "cpp", "train_mirror_test")


def test_null_arguments_are_refused_before_any_device_call():
    lib = _lib.load()
    p = C.c_void_p()
    ref = C.byref(p)
    calls = [lambda: lib.rg_cast(None, None, 0, ref), lambda: lib.rg_from_device(None, None, 0, None, 0, ref),
             lambda: lib.rg_to_dlpack(None, ref), lambda: lib.rg_layer_norm_fwd(None, None, None, None, 1e-5, ref, ref, ref),
             lambda: lib.rg_layer_norm_bwd(None, None, None, None, None, None, ref, ref, ref),
             lambda: lib.rg_linear_cross_entropy(None, None, None, None, None, -100, ref, ref),
             lambda: lib.rg_linear_cross_entropy_bwd(None, None, None, None, None, -100, None, None, ref, ref, ref),
             lambda: lib.rg_clip_grad_norm(None, None, 0, 1.0, None, ref), lambda: lib.rg_ctx_create_on_stream(0, None, None)]
    for call in calls:
        assert call() == _lib.RG_ERR_INVALID_INPUT and lib.rg_last_error()
    assert lib.rg_storage_dtype(None) == _lib.RG_DTYPE_F32 and lib.rg_storage_free(None) == _lib.RG_OK


def test_no_gpu_is_an_error_on_a_caller_stream_too():
    import rustygradients_b200 as rg
    if rg.B200Backend.device_count() > 0:
        pytest.skip("a GPU is present")
    with pytest.raises(rg.BackendError):
        rg.B200Backend(0, stream=0)


def test_dlpack_requests_that_an_alias_cannot_fulfil_are_refused():
    import rustygradients_b200.backend as B

    class Owner:
        _ctx, stream, device_index = None, 0, 1

    class Shared(B.Storage):
        def to_dlpack(self):
            return "capsule"

    st = Shared(Owner(), 0)
    assert st.__dlpack_device__() == (2, 1)
    for asked in ({}, {"stream": 1}, {"stream": -1}, {"copy": None}, {"copy": False}, {"dl_device": (2, 1), "max_version": (1, 0)}):
        assert st.__dlpack__(**asked) == "capsule"
    for asked in ({"copy": True}, {"dl_device": (1, 0)}, {"dl_device": (2, 0)}, {"stream": 5}):
        with pytest.raises(BufferError):
            st.__dlpack__(**asked)
    with pytest.raises(TypeError):
        st.__dlpack__(something="else")


def test_timing_cases_follow_the_current_stream_and_device(monkeypatch):
    import importlib

    import rustygradients_b200 as rg
    P = importlib.import_module("perf.operators")
    made = []

    class Backend:
        def __init__(self, device, stream):
            self.at = (device, stream)
            made.append(self.at)

        def from_device(self, t):
            return t

        def layer_norm_fwd(self, x, gamma, beta, eps):
            raise LookupError(self.at)

    now = [0, 0]
    monkeypatch.setattr(rg, "B200Backend", Backend)
    monkeypatch.setattr(P, "_backends", {})
    monkeypatch.setattr(P, "own", True)
    monkeypatch.setattr(P.torch.cuda, "current_device", lambda: now[0])
    monkeypatch.setattr(P.torch.cuda, "current_stream", lambda: type("S", (), {"cuda_stream": now[1]})())
    state = {"op": "ln_fwd", "x": 0, "gamma": 0, "beta": 0}
    for now[:] in ([0, 0], [0, 7], [0, 0], [1, 0], [0, 7]):
        with pytest.raises(LookupError) as at:
            P.run(state)
        assert at.value.args[0] == tuple(now)
    assert made == [(0, 0), (0, 7), (1, 0)]


def test_the_per_thread_default_stream_is_refused():
    lib, p = _lib.load(), C.c_void_p()
    assert lib.rg_ctx_create_on_stream(0, C.c_void_p(2), C.byref(p)) == _lib.RG_ERR_UNSUPPORTED and not p.value   # cudaStreamPerThread
    assert b"per-thread" in lib.rg_last_error()


def _bits(a):
    return np.ascontiguousarray(a, np.float32).view(np.uint32)


def test_three_truncated_bf16_planes_hold_an_f32():
    """What the gradients' products rest on: each plane takes the leading 8 bits of what the planes before leave, exactly."""
    rng = np.random.default_rng(0)
    x = np.concatenate([rng.standard_normal(20000) * 10.0 ** rng.integers(-20, 20, 20000), [0.0, 1.0, 3.4028235e38, -3.4028235e38]]).astype(np.float32)
    rest, planes = x.copy(), []
    for _ in range(3):
        hi = (_bits(rest) & 0xFFFF0000).view(np.float32)
        planes.append(hi)
        rest = rest - hi
    assert not rest.any() and np.isfinite(planes).all()
    assert np.array_equal(sum(p.astype(np.float64) for p in planes), x.astype(np.float64))
    a, b = rng.permutation(x[:20000]).astype(np.float64), x[:20000].astype(np.float64)
    pa, pb = [], []
    for v, out in ((a, pa), (b, pb)):
        r = v.astype(np.float32)
        for _ in range(3):
            hi = (_bits(r) & 0xFFFF0000).view(np.float32)
            out.append(hi.astype(np.float64))
            r = r - hi
    taken = sum(pa[i] * pb[j] for i, j in ((0, 0), (0, 1), (1, 0), (1, 1), (0, 2), (2, 0)))
    live = np.abs(a * b) > 0
    assert (np.abs(taken - a * b)[live] <= 2.0 ** -21 * np.abs(a * b)[live]).all()


def test_two_scaled_f16_planes_hold_22_bits():
    """What the logits' products rest on: with the largest magnitude of a group at 2^14..2^15, two f16 are within 2^-22 of a
    value, or within 2^-40 of the largest one."""
    rng = np.random.default_rng(1)
    for scale in (1e-30, 1.0, 1e25):
        x = (rng.standard_normal(5000) * 10.0 ** rng.uniform(-12, 0, 5000) * scale).astype(np.float32)
        m = np.abs(x).max()
        a = 14 - (int(_bits(m)[()] >> 23) - 127) if np.ndim(m) == 0 else None
        s = x.astype(np.float64) * 2.0 ** a
        assert 2 ** 14 <= np.abs(s).max() < 2 ** 15
        hi = s.astype(np.float16)
        lo = (s - hi.astype(np.float64)).astype(np.float16)
        err = np.abs(hi.astype(np.float64) + lo.astype(np.float64) - s)
        assert (err <= np.maximum(2.0 ** -22 * np.abs(s), 2.0 ** -40 * 2 ** 15)).all()


def _pair_logits(x, w):
    """The three products of scaled f16 pairs, summed in 64 bits: a power of two per row of x, one for w."""
    def split(a, m):
        up = 2.0 ** (14 - np.floor(np.log2(m)))
        s = a.astype(np.float64) * up
        hi = s.astype(np.float16).astype(np.float64)
        return hi, (s - hi).astype(np.float16).astype(np.float64), up
    x0, x1, xs = split(x, np.abs(x).max(-1, keepdims=True))
    w0, w1, ws = split(w, np.abs(w).max())
    return (x0 @ w0 + x0 @ w1 + x1 @ w0) / xs / ws


@pytest.mark.parametrize("D", [8, 64, 768])
def test_logits_of_pairs_within_the_rule(D):
    """Up to D max|x| max|w| = 2^22 a logit from f16 pairs is off by at most 2^-16 and 2^-21 of its products' magnitudes, also where
    all roundings go the same way; far beyond, one large weight costs the other logits their digits."""
    rng = np.random.default_rng(D)
    x, w = rng.standard_normal((40, D)).astype(np.float32), (rng.standard_normal((D, 50)) * 0.1).astype(np.float32)
    x[:, 0] = 0
    w[1:, 7] = 0.1                      # one rounding for a whole column
    for size, inside in ((1.0, True), (1.0 / 64, True), (2.0 ** 20, False)):
        w[0, 3] = size * 2.0 ** 22 / D / np.abs(x).max()
        exact, mags = x.astype(np.float64) @ w.astype(np.float64), np.abs(x).astype(np.float64) @ np.abs(w).astype(np.float64)
        err = np.abs(_pair_logits(x, w) - exact)
        assert (err <= 2.0 ** -16 + 2.0 ** -21 * mags).all() == inside, (size, err.max())


def _compile():
    lib = build.build()
    cmd = ["g++", "-std=c++17", "-O1", "-I", os.path.join(ROOT, "include"), os.path.join(ROOT, "tests", "cpp", "train_mirror_test.cpp"),
           "-o", EXE, "-L", os.path.dirname(lib), "-lrg_b200", "-Wl,-rpath," + os.path.dirname(lib)]
    r = subprocess.run(cmd, capture_output=True, text=True)
    assert r.returncode == 0, r.stderr
    return EXE


def test_cpp_mirror_of_the_training_ops_compiles():
    assert os.path.exists(_compile())


@pytest.mark.gpu
def test_cpp_mirror_of_the_training_ops_runs():
    r = subprocess.run([_compile()], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "OK" in r.stdout, r.stdout + r.stderr


def _run_host_test(name, tmp_path):
    exe = str(tmp_path / name)
    r = subprocess.run(["g++", "-std=c++17", "-O1", "-I", os.path.join(ROOT, "rustygradients_b200", "csrc"),
                        os.path.join(ROOT, "tests", "cpp", name + ".cpp"), "-o", exe], capture_output=True, text=True)
    assert r.returncode == 0, r.stderr
    r = subprocess.run([exe], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0 and "OK" in r.stdout, r.stdout


def test_few_row_reads_stay_inside_the_matrix(tmp_path):
    """Every 16-byte read that the form for few rows makes without a guard, for matrices down to one column and one row."""
    _run_host_test("lce_plan_test", tmp_path)


def test_the_current_device_is_put_back(tmp_path):
    _run_host_test("device_scope_test", tmp_path)
    # every entry point sets the device through that class
    csrc = os.path.join(ROOT, "rustygradients_b200", "csrc")
    calls = [f"{f}: {line.strip()}" for f in sorted(os.listdir(csrc)) for line in open(os.path.join(csrc, f)) if "cudaSetDevice(" in line]
    assert calls == ["rg_internal.cuh: static int set(int d) { return (int)cudaSetDevice(d); }"]


def test_kernels_that_start_early_read_only_finished_data_as_constant():
    """A `const __restrict__` parameter of a kernel that waits for its predecessor may be read in front of the wait: only what was
    complete before the chain began (a caller's matrices, weights, LayerNorm parameters) is passed that way."""
    import re
    csrc = os.path.join(ROOT, "rustygradients_b200", "csrc")
    found = set()
    for f in sorted(os.listdir(csrc)):
        text = open(os.path.join(csrc, f)).read()
        text = re.sub(r"__launch_bounds__\((?:[^()]|\([^()]*\))*\)|__cluster_dims__\([^()]*\)", "", text)
        for m in re.finditer(r"__global__[^;{]*?(\w+)\(([^;{]*?)\)\s*\{", text):
            end = text.find("\n}", m.end())
            if re.search(r"rg_pdl_sync\(\)|griddepcontrol\.wait", text[m.end():end]):
                found |= {(m.group(1), p) for p in re.findall(r"const [\w:]+\s*\*\s*__restrict__ (\w+)", m.group(2))}
    assert found == {("lt_align_kernel", "src"), ("lt_max_kernel", "w"), ("lt_max_kernel", "x"), ("lt_pack_kernel", "src"),
                     ("rg_embed_step_kernel", "wte"), ("rg_embed_step_kernel", "wpe"),
                     ("rg_rows_res_ln_bf16_kernel", "bias"), ("rg_rows_res_ln_bf16_kernel", "gamma"), ("rg_rows_res_ln_bf16_kernel", "beta"),
                     ("rg_rows_act_bf16_kernel", "bias"), ("rg_rows_res_ln_tp_bf16_kernel", "bias"),
                     ("rg_rows_res_ln_tp_bf16_kernel", "gamma"), ("rg_rows_res_ln_tp_bf16_kernel", "beta")}
