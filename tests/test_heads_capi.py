"""The operators over heads and the Muon step without a GPU: the C entries' refusals, before
any HIP call, in a child process that sees no GPU."""
import ctypes
import os
import subprocess
import sys

import pytest
import torch

import cpab
from cpab.pytorch import _native

HERE = os.path.dirname(os.path.realpath(__file__))
ROOT = os.path.dirname(HERE)
I, L, V, F = ctypes.c_int, ctypes.c_int64, ctypes.c_void_p, ctypes.c_float
P, ODD = 64, 65   # made up: validation comes first


class QkNorm(ctypes.Structure):
    _fields_ = ([(n, I) for n in ("dtype", "weight_dtype", "neighbours", "position_type")]
                + [(n, L) for n in ("B", "T", "heads", "key_heads", "width", "turned")]
                + [("q", V), ("k", V), ("q_strides", L * 3), ("k_strides", L * 3), ("q_weight", V), ("k_weight", V),
                   ("freqs", V), ("positions", V), ("position_strides", L * 2), ("eps", F)])


class DeltaRule(ctypes.Structure):
    _fields_ = ([(n, I) for n in ("dtype", "gate_dtype", "lengths64")]
                + [(n, L) for n in ("B", "T", "heads", "key_heads", "dk", "dv")]
                + [(n, V) for n in ("q", "k", "v", "decay", "beta")]
                + [(n + "_strides", L * 3) for n in ("q", "k", "v", "decay", "beta")]
                + [("h0", V), ("lengths", V), ("scale", F)])


class Matrix(ctypes.Structure):
    _fields_ = [("param", V), ("grad", V), ("momentum", V), ("master", V), ("rows", L), ("cols", L)]


def qk_norm(**kw):
    st = (L * 3)(64, 16, 8)
    args = dict(B=2, T=4, heads=2, key_heads=1, width=8, turned=4, q=P, k=P, q_strides=st, k_strides=st, q_weight=P,
                k_weight=P, freqs=P, eps=1e-6)
    args.update(kw)
    return ctypes.byref(QkNorm(**args))


def delta_rule(**kw):
    st = (L * 3)(64, 16, 8)
    args = dict(B=2, T=4, heads=2, key_heads=1, dk=8, dv=8, q=P, k=P, v=P, decay=P, beta=P, scale=1.0,
                **{n + "_strides": st for n in ("q", "k", "v", "decay", "beta")})
    args.update(kw)
    return ctypes.byref(DeltaRule(**args))


def _run_without_gpu(check):
    env = dict(os.environ, HIP_VISIBLE_DEVICES="-1", ROCR_VISIBLE_DEVICES="-1", CUDA_VISIBLE_DEVICES="-1")
    paths = [HERE, ROOT, os.path.join(ROOT, "fg-cpab_amd")]
    code = f"import sys; sys.path[:0] = {paths!r}; import test_heads_capi as t; t.{check}()"
    r = subprocess.run([sys.executable, "-c", code], env=env, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stdout + r.stderr


def _refused(rc, word):
    msg = _native.load_library().cpab_last_error_string().decode()
    assert rc == 1 and word in msg, (rc, msg)


def test_qk_norm_refusals():
    _run_without_gpu("_check_qk_norm")


def _check_qk_norm():
    lib = _native.load_library()

    def forward(q_out=P, k_out=P, **kw):
        return lib.cpab_qk_norm_forward(qk_norm(**kw), q_out, k_out, None)

    def backward(grads=(P, P), outs=(P, P), weights=(P, P), strides=(8,) * 6, ws=P, n=0, **kw):
        return lib.cpab_qk_norm_backward(qk_norm(**kw), (V * 2)(*grads), (L * 6)(*strides), (V * 2)(*outs),
                                         (V * 2)(*weights), ws, n, None)
    down = (L * 3)(64, -16, 8)
    for call in (forward, backward):
        for kw, word in ((dict(dtype=2), "dtype"), (dict(weight_dtype=-1), "weight_dtype"), (dict(B=-1), "negative size"),
                         (dict(heads=-2), "negative size"), (dict(width=0), "width"), (dict(width=513), "width"),
                         (dict(turned=3), "turned"), (dict(turned=10), "turned"), (dict(T=1 << 31), "too large"),
                         (dict(B=1 << 16, T=1 << 16), "too large"), (dict(heads=65536), "too large"),
                         (dict(eps=-1.0), "eps"), (dict(eps=float("nan")), "eps"), (dict(q=None), "n.q"),
                         (dict(k=None), "n.k"), (dict(q_weight=None), "q_weight"), (dict(k_weight=None), "k_weight"),
                         (dict(freqs=None), "freqs"), (dict(q=ODD), "aligned"), (dict(k=66), "aligned"),
                         (dict(k_weight=66), "aligned"), (dict(freqs=66), "aligned"), (dict(position_type=3), "position_type"),
                         (dict(positions=68, position_type=1), "aligned"), (dict(q_strides=down), "strides of q"),
                         (dict(k_strides=down), "strides of k"),
                         (dict(position_strides=(L * 2)(-1, 1)), "strides of positions")):
            _refused(call(**kw), word)
        _refused(lib.cpab_qk_norm_forward(None, P, P, None), "norm")
    _refused(forward(q_out=None), "q_out")
    _refused(forward(k_out=None), "k_out")
    _refused(forward(q_out=ODD), "aligned")
    _refused(backward(grads=(None, P)), "grads")
    _refused(backward(grads=(P, ODD)), "aligned")
    _refused(backward(outs=(ODD, P)), "aligned")
    _refused(backward(weights=(P, 66)), "aligned")
    _refused(backward(strides=(8, 8, 8, 8, -1, 8)), "strides of the gradients")
    _refused(lib.cpab_qk_norm_backward(qk_norm(), None, None, None, None, P, 0, None), "grads")
    need = lib.cpab_qk_norm_backward_workspace_size(qk_norm())
    assert need > 0 and lib.cpab_qk_norm_backward_workspace_size(qk_norm(width=0)) == 0
    assert lib.cpab_qk_norm_backward_workspace_size(None) == 0
    _refused(backward(n=need - 1), "workspace too small")
    _refused(backward(ws=None, n=need), "workspace")
    _refused(backward(ws=72, n=need), "aligned")
    assert forward(B=0) == 0 and forward(T=0, q=None, k=None) == 0


def test_delta_rule_refusals():
    _run_without_gpu("_check_delta_rule")


def _check_delta_rule():
    lib = _native.load_library()

    def forward(o=P, h=P, kept=None, ws=P, n=1 << 40, **kw):
        return lib.cpab_delta_rule_forward(delta_rule(**kw), o, h, kept, ws, n, None)

    def backward(kept=P, go=P, gh=P, gq=P, gk=P, gv=P, gd=P, gb=P, g0=P, ws=P, n=1 << 40, **kw):
        return lib.cpab_delta_rule_backward(delta_rule(**kw), kept, go, gh, gq, gk, gv, gd, gb, g0, ws, n, None)
    down, far = (L * 3)(64, -16, 8), (L * 3)(64, 4194305, 8)
    for call in (forward, backward):
        for kw, word in ((dict(dtype=2), "dtype"), (dict(gate_dtype=5), "gate_dtype"), (dict(B=-1), "negative size"),
                         (dict(dv=-1), "negative size"), (dict(dk=0), "dk"), (dict(dk=129), "dk"), (dict(dv=0), "dv"),
                         (dict(heads=3, key_heads=2), "multiple"), (dict(key_heads=0), "multiple"),
                         (dict(T=1 << 31), "too large"), (dict(T=(1 << 31) - 64), "too large"),
                         (dict(B=1 << 22, T=1 << 12), "too large"), (dict(heads=65536), "too large"),
                         (dict(dv=1 << 22), "too large"), (dict(scale=float("inf")), "scale"),
                         (dict(scale=float("nan")), "scale"), (dict(q=None), "r.q"), (dict(k=None), "r.k"),
                         (dict(v=None), "r.v"), (dict(decay=None), "decay"), (dict(beta=None), "beta"),
                         (dict(q=66), "aligned"), (dict(v=ODD), "aligned"), (dict(beta=66), "aligned"),
                         (dict(h0=66), "aligned"), (dict(lengths=68, lengths64=1), "aligned"),
                         (dict(lengths=66), "aligned"), (dict(v_strides=far), "too far"), (dict(q_strides=far), "too far"),
                         *((dict(**{n + "_strides": down}), "strides of " + n) for n in ("q", "k", "v", "decay", "beta"))):
            _refused(call(**kw), word)
    _refused(lib.cpab_delta_rule_forward(None, P, P, None, P, 0, None), "rule")
    _refused(forward(o=None), "o must not be NULL")
    _refused(forward(h=None), "h must not be NULL")
    _refused(forward(o=ODD), "aligned")
    _refused(forward(kept=66), "aligned")
    _refused(backward(kept=None), "kept")
    for name in ("go", "gh", "gq", "gk", "gv", "gd", "gb", "g0"):
        _refused(backward(**{name: 66}), "aligned")
    for keep, back, call in ((0, 0, forward), (1, 1, backward)):
        need = lib.cpab_delta_rule_workspace_size(delta_rule(T=100), keep, back)
        assert need > 0
        _refused(call(T=100, n=need - 1), "workspace too small")
        _refused(call(T=100, ws=None, n=need), "workspace")
        _refused(call(T=100, ws=72, n=need), "aligned")
    assert lib.cpab_delta_rule_workspace_size(delta_rule(dk=200), 0, 0) == 0
    # 2^22 chunks of up to 1024 lanes would pass 2^32 lanes
    one = dict(heads=1, key_heads=1, B=1 << 16)
    assert lib.cpab_delta_rule_workspace_size(delta_rule(T=62 * 64, **one), 1, 1) > 0
    _refused(forward(T=63 * 64, **one), "too large")
    assert lib.cpab_delta_rule_kept(delta_rule(T=100)) > 0 and lib.cpab_delta_rule_kept(delta_rule(B=0)) == 0
    assert lib.cpab_delta_rule_kept(None) == 0
    assert forward(B=0) == 0 and forward(heads=0, key_heads=0) == 0 and backward(B=0) == 0


def test_muon_refusals():
    _run_without_gpu("_check_muon")


def _check_muon():
    lib = _native.load_library()
    ok = dict(param=P, grad=1 << 10, momentum=1 << 11, master=None, rows=70, cols=90)
    coefficients = (ctypes.c_double * 3)(3.4445, -4.775, 2.0315)

    def step(matrices=(ok,), dtype=0, n=None, rates=None, lr=0.1, wd=0.0, mu=0.9, c=coefficients, eps=1e-7, steps=5,
             ws=256, room=1 << 50):
        entries = (Matrix * len(matrices))(*[Matrix(**{**ok, **m}) for m in matrices])
        rates = (ctypes.c_double * len(matrices))(*(rates or [0.1] * len(matrices)))
        return lib.cpab_muon_step(dtype, len(matrices) if n is None else n, entries, rates, lr, wd, mu, 1, c, eps, steps,
                                  ws, room, None)
    nan = float("nan")
    for kw, word in ((dict(dtype=2), "dtype"), (dict(n=-1), "negative number"), (dict(n=1 << 31), "too many"),
                     (dict(mu=1.0), "momentum"), (dict(mu=-0.1), "momentum"), (dict(mu=nan), "momentum"),
                     (dict(lr=-1.0), "lr"), (dict(wd=nan), "weight_decay"), (dict(eps=-1.0), "eps"),
                     (dict(steps=0), "ns_steps"), (dict(steps=101), "ns_steps"), (dict(c=None), "coefficients"),
                     (dict(c=(ctypes.c_double * 3)(1, nan, 1)), "coefficients"), (dict(rates=[nan]), "rates"),
                     (dict(ws=None), "workspace"), (dict(ws=272), "aligned"), (dict(room=1000), "workspace too small")):
        _refused(step(**kw), word)
    for m, word in ((dict(rows=-1), "negative size"), (dict(cols=1 << 40), "too large"),
                    (dict(rows=1 << 20, cols=1 << 20), "too large"), (dict(param=None), "param"), (dict(grad=None), "grad"),
                    (dict(momentum=None), "momentum"), (dict(param=66), "aligned"), (dict(grad=ODD), "aligned"),
                    (dict(momentum=66), "aligned"), (dict(master=66), "aligned"), (dict(master=P), "comes twice"),
                    (dict(momentum=P), "comes twice")):
        _refused(step([m]), word)
    _refused(step([{}, {}]), "comes twice")
    _refused(step([dict(grad=P)]), "the gradient of matrix 0 is an array")
    _refused(step([dict(param=1 << 12, momentum=1 << 13), dict(grad=1 << 13)]), "the gradient of matrix 1 is an array")
    _refused(lib.cpab_muon_step(0, 1, None, None, 0.1, 0.0, 0.9, 1, coefficients, 1e-7, 5, 256, 1 << 50, None), "matrices")
    assert step([dict(rows=0), dict(cols=0)], ws=None, room=0) == 0 and step([], n=0) == 0
    size = lib.cpab_muon_workspace_size
    assert size(1, (Matrix * 1)(Matrix(**{**ok, "rows": -1}))) == 0
    # a matrix that one workgroup keeps needs none; one value more on either side does
    assert [size(1, (Matrix * 1)(Matrix(**{**ok, "rows": r, "cols": c}))) > 0
            for r, c in ((64, 256), (256, 64), (65, 65), (257, 64), (1, 257))] == [False, False, True, True, True]


@pytest.mark.parametrize("call", [
    lambda t: cpab.gated_delta_rule(t, t, t, t[..., 0], t[..., 0]),
    lambda t: cpab.qk_norm(t, t, t[0, 0, 0], t[0, 0, 0]),
    lambda t: cpab.muon_step([t[0, 0]], [t[0, 0]], [t[0, 0]]),
])
def test_no_fallback_without_a_gpu(call):
    with pytest.raises(RuntimeError):
        call(torch.zeros(1, 2, 2, 4))
