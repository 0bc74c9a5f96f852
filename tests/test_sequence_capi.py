"""The operators around the transform without a GPU: the C entries' refusals, before any
HIP call, in a child process that sees no GPU; and the oracle's own formulas."""
import ctypes
import os
import subprocess
import sys

import numpy as np
import torch

import sequence_oracle as so
from cpab.pytorch import _native

HERE = os.path.dirname(os.path.realpath(__file__))
ROOT = os.path.dirname(HERE)


def _run_without_gpu(check):
    env = dict(os.environ, HIP_VISIBLE_DEVICES="-1", ROCR_VISIBLE_DEVICES="-1", CUDA_VISIBLE_DEVICES="-1")
    paths = [HERE, ROOT, os.path.join(ROOT, "fg-cpab_amd")]
    code = f"import sys; sys.path[:0] = {paths!r}; import test_sequence_capi as t; t.{check}()"
    r = subprocess.run([sys.executable, "-c", code], env=env, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stdout + r.stderr


P = ctypes.c_void_p(64)   # made up: validation comes first
ODD = ctypes.c_void_p(65)


def _refused(rc, word):
    msg = _native.load_library().cpab_last_error_string().decode()
    assert rc == 1 and word in msg, (rc, msg)


def test_recurrence_refusals():
    _run_without_gpu("_check_recurrence")


def _check_recurrence():
    lib = _native.load_library()
    st = (ctypes.c_int64 * 6)(8, 4, 8, 4, 8, 4)

    def forward(dtype=0, B=1, T=2, C=4, x=P, f=P, g=P, strides=st, h0=P, y=P, h=P, lengths=None, l64=0):
        return lib.cpab_recurrence_forward(dtype, B, T, C, x, f, g, strides, h0, lengths, l64, y, h, None,
                                           None, 0, None)
    _refused(forward(dtype=2), "dtype")
    _refused(forward(B=-1), "negative")
    _refused(forward(T=1 << 31), "too large")
    _refused(forward(B=1 << 20, T=1 << 20, C=1 << 10), "too large")
    _refused(forward(x=None), "x must not be NULL")
    _refused(forward(f=None), "f must not be NULL")
    _refused(forward(strides=None), "strides")
    _refused(forward(y=None), "y must not be NULL")
    _refused(forward(h=None), "h_last")
    _refused(forward(x=ODD), "aligned")
    _refused(forward(lengths=ctypes.c_void_p(68), l64=1), "aligned")
    assert forward(B=0) == 0 and forward(C=0) == 0

    def backward(dtype=0, B=1, T=2, C=4, carries=P, g=P, dg=P, dx=P):
        return lib.cpab_recurrence_backward(dtype, B, T, C, P, P, g, st, P, None, 0, carries, P, P, dx, P,
                                            dg, P, None, 0, None)
    _refused(backward(dtype=-1), "dtype")
    _refused(backward(carries=None), "carries")
    _refused(backward(g=None), "grad_g")
    _refused(backward(dx=ODD), "aligned")
    assert backward(B=0) == 0
    # a workspace that is needed has to be there, aligned and large enough
    need = lib.cpab_recurrence_workspace_size(0, 1, 100000, 64, 0)
    if need > 0:
        args = [0, 1, 100000, 64, P, P, P, st, P, None, 0, P, P, None]
        _refused(lib.cpab_recurrence_forward(*args, None, need, None), "workspace")
        _refused(lib.cpab_recurrence_forward(*args, P, need - 1, None), "workspace too small")
        _refused(lib.cpab_recurrence_forward(*args, ctypes.c_void_p(72), need, None), "aligned")
    assert lib.cpab_recurrence_workspace_size(0, -1, 1, 1, 0) == 0
    assert lib.cpab_recurrence_carries(7, 1, 1, 1) == 0


def test_norm_refusals():
    _run_without_gpu("_check_norm")


def _check_norm():
    lib = _native.load_library()

    def forward(dtype=0, rtype=0, wtype=0, rows=2, C=4, x=P, res=P, w=P, eps=1e-6, y=P, rout=P):
        return lib.cpab_rms_norm_forward(dtype, rtype, wtype, rows, C, x, 4, res, 4, w, eps, y, rout, P, None)
    _refused(forward(dtype=5), "dtype")
    _refused(forward(rtype=1), "residual_dtype")
    _refused(forward(wtype=9), "weight_dtype")
    _refused(forward(rows=-1), "negative")
    _refused(forward(rows=1 << 31), "too large")
    _refused(forward(eps=-1.0), "eps")
    _refused(forward(eps=float("nan")), "eps")
    _refused(forward(x=None), "x must not be NULL")
    _refused(forward(w=None), "weight")
    _refused(forward(y=None), "y must not be NULL")
    _refused(forward(rout=None), "residual_out")
    _refused(forward(res=None), "without a residual")
    _refused(forward(x=ODD), "aligned")
    assert forward(rows=0) == 0 and forward(C=0) == 0
    _refused(lib.cpab_rms_norm_e4m3(0, 0, 0, 2, 4, P, 4, P, 4, P, 1e-6, P, None, P, None), "scale")

    def backward(rows=2, C=4, r=P, rstd=P, dw=None):
        return lib.cpab_rms_norm_backward(0, 0, 0, rows, C, r, 4, None, 0, rstd, P, P, 4, P, 4, P, P, dw, None, 0,
                                          None)
    _refused(backward(r=None), "r must not be NULL")
    _refused(backward(rstd=None), "rstd")
    need = lib.cpab_rms_norm_backward_workspace_size(100000, 64)
    if need > 0:
        _refused(backward(rows=100000, C=64, dw=P), "workspace")
    assert backward(C=0) == 0


def test_adamw_refusals():
    _run_without_gpu("_check_adamw")


class _Tensor(ctypes.Structure):
    _fields_ = [(k, ctypes.c_void_p) for k in ("param", "grad", "exp_avg", "exp_avg_sq", "exp_avg_scale",
                                               "exp_avg_sq_scale", "master")] + [("n", ctypes.c_int64)]


def _check_adamw():
    lib = _native.load_library()

    def step(dtype=0, bits=32, count=1, t=1, lr=1e-3, b1=0.9, b2=0.999, eps=1e-8, wd=0.0, **kw):
        one = dict(param=64, grad=64, exp_avg=64, exp_avg_sq=64, exp_avg_scale=64, exp_avg_sq_scale=64,
                   master=None, n=8)
        one.update(kw)
        arr = (_Tensor * 1)(_Tensor(**one))
        return lib.cpab_adamw_step(dtype, bits, count, ctypes.cast(arr, ctypes.c_void_p), t, lr, b1, b2, eps,
                                   wd, 0, None)
    _refused(step(dtype=3), "dtype")
    _refused(step(bits=16), "state_bits")
    _refused(step(count=-1), "negative")
    _refused(step(t=0), "step")
    _refused(step(b1=1.0), "beta1")
    _refused(step(b2=float("nan")), "beta")
    _refused(step(lr=-1.0), "lr")
    _refused(step(wd=-1.0), "weight_decay")
    _refused(step(param=None), "param")
    _refused(step(grad=None), "grad")
    _refused(step(exp_avg=None), "exp_avg")
    _refused(step(bits=8, exp_avg_scale=None), "exp_avg_scale")
    _refused(step(grad=66), "aligned")
    _refused(step(exp_avg=65), "aligned")
    _refused(step(master=66), "aligned")
    _refused(step(n=-1), "values")
    assert lib.cpab_adamw_step(0, 32, 0, None, 1, 1e-3, 0.9, 0.999, 1e-8, 0.0, 0, None) == 0


def test_oracle_recurrence_gradient_formula():
    # the gradient as the definition's adjoint gives it, against autograd and differences
    torch.manual_seed(0)
    B, T, C = 2, 9, 3
    x, f, g, dy = (torch.randn(B, T, C, dtype=torch.float64) for _ in range(4))
    h0, dh = (torch.randn(B, C, dtype=torch.float64) for _ in range(2))
    n = torch.tensor([9, 4])
    got = so.recurrence_grads(x, f, g, h0, n, dy, dh)
    _, _, H = so.recurrence(x, f, g, h0, n)
    a, s = torch.sigmoid(f), torch.sigmoid(g)
    lam = dh.clone()
    for t in range(T - 1, -1, -1):
        live = (t < n)[:, None].double()
        lam = lam + live * dy[:, t] * g[:, t] * s[:, t]
        torch.testing.assert_close(got["x"][:, t], live * (1 - a[:, t]) * lam)
        torch.testing.assert_close(got["f"][:, t], live * lam * (H[:, t] - x[:, t]) * a[:, t] * (1 - a[:, t]))
        torch.testing.assert_close(got["g"][:, t], live * dy[:, t] * H[:, t + 1] * s[:, t] * (1 + g[:, t] * (1 - s[:, t])))
        lam = torch.where(t < n[:, None], a[:, t] * lam, lam)
    torch.testing.assert_close(got["h0"], lam)

    def value(x_):
        y, h, _ = so.recurrence(x_, f, g, h0, n)
        return float((y * dy).sum() + (h * dh).sum())
    d = torch.randn_like(x)
    slope = (value(x + 1e-6 * d) - value(x - 1e-6 * d)) / 2e-6
    assert abs(slope - float((got["x"] * d).sum())) < 1e-6


def test_oracle_rounding():
    # the codes are E4M3 values, never further than a step, up and down in proportion
    rng = np.random.default_rng(0)
    x = np.concatenate([rng.standard_normal(960) * np.exp(3 * rng.standard_normal(960)), np.zeros(32)])
    for r in (0, 1, 0x8000, 0xFFFF):
        z, s = so.mx_round(x, np.full(x.shape, float(r)))
        back = torch.tensor(z, dtype=torch.float32).to(torch.float8_e4m3fn).float().numpy()
        assert np.array_equal(back, z.astype(np.float32)) and np.abs(z).max() <= 448
        top = np.abs(x).reshape(-1, 32).max(1)
        live = top > 0
        assert (top[live] <= 448 * s[live]).all() and (top[live] > 224 * s[live]).all()
    bits = so.random_bits(200000, 7, 3, 2)
    assert abs((bits & 0xFFFF).mean() / 65536 - 0.5) < 0.005 and abs((bits >> 16).mean() / 65536 - 0.5) < 0.005
    assert abs(np.corrcoef(bits & 0xFFFF, bits >> 16)[0, 1]) < 0.01
    assert abs(np.corrcoef(bits[1:] >> 16, bits[:-1] >> 16)[0, 1]) < 0.01
