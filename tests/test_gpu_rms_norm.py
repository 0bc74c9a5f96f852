"""Root-mean-square norm against its definition in 64 bits.

Bounds, from the arithmetic (u = 2^-24).  A lane adds C / 64 squares, or in narrow rows
up to 24, one after the other (growing sums: half as many units) and a tree the lanes'
sums: the mean of squares carries (C / 64 + 20) u at most, its root half of that and the
root's and division's roundings 3 u; r, the two products and the store a unit each.  So y
carries e = (C / 128 + 16) u of its value
(and 16-bit outputs half a unit of their last place, at most 2^-8 of the value, besides).  In the backward
the mean of u r s carries (C / 64 + 20) u of the mean of |u r s|, and a term of the
weight's gradient 8 u before `rows` are added in some order: rows u of the sum of the
terms' sizes.  r of 16 bits, as it is kept for the backward, is off by 2^-8."""
import time

import pytest
import torch

import cpab
import sequence_oracle as so

pytestmark = pytest.mark.gpu
U = so.U
F32, BF16, E4M3 = torch.float32, torch.bfloat16, torch.float8_e4m3fn


def make(cuda, dtype, rows, C, residual, wtype, seed):
    gen = torch.Generator().manual_seed(seed * 977 + rows * 13 + C)
    x = torch.randn(rows, C, generator=gen) * torch.exp(torch.randn(rows, 1, generator=gen))
    w = 1 + 0.3 * torch.randn(C, generator=gen)
    r = None if residual is None else torch.randn(rows, C, generator=gen).to(residual).to(cuda)
    return x.to(dtype).to(cuda), w.to(wtype).to(cuda), r


def check(got, want, bound, what):
    got = so.f64(got)
    assert got.shape == want.shape, what
    over = (got - want).abs() - bound
    assert got.numel() == 0 or over.max() <= 0, (what, float((got - want).abs().max()), float(over.max()))


def unit(dtype):
    return 0.0 if dtype == F32 else 2.0 ** -8 * 1.01


def compare(cuda, dtype, rows, C, residual=None, wtype=None, seed=0, eps=1e-6):
    x, w, res = make(cuda, dtype, rows, C, residual, wtype or dtype, seed)
    leaves = [t.detach().requires_grad_() for t in (x, w, res) if t is not None]
    out = cpab.rms_norm(leaves[0], leaves[1], leaves[2] if res is not None else None, eps=eps)
    y, rout = out if res is not None else (out, None)
    assert y.dtype == dtype and (rout is None or rout.dtype == residual)
    gen = torch.Generator().manual_seed(3)
    dy = torch.randn(rows, C, generator=gen).to(dtype).to(cuda)
    dres = torch.randn(rows, C, generator=gen).to(residual).to(cuda) if res is not None else None
    grads = torch.autograd.grad(out, leaves, (dy, dres) if res is not None else dy)
    X, W, R, DY, DR = (so.f64(t) for t in (x, w, res, dy, dres))
    ry, rr, s = so.rms_norm(X, W, R, eps)
    want = so.rms_norm_grads(X, W, R, eps, DY, DR)
    e = (C / 128 + 16) * U
    check(y, ry, (e + unit(dtype)) * ry.abs() + 1e-38, "y")
    if rout is not None:
        check(rout, rr, (U + unit(residual)) * rr.abs(), "residual")
    n = rr * s
    v = (DY * W).abs()
    kept = unit(residual) if residual is not None else 0.0
    mean = (v * n.abs()).mean(-1, keepdim=True)
    bound = s * ((e + 8 * U) * v + n.abs() * mean * ((C / 64 + 40) * U + 2 * kept + 2 * e))
    if DR is not None:
        bound = bound + 4 * U * DR.abs()
    check(grads[0], want[0], bound * 1.001 + (unit(dtype) + 4 * U) * want[0].abs(), "grad x")
    if res is not None:
        check(grads[2], want[2], bound * 1.001 + (unit(residual) + 4 * U) * want[2].abs(), "grad residual")
    size = (DY * n).abs().sum(0)
    check(grads[1], want[1], ((rows + 8) * U + e + kept) * size + (unit(w.dtype) + U) * want[1].abs(),
          "grad weight")
    # the 8-bit output: its scale is y's largest size, the value within half a step of
    # 3 bits of mantissa (2^-4), and of 2^-10 below the normal ones
    with torch.no_grad():
        got = cpab.rms_norm(x, w, res, eps=eps, out_dtype=E4M3)
    q, scale = got[0], so.f64(got[1])
    assert q.dtype == E4M3 and q.shape == x.shape and got[1].shape == x.shape[:-1]
    top = ry.abs().amax(-1) / 448
    top = torch.where(top == 0, torch.ones_like(top), top)
    check(got[1], top, (e + 4 * U) * top, "scale")
    value = so.f64(q.float()) * scale[:, None]
    check(value, ry, (2.0 ** -4 + 4 * e) * ry.abs() + 2.0 ** -10 * scale[:, None] * (1 + e), "8 bits")
    assert (so.f64(q.float()).abs() <= 448).all()
    if res is not None:
        assert torch.equal(got[2], rout)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("C", [1, 2, 7, 63, 64, 65, 333, 1000, 1024, 2047])
@pytest.mark.parametrize("rows", [1, 5])
def test_widths(cuda, dtype, C, rows):
    compare(cuda, dtype, rows, C, residual=dtype)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("rows,C", [(1, 8192), (3, 16384), (2, 16383), (2, 20000), (1, 40001), (3, 4100)])
def test_wide_rows(cuda, dtype, rows, C):
    compare(cuda, dtype, rows, C, residual=dtype, seed=1)


@pytest.mark.parametrize("dtype,C", [(F32, 20), (F32, 100), (F32, 600), (F32, 1536), (F32, 5000), (F32, 9000),
                                     (F32, 12288), (F32, 16389), (F32, 32768), (BF16, 180), (BF16, 1040),
                                     (BF16, 2100), (BF16, 4200), (BF16, 5000), (BF16, 7168), (BF16, 8200),
                                     (BF16, 14000), (BF16, 24600)])
@pytest.mark.parametrize("rows", [1, 3, 19, 130])
def test_widths_between_the_powers_of_two(cuda, dtype, C, rows):
    compare(cuda, dtype, rows, C, residual=dtype, seed=4)


@pytest.mark.parametrize("rows,C", [(1000, 64), (4099, 32), (700, 513), (20000, 8), (9000, 128)])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_many_rows(cuda, dtype, rows, C):
    compare(cuda, dtype, rows, C, residual=dtype, seed=2)


@pytest.mark.parametrize("C", [48, 129, 2100])
@pytest.mark.parametrize("dtype,residual,wtype", [(F32, None, F32), (F32, F32, BF16), (BF16, None, BF16),
                                                  (BF16, None, F32), (BF16, F32, BF16),
                                                  (BF16, F32, F32), (BF16, BF16, F32)])
def test_types(cuda, dtype, residual, wtype, C):
    compare(cuda, dtype, 17, C, residual=residual, wtype=wtype, seed=3)


def test_zero_rows_and_tiny_ones(cuda):
    # a row of zeros: y = 0, 8-bit scale 1; eps takes over below its root
    x = torch.zeros(3, 100, device=cuda)
    x[1] = 1e-12
    w = torch.ones(100, device=cuda)
    y = cpab.rms_norm(x, w)
    assert (y[0] == 0).all()
    torch.testing.assert_close(y[1], torch.full((100,), 1e-9, device=cuda), rtol=1e-5, atol=0)
    q, scale = cpab.rms_norm(x, w, out_dtype=E4M3)
    assert (q.float()[0] == 0).all() and scale[0] == 1 and (q.float()[1] == 448).all()
    g = torch.autograd.grad(cpab.rms_norm(x.requires_grad_(), w).sum(), x)[0]
    assert torch.isfinite(g).all()
    # large values: the squares overflow 32 bits, as the definition in 32 bits says
    z = torch.full((1, 4), 3e38, device=cuda)
    assert (cpab.rms_norm(z, w[:4]) == 0).all()


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("C", [100, 20000])
@pytest.mark.parametrize("size,weight,eps", [(1e-37, 1.0, 1e-6), (1e-15, 1e-27, 1e-32),
                                             (1e-19, 1e19, 1e-30), (1e17, 1e22, 1e-6), (1.0, 1e-33, 1e-6)])
def test_8_bits_of_sizes_at_the_types_ends(cuda, dtype, C, size, weight, eps):
    # rows whose norm and scale 32 bits hold as normal numbers, and r, r w or its inverse not
    # in between: the bounds of compare(), and what rounding below 2^-126 adds to r w
    x = (torch.randn(3, C, device=cuda) * size).to(dtype)
    w = ((torch.rand(C, device=cuda) + 0.5) * weight).to(dtype)
    q, scale = cpab.rms_norm(x, w, eps=eps, out_dtype=E4M3)
    ry = so.rms_norm(so.f64(x), so.f64(w), None, eps)[0]
    e = (C / 128 + 16) * U
    top = ry.abs().amax(-1) / 448
    assert (top > 2.0 ** -126).all()
    check(scale, top, (e + 4 * U) * top + 2.0 ** -148, "scale")
    value = so.f64(q.float()) * so.f64(scale)[:, None]
    check(value, ry, (2.0 ** -4 + 4 * e) * ry.abs() + 2.0 ** -10 * so.f64(scale)[:, None] * (1 + e), "8 bits")
    assert (so.f64(q.float()).abs() <= 448).all()


def test_not_finite_rows(cuda):
    x = torch.randn(6, 70, device=cuda)
    w = torch.ones(70, device=cuda)
    ref = cpab.rms_norm(x, w)
    q0, s0 = cpab.rms_norm(x, w, out_dtype=E4M3)
    bad = x.clone()
    bad[1, 3], bad[4, 69] = float("nan"), float("inf")
    y = cpab.rms_norm(bad, w)
    rows = [0, 2, 3, 5]
    assert torch.equal(y[rows], ref[rows])
    assert torch.isnan(y[1]).all() and torch.isnan(y[4, 69]) and (y[4, :69] == 0).all()
    q, s = cpab.rms_norm(bad, w, out_dtype=E4M3)
    assert torch.equal(q.view(torch.uint8)[rows], q0.view(torch.uint8)[rows]) and torch.equal(s[rows], s0[rows])
    assert torch.isnan(q.float()[1]).all() and torch.isnan(s[1])
    assert torch.isnan(q.float()[4] * s[4])[69]


def test_layouts(cuda):
    gen = torch.Generator(device=cuda).manual_seed(1)
    big = torch.randn(12, 3, 5, 200, device=cuda, generator=gen)
    w = torch.randn(65, device=cuda, generator=gen)
    views = [big[..., 7:72], big[:, 1, :, 100:165], big.transpose(0, 2)[..., :65],
             torch.randn(65, 20, device=cuda, generator=gen).t(), big[0, 0, 0, 3:68],
             torch.randn(1, 65, device=cuda, generator=gen).expand(9, 65)]
    for x in views:
        want = cpab.rms_norm(x.contiguous(), w)
        assert torch.equal(cpab.rms_norm(x, w), want)
        y, r = cpab.rms_norm(x, w, residual=x)
        z, s = cpab.rms_norm(x.contiguous(), w, residual=x.contiguous())
        assert torch.equal(y, z) and torch.equal(r, s)
        a, b = (x.detach().requires_grad_(), x.detach().contiguous().requires_grad_())
        dy = torch.randn_like(want)
        ga = torch.autograd.grad(cpab.rms_norm(a, w), a, dy.t().contiguous().t() if dy.dim() == 2 else dy)[0]
        gb = torch.autograd.grad(cpab.rms_norm(b, w), b, dy)[0]
        assert torch.equal(ga, gb)
        q, sc = cpab.rms_norm(x, w, out_dtype=E4M3)
        assert q.shape == x.shape and sc.shape == x.shape[:-1]
    x = torch.randn(4, 66, device=cuda).bfloat16()
    odd = x.reshape(-1)[1:1 + 4 * 65].view(4, 65)   # aligned to 2 bytes
    assert torch.equal(cpab.rms_norm(odd, w), cpab.rms_norm(odd.clone(), w))


def test_parts_of_the_gradient(cuda):
    x, w, r = make(cuda, BF16, 40, 96, BF16, BF16, 4)
    leaves = [t.detach().requires_grad_() for t in (x, w, r)]
    y, s = cpab.rms_norm(*leaves)
    dy, ds = torch.randn_like(y), torch.randn_like(s)
    whole = torch.autograd.grad((y, s), leaves, (dy, ds), retain_graph=True)
    only_y = torch.autograd.grad(y, leaves, dy, retain_graph=True)
    only_s = torch.autograd.grad(s, leaves, ds, allow_unused=True)
    assert torch.equal(only_s[0], ds) and torch.equal(only_s[2], ds)
    assert torch.equal(only_y[1], whole[1])
    torch.testing.assert_close((only_y[0].float() + ds.float()), whole[0].float(), rtol=2 ** -7, atol=2 ** -7)
    for i in range(3):
        args = [t.detach().requires_grad_(j == i) for j, t in enumerate(leaves)]
        y, s = cpab.rms_norm(*args)
        assert torch.equal(torch.autograd.grad((y, s), args[i], (dy, ds), allow_unused=True)[0], whole[i])
    # x + residual and the norm share a gradient: both leaves accumulate it apart
    y, s = cpab.rms_norm(*leaves)
    torch.autograd.backward((y, s), (dy, ds))
    y, s = cpab.rms_norm(*leaves)
    torch.autograd.backward((y, s), (dy, ds))
    for t, g in zip(leaves, whole):
        torch.testing.assert_close(t.grad.float(), 2 * g.float(), rtol=2 ** -7, atol=0)


@pytest.mark.parametrize("rows,C", [(37, 100), (700, 513), (3, 40001)])
def test_weight_of_32_bits_beside_16(cuda, rows, C):
    # its gradient does not show the rounding of a 16-bit residual: the bound of a
    # 32-bit sum of the terms
    x, w, res = make(cuda, BF16, rows, C, BF16, F32, 8)
    leaves = [t.detach().requires_grad_() for t in (x, w, res)]
    dy = torch.randn(rows, C, generator=torch.Generator().manual_seed(4)).bfloat16().to(cuda)
    out = cpab.rms_norm(*leaves)
    got = torch.autograd.grad(out, leaves, (dy, torch.zeros_like(out[1])))
    X, W, R, DY = (so.f64(t) for t in (x, w, res, dy))
    _, rr, s = so.rms_norm(X, W, R)
    want = so.rms_norm_grads(X, W, R, 1e-6, DY, None)
    size = (DY * rr * s).abs().sum(0)
    check(got[1], want[1], ((rows + 8) * U + (C / 128 + 16) * U) * size + U * want[1].abs(), "grad weight")
    # the inputs are what is kept then: changed in place they are refused
    out = cpab.rms_norm(*leaves)
    with torch.no_grad():
        leaves[2].mul_(1.0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        out[0].sum().backward()


def test_gradient_against_differences(cuda):
    # central differences of the kernel's own forward; with a step of 2^-7 the
    # third-order term is under 2^-12 of the derivative's scale
    x, w, r = make(cuda, F32, 30, 45, F32, F32, 5)
    leaves = [t.detach().requires_grad_() for t in (x, w, r)]
    gen = torch.Generator(device=cuda).manual_seed(9)
    y, s = cpab.rms_norm(*leaves)
    dy, ds = (torch.randn(y.shape, device=cuda, generator=gen) for _ in range(2))
    grads = torch.autograd.grad((y, s), leaves, (dy, ds))
    eps = 2.0 ** -7
    for i, grad in enumerate(grads):
        d = torch.randn(leaves[i].shape, device=cuda, generator=gen)

        def value(sign):
            args = [t.detach() + (sign * eps * d if j == i else 0) for j, t in enumerate(leaves)]
            a, b = cpab.rms_norm(*args)
            return float((a.double() * dy).sum() + (b.double() * ds).sum())
        with torch.no_grad():
            slope = (value(1) - value(-1)) / (2 * eps)
        scale = float(grad.double().norm() * d.double().norm()) / d.numel() ** 0.5
        assert abs(slope - float((grad.double() * d).sum())) <= 2e-2 * scale, (i, slope, scale)


def test_same_call_same_bits(cuda):
    x, w, r = make(cuda, BF16, 5000, 320, BF16, F32, 6)
    leaves = [t.detach().requires_grad_() for t in (x, w, r)]
    runs = []
    for _ in range(3):
        y, s = cpab.rms_norm(*leaves)
        runs.append((y, s) + torch.autograd.grad((y, s), leaves, (torch.ones_like(y), torch.ones_like(s))))
    for other in runs[1:]:
        assert all(torch.equal(a, b) for a, b in zip(runs[0], other))


def test_more_than_32_bits_of_values(cuda):
    rows, C = 2_100_000, 1027
    x = torch.randn(1, C, device=cuda).bfloat16()
    w = torch.ones(C, device=cuda).bfloat16()
    one = cpab.rms_norm(x, w)
    y = cpab.rms_norm(x.expand(rows, C), w)
    assert y.numel() > 2 ** 31
    for k in (0, 1, rows // 2, rows - 1):
        assert torch.equal(y[k], one[0])


def test_side_stream_and_graph(cuda):
    x, w, r = make(cuda, BF16, 300, 256, BF16, BF16, 7)
    leaves = [t.detach().requires_grad_() for t in (x, w, r)]
    y, s = cpab.rms_norm(*leaves)
    ref = torch.autograd.grad((y, s), leaves, (torch.ones_like(y), torch.ones_like(s)))
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        z, t = cpab.rms_norm(*leaves)
        got = torch.autograd.grad((z, t), leaves, (torch.ones_like(z), torch.ones_like(t)))
    side.synchronize()
    assert torch.equal(y, z) and torch.equal(s, t) and all(torch.equal(a, b) for a, b in zip(ref, got))
    graph = torch.cuda.CUDAGraph()
    with torch.no_grad():
        with torch.cuda.graph(graph):
            q, scale, t = cpab.rms_norm(x, w, r, out_dtype=E4M3)
        for k in range(4):
            x.copy_(torch.randn(x.shape, device=cuda))
            graph.replay()
            want = cpab.rms_norm(x, w, r, out_dtype=E4M3)
            torch.cuda.synchronize()
            assert torch.equal(q.view(torch.uint8), want[0].view(torch.uint8))
            assert torch.equal(scale, want[1]) and torch.equal(t, want[2])


def test_nothing_is_left_behind(cuda):
    # the sum is an output and kept for the backward: neither a dropped graph nor a used
    # one holds it
    x, w, r = make(cuda, BF16, 500, 1000, BF16, BF16, 9)
    leaves = [t.detach().requires_grad_() for t in (x, w, r)]
    dy = torch.ones_like(x)
    before = torch.cuda.memory_allocated()
    for _ in range(5):
        cpab.rms_norm(*leaves)
        torch.autograd.grad(cpab.rms_norm(*leaves), leaves, (dy, dy))
    # the engine's thread lets go of the last pass's tensors a little after grad returns
    for _ in range(100):
        if torch.cuda.memory_allocated() <= before:
            break
        time.sleep(0.01)
    assert torch.cuda.memory_allocated() <= before


def test_refusals(cuda):
    x = torch.randn(3, 8, device=cuda)
    w = torch.ones(8, device=cuda)
    for args, kw, word in (((x.cpu(), w.cpu()), {}, "GPU"), ((x.half(), w), {}, "bfloat16"),
                           ((x, w[:7]), {}, "weight must"), ((x, w.half()), {}, "weight must"),
                           ((x, w.cpu()), {}, "weight must"), ((x, w[None]), {}, "weight must"),
                           ((x, w, x[:2]), {}, "residual must"), ((x, w, x.bfloat16()), {}, "residual must"),
                           ((x, w, x.cpu()), {}, "residual must"), ((x, w), {"eps": -1.0}, "eps"),
                           ((x, w), {"eps": float("nan")}, "eps"),
                           ((x[:, :0], w[:0]), {}, "no values"),
                           ((x.clone().requires_grad_(), w), {"out_dtype": E4M3}, "no gradient")):
        with pytest.raises(RuntimeError, match=word):
            cpab.rms_norm(*args, **kw)
    with pytest.raises(AssertionError, match="out_dtype"):
        cpab.rms_norm(x, w, out_dtype=BF16)


def test_no_rows(cuda):
    x = torch.randn(0, 8, device=cuda).requires_grad_()
    w = torch.ones(8, device=cuda).requires_grad_()
    y = cpab.rms_norm(x, w)
    gx, gw = torch.autograd.grad(y.sum(), (x, w))
    assert y.shape == (0, 8) and gx.shape == (0, 8) and (gw == 0).all()

class NoGradient(torch.autograd.Function):
    @staticmethod
    def forward(ctx, *outputs):
        return sum(t.float().sum() for t in outputs)

    @staticmethod
    def backward(ctx, g):
        return (None,) * len(ctx.needs_input_grad)


@pytest.mark.parametrize("residual", [False, True])
def test_no_gradient_comes(cuda, residual):
    # what stands behind the outputs has no gradient to give: then neither has the norm
    x, r = (torch.randn(5, 8, device=cuda).requires_grad_() for _ in range(2))
    w = torch.ones(8, device=cuda).requires_grad_()
    out = cpab.rms_norm(x, w, r) if residual else (cpab.rms_norm(x, w),)
    leaves = (x, w, r)[:3 if residual else 2]
    grads = torch.autograd.grad(NoGradient.apply(*out), leaves, allow_unused=True)
    assert all(g is None for g in grads)
