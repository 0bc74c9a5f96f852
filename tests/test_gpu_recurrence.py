"""Gated linear recurrence against its definition in 64 bits.

Bounds, from the arithmetic (u = 2^-24).  A gate and its complement carry a few u each:
|f| u from the scaling of exp's argument, for |f| up to 8 at most 12 u, and 4 u from
exp, the sum and the reciprocal.  A state's error e then obeys
e_t <= a e_{t-1} + 16 u (a |h| + (1 - a) |x|) + u |h|: with M = max(|x|, |h0|) >= |h|
and N the samples over which 1 / (1 - a) lets that add up (at most T),
e <= 18 u N M.  The gradient through time obeys the same with its own largest value L.
bfloat16 results carry half a unit of their last place, at most 2^-8 of the value, besides."""
import numpy as np
import pytest
import torch

import cpab
import sequence_oracle as so

pytestmark = pytest.mark.gpu
U = so.U


def make(cuda, dtype, B, T, C, gate=True, start=True, lengths=None, layout="own", seed=0, keep=3.0):
    """Inputs on the GPU in one of the layouts a program has them in."""
    gen = torch.Generator().manual_seed(1000 * seed + 31 * T + C)
    k = 3 if gate else 2
    whole = torch.randn(B, T, k * C, generator=gen)
    whole[..., C:2 * C] += torch.rand(C, generator=gen) * keep
    whole = whole.clamp(-8, 8)
    if lengths is not None:
        lengths = torch.tensor(lengths)
        pad = torch.arange(T)[None, :] >= lengths.clamp(0, T)[:, None]
        junk = torch.tensor([float("nan"), float("inf"), -float("inf"), 3.4e38])
        fill = junk[torch.randint(0, 4, whole.shape, generator=gen)]
        whole = torch.where(pad[..., None], fill, whole)
        lengths = lengths.to(cuda)
    whole = whole.to(cuda).to(dtype)
    parts = [whole[..., j * C:(j + 1) * C] for j in range(k)]
    if layout == "own":
        parts = [p.contiguous() for p in parts]
    elif layout == "time":      # [T, B, C] in memory
        parts = [p.transpose(0, 1).contiguous().transpose(0, 1) for p in parts]
    elif layout == "channel":   # [B, C, T] in memory
        parts = [p.transpose(1, 2).contiguous().transpose(1, 2) for p in parts]
    elif layout == "offset":    # not aligned to more than a value
        parts = [torch.cat([p.new_zeros(1), p.reshape(-1)])[1:].view(B, T, C) for p in parts]
    else:
        assert layout == "packed"
    h0 = torch.randn(B, C, generator=gen).to(cuda) if start else None
    return parts[0], parts[1], parts[2] if gate else None, h0, lengths


def check(got, want, bound, what):
    got, want, bound = so.f64(got), want.detach(), torch.as_tensor(bound)
    assert got.shape == want.shape, (what, got.shape, want.shape)
    assert torch.isfinite(got).all(), what
    over = (got - want).abs() - bound
    assert got.numel() == 0 or over.max() <= 0, (
        f"{what}: off by {float((got - want).abs().max()):.3g}, bound there "
        f"{float(bound.expand_as(over).reshape(-1)[over.argmax()]):.3g}")


def compare(cuda, dtype, B, T, C, **kw):
    x, f, g, h0, lengths = make(cuda, dtype, B, T, C, **kw)
    leaves = {k: v.detach().requires_grad_() for k, v in
              (("x", x), ("f", f), ("g", g), ("h0", h0)) if v is not None}
    y, h = cpab.gated_recurrence(leaves["x"], leaves["f"], leaves.get("g"), leaves.get("h0"), lengths)
    assert y.dtype == dtype and h.dtype == torch.float32
    gen = torch.Generator().manual_seed(5)
    dy = torch.randn(B, T, C, generator=gen).to(dtype).to(cuda)
    dh = torch.randn(B, C, generator=gen).to(cuda)
    names = list(leaves)
    grads = dict(zip(names, torch.autograd.grad((y, h), [leaves[k] for k in names], (dy, dh))))
    # the definition
    cl = None if lengths is None else lengths.cpu()
    ref = [so.padding_zeroed(so.f64(t), cl) for t in (x, f, g)]
    X, F, G = ref
    H0 = so.f64(h0)
    ry, rh, states = so.recurrence(X, F, G, H0, cl)
    want = so.recurrence_grads(X, F, G, H0, cl, so.f64(dy), so.f64(dh))
    M = max([float(v.abs().max()) for v in (X, H0) if v is not None and v.numel()] or [0.0])
    N = so.recurrence_memory(F, T)
    unit = so.UNIT[dtype] if dtype != torch.float32 else 0.0
    eh = 18 * U * N * M
    check(h, rh, eh, "h")
    silu = 1.0 if G is None else G.abs()
    check(y, ry, eh * silu + (40 * U + unit) * ry.abs() + 1e-38, "y")
    # L bounds the gradient of any state: what arrives, over the samples that remember it
    live = so.f64(dy) if G is None else so.f64(dy) * G * torch.sigmoid(G)
    L = (float(live.abs().max()) if live.numel() else 0.0) * N + float(so.f64(dh).abs().max() if dh.numel() else 0)
    el = 18 * U * N * L
    if "h0" in want and want["h0"] is not None:
        check(grads["h0"], want["h0"], el + 20 * U * want["h0"].abs(), "grad h0")
    if T == 0:
        return
    a = torch.sigmoid(F)
    ab = a * (1 - a)
    check(grads["x"], want["x"], (1 - a) * el + (40 * U + unit) * want["x"].abs() + 1e-38, "grad x")
    check(grads["f"], want["f"], ab * (2 * M * el + L * 2 * eh + 40 * U * 2 * M * L)
          + unit * want["f"].abs() + 1e-38, "grad f")
    if G is not None:
        s = torch.sigmoid(G)
        slope = (s * (1 + G * (1 - s))).abs()
        check(grads["g"], want["g"], so.f64(dy).abs() * (slope * eh + 60 * U * M * (1 + G.abs()))
              + unit * want["g"].abs() + 1e-38, "grad g")


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("T", [0, 1, 2, 15, 16, 17, 64, 127, 129, 300])
@pytest.mark.parametrize("C", [1, 5, 64, 131])
def test_lengths_and_widths(cuda, dtype, T, C):
    compare(cuda, dtype, 3, T, C, seed=1)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("B,T,C", [(1, 1500, 40), (2, 2049, 130), (5, 1023, 16), (1, 1, 700),
                                   (300, 3, 9), (70, 33, 257), (1, 4096, 2)])
def test_long_and_wide(cuda, dtype, B, T, C):
    compare(cuda, dtype, B, T, C, seed=2)


@pytest.mark.parametrize("B,T,C", [(12, 2600, 300), (9, 1000, 1111)])
def test_rows_that_are_not_whole_lines(cuda, B, T, C):
    # such rows are laid out in another way where there are many: the whole batch against
    # its rows a few at a time, whose layout the other tests hold to the definition; either
    # is within compare()'s bounds, so they are within twice those of each other
    lengths = [T - 7 * k * k for k in range(B)]
    x, f, g, h0, n = make(cuda, torch.float32, B, T, C, lengths=lengths, seed=3)
    dy, dh = torch.randn(B, T, C, device=cuda), torch.randn(B, C, device=cuda)

    def run(rows):
        leaves = [t[rows].detach().requires_grad_() for t in (x, f, g, h0)]
        out = cpab.gated_recurrence(*leaves, n[rows])
        return (*out, *torch.autograd.grad(out, leaves, (dy[rows], dh[rows])))

    whole = run(slice(None))
    few = [torch.cat(t) for t in zip(*(run(slice(k, k + 3)) for k in range(0, B, 3)))]
    X, F, G = (so.padding_zeroed(so.f64(t), n.cpu()) for t in (x, f, g))
    y, h, gx, gf, gg, gh = (so.f64(t) for t in few)
    M, N = max(float(X.abs().max()), float(h0.abs().max())), so.recurrence_memory(F, T)
    L = float((so.f64(dy) * G * torch.sigmoid(G)).abs().max()) * N + float(dh.abs().max())
    eh, el, a, s = 18 * U * N * M, 18 * U * N * L, torch.sigmoid(F), torch.sigmoid(G)
    for what, got, want, bound in (
            ("h", whole[1], h, eh), ("y", whole[0], y, eh * G.abs() + 40 * U * y.abs() + 1e-38),
            ("grad x", whole[2], gx, (1 - a) * el + 40 * U * gx.abs() + 1e-38),
            ("grad f", whole[3], gf, a * (1 - a) * (2 * M * el + 2 * L * eh + 80 * U * M * L) + 1e-38),
            ("grad g", whole[4], gg, so.f64(dy).abs() * ((s * (1 + G * (1 - s))).abs() * eh
                                                        + 60 * U * M * (1 + G.abs())) + 1e-38),
            ("grad h0", whole[5], gh, el + 20 * U * gh.abs())):
        check(got, want, 2 * torch.as_tensor(bound), what)


@pytest.mark.parametrize("gate,start", [(True, False), (False, True), (False, False)])
@pytest.mark.parametrize("T", [1, 37, 520])
def test_without_gate_or_start(cuda, gate, start, T):
    compare(cuda, torch.float32, 2, T, 66, gate=gate, start=start, seed=3)
    compare(cuda, torch.bfloat16, 2, T, 66, gate=gate, start=start, seed=3)


@pytest.mark.parametrize("layout", ["packed", "time", "channel", "offset"])
@pytest.mark.parametrize("dtype,C", [(torch.float32, 64), (torch.bfloat16, 64), (torch.bfloat16, 33)])
def test_layouts(cuda, layout, dtype, C):
    compare(cuda, dtype, 3, 150, C, layout=layout, seed=4)
    compare(cuda, dtype, 3, 1, C, layout=layout, seed=4)


@pytest.mark.parametrize("T", [1, 16, 40, 700])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("kind", [torch.int32, torch.int64])
def test_ragged_rows(cuda, T, dtype, kind):
    # empty rows, whole ones, ends inside and at the ends of tiles, lengths out of range
    lengths = [0, T, T // 2, 1, min(T, 16), min(T, 128), T + 9, -3, max(0, T - 1), T // 3]
    x, f, g, h0, n = make(cuda, dtype, len(lengths), T, 37, lengths=lengths, seed=5)
    y, _ = cpab.gated_recurrence(x, f, g, h0, n.to(kind))
    for b, k in enumerate(lengths):
        assert (y[b, max(0, min(k, T)):] == 0).all()
    compare(cuda, dtype, len(lengths), T, 37, lengths=lengths, seed=5)


def test_long_memory_and_no_memory(cuda):
    # gates at both ends: a rounds to 1 (the state stays) and to 0 (the state is x)
    B, T, C = 2, 400, 70
    x = torch.randn(B, T, C, device=cuda)
    h0 = torch.randn(B, C, device=cuda)
    y, h = cpab.gated_recurrence(x, torch.full_like(x, 200.0), h0=h0)
    assert torch.equal(y, h0[:, None].expand_as(y)) and torch.equal(h, h0)
    y, h = cpab.gated_recurrence(x, torch.full_like(x, -200.0), h0=h0)
    assert torch.equal(y, x) and torch.equal(h, x[:, -1])
    y, _ = cpab.gated_recurrence(x, torch.full_like(x, float("-inf")), h0=h0)
    assert torch.equal(y, x)
    y, _ = cpab.gated_recurrence(x, torch.full_like(x, float("inf")), h0=h0)
    assert torch.equal(y, h0[:, None].expand_as(y))


def test_not_finite_stays_in_its_row_and_channel(cuda):
    B, T, C = 3, 300, 40
    x, f, g, h0, _ = make(cuda, torch.float32, B, T, C, seed=6)
    ref, href = cpab.gated_recurrence(x, f, g, h0)
    bad = x.clone()
    bad[1, 200, 7] = float("nan")
    y, h = cpab.gated_recurrence(bad, f, g, h0)
    hit = torch.zeros(B, T, C, dtype=torch.bool, device=cuda)
    hit[1, 200:, 7] = True
    assert torch.isnan(y[hit]).all() and torch.equal(y[~hit], ref[~hit])
    assert torch.isnan(h[1, 7]) and int(torch.isnan(h).sum()) == 1


def test_in_pieces(cuda):
    # a signal read in pieces, down to single samples, gives the whole's results to
    # rounding: the state handed on is the 32-bit one
    B, T, C = 2, 260, 96
    x, f, g, h0, _ = make(cuda, torch.float32, B, T, C, seed=7)
    y, h = cpab.gated_recurrence(x, f, g, h0)
    parts, s, t = [], h0, 0
    for n in (1, 1, 5, 128, 0, 64, 61):
        p, s = cpab.gated_recurrence(x[:, t:t + n], f[:, t:t + n], g[:, t:t + n], s)
        parts.append(p)
        t += n
    assert t == T
    bound = 36 * U * so.recurrence_memory(so.f64(f), T) * float(max(x.abs().max(), h0.abs().max()))
    check(s, so.f64(h), bound, "h")
    check(torch.cat(parts, 1), so.f64(y), bound * so.f64(g).abs() + 40 * U * so.f64(y).abs(), "y")


@pytest.mark.parametrize("dtype,C", [(torch.float32, 40), (torch.bfloat16, 130)])
def test_hundreds_of_tiles_in_pieces(cuda, dtype, C):
    # a state passes hundreds of tiles: against the same signal read in short pieces,
    # whose states and gradients autograd hands on.  Both sides carry the bounds above
    # (twice); bfloat16 gradients half a unit each besides.
    B, T = 2, 70001
    lengths = [T, 33333]
    x, f, g, h0, n = make(cuda, dtype, B, T, C, lengths=lengths, seed=17)
    x, f, g = (torch.nan_to_num(t, 0.0, 0.0, 0.0) for t in (x, f, g))
    x, f = x.clamp(-8, 8), f.clamp(-8, 8)
    gen = torch.Generator(device=cuda).manual_seed(1)
    dy = torch.randn(B, T, C, device=cuda, generator=gen).to(dtype)
    dh = torch.randn(B, C, device=cuda, generator=gen)
    one = [t.detach().requires_grad_() for t in (x, f, g, h0)]
    y, h = cpab.gated_recurrence(*one, n)
    grads = torch.autograd.grad((y, h), one, (dy, dh))
    two = [t.detach().requires_grad_() for t in (x, f, g, h0)]
    s, parts, step = two[3], [], 3001
    for t in range(0, T, step):
        p, s = cpab.gated_recurrence(*(v[:, t:t + step] for v in two[:3]), s, (n - t).clamp(min=0))
        parts.append(p)
    want = torch.autograd.grad((torch.cat(parts, 1), s), two, (dy, dh))
    M = float(max(x.abs().max(), h0.abs().max()))
    N = so.recurrence_memory(so.f64(f), T)
    unit = 2 * so.UNIT[dtype] if dtype != torch.float32 else 0.0
    eh = 36 * U * N * M
    silu = so.f64(g).abs()
    check(h, so.f64(s), eh, "h")
    ry = so.f64(torch.cat(parts, 1))
    check(y, ry, eh * silu + (80 * U + unit) * ry.abs() + 1e-38, "y")
    L = float((dy.float() * g.float() * torch.sigmoid(g.float())).abs().max()) * N + float(dh.abs().max())
    el = 36 * U * N * L
    for k, (a, b) in enumerate(zip(grads, want)):
        b = so.f64(b)
        scale = (el, 0.25 * (2 * M * el + 4 * L * eh + 160 * U * M * L),
                 so.f64(dy).abs() * (1.1 * eh + 120 * U * M * (1 + silu)), el)[k]
        check(a, b, scale + (unit + 80 * U) * b.abs() + 1e-38, f"grad {k}")


def test_same_call_same_bits(cuda):
    x, f, g, h0, _ = make(cuda, torch.float32, 2, 3000, 65, seed=8)
    leaves = [t.detach().requires_grad_() for t in (x, f, g, h0)]
    runs = []
    for _ in range(3):
        y, h = cpab.gated_recurrence(*leaves)
        runs.append((y, h) + torch.autograd.grad((y, h), leaves, (torch.ones_like(y), torch.ones_like(h))))
    for other in runs[1:]:
        assert all(torch.equal(a, b) for a, b in zip(runs[0], other))


@pytest.mark.parametrize("B,T,C", [(2, 300, 8), (1, 37, 5)])
def test_gradient_against_differences(cuda, B, T, C):
    # central differences of the kernel's own forward along random directions.  The
    # sum of y * dy over n = B T C values carries about sqrt(n) roundings; with a step of
    # 2^-6 the third-order term is 2^-12 of the derivative's scale.
    x, f, g, h0, _ = make(cuda, torch.float32, B, T, C, seed=9, keep=1.0)
    leaves = [t.detach().requires_grad_() for t in (x, f, g, h0)]
    gen = torch.Generator(device=cuda).manual_seed(3)
    y, h = cpab.gated_recurrence(*leaves)
    dy = torch.randn(y.shape, device=cuda, generator=gen)
    dh = torch.randn(h.shape, device=cuda, generator=gen)
    grads = torch.autograd.grad((y, h), leaves, (dy, dh))
    eps = 2.0 ** -6
    for i, grad in enumerate(grads):
        d = torch.randn(leaves[i].shape, device=cuda, generator=gen)

        def value(sign):
            args = [t.detach() + (sign * eps * d if j == i else 0) for j, t in enumerate(leaves)]
            with torch.no_grad():
                a, b = cpab.gated_recurrence(*args)
            return float((a.double() * dy).sum() + (b.double() * dh).sum())
        slope = (value(1) - value(-1)) / (2 * eps)
        scale = float(grad.double().norm() * d.double().norm()) / d.numel() ** 0.5
        assert abs(slope - float((grad.double() * d).sum())) <= 2e-2 * scale, (i, slope, scale)


def test_parts_of_the_gradient(cuda):
    # only one output used, only some inputs asked for
    x, f, g, h0, _ = make(cuda, torch.float32, 2, 200, 20, seed=10)
    leaves = [t.detach().requires_grad_() for t in (x, f, g, h0)]
    y, h = cpab.gated_recurrence(*leaves)
    dy, dh = torch.randn_like(y), torch.randn_like(h)
    both = torch.autograd.grad((y, h), leaves, (dy, dh))
    y, h = cpab.gated_recurrence(*leaves)
    a = torch.autograd.grad(y, leaves, dy, retain_graph=True)
    b = torch.autograd.grad(h, leaves, dh, allow_unused=True)
    for p, q, r in zip(both, a, b):
        r = torch.zeros_like(p) if r is None else r
        torch.testing.assert_close(q + r, p, rtol=1e-4, atol=1e-4 * float(p.abs().max()))
    for i in range(4):
        args = [t.detach().requires_grad_(j == i) for j, t in enumerate(leaves)]
        y, h = cpab.gated_recurrence(*args)
        one = torch.autograd.grad((y, h), args[i], (dy, dh))[0]
        assert torch.equal(one, both[i])
    # an upstream gradient that is one number, expanded
    y, _ = cpab.gated_recurrence(*leaves)
    one = torch.autograd.grad(y.sum(), leaves)
    y, _ = cpab.gated_recurrence(*leaves)
    for p, q in zip(one, torch.autograd.grad(y, leaves, torch.ones_like(y))):
        assert torch.equal(p, q)


def test_broadcast_inputs(cuda):
    # one signal and one gate for all rows, as expanded views: the gradient of the
    # shared tensor is the sum over the rows
    B, T, C = 4, 90, 24
    x1, f1, _, h0, _ = make(cuda, torch.float32, 1, T, C, gate=False, seed=11)
    h0 = torch.randn(B, C, device=cuda)
    x1, f1 = x1.detach().requires_grad_(), f1.detach().requires_grad_()
    y, _ = cpab.gated_recurrence(x1.expand(B, T, C), f1.expand(B, T, C), h0=h0)
    dy = torch.randn_like(y)
    gx, gf = torch.autograd.grad(y, (x1, f1), dy)
    xc, fc = (t.detach().expand(B, T, C).contiguous().requires_grad_() for t in (x1, f1))
    z, _ = cpab.gated_recurrence(xc, fc, h0=h0)
    assert torch.equal(y, z)
    hx, hf = torch.autograd.grad(z, (xc, fc), dy)
    assert torch.equal(gx, hx.sum(0, keepdim=True)) and torch.equal(gf, hf.sum(0, keepdim=True))


def test_more_than_32_bits_of_values(cuda):
    # 2.2e9 outputs: every row the same, the inputs one row's, expanded
    B, T, C = 33600, 1024, 64
    x, f, _, _, _ = make(cuda, torch.bfloat16, 1, T, C, gate=False, start=False, seed=12)
    with torch.no_grad():
        one, h1 = cpab.gated_recurrence(x, f)
        y, h = cpab.gated_recurrence(x.expand(B, T, C), f.expand(B, T, C))
    assert y.numel() > 2 ** 31
    for b in (0, 1, B // 2, B - 1):
        assert torch.equal(y[b], one[0])
    assert torch.equal(h, h1.expand_as(h))


def test_side_stream(cuda):
    x, f, g, h0, _ = make(cuda, torch.bfloat16, 4, 1000, 128, seed=13)
    leaves = [t.detach().requires_grad_() for t in (x, f, g, h0)]
    y, h = cpab.gated_recurrence(*leaves)
    ref = torch.autograd.grad((y, h), leaves, (torch.ones_like(y), torch.ones_like(h)))
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        for _ in range(3):
            z, k = cpab.gated_recurrence(*leaves)
            got = torch.autograd.grad((z, k), leaves, (torch.ones_like(z), torch.ones_like(k)))
    s.synchronize()
    assert torch.equal(y, z) and torch.equal(h, k) and all(torch.equal(a, b) for a, b in zip(ref, got))


def test_graph_replays(cuda):
    # recorded into a graph and replayed with other inputs, with eager work between
    x, f, g, h0, _ = make(cuda, torch.bfloat16, 2, 900, 64, seed=14)
    with torch.no_grad():
        cpab.gated_recurrence(x, f, g, h0)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y, h = cpab.gated_recurrence(x, f, g, h0)
        for k in range(4):
            x.copy_(torch.randn(x.shape, device=cuda).bfloat16() * (k + 1))
            graph.replay()
            want_y, want_h = cpab.gated_recurrence(x, f, g, h0)
            torch.cuda.synchronize()
            assert torch.equal(y, want_y) and torch.equal(h, want_h)


def test_autograd_manner(cuda):
    x, f, g, h0, _ = make(cuda, torch.float32, 2, 50, 8, seed=15)
    leaves = [t.detach().requires_grad_() for t in (x, f, g, h0)]
    y, _ = cpab.gated_recurrence(*leaves)
    grads = torch.autograd.grad(y.sum(), leaves, create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable"):
        grads[0].sum().backward()
    y, _ = cpab.gated_recurrence(*leaves)
    with torch.no_grad():
        leaves[0].mul_(1.0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()
    f0 = torch.randn(2, 50, 8, device=cuda)
    m = torch.jit.trace(lambda t: cpab.gated_recurrence(2 * t, f0)[0], (leaves[0],))
    other = torch.randn_like(leaves[0]).requires_grad_()
    assert torch.equal(m(other), cpab.gated_recurrence(2 * other, f0)[0])
    a = torch.autograd.grad(m(other).sum(), other)[0]
    b = torch.autograd.grad(cpab.gated_recurrence(2 * other, f0)[0].sum(), other)[0]
    assert torch.equal(a, b)


def test_nothing_kept_without_gradients(cuda):
    x, f, g, h0, _ = make(cuda, torch.float32, 2, 4096, 64, seed=16)
    before = torch.cuda.memory_allocated()
    y, h = cpab.gated_recurrence(x, f, g, h0)
    assert torch.cuda.memory_allocated() - before <= y.numel() * 4 + h.numel() * 4 + 1024


def test_refusals(cuda):
    x = torch.randn(2, 5, 4, device=cuda)
    h = torch.zeros(2, 4, device=cuda)
    for args, word in (((x.cpu(), x.cpu()), "GPU"), ((x.half(), x.half()), "bfloat16"),
                       ((x[0], x[0]), r"\[B, T, C\]"), ((x, x[:, :4]), "f must have"),
                       ((x, x.bfloat16()), "f must have"), ((x, x.cpu()), "f must have"),
                       ((x, x, x[..., :3]), "g must have"), ((x, x, x, h[:1]), "h0 must"),
                       ((x, x, x, h.double()), "h0 must"), ((x, x, x, h.cpu()), "h0 must"),
                       ((x, x, x, h, torch.ones(2, device=cuda)), "lengths must"),
                       ((x, x, x, h, torch.ones(3, device=cuda).int()), "lengths must"),
                       ((x, x, x, h, torch.ones(2).int()), "lengths must")):
        with pytest.raises(RuntimeError, match=word):
            cpab.gated_recurrence(*args)


def test_empty(cuda):
    for shape in ((0, 5, 4), (2, 0, 4), (2, 5, 0)):
        x = torch.randn(shape, device=cuda).requires_grad_()
        h0 = torch.randn(shape[0], shape[2], device=cuda).requires_grad_()
        y, h = cpab.gated_recurrence(x, x, h0=h0)
        assert y.shape == shape and torch.equal(h, h0) if shape[1] == 0 else y.numel() == 0
        gx, gh = torch.autograd.grad((y, h), (x, h0), (torch.ones_like(y), torch.ones_like(h)))
        assert gx.shape == shape and (gh == 1).all()
    assert np.isfinite(float(h.sum()))

class NoGradient(torch.autograd.Function):
    @staticmethod
    def forward(ctx, *outputs):
        return sum(t.float().sum() for t in outputs)

    @staticmethod
    def backward(ctx, g):
        return (None,) * len(ctx.needs_input_grad)


def test_no_gradient_comes(cuda):
    # what stands behind the outputs has no gradient to give: then neither has the scan
    leaves = [torch.randn(2, 9, 4, device=cuda).requires_grad_() for _ in range(3)]
    leaves.append(torch.randn(2, 4, device=cuda).requires_grad_())
    out = cpab.gated_recurrence(*leaves)
    grads = torch.autograd.grad(NoGradient.apply(*out), leaves, allow_unused=True)
    assert all(g is None for g in grads)
