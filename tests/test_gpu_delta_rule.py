"""Gated delta rule against its definition in 64 bits, sample by sample.

Bounds, from the arithmetic, with keys of length 1 at most, beta in [0, 1] and decays at
most 1.  u is what an operand is held to: 2^-24 in 32 bits; with 16-bit inputs 2^-16, room for
products whose 32-bit operands go as two 16-bit parts of 8 bits each, the second's rounding
2^-18 of the value and the product of the two second parts, 2^-16, left out.  A dot product
of n values is within n u |a| |b| (Cauchy).  A chunk's inverse has entries of at most 1 (what
a sample writes is at most read again), so that a difference x is within 64 times its
operands' errors.  With N = dk + 64 + 16 >= n and c chunks, whose errors add up at most:
every result is within 64 N c u of the product of the norms that it is a sum of, in which S
and L are the states' and their gradients' largest norms.  In 16 bits the u's own term does
not grow with n as every operand's error is relative: N = 16 there (the products in a row,
twice).  bfloat16 results carry half a unit of their last place, 2^-8 of the value, besides.

Those bounds hold for the worst signs.  A loss of bits everywhere shows in the whole: over a
result's values the roundings are independent, so that n of them leave sqrt(n) u and some ten
stages in a row sqrt(10 n) u < 50 u of the norm, 3e-6 in 32 bits: taken as 1e-5, and as 1e-5
too where a 16-bit part's rounding, 2^-18 / sqrt(3) = 2.2e-6 at a stage, adds to it.  That is
so of many values, whose norm is that of their terms; a few (below 64) can be small beside
their terms by chance.  A term t then still carries u t, and the root of their squares' sum
is at most the product of norms above: sqrt(10) 2.2e-6 = 7e-6 of that, taken as 1e-5."""
import pytest
import torch

import cpab
import heads_oracle as ho

pytestmark = pytest.mark.gpu
F32, BF16 = torch.float32, torch.bfloat16
NAMES = ("q", "k", "v", "decay", "beta", "h0")


def make(cuda, dtype, B, T, H, K, dk, dv, gates=None, start=True, lengths=None, layout="own", seed=0,
         keep=3.0, near=0.5):
    gen = torch.Generator().manual_seed(1000 * seed + 31 * T + dk)
    q, k = torch.randn(B, T, K, dk, generator=gen), torch.randn(B, T, K, dk, generator=gen)
    k = k + near * torch.randn(B, 1, K, dk, generator=gen)
    # a little shorter than 1, so that their rounding does not pass it
    q, k = (0.99 * t / t.norm(dim=-1, keepdim=True).clamp(min=1e-6) for t in (q, k))
    v = torch.randn(B, T, H, dv, generator=gen)
    decay = -torch.nn.functional.softplus(-(torch.randn(B, T, H, generator=gen) +
                                            keep * torch.rand(H, generator=gen)))
    beta = torch.rand(B, T, H, generator=gen)
    if lengths is not None:
        lengths = torch.tensor(lengths)
        pad = torch.arange(T)[None, :] >= lengths.clamp(0, T)[:, None]
        junk = torch.tensor([float("nan"), float("inf"), -float("inf"), 3.4e38])

        def spoiled(t):
            fill = junk[torch.randint(0, 4, t.shape, generator=gen)]
            return torch.where(pad.view(B, T, *[1] * (t.dim() - 2)), fill, t)
        q, k, v, decay, beta = (spoiled(t) for t in (q, k, v, decay, beta))
        lengths = lengths.to(cuda)
    if layout == "packed":
        whole = torch.cat([q.flatten(2), k.flatten(2), v.flatten(2)], -1).to(cuda, dtype)
        n = K * dk
        q, k, v = (whole[..., a:b].unflatten(-1, s) for a, b, s in
                   ((0, n, (K, dk)), (n, 2 * n, (K, dk)), (2 * n, 2 * n + H * dv, (H, dv))))
    else:
        q, k, v = (t.to(cuda, dtype) for t in (q, k, v))
        order = {"time": (0, 1), "head": (1, 2), "width": (2, 3)}.get(layout)
        if order:
            q, k, v = (t.transpose(*order).contiguous().transpose(*order) for t in (q, k, v))
        if layout == "offset":
            q, k, v = (torch.cat([t.new_zeros(1), t.flatten()])[1:].view(t.shape) for t in (q, k, v))
    decay, beta = (t.to(cuda, gates or dtype) for t in (decay, beta))
    if layout == "head":
        decay, beta = (t.transpose(1, 2).contiguous().transpose(1, 2) for t in (decay, beta))
    h0 = torch.randn(B, H, dk, dv, generator=gen).to(cuda) if start else None
    return [q, k, v, decay, beta, h0], lengths


def check(got, want, c, size, what, whole=True):
    bound = c * size
    out = got.dtype
    got = ho.f64(got)
    assert got.shape == want.shape, (what, got.shape, want.shape)
    if got.numel() == 0:
        return
    assert torch.isfinite(got).all(), what
    unit = 2.0 ** -8 if out == BF16 else 0.0
    over = (got - want).abs() - bound - unit * want.abs()
    assert over.max() <= 0, f"{what}: off by {float((got - want).abs().max()):.3g}, {float(over.max()):.3g} too much"
    n = want.numel()
    norm = max(float(want.norm()), size * n ** 0.5 if n < 64 else 0.0)
    rel = float((got - want).norm()) / max(norm, 1e-30)
    if whole and norm > 1e-3 * bound * n ** 0.5:
        assert rel <= (2.0 ** -8 if out == BF16 else 1e-5), f"{what}: {rel:.3g} of the whole"


def zeroed(t, lengths):
    t = ho.f64(t)
    if lengths is None:
        return t
    live = torch.arange(t.shape[1])[None] < lengths.cpu().long()[:, None]
    return torch.where(live.view(*live.shape, *[1] * (t.dim() - 2)), t, torch.zeros(()).double())


def most(t):
    return float(t.norm(dim=-1).max()) if t.numel() else 0.0


def compare(cuda, dtype, B, T, H, K, dk, dv, scale=None, whole=True, given=None, **kw):
    args, lengths = given or make(cuda, dtype, B, T, H, K, dk, dv, **kw)
    with torch.no_grad():
        o_only, h_only = cpab.gated_delta_rule(*args, lengths, scale)
    leaves = [None if t is None else t.detach().requires_grad_() for t in args]
    o, h = cpab.gated_delta_rule(*leaves, lengths, scale)
    assert o.dtype == dtype and h.dtype == F32
    gen = torch.Generator().manual_seed(5)
    do = torch.randn(B, T, H, dv, generator=gen).to(cuda, dtype)
    dh = torch.randn(B, H, dk, dv, generator=gen).to(cuda)
    asked = [t for t in leaves if t is not None]
    grads = dict(zip([n for n, t in zip(NAMES, leaves) if t is not None],
                     torch.autograd.grad((o, h), asked, (do, dh))))
    cl = None if lengths is None else lengths.cpu()
    ref = [zeroed(t, lengths) for t in args[:5]] + [ho.f64(args[5])]
    ro, rh = ho.delta_rule(*ref, cl, scale)
    want, size = ho.delta_rule_grads(*ref, cl, scale, ho.f64(do), ho.f64(dh))
    s = dk ** -0.5 if scale is None else abs(scale)
    S, L = max(size["S"], float(rh.norm(dim=(2, 3)).max()) if rh.numel() else 0.0), size["L"]
    chunks = -(-T // 64)
    c = 64 * chunks * ((dk + 80) * 2.0 ** -24 if dtype == F32 else 16 * 2.0 ** -16)
    Q, K1, V, D = most(ref[0]), most(ref[1]), most(ref[2]), most(ho.f64(do))
    for got, name in ((o, "o"), (o_only, "o alone")):
        check(got, ro, c, s * Q * (S + V), name, whole)
    for got, name in ((h, "h"), (h_only, "h alone")):
        check(got, rh, c, S + V, name, whole)
    M = s * Q * D + L
    check(grads["q"], want["q"], c, s * D * (S + V) * (H // K), "grad q", whole)
    check(grads["k"], want["k"], c, (H // K) * (M * (size["x"] + V + S) + (size["e"] + M) * S), "grad k", whole)
    check(grads["v"], want["v"], c, M, "grad v", whole)
    check(grads["beta"], want["beta"], c, (M + size["e"]) * (V + S + size["x"]), "grad beta", whole)
    check(grads["decay"], want["decay"], c, M * (S + V), "grad decay", whole)
    if "h0" in grads:
        check(grads["h0"], want["h0"], c, M, "grad h0", whole)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("T", [1, 2, 16, 17, 63, 64, 65, 130, 300])
@pytest.mark.parametrize("dk,dv", [(16, 16), (33, 70), (128, 64)])
def test_lengths_and_widths(cuda, dtype, T, dk, dv):
    compare(cuda, dtype, 2, T, 2, 1, dk, dv, seed=1)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("dk,dv", [(1, 1), (2, 200), (31, 32), (32, 31), (64, 33), (65, 128), (100, 5), (127, 129), (128, 257)])
def test_widths(cuda, dtype, dk, dv):
    compare(cuda, dtype, 1, 70, 2, 2, dk, dv, seed=2)
    compare(cuda, dtype, 3, 3, 2, 2, dk, dv, seed=2)


@pytest.mark.parametrize("dtype,gates", [(F32, BF16), (BF16, F32)])
@pytest.mark.parametrize("T", [5, 100])
def test_gates_of_another_type(cuda, dtype, gates, T):
    compare(cuda, dtype, 2, T, 4, 2, 24, 40, gates=gates, seed=3)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("B,T,H,K", [(1, 1, 1, 1), (70, 1, 4, 4), (5, 65, 6, 2), (1, 1000, 3, 1), (9, 20, 8, 1)])
def test_heads_and_rows(cuda, dtype, B, T, H, K):
    compare(cuda, dtype, B, T, H, K, 20, 24, seed=4)


def test_without_start_and_scale(cuda):
    compare(cuda, F32, 2, 80, 2, 2, 32, 32, start=False, seed=5)
    compare(cuda, BF16, 2, 80, 2, 2, 32, 32, start=False, scale=0.7, seed=5)
    compare(cuda, F32, 2, 4, 2, 2, 32, 32, start=False, scale=-1.5, seed=5)


@pytest.mark.parametrize("layout", ["packed", "time", "head", "width", "offset"])
@pytest.mark.parametrize("dtype,dk,dv", [(F32, 32, 32), (BF16, 64, 64), (BF16, 33, 21)])
def test_layouts(cuda, layout, dtype, dk, dv):
    compare(cuda, dtype, 2, 100, 4, 2, dk, dv, layout=layout, seed=6)
    compare(cuda, dtype, 2, 2, 4, 2, dk, dv, layout=layout, seed=6)


def test_samples_far_apart(cuda):
    # as far as the kernels reach, and one value further, where inputs are copied first
    for stride in (4194304, 4194305):
        args, _ = make(cuda, BF16, 1, 3, 1, 1, 8, 8, seed=29)
        want = cpab.gated_delta_rule(*args)
        far = []
        for t in args[:3]:
            room = torch.zeros(2 * stride + 8, device=cuda, dtype=BF16)
            view = room.as_strided((1, 3, 1, 8), (0, stride, 0, 1))
            view.copy_(t)
            far.append(view)
        for grad in (False, True):
            leaves = [t.detach().requires_grad_(grad) for t in (*far, *args[3:])]
            got = cpab.gated_delta_rule(*leaves)
            if not grad:
                assert all(torch.equal(a, b) for a, b in zip(got, want))
            else:
                near = [t.detach().requires_grad_() for t in args]
                ups = [torch.ones_like(t) for t in want]
                a = torch.autograd.grad(got, leaves, ups)
                b = torch.autograd.grad(cpab.gated_delta_rule(*near), near, ups)
                assert all(torch.equal(x, y) for x, y in zip(a, b))


@pytest.mark.parametrize("T", [1, 16, 40, 200])
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("kind", [torch.int32, torch.int64])
def test_ragged_rows(cuda, T, dtype, kind):
    lengths = [0, T, T // 2, 1, min(T, 64), min(T, 65), T + 9, -3, max(0, T - 1), T // 3]
    args, n = make(cuda, dtype, len(lengths), T, 2, 1, 20, 12, lengths=lengths, seed=7)
    n = n.to(kind)
    with torch.no_grad():
        o, h = cpab.gated_delta_rule(*args, n)
    leaves = [t.detach().requires_grad_() for t in args]
    grads = torch.autograd.grad(cpab.gated_delta_rule(*leaves, n), leaves, (torch.ones_like(o), torch.ones_like(h)))
    for b, k in enumerate(lengths):
        k = max(0, min(k, T))
        assert (o[b, k:] == 0).all()
        for g in grads[:5]:
            assert (g[b, k:] == 0).all()
        if k == 0:
            assert torch.equal(h[b], args[5][b]) and (grads[5][b] == 1).all()
    compare(cuda, dtype, len(lengths), T, 2, 1, 20, 12, given=(args, n.clamp(0, T)))


@pytest.mark.parametrize("T", [9, 150])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_cleared_and_kept_states(cuda, dtype, T):
    # decays at both ends: exp(0) = 1, and what clears the state; beta 0 (nothing is
    # written) and 1; the same key again and again
    args, _ = make(cuda, dtype, 2, T, 2, 1, 24, 16, seed=8)
    q, k, v, decay, beta, h0 = args
    compare(cuda, dtype, 2, T, 2, 1, 24, 16, given=([q, k, v, torch.zeros_like(decay), beta, h0], None))
    compare(cuda, dtype, 2, T, 2, 1, 24, 16, given=([q, k, v, decay, torch.zeros_like(beta), h0], None), whole=False)
    compare(cuda, dtype, 2, T, 2, 1, 24, 16, given=([q, k, v, decay, torch.ones_like(beta), h0], None))
    same = k[:, :1].expand_as(k).contiguous()
    compare(cuda, dtype, 2, T, 2, 1, 24, 16, given=([q, same, v, torch.zeros_like(decay), torch.ones_like(beta), h0], None))
    # a state that is cleared: what came before has no part in what comes after
    for low in (-float("inf"), -3e38, -200.0):
        cleared = decay.clone()
        cleared[:, T // 2] = low
        compare(cuda, dtype, 2, T, 2, 1, 24, 16, given=([q, k, v, cleared.clamp(min=-1e30), beta, h0], None))
        o, h = cpab.gated_delta_rule(q, k, v, cleared, beta, h0)
        rest = [t[:, T // 2:] for t in (q, k, v, decay, beta)]
        rest[3] = rest[3].clone()
        rest[3][:, 0] = 0
        leaves = [t.detach().requires_grad_() for t in (q, k, v, cleared, beta, h0)]
        out = cpab.gated_delta_rule(*leaves)
        grads = torch.autograd.grad(out, leaves, (torch.ones_like(out[0]), torch.ones_like(out[1])))
        assert all(torch.isfinite(g).all() for g in grads)
        assert (grads[3][:, T // 2] == 0).all() and torch.isfinite(h).all()
    # cleared at every sample: only the sample itself
    o, h = cpab.gated_delta_rule(q, k, v, torch.full_like(decay, -float("inf")), beta, h0)
    ro, rh = ho.delta_rule(ho.f64(q), ho.f64(k), ho.f64(v), torch.full(decay.shape, -1e4).double(), ho.f64(beta), ho.f64(h0))
    check(o, ro, 1e-3, float(ro.abs().max()), "o cleared")
    check(h, rh, 1e-3, float(rh.abs().max()), "h cleared")


def test_differences_after_a_clearing(cuda):
    # the decays after a cleared state keep their last places
    args, _ = make(cuda, F32, 1, 64, 1, 1, 16, 16, seed=9)
    args[3] = torch.full_like(args[3], -1e-3)
    args[3][:, :40] = -128.0
    compare(cuda, F32, 1, 64, 1, 1, 16, 16, given=(args, None))


def test_not_finite_stays_in_its_row_and_head(cuda):
    for T, t in ((200, 100), (5, 2)):
        args, _ = make(cuda, F32, 2, T, 2, 2, 16, 16, seed=10)
        ref, href = cpab.gated_delta_rule(*args)
        bad = [t.clone() for t in args]
        bad[2][1, t, 1, 3] = float("nan")
        o, h = cpab.gated_delta_rule(*bad)
        assert torch.equal(o[0], ref[0]) and torch.equal(o[1, :, 0], ref[1, :, 0])
        assert torch.equal(h[0], href[0]) and torch.equal(h[1, 0], href[1, 0])
        assert torch.isnan(h[1, 1, :, 3]).all() and torch.isnan(o[1, -1, 1, 3])


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_in_pieces(cuda, dtype):
    # a signal read in pieces, down to single samples: the state handed on is the 32-bit one
    args, _ = make(cuda, dtype, 2, 260, 2, 1, 32, 48, seed=11)
    *inputs, h0 = args
    o, h = cpab.gated_delta_rule(*inputs, h0)
    parts, s, t = [], h0, 0
    for n in (1, 1, 5, 128, 0, 64, 61):
        p, s = cpab.gated_delta_rule(*(x[:, t:t + n] for x in inputs), s)
        parts.append(p)
        t += n
    assert t == 260
    ro, rh = ho.delta_rule(*(ho.f64(x) for x in inputs), ho.f64(h0))
    for got, want in ((s, rh), (h, rh), (torch.cat(parts, 1), ro), (o, ro)):
        check(got, want, 64 * 7 * (112 * 2.0 ** -24 if dtype == F32 else 2.0 ** -12), float(h.norm(dim=(2, 3)).max()) + 10, "piece")


@pytest.mark.parametrize("dtype,B,H,K,T", [(F32, 1, 1, 1, 20011), (BF16, 1, 2, 1, 30001), (BF16, 2, 1, 1, 4095)])
def test_long_rows_in_pieces(cuda, dtype, B, H, K, T):
    # hundreds of chunks of few heads: against the same signal in shorter pieces, whose states
    # and gradients autograd hands on.  Each side is within 1e-5 of the norm (bfloat16 results
    # within half a unit, 2^-8)
    args, _ = make(cuda, dtype, B, T, H, K, 64, 64, gates=F32, seed=12, keep=5.0)
    one = [t.detach().requires_grad_() for t in args]
    o, h = cpab.gated_delta_rule(*one)
    do, dh = torch.randn_like(o), torch.randn_like(h)
    grads = torch.autograd.grad((o, h), one, (do, dh))
    with torch.no_grad():
        alone = cpab.gated_delta_rule(*args)
    two = [t.detach().requires_grad_() for t in args]
    s, parts = two[5], []
    for t in range(0, T, 997):
        p, s = cpab.gated_delta_rule(*(x[:, t:t + 997] for x in two[:5]), s)
        parts.append(p)
    want = torch.autograd.grad((torch.cat(parts, 1), s), two, (do, dh))
    pairs = [(o, torch.cat(parts, 1)), (h, s), (alone[0], torch.cat(parts, 1)), (alone[1], s), *zip(grads, want)]
    for k, (a, b) in enumerate(pairs):
        a, b = a.detach(), b.detach()
        rel = float((a.double() - b.double()).norm() / b.double().norm())
        assert rel <= (2 * 2.0 ** -8 if a.dtype == BF16 else 2e-5), (k, rel)


def test_same_call_same_bits(cuda):
    args, n = make(cuda, BF16, 3, 400, 4, 2, 64, 64, lengths=[400, 133, 250], seed=13)
    leaves = [t.detach().requires_grad_() for t in args]

    def run():
        out = cpab.gated_delta_rule(*leaves, n)
        return (*out, *torch.autograd.grad(out, leaves, [torch.ones_like(t) for t in out]))
    first = run()
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(first, run()))


@pytest.mark.parametrize("T", [3, 70])
def test_gradient_against_differences(cuda, T):
    args, _ = make(cuda, F32, 1, T, 2, 1, 4, 3, seed=14)
    gen = torch.Generator().manual_seed(15)
    do, dh = torch.randn(1, T, 2, 3, generator=gen).to(cuda), torch.randn(1, 2, 4, 3, generator=gen).to(cuda)
    leaves = [t.detach().requires_grad_() for t in args]
    grads = torch.autograd.grad(cpab.gated_delta_rule(*leaves), leaves, (do, dh))

    def loss(given):
        o, h = cpab.gated_delta_rule(*given)
        return float((o.double() * do).sum() + (h.double() * dh).sum())
    step = 2.0 ** -8
    for k, (x, g) in enumerate(zip(args, grads)):
        gen = torch.Generator(device=cuda).manual_seed(k)
        for _ in range(2):   # along directions over all of an input, of length 1
            way = torch.randn(x.shape, device=cuda, generator=gen)
            way = way / way.norm()
            up, down = [t.clone() for t in args], [t.clone() for t in args]
            up[k] += step * way
            down[k] -= step * way
            slope = (loss(up) - loss(down)) / (2 * step)
            exact = float((g.double() * way).sum())
            # the third derivative's step^2 / 6, of some hundred times the slope's own size at
            # most, and the sums' roundings over 2 step
            size = float(g.norm()) + 1.0
            assert abs(slope - exact) < 100 * step ** 2 / 6 * size + 64 * 2.0 ** -24 * size / step, (k, slope, exact)


def test_parts_of_the_gradient(cuda):
    args, _ = make(cuda, F32, 2, 90, 2, 1, 16, 16, seed=16)
    leaves = [t.detach().requires_grad_() for t in args]
    out = cpab.gated_delta_rule(*leaves)
    ups = [torch.randn_like(t) for t in out]
    full = torch.autograd.grad(out, leaves, ups)
    for wanted in ([0], [1], [2], [3], [4], [5], [2, 5], [0, 3]):
        some = [t.detach().requires_grad_(i in wanted) for i, t in enumerate(args)]
        got = torch.autograd.grad(cpab.gated_delta_rule(*some), [some[i] for i in wanted], ups)
        assert all(torch.equal(g, full[i]) for g, i in zip(got, wanted))
    for k in (0, 1):   # one output alone is the other's gradient as zeros
        out = cpab.gated_delta_rule(*leaves)
        got = torch.autograd.grad(out[k], leaves, ups[k])
        out = cpab.gated_delta_rule(*leaves)
        want = torch.autograd.grad(out, leaves, [u if j == k else torch.zeros_like(u) for j, u in enumerate(ups)])
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_broadcast_inputs(cuda):
    args, _ = make(cuda, F32, 2, 80, 2, 1, 16, 16, seed=17)
    small = args[1][:, :1].detach().requires_grad_()
    given = [args[0], small.expand(2, 80, 1, 16), *args[2:]]
    o, h = cpab.gated_delta_rule(*given)
    got, = torch.autograd.grad((o.sum(), h.sum()), small, (torch.ones((), device=cuda),) * 2)
    many = small.detach().expand(2, 80, 1, 16).contiguous().requires_grad_()
    o, h = cpab.gated_delta_rule(args[0], many, *args[2:])
    want, = torch.autograd.grad((o.sum(), h.sum()), many, (torch.ones((), device=cuda),) * 2)
    assert torch.equal(got, want.sum(1, keepdim=True))
    gate = args[3][:1, :1, :1].expand(2, 80, 2)
    a = cpab.gated_delta_rule(*args[:3], gate, *args[4:])
    b = cpab.gated_delta_rule(*args[:3], gate.contiguous(), *args[4:])
    assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_two_calls_at_once_and_side_stream(cuda):
    args, _ = make(cuda, BF16, 2, 300, 4, 2, 64, 64, seed=18)
    other, _ = make(cuda, BF16, 2, 300, 4, 2, 64, 64, seed=19)
    want, want2 = cpab.gated_delta_rule(*args), cpab.gated_delta_rule(*other)
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = []
    for s, a in zip(streams, (args, other)):
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            outs.append([cpab.gated_delta_rule(*a) for _ in range(3)])
    for s in streams:
        s.synchronize()
    for got, w in zip(outs, (want, want2)):
        for o in got:
            assert all(torch.equal(a, b) for a, b in zip(o, w))


@pytest.mark.parametrize("T", [2, 150])
def test_graph_replays(cuda, T):
    args, _ = make(cuda, BF16, 2, T, 4, 2, 32, 32, seed=20)

    def passes(given):
        leaves = [t.detach().requires_grad_() for t in given]
        out = cpab.gated_delta_rule(*leaves)
        return (*out, *torch.autograd.grad(out, leaves, [torch.ones_like(o) for o in out]))

    def serve(given):
        with torch.no_grad():
            return cpab.gated_delta_rule(*given)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        passes(args)
        serve(args)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = (*passes(args), *serve(args))
    for seed in range(21, 25):
        new, _ = make(cuda, BF16, 2, T, 4, 2, 32, 32, seed=seed)
        for a, b in zip(args, new):
            a.copy_(b)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(captured, (*passes(new), *serve(new))))


def test_more_than_32_bits_of_values(cuda):
    # v and o of more than 2^31 values; every row is the same
    B, T, H, dk, dv = 1030, 64, 128, 8, 256
    args, _ = make(cuda, BF16, 1, T, H, 1, dk, dv, start=False, seed=26)
    wide = [t.expand(B, *t.shape[1:]) for t in args[:2]]
    v = args[2].expand(B, T, H, dv).contiguous()
    assert v.numel() > 1 << 31
    gates = [t.expand(B, T, H) for t in args[3:5]]
    with torch.no_grad():
        o, h = cpab.gated_delta_rule(*wide, v, *gates)
        one = cpab.gated_delta_rule(*args[:5])
    assert all(torch.equal(o[b], one[0][0]) for b in (0, 500, B - 1)) and torch.equal(h[-1], one[1][0])


def test_nothing_kept_without_gradients(cuda):
    args, _ = make(cuda, BF16, 2, 200, 2, 2, 64, 64, seed=27)
    o, h = cpab.gated_delta_rule(*args)
    assert o.grad_fn is None and h.grad_fn is None
    with torch.no_grad():
        o, h = cpab.gated_delta_rule(*(t.detach().requires_grad_() for t in args))
    assert o.grad_fn is None and not o.requires_grad


def test_refusals(cuda):
    (q, k, v, decay, beta, h0), _ = make(cuda, F32, 2, 5, 4, 2, 16, 8, seed=28)
    n = torch.tensor([5, 5], device=cuda)
    for args, word in (((q, k, v.cpu(), decay, beta), "GPU"), ((q, k, v.half(), decay, beta), "float32 or bfloat16"),
                       ((q, k, v[0], decay, beta), "v must be"), ((q.bfloat16(), k, v, decay, beta), "q must be"),
                       ((q[:, :, :1], k, v, decay, beta), "k must be"), ((q, k[..., :8], v, decay, beta), "k must be"),
                       ((q[:, :3], k[:, :3], v, decay, beta), "q must be"),
                       ((q, k, v[:, :, :3], decay[..., :3], beta[..., :3]), "multiple"),
                       ((q, k, v, decay[..., :2], beta), "decay"), ((q, k, v, decay.double(), beta), "decay"),
                       ((q, k, v, decay, beta.bfloat16()), "beta"), ((q, k, v, decay, beta.cpu()), "beta"),
                       ((q, k, v, decay, beta, h0.bfloat16()), "h0"), ((q, k, v, decay, beta, h0[:, :2]), "h0"),
                       ((q, k, v, decay, beta, h0.cpu()), "h0"),
                       ((q, k, v, decay, beta, h0, n.float()), "lengths"), ((q, k, v, decay, beta, h0, n[:1]), "lengths"),
                       ((q, k, v, decay, beta, h0, n.cpu()), "lengths"),
                       ((q, k, v, decay, beta, h0, n, float("nan")), "scale")):
        with pytest.raises(RuntimeError, match=word):
            cpab.gated_delta_rule(*args)
    wide = torch.zeros(1, 1, 1, 129, device=cuda)
    for keys in (wide, wide[..., :0]):
        with pytest.raises(RuntimeError, match="from 1 to 128"):
            cpab.gated_delta_rule(keys, keys, v[:1, :1, :1], decay[:1, :1, :1], beta[:1, :1, :1])
    with pytest.raises(RuntimeError, match="no values"):
        cpab.gated_delta_rule(q, k, v[..., :0], decay, beta)
    leaf = v.detach().requires_grad_()
    g, = torch.autograd.grad(cpab.gated_delta_rule(q, k, leaf, decay, beta)[0].sum(), leaf, create_graph=True)
    with pytest.raises(RuntimeError, match="differentiate twice"):
        g.sum().backward()


@pytest.mark.parametrize("B,T,H,K,dk,dv", [(0, 5, 2, 2, 16, 8), (2, 0, 2, 1, 16, 8), (2, 5, 0, 1, 16, 8)])
def test_empty(cuda, B, T, H, K, dk, dv):
    args, _ = make(cuda, F32, B, T, H, K, dk, dv)
    for grad in (False, True):
        leaves = [t.detach().requires_grad_(grad) for t in args]
        o, h = cpab.gated_delta_rule(*leaves)
        assert o.shape == (B, T, H, dv) and h.shape == (B, H, dk, dv)
        if T == 0:
            assert torch.equal(h, args[5])
    grads = torch.autograd.grad((o.sum() + h.sum()), leaves)
    if T == 0:
        assert (grads[5] == 1).all()


def test_no_gradient_comes(cuda):
    args, _ = make(cuda, F32, 2, 70, 2, 1, 16, 8)
    leaves = [t.detach().requires_grad_() for t in args]

    class Nothing(torch.autograd.Function):
        @staticmethod
        def forward(ctx, x):
            return x.sum()

        @staticmethod
        def backward(ctx, g):
            return None
    o, h = cpab.gated_delta_rule(*leaves)
    (Nothing.apply(o) + Nothing.apply(h) + leaves[0].sum()).backward()
    assert leaves[1].grad is None and torch.equal(leaves[0].grad, torch.ones_like(leaves[0]))


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("T", [7, 8, 9])
def test_on_both_sides_of_sample_by_sample(cuda, dtype, T):
    compare(cuda, dtype, 3, T, 4, 2, 40, 72, seed=31)


@pytest.mark.parametrize("dtype,gates", [(F32, F32), (BF16, BF16), (BF16, F32)])
@pytest.mark.parametrize("dk,dv", [(20, 70), (64, 96), (128, 130)])
def test_many_heads_to_a_key(cuda, dtype, gates, dk, dv):
    # three heads of several blocks of columns to each key, rows that end within a chunk or have none
    args, n = make(cuda, dtype, 4, 140, 6, 2, dk, dv, gates=gates, lengths=[140, 0, 64, 77], seed=33)
    compare(cuda, dtype, 4, 140, 6, 2, dk, dv, given=(args, n))


@pytest.mark.parametrize("T", [1000, 1023, 1025, 2100])
def test_segments(cuda, T):
    # where a head's axis begins to be cut, in four to eight pieces
    compare(cuda, F32, 1, T, 2, 1, 32, 40, seed=34)
    compare(cuda, BF16, 2, T, 1, 1, 64, 64, seed=35)
