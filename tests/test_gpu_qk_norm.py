"""Norms of queries and keys with their rotation against the definition in 64 bits.

Bounds, from the arithmetic (u = 2^-24).  The sum of D <= 512 squares: a lane adds at most
16, the lanes 6 more times: 24 u; its root halves that, the division, the root and two
products add 4 u: y before turning is within 16 u, taken as 20 u.  A sine or cosine: the
part of a turn, rounded to 32 bits, is off by u / 2 turns, 3.2 u radians; sincospi by 2 u;
the angle p itself, three roundings in 64 bits, by 3 2^-53 |p|.  Turning adds 3 u of each
product.  So a turned value is within (30 u + 2^-51 |p|) (|a| + |b|).  The gradient turned
back carries as much (10 u, without the norm's), and dx = s (w g - n mean(w g n)) 16 u for s
and 30 u for the mean of D products: 60 u of the sizes of both terms.  The weight's
gradient adds N rows in at most N steps: (N + 60) u of the sum of sizes.
bfloat16 results carry half a unit of their last place, 2^-8 of the value, besides."""
import pytest
import torch

import cpab
import heads_oracle as ho

pytestmark = pytest.mark.gpu
U = ho.U
F32, BF16 = torch.float32, torch.bfloat16


def make(cuda, dtype, B, T, H, K, D, wtype=None, layout="own", seed=0, size=1.0):
    gen = torch.Generator().manual_seed(100 * seed + 7 * D + T)
    q, k = (torch.randn(B, T, n, D, generator=gen) * size for n in (H, K))
    if layout == "packed":
        whole = torch.cat([q.flatten(2), k.flatten(2)], -1).to(cuda, dtype)
        q, k = whole[..., :H * D].unflatten(-1, (H, D)), whole[..., H * D:].unflatten(-1, (K, D))
    else:
        q, k = q.to(cuda, dtype), k.to(cuda, dtype)
        if layout == "time":      # [T, B, H, D] in memory
            q, k = (t.transpose(0, 1).contiguous().transpose(0, 1) for t in (q, k))
        elif layout == "head":    # [B, H, T, D] in memory
            q, k = (t.transpose(1, 2).contiguous().transpose(1, 2) for t in (q, k))
        elif layout == "width":   # the width not contiguous
            q, k = (t.transpose(2, 3).contiguous().transpose(2, 3) for t in (q, k))
        elif layout == "offset":  # aligned to a value alone
            q, k = (torch.cat([t.new_zeros(1), t.flatten()])[1:].view(t.shape) for t in (q, k))
    w = [(1 + 0.2 * torch.randn(D, generator=gen)).to(cuda, wtype or dtype) for _ in range(2)]
    return q, k, w[0], w[1]


def check(got, want, bound, what):
    got = ho.f64(got)
    assert got.shape == want.shape, (what, got.shape, want.shape)
    if got.numel() == 0:
        return
    assert torch.isfinite(got).all(), what
    over = (got - want).abs() - torch.as_tensor(bound)
    assert over.max() <= 0, f"{what}: off by {float((got - want).abs().max()):.3g}, {float(over.max()):.3g} too much"


def beside(x, R, neighbours):
    """For each value of x >= 0: its own and, where it turns, its pair's added."""
    out = x.clone()
    a, b = ho.pairs(R, neighbours)
    out[..., a] = out[..., b] = x[..., a] + x[..., b]
    return out


def compare(cuda, dtype, B, T, H, K, D, R, neighbours=False, positions=None, eps=1e-6, **kw):
    given = [t.detach().requires_grad_() for t in make(cuda, dtype, B, T, H, K, D, **kw)]
    gen = torch.Generator().manual_seed(3)
    freqs = None
    if R:
        freqs = (10000.0 ** (-torch.arange(0, R, 2) / R)).to(cuda)
    out = cpab.qk_norm(*given, freqs=freqs, positions=positions, neighbours=neighbours, eps=eps)
    ups = [torch.randn(t.shape, generator=gen).to(cuda, dtype) for t in out]
    grads = torch.autograd.grad(out, given, ups)
    P, Fq = ho.f64(positions), ho.f64(freqs)
    angle = torch.zeros(B, T)
    if R:
        p = torch.arange(T).expand(B, T) if P is None else P.expand(B, T)
        angle = p.abs() * float(Fq.abs().max())
    angle = angle[:, :, None, None].double() * 2.0 ** -51
    unit = ho.UNIT[dtype] if dtype != F32 else 0.0
    for side in (0, 1):
        x, w, g = ho.f64(given[side]), ho.f64(given[2 + side]), ho.f64(ups[side])
        assert out[side].dtype == dtype and out[side].is_contiguous()
        s = 1 / torch.sqrt((x * x).mean(-1, keepdim=True) + eps)
        n = x * s
        y = ho.turned(n * w, Fq, P, neighbours)
        check(out[side], y, (30 * U + angle) * beside((n * w).abs(), R, neighbours) + unit * y.abs() + 1e-37,
              f"y {side}")
        g_back = ho.turned(g, Fq, P, neighbours, -1.0)
        eg = (10 * U + angle) * beside(g.abs(), R, neighbours)
        u, eu = g_back * w, eg * w.abs()
        dx = s * (u - n * (u * n).mean(-1, keepdim=True))
        size = u.abs() + n.abs() * (u * n).abs().mean(-1, keepdim=True)
        err = eu + n.abs() * (eu * n.abs()).mean(-1, keepdim=True)
        check(grads[side], dx, s * (60 * U * size + err) + unit * dx.abs() + 1e-37, f"dx {side}")
        dw = (g_back * n).sum((0, 1, 2))
        rows = x[..., 0].numel()
        wunit = ho.UNIT[given[2].dtype] if given[2].dtype != F32 else 0.0
        check(grads[2 + side], dw, (eg * n.abs()).sum((0, 1, 2)) +
              (rows + 60) * U * (g_back * n).abs().sum((0, 1, 2)) + wunit * dw.abs() + 1e-37, f"dw {side}")


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("neighbours", [False, True])
@pytest.mark.parametrize("D,R", [(1, 0), (2, 2), (3, 2), (7, 4), (8, 8), (16, 16), (32, 8), (50, 24), (64, 64), (65, 64),
                                 (96, 32), (128, 128), (200, 100), (255, 254), (257, 128), (511, 510), (512, 512)])
def test_widths(cuda, dtype, neighbours, D, R):
    compare(cuda, dtype, 2, 5, 3, 2, D, R, neighbours)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("B,T,H,K,D", [(1, 1, 1, 1, 64), (64, 1, 8, 2, 64), (3, 700, 5, 1, 32), (1, 4099, 2, 2, 8),
                                       (1, 3, 200, 7, 16)])
def test_sizes(cuda, dtype, B, T, H, K, D):
    compare(cuda, dtype, B, T, H, K, D, D, seed=1)


@pytest.mark.parametrize("layout", ["packed", "time", "head", "width", "offset"])
@pytest.mark.parametrize("dtype,D", [(F32, 64), (BF16, 64), (BF16, 33)])
def test_layouts(cuda, layout, dtype, D):
    compare(cuda, dtype, 3, 20, 4, 2, D, D // 4 * 2, layout=layout, seed=2)


@pytest.mark.parametrize("kind", [torch.int32, torch.int64, torch.float32])
def test_positions(cuda, kind):
    B, T = 3, 11
    near = torch.arange(B * T, device=cuda).view(B, T)
    compare(cuda, F32, B, T, 2, 1, 24, 16, positions=(near * 7 - 100).to(kind))
    compare(cuda, F32, B, T, 2, 1, 24, 16, positions=(near[0] * 7).to(kind))          # [T]
    compare(cuda, F32, B, T, 2, 1, 24, 16, positions=near[:, :1].to(kind))            # [B, 1]
    compare(cuda, F32, B, T, 2, 1, 24, 16, positions=(near.T.contiguous().T * 3).to(kind))
    # far ones, whose product with a frequency 32 bits do not hold
    compare(cuda, F32, B, T, 2, 1, 24, 16, positions=(near * 8 + (1 << 30)).to(kind))
    if kind == torch.float32:
        compare(cuda, F32, B, T, 2, 1, 24, 16, positions=near.float() * 0.37)


@pytest.mark.parametrize("dtype,wtype", [(F32, BF16), (BF16, F32)])
def test_weights_of_another_type(cuda, dtype, wtype):
    compare(cuda, dtype, 2, 30, 3, 2, 40, 20, wtype=wtype)


def test_small_and_large_rows(cuda):
    compare(cuda, F32, 1, 4, 2, 2, 16, 8, size=1e-12)
    compare(cuda, F32, 1, 4, 2, 2, 16, 8, size=1e15)
    q, k, w, v = make(cuda, F32, 1, 4, 2, 2, 16)
    out = cpab.qk_norm(torch.zeros_like(q), k, w, v)
    assert (out[0] == 0).all()
    bad = q.clone()
    bad[0, 2, 1, 5] = float("nan")
    a, b = cpab.qk_norm(q, k, w, v), cpab.qk_norm(bad, k, w, v)
    hit = torch.zeros(1, 4, 2, 16, dtype=torch.bool, device=cuda)
    hit[0, 2, 1] = True
    assert torch.isnan(b[0][hit]).all() and torch.equal(a[0][~hit], b[0][~hit]) and torch.equal(a[1], b[1])


def test_one_sample_at_a_time(cuda):
    # as signals arrive: each sample with its position, bit for bit as the whole
    q, k, w, v = make(cuda, BF16, 3, 9, 4, 2, 64)
    freqs = torch.linspace(1, 0.01, 32, device=cuda)
    whole = cpab.qk_norm(q, k, w, v, freqs)
    for t in range(9):
        at = torch.full((3, 1), t, device=cuda)
        part = cpab.qk_norm(q[:, t:t + 1], k[:, t:t + 1], w, v, freqs, at)
        assert all(torch.equal(a, b[:, t:t + 1]) for a, b in zip(part, whole))


def test_gradient_against_differences(cuda):
    given = [t.double() for t in make(cuda, F32, 1, 3, 2, 1, 6)]
    freqs = torch.tensor([1.0, 0.3], device=cuda)
    gen = torch.Generator().manual_seed(9)
    ups = [torch.randn(1, 3, n, 6, generator=gen).to(cuda) for n in (2, 1)]

    def loss(args):
        out = cpab.qk_norm(*(a.float() for a in args), freqs)
        return sum(float((o.double() * u).sum()) for o, u in zip(out, ups))

    leaves = [t.float().requires_grad_() for t in given]
    grads = torch.autograd.grad(cpab.qk_norm(*leaves, freqs), leaves, ups)
    h = 2.0 ** -7
    for t, g in zip(given, grads):
        for i in range(0, t.numel(), 3):
            up, down = t.clone(), t.clone()
            up.view(-1)[i] += h
            down.view(-1)[i] -= h
            args = [[up if a is t else a for a in given], [down if a is t else a for a in given]]
            slope = (loss(args[0]) - loss(args[1])) / (2 * h)
            # h^2 / 6 of a third derivative below 60 here, and 36 values' roundings over 2 h
            assert abs(slope - float(g.view(-1)[i])) < 60 * h * h / 6 + 36 * 4 * U * 4 / (2 * h) + 1e-3


def test_parts_of_the_gradient(cuda):
    args = make(cuda, F32, 2, 9, 3, 2, 20)
    freqs = torch.linspace(1, 0.1, 5, device=cuda)
    leaves = [t.detach().requires_grad_() for t in args]
    out = cpab.qk_norm(*leaves, freqs)
    ups = [torch.randn_like(o) for o in out]
    full = torch.autograd.grad(out, leaves, ups)
    for wanted in ([0], [1], [2], [3], [0, 3], [1, 2]):
        some = [t.detach().requires_grad_(i in wanted) for i, t in enumerate(args)]
        got = torch.autograd.grad(cpab.qk_norm(*some, freqs), [some[i] for i in wanted], ups)
        assert all(torch.equal(g, full[i]) for g, i in zip(got, wanted))
    # one output alone
    leaves = [t.detach().requires_grad_() for t in args]
    q, k = cpab.qk_norm(*leaves, freqs)
    got = torch.autograd.grad(q, leaves, ups[0])
    assert torch.equal(got[0], full[0]) and torch.equal(got[2], full[2])
    assert (got[1] == 0).all() and (got[3] == 0).all()


def test_broadcast_inputs(cuda):
    # one query for all samples: autograd adds its gradients up
    q, k, w, v = make(cuda, F32, 2, 6, 2, 2, 16)
    one = q[:, :1].detach().requires_grad_()
    out, _ = cpab.qk_norm(one.expand(2, 6, 2, 16), k, w, v, torch.ones(4, device=cuda))
    up = torch.randn_like(out)
    got, = torch.autograd.grad(out, one, up)
    many = one.detach().expand(2, 6, 2, 16).contiguous().requires_grad_()
    out, _ = cpab.qk_norm(many, k, w, v, torch.ones(4, device=cuda))
    want, = torch.autograd.grad(out, many, up)
    assert torch.equal(got, want.sum(1, keepdim=True))


def test_same_call_same_bits(cuda):
    given = [t.detach().requires_grad_() for t in make(cuda, BF16, 4, 500, 6, 2, 64)]
    freqs = torch.linspace(1, 0.01, 32, device=cuda)

    def run():
        out = cpab.qk_norm(*given, freqs)
        return (*out, *torch.autograd.grad(out, given, [torch.ones_like(o) for o in out]))
    first = run()
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(first, run()))


def test_side_stream_and_graph(cuda):
    q, k, w, v = make(cuda, BF16, 2, 40, 4, 2, 64)
    freqs = torch.linspace(1, 0.01, 32, device=cuda)
    at = torch.arange(40, device=cuda)
    want = cpab.qk_norm(q, k, w, v, freqs, at)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        got = cpab.qk_norm(q, k, w, v, freqs, at)
    stream.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))

    def passes(*args):
        leaves = [t.detach().requires_grad_() for t in args]
        out = cpab.qk_norm(*leaves, freqs, at)
        return (*out, *torch.autograd.grad(out, leaves, [torch.ones_like(o) for o in out]))
    with torch.cuda.stream(stream):
        passes(q, k, w, v)
    torch.cuda.current_stream().wait_stream(stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = passes(q, k, w, v)
    for seed in range(3):
        new = make(cuda, BF16, 2, 40, 4, 2, 64, seed=seed + 5)
        for a, b in zip((q, k, w, v), new):
            a.copy_(b)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(captured, passes(*new)))


def test_more_than_32_bits_of_values(cuda):
    B, T, H, D = 1, 8192, 64, 512
    q = torch.randn(B, 1, H, D, device=cuda, dtype=BF16).expand(B, 2 * T, H, D)
    w = torch.ones(D, device=cuda, dtype=BF16)
    freqs = torch.zeros(D // 2, device=cuda)
    big = torch.empty(9 * T, H, D, device=cuda, dtype=BF16)   # 2.4e9 values
    big.copy_(q[0, :1].expand(9 * T, H, D))
    out, _ = cpab.qk_norm(big[None], big[None, :, :1], w, w, freqs)
    assert out.numel() > 1 << 31
    assert torch.equal(out[0, -1], out[0, 0]) and torch.equal(out[0, 5 * T], out[0, 0])


def test_refusals(cuda):
    q, k, w, v = make(cuda, F32, 2, 5, 3, 2, 16)
    freqs = torch.ones(4, device=cuda)
    at = torch.arange(5, device=cuda)
    for args, word in (((q.cpu(), k, w, v), "GPU"), ((q.half(), k, w, v), "float32 or bfloat16"),
                       ((q[0], k, w, v), "q must be"), ((q, k.bfloat16(), w, v), "k must be"),
                       ((q, k[:, :4], w, v), "k must be"), ((q, k[..., :8], w, v), "k must be"),
                       ((q, k, w[:8], v), "q_weight"), ((q, k, w, v.bfloat16()), "k_weight"),
                       ((q, k, w, v.cpu()), "k_weight"),
                       ((q, k, w, v, torch.ones(9, device=cuda)), "freqs"),
                       ((q, k, w, v, freqs.double()), "freqs"), ((q, k, w, v, freqs.cpu()), "freqs"),
                       ((q, k, w, v, freqs.clone().requires_grad_()), "no gradient"),
                       ((q, k, w, v, None, at), "without freqs"),
                       ((q, k, w, v, freqs, at.double()), "positions"), ((q, k, w, v, freqs, at[:3]), "positions"),
                       ((q, k, w, v, freqs, at.cpu()), "positions"),
                       ((q, k, w, v, freqs, at.float().requires_grad_()), "no gradient"),
                       ((q, k, w, v, freqs, at, False, -1.0), "eps")):
        with pytest.raises(RuntimeError, match=word):
            cpab.qk_norm(*args)
    wide = torch.zeros(1, 1, 1, 513, device=cuda)
    with pytest.raises(RuntimeError, match="width"):
        cpab.qk_norm(wide, wide, wide[0, 0, 0], wide[0, 0, 0])
    leaf = q.detach().requires_grad_()
    g, = torch.autograd.grad(cpab.qk_norm(leaf, k, w, v)[0].sum(), leaf, create_graph=True)
    with pytest.raises(RuntimeError, match="differentiate twice"):
        g.sum().backward()


def test_empty(cuda):
    for B, T, H, K in ((0, 3, 2, 2), (2, 0, 2, 2), (2, 3, 0, 1), (2, 3, 1, 0)):
        given = [t.detach().requires_grad_() for t in make(cuda, F32, B, T, H, K, 16)]
        out = cpab.qk_norm(*given, torch.ones(4, device=cuda))
        assert out[0].shape == (B, T, H, 16) and out[1].shape == (B, T, K, 16)
        grads = torch.autograd.grad([o.sum() for o in out], given)
        if B * T * H == 0:
            assert (grads[2] == 0).all()
        if B * T * K == 0:
            assert (grads[3] == 0).all()


def test_no_gradient_comes(cuda):
    given = [t.detach().requires_grad_() for t in make(cuda, F32, 2, 3, 2, 2, 16)]

    class Nothing(torch.autograd.Function):
        @staticmethod
        def forward(ctx, x):
            return x.sum()

        @staticmethod
        def backward(ctx, g):
            return None
    q, k = cpab.qk_norm(*given)
    (Nothing.apply(q) + Nothing.apply(k) + given[0].sum()).backward()
    assert given[1].grad is None and torch.equal(given[0].grad, torch.ones_like(given[0]))
