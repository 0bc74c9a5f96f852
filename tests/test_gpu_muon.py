"""A Muon step against its formula in 64 bits.

Bounds, from the arithmetic.  X and A are held to 22 bits, a product to 2^-21 of its
operands' norms and its sums in 32 bits: each of the three products of a step is off by at
most 2^-20 of what it is made of, which the coefficients' sum, 10.3, weighs: 1e-5 of a
largest singular value that stays below 1.3.  The polynomial's slope, at most 3.5, grows an
error from step to step: 5 steps, 1.3e-5 (1 + 3.5 + ... + 3.5^4) = 2.8e-3 in the worst case,
of any value of X (a value is at most the norm).  That is where all errors align with the
direction that grows most; independent roundings (2^-23 of a value, relative errors grow by
at most |s p'(s) / p(s)| < 3 and by 1 where s is small) leave some 15 x 2^-23 = 2e-6 of the
whole: taken as 1e-5.  The parameter's own rounding is half a unit, and its two products
half a unit each: 2^-22 of the largest of the terms in 32 bits."""
import pytest
import torch

import cpab
import heads_oracle as ho

pytestmark = pytest.mark.gpu
F32, BF16 = torch.float32, torch.bfloat16
C = (3.4445, -4.775, 2.0315)


def make(cuda, dtype, shapes, seed=0, rank=None, masters=False, size=1e-3):
    gen = torch.Generator().manual_seed(seed)
    out = {"params": [], "grads": [], "momenta": [], "masters": [] if masters else None}
    for r, c in shapes:
        w = torch.randn(r, c, generator=gen) * 0.02
        g = torch.randn(r, c, generator=gen)
        if rank:
            g = g * 0.1 + torch.randn(r, rank, generator=gen) @ torch.randn(rank, c, generator=gen)
        out["params"].append(w.to(cuda, dtype))
        out["grads"].append((g * size).to(cuda, dtype))
        out["momenta"].append((torch.randn(r, c, generator=gen) * size).to(cuda))
        if masters:
            out["masters"].append(w.to(cuda))
    return out


def compare(cuda, dtype, shapes, masters=False, seed=0, **kw):
    args = dict(lr=1.0, weight_decay=0.0, momentum=0.95, nesterov=True, ns_coefficients=C, eps=1e-7, ns_steps=5)
    make_kw = {k: kw.pop(k) for k in ("rank", "size") if k in kw}
    args.update(kw)
    st = make(cuda, dtype, shapes, seed, masters=masters, **make_kw)
    values = st["masters"] if masters else st["params"]
    before = [(ho.f64(w), ho.f64(g), ho.f64(m)) for w, g, m in zip(values, st["grads"], st["momenta"])]
    adjust = args.pop("adjust_lr_fn", None)
    cpab.muon_step(st["params"], st["grads"], st["momenta"], masters=st["masters"], adjust_lr_fn=adjust, **args)
    for k, (w, g, m) in enumerate(before):
        rows, cols = w.shape
        if w.numel() == 0:
            continue
        rate = args["lr"] * (0.2 * max(rows, cols) ** 0.5 if adjust == "match_rms_adamw" else max(1.0, rows / cols) ** 0.5)
        want, mom = ho.muon(w, g, m, args["lr"], args["weight_decay"], args["momentum"], args["nesterov"],
                            args["ns_coefficients"], args["eps"], args["ns_steps"], rate)
        got = ho.f64(values[k])
        assert torch.isfinite(got).all()
        off = (got - want).abs()
        unit = 2.0 ** -8 if values[k].dtype == BF16 else 0.0
        assert (off <= 2.8e-3 * rate + 2.0 ** -22 * (w.abs() + want.abs()) + unit * want.abs()).all(), (k, float(off.max()))
        if values[k].dtype == F32:
            # what rounding the parameter itself leaves is not the product's
            rest = float((got - want).norm()) - 2.0 ** -22 * float(w.norm() + want.norm())
            move = float((want - w * (1 - args["lr"] * args["weight_decay"])).norm())
            assert rest <= 1e-5 * move, (k, rest / max(move, 1e-30))
        em = (ho.f64(st["momenta"][k]) - mom).abs()
        assert (em <= 2.0 ** -22 * (m.abs() + g.abs())).all()
        if masters:
            assert torch.equal(st["params"][k], st["masters"][k].to(dtype))


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("shape", [(1, 1), (1, 7), (7, 1), (2, 3), (16, 16), (31, 33), (63, 65), (64, 64), (65, 64),
                                   (49, 200), (200, 49), (128, 300), (257, 129), (1000, 3), (5, 4099)])
def test_shapes(cuda, dtype, shape):
    compare(cuda, dtype, [shape], seed=1)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_many_matrices(cuda, dtype):
    shapes = [(3 * w, w) for w in (5, 17, 64, 100)] + [(64, 64)] * 50 + [(0, 4), (70, 20), (20, 70), (4, 0)]
    compare(cuda, dtype, shapes, seed=2)
    compare(cuda, dtype, [(300, 500), (640, 512), (33, 40)], seed=2)


@pytest.mark.parametrize("shape", [(512, 512), (700, 333), (640, 1900), (1500, 1300)])
def test_large(cuda, shape):
    compare(cuda, F32, [shape], seed=3, rank=3)
    compare(cuda, BF16, [shape], seed=3, masters=True)


@pytest.mark.parametrize("kw", [dict(nesterov=False), dict(momentum=0.0), dict(ns_steps=1), dict(ns_steps=2),
                                dict(ns_steps=8), dict(adjust_lr_fn="match_rms_adamw"), dict(lr=0.02, weight_decay=0.5),
                                dict(ns_coefficients=(1.875, -1.25, 0.375), ns_steps=5), dict(rank=1), dict(rank=5),
                                dict(size=1e-20), dict(size=1e12), dict(size=1e-3, eps=10.0)])
def test_options(cuda, kw):
    for masters in (False, True):
        compare(cuda, BF16 if masters else F32, [(40, 90), (130, 64)], masters=masters, seed=4, **kw)


def test_zero_update_and_not_finite(cuda):
    st = make(cuda, F32, [(20, 30), (20, 30)], seed=5)
    for t in st["grads"] + st["momenta"]:
        t.zero_()
    st["grads"][1][3, 4] = float("nan")
    before = [p.clone() for p in st["params"]]
    cpab.muon_step(st["params"], st["grads"], st["momenta"], lr=0.1, weight_decay=0.0)
    assert torch.equal(st["params"][0], before[0])
    assert torch.isnan(st["params"][1]).all()


def test_layouts(cuda):
    # tensors one after another at any offset; gradients in another order
    sizes = [(3, 5), (70, 33), (64, 64), (1, 9)]
    st = make(cuda, F32, sizes, seed=6)
    want = make(cuda, F32, sizes, seed=6)
    cpab.muon_step(want["params"], want["grads"], want["momenta"])

    def tight(ts):
        flat = torch.cat([ts[0].new_zeros(1)] + [t.flatten() for t in ts])
        out, at = [], 1
        for t in ts:
            out.append(flat[at:at + t.numel()].view(t.shape))
            at += t.numel()
        return out
    params, momenta = tight(st["params"]), tight(st["momenta"])
    grads = [g.T.contiguous().T for g in st["grads"]]
    cpab.muon_step(params, grads, momenta)
    for a, b in zip(params + momenta, want["params"] + want["momenta"]):
        assert torch.equal(a, b)


def test_same_call_same_bits_and_alone(cuda):
    # a matrix's step does not depend on those beside it
    shapes = [(100, 60), (64, 640), (33, 33)]
    one = make(cuda, F32, shapes, seed=7)
    two = make(cuda, F32, shapes, seed=7)
    cpab.muon_step(one["params"], one["grads"], one["momenta"])
    for k in range(3):
        cpab.muon_step(two["params"][k:k + 1], two["grads"][k:k + 1], two["momenta"][k:k + 1])
    for a, b in zip(one["params"], two["params"]):
        assert torch.equal(a, b)


def test_side_stream_and_graph(cuda):
    shapes = [(100, 60), (192, 64), (64, 64)]
    one, two = make(cuda, BF16, shapes, seed=8, masters=True), make(cuda, BF16, shapes, seed=8, masters=True)

    def step(s):
        cpab.muon_step(s["params"], s["grads"], s["momenta"], masters=s["masters"])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(one)
    torch.cuda.current_stream().wait_stream(side)
    step(two)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(one)
    for k in range(4):
        for a, b in zip(one["grads"], two["grads"]):
            new = torch.randn(a.shape, device=cuda) * 1e-3
            a.copy_(new)
            b.copy_(new)
        graph.replay()
        torch.cuda.synchronize()
        step(two)
        for name in ("params", "momenta", "masters"):
            assert all(torch.equal(a, b) for a, b in zip(one[name], two[name])), (k, name)


def test_optimiser(cuda):
    torch.manual_seed(9)
    for dtype in (F32, BF16):
        net = torch.nn.Sequential(torch.nn.Linear(20, 40, bias=False), torch.nn.Linear(40, 8, bias=False)).to(cuda, dtype)
        opt = cpab.Muon(net.parameters(), lr=0.01, weight_decay=0.1)
        values = [p.detach().double().cpu() for p in net.parameters()]
        moms = [torch.zeros_like(v) for v in values]
        for _ in range(3):
            x = torch.randn(16, 20, device=cuda, dtype=dtype)
            opt.zero_grad()
            net(x).float().square().mean().backward()
            grads = [p.grad.double().cpu() for p in net.parameters()]
            opt.step()
            for k, g in enumerate(grads):
                rows, cols = g.shape
                values[k], moms[k] = ho.muon(values[k], g, moms[k], 0.01, 0.1, 0.95, True, C, 1e-7, 5,
                                             0.01 * max(1.0, rows / cols) ** 0.5)
        for k, p in enumerate(net.parameters()):
            state = opt.state[p]
            kept = state.get("master", p.detach()).double().cpu()
            assert ("master" in state) == (dtype == BF16)
            # three steps of 0.01, each within the bound above, and the value's roundings
            assert (kept - values[k]).abs().max() <= 3 * 0.015 * 2.8e-3 + 1e-6
        again = cpab.Muon(net.parameters(), lr=0.5)
        again.load_state_dict(opt.state_dict())
        assert again.param_groups[0]["lr"] == 0.01
        for p in net.parameters():
            for name, t in opt.state[p].items():
                assert again.state[p][name].dtype == F32 and torch.equal(again.state[p][name], t)


def test_changes_are_seen(cuda):
    st = make(cuda, F32, [(8, 8)], seed=10)
    p = st["params"][0]
    x = torch.ones(8, 8, device=cuda, requires_grad=True)
    y = (x * p).sum()
    cpab.muon_step(st["params"], st["grads"], st["momenta"])
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()


def test_refusals(cuda):
    def call(change=None, **kw):
        st = make(cuda, F32, [(8, 9), (9, 8)], seed=11)
        if change:
            change(st)
        before = [t.clone() for t in st["params"] + st["momenta"]]
        try:
            cpab.muon_step(st["params"], st["grads"], st["momenta"], masters=st["masters"], **kw)
        finally:
            now = st["params"] + st["momenta"]
            assert all(torch.equal(a.cpu(), b.cpu()) for a, b in zip(now, before))

    def put(name, k, f):
        def change(st):
            st[name][k] = f(st[name][k])
        return change
    for change, word in ((put("params", 0, lambda t: t.cpu()), "GPU"), (put("params", 0, lambda t: t.double()), "float32 or bfloat16"),
                         (put("params", 1, lambda t: t.bfloat16()), "one type"), (put("params", 1, lambda t: t.T.contiguous().T), "contiguous"),
                         (put("grads", 1, lambda t: t[:3]), "gradient"), (put("grads", 1, lambda t: t.bfloat16()), "gradient"),
                         (put("grads", 0, lambda t: t.to_sparse()), "gradient"), (put("grads", 0, lambda t: t.cpu()), "gradient"),
                         (put("momenta", 0, lambda t: t.bfloat16()), "momentum"), (put("momenta", 1, lambda t: t.T), "momentum"),
                         (put("momenta", 1, lambda t: t.cpu()), "momentum"),
                         (lambda st: st["grads"].pop(), "one entry"),
                         (lambda st: st.update(masters=[torch.zeros(8, 9, device=cuda)]), "one entry"),
                         (lambda st: st.update(masters=[torch.zeros(8, 9, device=cuda), torch.zeros(9, 8, device=cuda).bfloat16()]), "master"),
                         (lambda st: st["params"].__setitem__(1, st["params"][0]) or st["grads"].__setitem__(1, st["grads"][0])
                          or st["momenta"].__setitem__(1, st["momenta"][0].clone()), "twice"),
                         (lambda st: st["momenta"].__setitem__(1, st["params"][0]) or st["params"].__setitem__(1, st["params"][0].clone())
                          or st["grads"].__setitem__(1, st["grads"][0]), "twice")):
        with pytest.raises(RuntimeError, match=word):
            call(change)
    for kw, word in ((dict(lr=-1.0), "lr"), (dict(weight_decay=-1.0), "weight_decay"), (dict(momentum=1.0), "momentum"),
                     (dict(eps=-1.0), "eps"), (dict(ns_steps=0), "ns_steps"), (dict(ns_steps=101), "ns_steps"),
                     (dict(ns_coefficients=(1.0, float("nan"), 0.0)), "coefficients")):
        with pytest.raises(RuntimeError, match=word):
            call(**kw)
    with pytest.raises(AssertionError):
        call(put("params", 0, lambda t: t[0]))
    with pytest.raises(AssertionError):
        call(adjust_lr_fn="other")
    with pytest.raises(AssertionError):
        cpab.Muon([torch.zeros(3, device=cuda, requires_grad=True)])
    with torch.inference_mode():
        made = torch.zeros(8, 9, device=cuda)
    with pytest.raises(RuntimeError, match="inference"):
        call(put("momenta", 0, lambda t: made))
    cpab.muon_step([], [], [])


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_on_both_sides_of_each_way(cuda, dtype):
    # one workgroup up to 64 x 256, then tiles of 64, of 128 past a shorter side of 256 and of
    # 256 past one of 1024; each way's own launches, in one call
    compare(cuda, dtype, [(64, 256), (256, 64), (1, 256), (64, 1), (50, 97), (130, 20)], seed=11)
    compare(cuda, dtype, [(64, 257), (257, 64), (65, 65), (65, 256)], seed=12)
    compare(cuda, dtype, [(256, 256), (256, 700), (257, 257), (1024, 1024), (1025, 1025), (48, 31)], seed=13,
            masters=dtype == BF16)


def test_whole_matrices_same_bits(cuda):
    def run(shapes):
        st = make(cuda, F32, shapes, seed=14)
        cpab.muon_step(st["params"], st["grads"], st["momenta"])
        return st["params"] + st["momenta"]
    a, b = run([(60, 200)] * 50), run([(60, 200)] * 50)
    assert all(torch.equal(x, y) for x, y in zip(a, b))
    # the first alone, and beside one that goes in tiles
    for shapes in ([(60, 200)], [(60, 200), (300, 300)]):
        c = run(shapes)
        assert torch.equal(c[0], a[0])
