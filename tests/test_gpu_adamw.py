"""AdamW over many tensors against its definition in 64 bits.

Bounds, from the arithmetic (u = 2^-24): m and v are two products and a sum, 3 u of the
sum of the terms' sizes; the update is a quotient of things a few roundings each, 12 u of
its value besides what m and v bring; the weight 2 u.  8-bit states are one of the two
values of 3 bits of mantissa around the 64-bit result, the one that the random bits say
except where the 32-bit result lies within a few u of their threshold."""
import numpy as np
import pytest
import torch

import cpab
import sequence_oracle as so

pytestmark = pytest.mark.gpu
U = so.U
F32, BF16, E4M3, E8M0 = torch.float32, torch.bfloat16, torch.float8_e4m3fn, torch.float8_e8m0fnu
BETAS, LR, EPS, WD = (0.9, 0.999), 1e-2, 1e-8, 0.1


def n64(t):
    return t.detach().double().cpu().numpy().reshape(-1)


def tensors(cuda, sizes, dtype, seed, master=False):
    gen = torch.Generator().manual_seed(seed)
    out = []
    for s in sizes:
        w = torch.randn(s, generator=gen)
        d = {"master": w.to(cuda) if master else None, "p": w.to(dtype).to(cuda),
             "g": (torch.randn(s, generator=gen) * torch.exp(2 * torch.randn(s, generator=gen))).to(dtype).to(cuda),
             "m": torch.randn(s, generator=gen).to(cuda), "v": torch.rand(s, generator=gen).to(cuda)}
        out.append(d)
    return out


def check_step(got, want, old, g, step, unit=0.0):
    """got, want: (p, m, v); old the same before."""
    m, v = want[1], want[2]
    em = 3 * U * (np.abs(BETAS[0] * old[1]) + np.abs((1 - BETAS[0]) * g))
    ev = 4 * U * np.abs(v)
    assert (np.abs(got[1] - m) <= em + 1e-40).all() and (np.abs(got[2] - v) <= ev + 1e-40).all()
    root = np.sqrt(v / (1 - BETAS[1] ** step)) + EPS
    upd = LR * np.abs(m) / (1 - BETAS[0] ** step) / root
    bound = 16 * U * upd + LR / (1 - BETAS[0] ** step) * em / root + 3 * U * np.abs(old[0]) + unit * np.abs(want[0])
    assert (np.abs(got[0] - want[0]) <= bound + 1e-40).all(), float(np.max(np.abs(got[0] - want[0]) - bound))


@pytest.mark.parametrize("dtype,master", [(F32, False), (BF16, False), (BF16, True), (F32, True)])
@pytest.mark.parametrize("step", [1, 7, 100000])
def test_32_bit_states(cuda, dtype, master, step):
    sizes = [(1,), (31,), (32,), (33,), (4, 5, 6), (255,), (1024,), (70, 1001), (0,), (65537,), ()]
    ts = tensors(cuda, sizes, dtype, 1, master)
    old = [[n64(t["master"] if master else t["p"]), n64(t["m"]), n64(t["v"])] for t in ts]
    cpab.adamw_step([t["p"] for t in ts], [t["g"] for t in ts], [t["m"] for t in ts], [t["v"] for t in ts],
                    step, LR, BETAS, EPS, WD, masters=[t["master"] for t in ts] if master else None)
    for t, o in zip(ts, old):
        g = n64(t["g"])
        want = so.adamw(*[o[0], g, o[1], o[2]], step, LR, BETAS, EPS, WD)
        p = n64(t["master"] if master else t["p"])
        unit = 2.0 ** -8 if dtype == BF16 and not master else 0.0
        check_step((p, n64(t["m"]), n64(t["v"])), want, o, g, step, unit)
        if master:
            assert torch.equal(t["p"], t["master"].to(dtype))


def states8(cuda, t):
    """8-bit states of the tensors' m and sqrt(v), through the oracle's rounding."""
    for name, full in (("m", n64(t["m"])), ("v", np.sqrt(n64(t["v"])))):
        z, s = so.mx_round(full, np.full(full.shape, 0x8000))
        t[name + "8"] = torch.tensor(z, dtype=F32, device=cuda).to(E4M3)
        t[name + "s"] = torch.tensor(np.log2(s) + 127, device=cuda).round().to(torch.uint8).view(E8M0)


@pytest.mark.parametrize("dtype,master", [(F32, False), (BF16, False), (BF16, True)])
@pytest.mark.parametrize("step", [1, 50])
def test_8_bit_states(cuda, dtype, master, step):
    sizes = [(1,), (31,), (32,), (33,), (9, 7), (256,), (1023,), (40, 1001), (0,), (65537,)]
    ts = tensors(cuda, sizes, dtype, 2, master)
    ts[3]["g"].zero_()
    ts[4]["m"].zero_()
    ts[4]["g"].zero_()
    ts[4]["v"].zero_()
    for t in ts:
        states8(cuda, t)
    old = [[n64(t["master"] if master else t["p"]), so.mx_values(t["m8"], t["ms"]),
            so.mx_values(t["v8"], t["vs"]) ** 2] for t in ts]
    seed = 0xC0FFEE
    cpab.adamw_step([t["p"] for t in ts], [t["g"] for t in ts], [t["m8"] for t in ts], [t["v8"] for t in ts],
                    step, LR, BETAS, EPS, WD, [t["ms"] for t in ts], [t["vs"] for t in ts],
                    [t["master"] for t in ts] if master else None, seed)
    differ = total = 0
    for k, (t, o) in enumerate(zip(ts, old)):
        g = n64(t["g"])
        want = so.adamw(o[0], g, o[1], o[2], step, LR, BETAS, EPS, WD)
        p = n64(t["master"] if master else t["p"])
        check_step((p, want[1], want[2]), want, o, g, step, 2.0 ** -8 if dtype == BF16 and not master else 0.0)
        if master:
            assert torch.equal(t["p"], t["master"].to(dtype))
        bits = so.random_bits(len(g), seed, step, k)
        for name, full, part, least in (("m", want[1], bits & 0xFFFF, False),
                                        ("v", np.sqrt(want[2]), bits >> 16, True)):
            z, s = so.mx_round(full, part.astype(np.float64), least)
            got = so.mx_values(t[name + "8"], t[name + "s"])
            ref = z * np.repeat(s, 32)[:len(z)]
            # never further off than a step of the value's own spacing
            step_size = np.maximum(2.0 ** -9 * np.repeat(s, 32)[:len(z)], 2.0 ** -3 * np.abs(full))
            assert (np.abs(got - full) <= step_size * 1.001 + 1e-45).all()
            differ += int((got != ref).sum())
            total += len(z)
    assert differ <= 1e-3 * total, (differ, total)
    assert (ts[4]["v8"].float() == 0).all() and (ts[4]["m8"].float() == 0).all()


def test_random_rounding_is_fair(cuda):
    # over 400 seeds the mean of a state is the value itself: a value x between two
    # codes d apart has a standard deviation of at most d / 2, the mean of 400 d / 40;
    # 6 of those, over a few thousand values
    n = 4096
    gen = torch.Generator().manual_seed(3)
    g = torch.randn(n, generator=gen).to(cuda)
    sums = {"m": 0.0, "v": 0.0}
    for seed in range(400):
        m8, v8 = (torch.zeros(n, dtype=torch.uint8, device=cuda).view(E4M3) for _ in range(2))
        ms, vs = (torch.zeros(n // 32, dtype=torch.uint8, device=cuda).view(E8M0) for _ in range(2))
        p = torch.zeros(n, device=cuda)
        cpab.adamw_step([p], [g], [m8], [v8], 1, LR, BETAS, EPS, WD, [ms], [vs], seed=seed)
        sums["m"] = sums["m"] + so.mx_values(m8, ms)
        sums["v"] = sums["v"] + so.mx_values(v8, vs)
    G = n64(g)
    for name, x in (("m", 0.1 * G), ("v", np.sqrt(0.001 * G * G))):
        scale = np.repeat(so.mx_scale(x), 32)
        d = np.maximum(2.0 ** -9 * scale, 2.0 ** -3 * np.abs(x))
        fine = np.abs(x) > 2.0 ** -9 * scale       # below it a root is held at the smallest code
        assert (np.abs(sums[name] / 400 - x)[fine] <= 6 * d[fine] / 40).all()
        # and none lean one way: the mean of the errors in units of d, over all values
        lean = ((sums[name] / 400 - x) / d)[fine].mean()
        assert abs(lean) <= 6 * 0.5 / np.sqrt(400 * fine.sum()), (name, lean)


def test_small_roots_are_not_lost(cuda):
    # a value whose second moment is far below its group's: the root is held at the
    # smallest code, so that the step stays of the learning rate's size
    n = 64
    g = torch.full((n,), 1e-9, device=cuda)
    g[0] = 1.0
    m8, v8 = (torch.zeros(n, dtype=torch.uint8, device=cuda).view(E4M3) for _ in range(2))
    ms, vs = (torch.zeros(2, dtype=torch.uint8, device=cuda).view(E8M0) for _ in range(2))
    p = torch.zeros(n, device=cuda)
    for step in range(1, 30):
        cpab.adamw_step([p], [g], [m8], [v8], step, LR, BETAS, EPS, 0.0, [ms], [vs], seed=step)
        assert (v8.float()[1:32] > 0).all()
        assert (p.abs() <= 1.1 * LR * step).all()


def test_not_finite_gradients(cuda):
    # 32 bits: the value's own; 8 bits: the value alone, not those that share its scale
    n = 96
    g = torch.randn(n, device=cuda)
    g[5], g[40], g[70] = float("nan"), float("inf"), 3e38
    m, v, p = (torch.zeros(n, device=cuda) for _ in range(3))
    cpab.adamw_step([p], [g], [m], [v], 1)
    bad = torch.zeros(n, dtype=torch.bool, device=cuda)
    bad[[5, 40]] = True
    assert torch.isnan(p[bad]).all() and torch.isfinite(p[~bad]).all()
    m8, v8 = (torch.zeros(n, dtype=torch.uint8, device=cuda).view(E4M3) for _ in range(2))
    ms, vs = (torch.zeros(3, dtype=torch.uint8, device=cuda).view(E8M0) for _ in range(2))
    q = torch.zeros(n, device=cuda)
    cpab.adamw_step([q], [g], [m8], [v8], 1, exp_avg_scales=[ms], exp_avg_sq_scales=[vs])
    assert torch.equal(torch.isnan(q), bad) and torch.equal(p[~bad], q[~bad])
    assert torch.equal(torch.isnan(m8.float()), bad)
    bad[70] = True                                   # its square is not finite
    assert torch.equal(torch.isnan(v8.float()), bad)


def test_layouts(cuda):
    gen = torch.Generator().manual_seed(5)
    base = torch.randn(6, 4, 5, 3, generator=gen).to(cuda)
    grad = torch.randn(6, 4, 5, 3, generator=gen).to(cuda)
    plain = [base.clone(), torch.zeros_like(base), torch.zeros_like(base)]
    cpab.adamw_step([plain[0]], [grad], [plain[1]], [plain[2]], 1, LR)
    last = [t.contiguous(memory_format=torch.channels_last) for t in (base, torch.zeros_like(base), torch.zeros_like(base))]
    for g in (grad, grad.contiguous(memory_format=torch.channels_last)):
        p, m, v = (t.clone(memory_format=torch.preserve_format) for t in last)
        cpab.adamw_step([p], [g], [m], [v], 1, LR)
        assert torch.equal(p, plain[0]) and torch.equal(m, plain[1]) and torch.equal(v, plain[2])
    # a transposed parameter with a gradient that is one number, expanded
    p = base[0, :, :, 0].clone().t()
    m, v = (torch.zeros_like(p, memory_format=torch.preserve_format) for _ in range(2))
    q, a, b = p.contiguous(), torch.zeros(5, 4, device=cuda), torch.zeros(5, 4, device=cuda)
    one = torch.ones((), device=cuda)
    cpab.adamw_step([p], [one.expand(5, 4)], [m], [v], 1, LR)
    cpab.adamw_step([q], [torch.ones(5, 4, device=cuda)], [a], [b], 1, LR)
    assert torch.equal(p, q) and torch.equal(m, a)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("bits", [32, 8])
def test_many_tensors_at_any_offset(cuda, dtype, bits):
    # 700 tensors one after another in one buffer: several launches, every alignment;
    # each as a call of its own gives it (the random bits go by its place in the list,
    # so in 8 bits that is compared through the weights alone)
    gen = torch.Generator().manual_seed(6)
    sizes = [int(s) for s in torch.randint(0, 700, (700,), generator=gen)]
    total = sum(sizes)
    flat = {k: torch.randn(total, generator=gen).to(dtype).to(cuda) for k in ("p", "g")}
    guard = flat["p"].clone()
    at = np.concatenate([[0], np.cumsum(sizes)])

    def views(t):
        return [t[a:b] for a, b in zip(at[:-1], at[1:])]

    def fresh():
        if bits == 32:
            return [[torch.zeros(n, device=cuda) for n in sizes] for _ in range(2)] + [None, None]
        return ([[torch.zeros(n, dtype=torch.uint8, device=cuda).view(E4M3) for n in sizes] for _ in range(2)]
                + [[torch.zeros(-(-n // 32), dtype=torch.uint8, device=cuda).view(E8M0) for n in sizes] for _ in range(2)])
    m, v, ms, vs = fresh()
    cpab.adamw_step(views(flat["p"]), views(flat["g"]), m, v, 1, LR, BETAS, EPS, WD, ms, vs)
    for k in range(0, 700, 37):
        p = views(guard)[k].clone()
        a, b, c, d = ([x[k]] if x is not None else None for x in fresh())
        cpab.adamw_step([p], [views(flat["g"])[k].clone()], a, b, 1, LR, BETAS, EPS, WD, c, d)
        assert torch.equal(p, views(flat["p"])[k]), k
        if bits == 32:
            assert torch.equal(a[0], m[k]) and torch.equal(b[0], v[k])


def test_more_than_32_bits_of_values(cuda):
    n = 2 ** 31 + 12345
    p = torch.ones(n, device=cuda, dtype=BF16)
    g = torch.ones(n, device=cuda, dtype=BF16)
    m8, v8 = (torch.zeros(n, dtype=torch.uint8, device=cuda).view(E4M3) for _ in range(2))
    ms, vs = (torch.zeros(-(-n // 32), dtype=torch.uint8, device=cuda).view(E8M0) for _ in range(2))
    cpab.adamw_step([p], [g], [m8], [v8], 1, 0.5, BETAS, EPS, 0.0, [ms], [vs])
    for part in (slice(0, 100), slice(2 ** 31 - 50, 2 ** 31 + 50), slice(n - 100, n)):
        assert (p[part] == 0.5).all()
        # 0.1 is 409.6 times its scale, 2^-12: 384 or 416
        got = m8[part].float()
        assert ((got == 384) | (got == 416)).all()
    codes = ms.view(torch.uint8)
    assert int(codes.min()) == int(codes.max()) == 127 - 12


def test_as_torch_adamw(cuda):
    # the class, several steps, two groups, parameters without gradients now and then
    gen = torch.Generator().manual_seed(7)
    sizes = [(20, 30), (30,), (7, 3, 3), (1,)]
    mine = [torch.nn.Parameter(torch.randn(s, generator=gen).to(cuda)) for s in sizes]
    ref = [torch.nn.Parameter(p.detach().clone()) for p in mine]

    def groups(ps):
        return [{"params": ps[:2], "lr": 3e-3, "weight_decay": 0.2}, {"params": ps[2:]}]
    a = cpab.AdamW(groups(mine), lr=1e-2)
    b = torch.optim.AdamW(groups(ref), lr=1e-2, foreach=False)
    for step in range(12):
        for k, (p, q) in enumerate(zip(mine, ref)):
            g = torch.randn(p.shape, generator=gen).to(cuda)
            p.grad, q.grad = (None, None) if (step + k) % 5 == 0 else (g, g.clone())
        version = mine[0]._version
        assert a.step(lambda: 3.5) == 3.5
        b.step()
        assert mine[0]._version > version or mine[0].grad is None
        for p, q in zip(mine, ref):
            torch.testing.assert_close(p, q, rtol=3e-6, atol=3e-7)


@pytest.mark.parametrize("bits", [32, 8])
def test_saved_and_loaded(cuda, bits, tmp_path):
    gen = torch.Generator().manual_seed(8)
    start = [torch.randn(s, generator=gen).to(BF16).to(cuda) for s in ((33, 65), (17,))]
    grads = [[torch.randn(p.shape, generator=gen).to(BF16).to(cuda) for p in start] for _ in range(6)]

    def run(params, opt, some):
        for gs in some:
            for p, g in zip(params, gs):
                p.grad = g.clone()
            opt.step()

    def new():
        params = [torch.nn.Parameter(p.clone()) for p in start]
        return params, cpab.AdamW(params, lr=1e-2, state_bits=bits, seed=5)
    whole, opt = new()
    run(whole, opt, grads)
    half, opt = new()
    run(half, opt, grads[:3])
    torch.save({"opt": opt.state_dict(), "p": [p.detach() for p in half]}, tmp_path / "s.pt")
    data = torch.load(tmp_path / "s.pt", weights_only=True)
    rest, opt = new()
    for p, q in zip(rest, data["p"]):
        p.data.copy_(q)
    opt.load_state_dict(data["opt"])
    state = opt.state[rest[0]]
    assert state["master"].dtype == F32 and state["exp_avg"].dtype == (F32 if bits == 32 else E4M3)
    run(rest, opt, grads[3:])
    for p, q in zip(whole, rest):
        assert torch.equal(p, q)


@pytest.mark.parametrize("bits", [32, 8])
def test_finds_a_minimum(cuda, bits):
    # a least-squares problem: 8-bit states come about as near as 32-bit ones
    gen = torch.Generator().manual_seed(9)
    A = torch.randn(256, 64, generator=gen).to(cuda)
    want = torch.randn(64, generator=gen).to(cuda)
    x = torch.nn.Parameter(torch.zeros(64, device=cuda))
    opt = cpab.AdamW([x], lr=0.05, weight_decay=0.0, state_bits=bits)
    for k in range(400):
        if k == 300:
            opt.param_groups[0]["lr"] = 0.005
        opt.zero_grad()
        ((A @ (x - want)) ** 2).mean().backward()
        opt.step()
    assert float((x - want).norm() / want.norm()) < 0.02


def test_same_call_same_bits(cuda):
    outs = []
    for _ in range(2):
        ts = tensors(cuda, [(5000,), (33,)], BF16, 10, True)
        for t in ts:
            states8(cuda, t)
        cpab.adamw_step([t["p"] for t in ts], [t["g"] for t in ts], [t["m8"] for t in ts], [t["v8"] for t in ts],
                        3, LR, BETAS, EPS, WD, [t["ms"] for t in ts], [t["vs"] for t in ts],
                        [t["master"] for t in ts], 11)
        outs.append([t[k].view(torch.uint8) for t in ts for k in ("p", "m8", "v8", "ms", "vs", "master")])
    assert all(torch.equal(a, b) for a, b in zip(*outs))


def test_side_stream(cuda):
    res = []
    for side in (False, True):
        ts = tensors(cuda, [(3000,), (77,)], F32, 12)
        torch.cuda.synchronize()
        s = torch.cuda.Stream() if side else torch.cuda.current_stream()
        with torch.cuda.stream(s):
            for k in range(1, 4):
                cpab.adamw_step([t["p"] for t in ts], [t["g"] for t in ts], [t["m"] for t in ts],
                                [t["v"] for t in ts], k)
        s.synchronize()
        res.append([t[k] for t in ts for k in ("p", "m", "v")])
    assert all(torch.equal(a, b) for a, b in zip(*res))


def test_refusals(cuda):
    p, g, m, v = (torch.zeros(8, device=cuda) for _ in range(4))
    c8 = torch.zeros(8, dtype=torch.uint8, device=cuda).view(E4M3)
    s8 = torch.zeros(1, dtype=torch.uint8, device=cuda).view(E8M0)
    ok = dict(params=[p], grads=[g], exp_avgs=[m], exp_avg_sqs=[v], step=1)
    for change, word in ((dict(step=0), "step must"), (dict(betas=(1.0, 0.9)), "beta"),
                         (dict(betas=(0.9, -0.1)), "beta"), (dict(lr=-1.0), "lr"),
                         (dict(lr=float("nan")), "lr"), (dict(eps=-1e-8), "eps"),
                         (dict(grads=[]), "one entry"), (dict(masters=[]), "one entry"),
                         (dict(exp_avg_scales=[s8]), "both lists"),
                         (dict(params=[p.cpu()]), "GPU"), (dict(params=[p.half()]), "bfloat16"),
                         (dict(grads=[g.bfloat16()]), "gradient"), (dict(grads=[g[:4]]), "gradient"),
                         (dict(grads=[g.cpu()]), "gradient"),
                         (dict(exp_avgs=[m.bfloat16()]), "exp_avg of parameter 0"),
                         (dict(exp_avg_sqs=[v[:7]]), "exp_avg_sq of parameter 0"),
                         (dict(masters=[v.bfloat16()]), "master"),
                         (dict(exp_avg_scales=[s8], exp_avg_sq_scales=[s8]), "exp_avg of parameter 0"),
                         (dict(exp_avgs=[c8], exp_avg_sqs=[c8.clone()], exp_avg_scales=[s8],
                               exp_avg_sq_scales=[torch.zeros(2, dtype=torch.uint8, device=cuda).view(E8M0)]),
                          "exp_avg_sq scale"),
                         (dict(params=[torch.zeros(16, device=cuda)[::2]]), "not dense"),
                         (dict(params=[p, p.bfloat16()], grads=[g, g.bfloat16()], exp_avgs=[m, m.clone()],
                               exp_avg_sqs=[v, v.clone()]), "one type")):
        with pytest.raises(RuntimeError, match=word):
            cpab.adamw_step(**dict(ok, **change))
    assert (p == 0).all() and (m == 0).all()
    cpab.adamw_step([], [], [], [], 1)
    for kw in (dict(state_bits=16), dict(lr=-1.0), dict(betas=(0.9, 1.0))):
        with pytest.raises(AssertionError):
            cpab.AdamW([torch.nn.Parameter(p)], **kw)
