"""The operators around the transform: a network that reads long signals and gives
theta, and the step that moves its weights.

Three operators: the gated linear recurrence (``cpab.gated_recurrence``), the
root-mean-square norm with the residual's addition (``cpab.rms_norm``) and an AdamW
step over many tensors (``cpab.adamw_step``).  ``run`` makes one pass as a program
makes it, with its gradients where the case trains, through the framework where
``own`` is true and in elementary torch operations in 32 bits where it is not.
"""
import math
import os
import sys

import torch

own = False

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
DEV = "cuda"
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
E4M3, E8M0 = torch.float8_e4m3fn, torch.float8_e8m0fnu
EPS = 1e-6
BETAS, ADAM_EPS, DECAY, LR = (0.9, 0.999), 1e-8, 1e-2, 1e-3


def _cpab():
    path = os.path.join(ROOT, "fg-cpab_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    import cpab
    return cpab


# --------------------------------------------------------------------------
# cases
# --------------------------------------------------------------------------

# A case's fields.
# recurrence: batch, time, width; gate: with the output gate; ragged: rows of
#   different lengths, padded; packed: the inputs are slices of one projection's
#   output; start: a state from before.
# norm: rows, width; residual; out: "same" or "e4m3"; weight: the weight's type.
# adamw: width, layers of the encoder; bits of the states; master: 32-bit master
#   weights beside the parameters; tight: the tensors lie one after another in one
#   buffer, at any offset, rather than in allocations of their own.
def _rec(dtype, batch, time, width, train, gate=True, ragged=False, packed=False, start=True, **kw):
    return dict(op="recurrence", dtype=dtype, batch=batch, time=time, width=width, train=train,
                gate=gate, ragged=ragged, packed=packed, start=start, **kw)


def _norm(dtype, rows, width, train, residual=True, out="same", weight=None, **kw):
    return dict(op="norm", dtype=dtype, rows=rows, width=width, train=train, residual=residual,
                out=out, weight=weight or dtype, **kw)


def _adamw(dtype, width, layers, bits, master=False, tight=False, **kw):
    return dict(op="adamw", dtype=dtype, width=width, layers=layers, bits=bits, master=master,
                tight=tight, **kw)


def listed():
    return [
        # One new sample of each of 64 signals that arrive as they are measured: the
        # smallest call, its latency is what counts.
        _rec("bf16", 64, 1, 512, False, name="rec_token"),
        # Training on 16 signals of up to 10,000 samples, ragged, in 32 bits.
        _rec("f32", 16, 10000, 64, True, ragged=True, start=False, name="rec_signals"),
        # Training a wider encoder, its inputs the slices of one projection.
        _rec("bf16", 8, 4096, 1280, True, packed=True, start=False, name="rec_train"),
        # Reading one very long recording: few channels in parallel, a long axis.
        _rec("bf16", 1, 131072, 512, False, name="rec_long"),
        # One new sample's norm on the way to an 8-bit product.
        _norm("bf16", 64, 1024, False, out="e4m3", name="norm_token"),
        # An odd width, the 28 x 28 inputs of a layer as rows, in 32 bits.
        _norm("f32", 12544, 333, True, name="norm_odd"),
        # Training a wide encoder.
        _norm("bf16", 32768, 1024, True, name="norm_train"),
        # Evaluating a very wide encoder with 8-bit products.
        _norm("bf16", 16384, 8192, False, out="e4m3", name="norm_quant"),
        # A small encoder that gives theta (49 numbers): many small tensors.
        _adamw("f32", 64, 8, 32, name="adamw_small"),
        # A large one, all in 32 bits.
        _adamw("f32", 2048, 8, 32, name="adamw_large"),
        # The same trained in bf16, with master weights and states of 8 bits.
        _adamw("bf16", 2048, 8, 8, master=True, name="adamw_8bit"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["recurrence", "norm", "adamw"])
    dtype = rng.choice(["f32", "bf16"])
    if op == "recurrence":
        width, batch = _log(rng, 16, 2048), _log(rng, 1, 64)
        time = _log(rng, 1, max(1, min(65536, 32_000_000 // (width * batch))))
        return _rec(dtype, batch, time, width, rng.random() < 0.6, gate=rng.random() < 0.7,
                    ragged=rng.random() < 0.4, packed=rng.random() < 0.4, start=rng.random() < 0.5)
    if op == "norm":
        width = _log(rng, 32, 16384)
        rows = _log(rng, 1, max(1, min(65536, 64_000_000 // width)))
        quant = rng.random() < 0.4
        return _norm(dtype, rows, width, not quant and rng.random() < 0.7, rng.random() < 0.7,
                     "e4m3" if quant else "same", rng.choice([dtype, "f32"]))
    width, layers = _log(rng, 16, 1800), rng.randint(1, 10)
    return _adamw(dtype, width, layers, rng.choice([8, 32]), dtype == "bf16" and rng.random() < 0.6,
                  rng.random() < 0.4)


# --------------------------------------------------------------------------
# inputs
# --------------------------------------------------------------------------

def _sizes(c):
    """The encoder's tensors: per layer a norm's weight, the projection to the
    recurrence's three inputs, and the one back; then the head that gives theta."""
    w = c["width"]
    layer = [(w,), (3 * w, w), (3 * w,), (w, w), (w,)]
    return layer * c["layers"] + [(49, w), (49,)]


def _offsets(sizes, step):
    """Where each tensor begins in one buffer, at multiples of `step`; and the whole."""
    at, offs = 0, []
    for s in sizes:
        offs.append(at)
        at += -(-math.prod(s) // step) * step
    return offs, at


def _views(flat, offs, sizes, shaped=True):
    parts = [flat[o:o + math.prod(s)] for o, s in zip(offs, sizes)]
    return [p.view(s) for p, s in zip(parts, sizes)] if shaped else parts


def _prepare_adamw(c, gen):
    sizes = _sizes(c)
    dt = TYPES[c["dtype"]]
    offs, total = _offsets(sizes, 1 if c["tight"] else 256)
    live = torch.zeros(total, device=DEV, dtype=torch.bool)
    for v in _views(live, offs, sizes):
        v.fill_(True)
    spread = torch.exp(torch.randn(total, device=DEV, generator=gen))
    master = torch.randn(total, device=DEV, generator=gen) * 0.02 * live
    grad = torch.randn(total, device=DEV, generator=gen) * spread * 1e-3 * live
    m = torch.randn(total, device=DEV, generator=gen) * spread * 3e-4 * live
    v = (spread * 1e-3 * live).square()
    st = {"step": 100, "seed": int(torch.randint(0, 2 ** 31, (1,), device=DEV, generator=gen)),
          "param": master.to(dt), "grad": grad.to(dt), "case": c, "sizes": sizes}
    if c["master"]:
        st["master"] = master
        st["masters"] = _views(master, offs, sizes)
    st["params"] = _views(st["param"], offs, sizes)
    st["grads"] = _views(st["grad"], offs, sizes)
    if c["bits"] == 32:
        st["exp_avg"], st["exp_avg_sq"] = m, v
        st["exp_avgs"], st["exp_avg_sqs"] = _views(m, offs, sizes), _views(v, offs, sizes)
        return st
    # 8-bit states, one value a byte, a scale to each 32 of a tensor's values
    eoffs, etotal = _offsets(sizes, 32)
    soffs = [o // 32 for o in eoffs]
    groups = [(-(-math.prod(s) // 32),) for s in sizes]
    for name, full in (("exp_avg", m), ("exp_avg_sq", v.sqrt())):
        codes = torch.zeros(etotal, device=DEV, dtype=torch.uint8).view(E4M3)
        scales = torch.zeros(etotal // 32, device=DEV, dtype=torch.uint8).view(E8M0)
        st[name], st[name + "_scale"] = codes, scales
        st[name + "s"] = _views(codes, eoffs, sizes, shaped=False)
        st[name + "_scales"] = _views(scales, soffs, groups)
        for i, part in enumerate(_views(full, offs, sizes, shaped=False)):
            _mx_store(part, st[name + "s"][i], st[name + "_scales"][i], None)
    return st


def prepare(case, seed):
    c = dict(case)
    gen = torch.Generator(device=DEV).manual_seed(int(seed))

    def normal(*shape):
        return torch.randn(*shape, device=DEV, generator=gen)

    if c["op"] == "adamw":
        return _prepare_adamw(c, gen)
    dt = TYPES[c["dtype"]]
    st = {"case": c}
    train = c["train"]
    if c["op"] == "norm":
        R, C = c["rows"], c["width"]
        # rows of different sizes, as a residual stream has them
        size = torch.exp(0.5 * normal(R, 1))
        st["x"] = (normal(R, C) * size).to(dt).requires_grad_(train)
        st["weight"] = (1 + 0.1 * normal(C)).to(TYPES[c["weight"]]).requires_grad_(train)
        if c["residual"]:
            st["residual"] = (normal(R, C) * 2).to(dt).requires_grad_(train)
        if train:
            st["dy"] = normal(R, C).to(dt)
            if c["residual"]:
                st["dres"] = normal(R, C).to(dt)
        return st
    B, T, C = c["batch"], c["time"], c["width"]
    # gates that remember from 2 samples to some hundreds, by channel
    keep = 6 * torch.rand(C, device=DEV, generator=gen)
    names = ["x", "f"] + (["g"] if c["gate"] else [])
    whole = normal(B, T, len(names) * C)
    whole[..., C:2 * C] += keep
    if c["ragged"]:
        low = max(1, T // 4)
        lengths = torch.randint(low, T + 1, (B,), device=DEV, generator=gen, dtype=torch.int32)
        lengths[0] = T
        if B >= 8:
            lengths[B // 2] = 0   # a signal that is missing
        st["lengths"] = lengths
        # what lies behind a signal's end is nobody's
        pad = torch.arange(T, device=DEV)[None, :] >= lengths[:, None]
        whole.masked_fill_(pad[..., None], float("nan"))
    whole = whole.to(dt)
    for k, name in enumerate(names):
        part = whole[..., k * C:(k + 1) * C]
        st[name] = (part if c["packed"] else part.contiguous()).detach().requires_grad_(train)
    if c["start"]:
        st["h0"] = (0.5 * normal(B, C)).requires_grad_(train)
    if train:
        st["dy"] = normal(B, T, C).to(dt)
        st["dh"] = normal(B, C)
    return st


# --------------------------------------------------------------------------
# one pass
# --------------------------------------------------------------------------

def _outputs_adamw(st):
    names = ("param", "master", "exp_avg", "exp_avg_sq", "exp_avg_scale", "exp_avg_sq_scale")
    return {k: st[k] for k in names if k in st}


def run(st):
    c = st["case"]
    if c["op"] == "adamw":
        st["step"] += 1
        if own:
            _cpab().adamw_step(st["params"], st["grads"], st["exp_avgs"], st["exp_avg_sqs"],
                               st["step"], lr=LR, betas=BETAS, eps=ADAM_EPS, weight_decay=DECAY,
                               exp_avg_scales=st.get("exp_avg_scales"),
                               exp_avg_sq_scales=st.get("exp_avg_sq_scales"),
                               masters=st.get("masters"), seed=st["seed"])
        else:
            _plain_adamw(st)
        return _outputs_adamw(st)
    if c["op"] == "norm":
        return _own_norm(st) if own else _plain_norm(st)
    return _own_recurrence(st) if own else _plain_recurrence(st)


def _own_norm(st):
    c = st["case"]
    cpab = _cpab()
    res = st.get("residual")
    if c["out"] == "e4m3":
        with torch.no_grad():
            got = cpab.rms_norm(st["x"], st["weight"], residual=res, eps=EPS, out_dtype=E4M3)
        return dict(zip(("y", "scale", "residual"), got))
    if not c["train"]:
        with torch.no_grad():
            got = cpab.rms_norm(st["x"], st["weight"], residual=res, eps=EPS)
        return dict(zip(("y", "residual"), got if res is not None else (got,)))
    got = cpab.rms_norm(st["x"], st["weight"], residual=res, eps=EPS)
    if res is None:
        gx, gw = torch.autograd.grad(got, (st["x"], st["weight"]), st["dy"])
        return {"y": got, "grad_x": gx, "grad_weight": gw}
    gx, gr, gw = torch.autograd.grad(got, (st["x"], res, st["weight"]), (st["dy"], st["dres"]))
    return {"y": got[0], "residual": got[1], "grad_x": gx, "grad_residual": gr, "grad_weight": gw}


def _own_recurrence(st):
    c = st["case"]
    cpab = _cpab()
    args = dict(g=st.get("g"), h0=st.get("h0"), lengths=st.get("lengths"))
    if not c["train"]:
        with torch.no_grad():
            y, h = cpab.gated_recurrence(st["x"], st["f"], **args)
        return {"y": y, "h": h}
    y, h = cpab.gated_recurrence(st["x"], st["f"], **args)
    wanted = [k for k in ("x", "f", "g", "h0") if k in st]
    grads = torch.autograd.grad((y, h), [st[k] for k in wanted], (st["dy"], st["dh"]))
    return dict({"y": y, "h": h}, **{"grad_" + k: v for k, v in zip(wanted, grads)})


# --------------------------------------------------------------------------
# the plain forms
# --------------------------------------------------------------------------

def _plain_norm(st):
    c = st["case"]
    with torch.no_grad():
        x, w = st["x"].float(), st["weight"].float()
        r = x + st["residual"].float() if "residual" in st else x
        s = torch.rsqrt(r.square().mean(-1, keepdim=True) + EPS)
        n = r * s
        y = n * w
        dt = st["x"].dtype
        if c["out"] == "e4m3":
            scale = y.abs().amax(-1) / 448
            scale = torch.where(scale == 0, torch.ones_like(scale), scale)
            out = {"y": (y / scale[:, None]).to(E4M3), "scale": scale}
        else:
            out = {"y": y.to(dt)}
        if "residual" in st:
            out["residual"] = r.to(dt)
        if c["train"]:
            dy = st["dy"].float()
            u = dy * w
            dr = s * (u - n * (u * n).mean(-1, keepdim=True))
            if "dres" in st:
                dr = dr + st["dres"].float()
                out["grad_residual"] = dr.to(dt)
            out["grad_x"] = dr.to(dt)
            out["grad_weight"] = (dy * n).sum(0).to(st["weight"].dtype)
        return out


def _scan(a, u):
    """h_t = a_t h_{t-1} + u_t along dimension 1 from h = 0, in steps that double."""
    d, T = 1, a.shape[1]
    while d < T:
        u = torch.cat([u[:, :d], u[:, d:] + a[:, d:] * u[:, :-d]], 1)
        a = torch.cat([a[:, :d], a[:, d:] * a[:, :-d]], 1)
        d *= 2
    return u


def _plain_recurrence(st):
    c = st["case"]
    with torch.no_grad():
        x, f = st["x"].float(), st["f"].float()
        B, T, C = x.shape
        a, u = torch.sigmoid(f), torch.sigmoid(-f) * x
        valid = None
        if "lengths" in st:
            valid = (torch.arange(T, device=x.device)[None, :] < st["lengths"][:, None])[..., None]
            zero, one = torch.zeros((), device=x.device), torch.ones((), device=x.device)
            a, u, x = torch.where(valid, a, one), torch.where(valid, u, zero), torch.where(valid, x, zero)
        h0 = st["h0"] if "h0" in st else torch.zeros(B, C, device=x.device)
        first = torch.cat([u[:, :1] + a[:, :1] * h0[:, None], u[:, 1:]], 1)
        h = _scan(a, first)
        y, s = h, None
        if "g" in st:
            g = st["g"].float()
            if valid is not None:
                g = torch.where(valid, g, zero)
            s = torch.sigmoid(g)
            y = h * (g * s)
        if valid is not None:
            y = torch.where(valid, y, zero)
        dt = st["x"].dtype
        out = {"y": y.to(dt), "h": h[:, -1].clone()}
        if not c["train"]:
            return out
        dy = st["dy"].float()
        if valid is not None:
            dy = torch.where(valid, dy, zero)
        if "g" in st:
            out["grad_g"] = (dy * h * s * (1 + g * (1 - s))).to(dt)
            dy = dy * (g * s)
        dy = torch.cat([dy[:, :-1], dy[:, -1:] + st["dh"][:, None]], 1)
        after = torch.cat([a[:, 1:], torch.ones_like(a[:, :1])], 1)
        lam = _scan(after.flip(1), dy.flip(1)).flip(1)
        before = torch.cat([h0[:, None], h[:, :-1]], 1)
        b = torch.sigmoid(-f)
        if valid is not None:
            b = torch.where(valid, b, zero)
        out["grad_x"] = (b * lam).to(dt)
        out["grad_f"] = (lam * (before - x) * a * b).to(dt)
        if "h0" in st:
            out["grad_h0"] = a[:, 0] * lam[:, 0]
        return out


_LOW = 0xFFFFFFFF


def _mix(z):
    """Scrambles 32-bit numbers (held in 64): xorshifts and odd multipliers, the leading
    digits of the golden section and of the square root of two."""
    z = z ^ (z >> 16)
    z = (z * 0x9E3779B1) & _LOW
    z = z ^ (z >> 15)
    z = (z * 0xB504F333) & _LOW
    return z ^ (z >> 16)


def _random(n, seed, step, ordinal):
    """32 random bits for each of a tensor's values, from the step's seed."""
    key = _mix((_mix((seed & _LOW) ^ ((step * 0x9E3779B1) & _LOW)) + ordinal) & _LOW)
    return _mix((torch.arange(n, device=DEV) + key) & _LOW)


def _mx_scale(x):
    """Exponents k of each 32 finite values' scale: the least with max |x| <= 448 2^k."""
    groups = torch.nn.functional.pad(x, (0, -x.numel() % 32)).view(-1, 32)
    top = torch.where(torch.isfinite(groups), groups.abs(), torch.zeros_like(groups)).amax(1)
    part, e = torch.frexp(top)            # top = part 2^e, 0.5 <= part < 1
    k = torch.where(part > 0.875, e - 8, e - 9)
    return torch.where(top == 0, torch.full_like(k, -127), k).clamp(min=-127)


def _mx_load(codes, scales):
    """The values that 8-bit codes and their groups' scales stand for."""
    k = scales.view(torch.uint8).int() - 127
    n = codes.numel()
    two = torch.where(k > -127, (k + 127) << 23, torch.full_like(k, 1 << 22)).view(torch.float32)
    return codes.float() * two.repeat_interleave(32)[:n]


def _mx_store(x, codes, scales, bits, least=False):
    """x in 8 bits: rounded up or down by 16 random bits (to nearest without them);
    `least`: positive values give at least the smallest positive code."""
    n = x.numel()
    k = _mx_scale(x)
    inv = ((127 - k) << 23).view(torch.float32).repeat_interleave(32)[:n]
    a = x.abs() * inv
    if bits is not None:
        small = a < 0.015625                  # below the least normal code: even spacing
        a = torch.where(small, a + 0.015625, a)
        a = ((a.view(torch.int32) + (bits << 4).int()) & ~0xFFFFF).view(torch.float32)
        a = torch.where(small, a - 0.015625, a)
    if least:
        a = torch.where(x > 0, a.clamp(min=0.001953125), a)
    a = torch.where(torch.isfinite(x), a, torch.full_like(a, float("nan")))
    codes.copy_(torch.copysign(a, x).to(E4M3))
    scales.copy_((k + 127).to(torch.uint8).view(E8M0))


def _plain_adamw(st):
    c = st["case"]
    b1, b2 = BETAS
    c1, c2 = 1 - b1 ** st["step"], 1 - b2 ** st["step"]
    for i, (p, g) in enumerate(zip(st["params"], st["grads"])):
        g = g.float().view(-1)
        w = (st["masters"][i] if c["master"] else p).float().view(-1)
        if c["bits"] == 32:
            m, v = st["exp_avgs"][i].view(-1), st["exp_avg_sqs"][i].view(-1)
        else:
            m = _mx_load(st["exp_avgs"][i], st["exp_avg_scales"][i])
            v = _mx_load(st["exp_avg_sqs"][i], st["exp_avg_sq_scales"][i]).square()
        m = b1 * m + (1 - b1) * g
        v = b2 * v + (1 - b2) * g * g
        w = w * (1 - LR * DECAY) - (LR / c1) * m / (torch.sqrt(v) / math.sqrt(c2) + ADAM_EPS)
        p.copy_(w.view(p.shape))
        if c["master"]:
            st["masters"][i].copy_(w.view(p.shape))
        if c["bits"] == 32:
            st["exp_avgs"][i].view(-1).copy_(m)
            st["exp_avg_sqs"][i].view(-1).copy_(v)
        else:
            r = _random(m.numel(), st["seed"], st["step"], i)
            _mx_store(m, st["exp_avgs"][i], st["exp_avg_scales"][i], r & 0xFFFF)
            _mx_store(v.sqrt(), st["exp_avg_sqs"][i], st["exp_avg_sq_scales"][i], r >> 16, True)


# --------------------------------------------------------------------------
# the same in 64 bits, from the definitions
# --------------------------------------------------------------------------

def _exact_norm(st):
    c = st["case"]
    x, w = st["x"].detach().double(), st["weight"].detach().double()
    r = x + (st["residual"].detach().double() if c["residual"] else 0)
    C = x.shape[1]
    power = (r * r).sum(1) / C + EPS
    y = r / power.sqrt()[:, None] * w
    out = {"y": y}
    if c["residual"]:
        out["residual"] = r
    if c["out"] == "e4m3":
        top = y.abs().max(1).values
        scale = torch.where(top > 0, top / 448, torch.ones_like(top))
        out.update(y=(y / scale[:, None]).float().to(E4M3), scale=scale)
    if c["train"]:
        dy = st["dy"].double()
        u = dy * w
        g = u / power.sqrt()[:, None] - r * ((u * r).sum(1) / C / power ** 1.5)[:, None]
        if c["residual"]:
            g = g + st["dres"].double()
            out["grad_residual"] = g
        out["grad_x"] = g
        out["grad_weight"] = (dy * r / power.sqrt()[:, None]).sum(0)
    return out


def _exact_recurrence(st):
    """Sample by sample, over [T, B, C]."""
    c = st["case"]
    wide = {k: st[k].detach().double().transpose(0, 1).contiguous() for k in ("x", "f", "g") if k in st}
    x, f = wide["x"], wide["f"]
    T, B, C = x.shape
    a = 1 / (1 + torch.exp(-f))
    u = x / (1 + torch.exp(f))
    live = None
    if "lengths" in st:
        live = (torch.arange(T, device=DEV)[:, None] < st["lengths"][None, :])[..., None]
        a = a.masked_fill(~live, 1.0)
        u = u.masked_fill(~live, 0.0)
    h0 = st["h0"].detach().double() if "h0" in st else torch.zeros(B, C, device=DEV).double()
    H = torch.empty(T + 1, B, C, device=DEV, dtype=torch.float64)
    H[0] = h0
    rows, gains, adds = H.unbind(0), a.unbind(0), u.unbind(0)
    for t in range(T):
        torch.addcmul(adds[t], gains[t], rows[t], out=rows[t + 1])
    gate = 1.0
    if "g" in wide:
        s = 1 / (1 + torch.exp(-wide["g"]))
        gate = wide["g"] * s
    y = H[1:] * gate
    out = {"y": (y if live is None else y.masked_fill(~live, 0.0)).transpose(0, 1), "h": H[T].clone()}
    if not c["train"]:
        return out
    dy = st["dy"].double().transpose(0, 1)
    if "g" in wide:
        dg = dy * H[1:] * (s + wide["g"] * s * (1 - s))
        out["grad_g"] = (dg if live is None else dg.masked_fill(~live, 0.0)).transpose(0, 1)
    dh = dy * gate
    if live is not None:
        dh = dh.masked_fill(~live, 0.0)
    # L[t] = dh[t] + a[t + 1] L[t + 1]
    L = torch.empty(T + 1, B, C, device=DEV, dtype=torch.float64)
    L[T] = st["dh"].double()
    follow = torch.cat([a[1:], torch.ones_like(a[:1])]).unbind(0)
    back, given = L.unbind(0), dh.unbind(0)
    for t in range(T - 1, -1, -1):
        torch.addcmul(given[t], follow[t], back[t + 1], out=back[t])
    gx = L[:T] / (1 + torch.exp(f))
    gf = L[:T] * (H[:T] - x) * a / (1 + torch.exp(f))
    if live is not None:
        gx, gf = gx.masked_fill(~live, 0.0), gf.masked_fill(~live, 0.0)
    out["grad_x"], out["grad_f"] = gx.transpose(0, 1), gf.transpose(0, 1)
    if "h0" in st:
        out["grad_h0"] = a[0] * L[0]
    return out


def _two_to(k):
    """2^k in 64 bits, exactly, for whole k."""
    return ((k.long() + 1023) << 52).view(torch.float64)


def _exact_mx(x, bits, least):
    """8-bit codes (as numbers) and scales of x [n] in 64 bits."""
    n = x.numel()
    groups = torch.zeros(-(-n // 32) * 32, device=DEV, dtype=torch.float64)
    groups[:n] = x.abs()
    top = groups.view(-1, 32).max(1).values
    k = torch.ceil(torch.log2(top / 448)).clamp(min=-127)
    k = torch.where(top > 448 * _two_to(k), k + 1, torch.where(top <= 448 * _two_to(k - 1), k - 1, k))
    k = k.clamp(min=-127)
    a = x.abs() / _two_to(k).repeat_interleave(32)[:n]
    spacing = _two_to(torch.frexp(a.clamp(min=2.0 ** -6))[1] - 4)
    a = torch.floor(a / spacing + bits.double() / 65536) * spacing
    if least:
        a = torch.where(x > 0, a.clamp(min=2.0 ** -9), a)
    return torch.copysign(a, x), _two_to(k)


def _exact_adamw(st):
    c = st["case"]
    t = st["step"] + 1
    b1, b2 = BETAS
    out = {k: v.clone() if k.endswith("scale") else v.double() for k, v in _outputs_adamw(st).items()}
    for k in out:
        if k.endswith("scale"):
            out[k] = _two_to(out[k].view(torch.uint8).long() - 127)

    def place(name, whole, part):
        # where the tensor `part` (a view) lies in its buffer
        at = (part.data_ptr() - st[name].data_ptr()) // st[name].element_size()
        return whole[at:at + part.numel()]

    for i, p in enumerate(st["params"]):
        g = st["grads"][i].double().reshape(-1)
        w = (st["masters"][i] if c["master"] else p).double().reshape(-1)
        m, v = (place(k, out[k], st[k + "s"][i]) for k in ("exp_avg", "exp_avg_sq"))
        new_m, new_v = m, v
        if c["bits"] == 8:
            ms, vs = (place(k + "_scale", out[k + "_scale"], st[k + "_scales"][i])
                      for k in ("exp_avg", "exp_avg_sq"))
            new_m = m * ms.repeat_interleave(32)[:m.numel()]
            new_v = (v * vs.repeat_interleave(32)[:v.numel()]) ** 2
        new_m = b1 * new_m + (1 - b1) * g
        new_v = b2 * new_v + (1 - b2) * g * g
        moved = new_m / (1 - b1 ** t) / ((new_v / (1 - b2 ** t)).sqrt() + ADAM_EPS)
        w = w - LR * DECAY * w - LR * moved
        place("param", out["param"], p).copy_(w)
        if c["master"]:
            place("master", out["master"], st["masters"][i]).copy_(w)
        if c["bits"] == 8:
            r = _random(m.numel(), st["seed"], t, i)
            new_m, k = _exact_mx(new_m, r & 0xFFFF, False)
            ms.copy_(k)
            new_v, k = _exact_mx(new_v.sqrt(), r >> 16, True)
            vs.copy_(k)
        m.copy_(new_m)
        v.copy_(new_v)
    return out


def exact(case, seed):
    st = prepare(case, seed)
    return {"norm": _exact_norm, "recurrence": _exact_recurrence, "adamw": _exact_adamw}[case["op"]](st)


# --------------------------------------------------------------------------
# work
# --------------------------------------------------------------------------

def work(case):
    """Bytes: every input read once, every output written once.  Operations: a
    multiplication, an addition or a call of exp, a division or a root counts as one."""
    c = case
    if c["op"] == "adamw":
        n = sum(math.prod(s) for s in _sizes(c))
        size = 4 if c["dtype"] == "f32" else 2
        state = 4.0 if c["bits"] == 32 else 1 + 1 / 32
        # without a master the parameter itself is read too
        each = size + (8 + size if c["master"] else 2 * size) + 4 * state
        return {"bytes": n * each, "flops": 16.0 * n + (40.0 * n if c["bits"] == 8 else 0)}
    e = 4 if c["dtype"] == "f32" else 2
    if c["op"] == "norm":
        n = float(c["rows"]) * c["width"]
        two = 2 if c["residual"] else 1
        back = 0 if not c["train"] else n * e * (1 + two + 1)   # dy, r (and dres); dr
        first = n * e * (two + two - 1) + n * (1 if c["out"] == "e4m3" else e)
        return {"bytes": first + back, "flops": n * (6 + (12 if c["train"] else 0))}
    n = float(c["batch"]) * c["time"] * c["width"]
    ins = 3 if c["gate"] else 2
    values = ins + 1 + ((ins + 1 + ins) if c["train"] else 0)
    ends = c["batch"] * c["width"] * 4.0 * ((1 + c["start"]) * (2 if c["train"] else 1))
    return {"bytes": n * e * values + ends,
            "flops": n * (6 + 6 * c["gate"] + (16 + 10 * c["gate"] if c["train"] else 0))}
