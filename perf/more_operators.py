"""More operators around the transform: a network that reads long signals with a matrix of
state for each head, what prepares its queries and keys, and the step that keeps the
updates of its matrices orthogonal.

Three operators: the gated delta rule (``cpab.gated_delta_rule``), the norms of queries
and keys with their rotation by the position (``cpab.qk_norm``) and a Muon step over many
matrices (``cpab.muon_step``).  ``run`` makes one pass as a program makes it, with its
gradients where the case trains, through the framework where ``own`` is true and in
elementary torch operations in 32 bits where it is not.
"""
import math
import os
import sys

import torch

own = False

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
DEV = "cuda"
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
EPS = 1e-6
BASE = 10000.0
MUON = dict(lr=2e-2, weight_decay=1e-2, momentum=0.95, ns_coefficients=(3.4445, -4.775, 2.0315),
            eps=1e-7, ns_steps=5)


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
# delta: batch, time; heads of the values, each `group` of them with one query and key;
#   dk, dv: values of a key and of a value; gates: the type of decay and beta; ragged: rows
#   of different lengths, padded; packed: q, k and v are slices of one projection's output;
#   start: a state from before.
# qk: batch, time; heads of queries and of keys; width: values of a head; turned: how many
#   of them the position rotates; neighbours: pairs side by side rather than half a head
#   apart; weight: the weights' type; packed: slices of one projection's output; given:
#   positions are given (a sample's place in its recording) rather than 0, 1, 2, ...
# muon: width, layers of the encoder; master: 32-bit master weights beside the parameters;
#   nesterov; tight: the tensors lie one after another in one buffer, at any offset.
def _delta(dtype, batch, time, heads, group, dk, dv, train, ragged=False, packed=False, start=True,
           gates="f32", **kw):
    return dict(op="delta", dtype=dtype, batch=batch, time=time, heads=heads, group=group, dk=dk,
                dv=dv, train=train, ragged=ragged, packed=packed, start=start, gates=gates, **kw)


def _qk(dtype, batch, time, heads, key_heads, width, turned, train, neighbours=False, packed=False,
        given=True, weight=None, **kw):
    return dict(op="qk", dtype=dtype, batch=batch, time=time, heads=heads, key_heads=key_heads,
                width=width, turned=turned, train=train, neighbours=neighbours, packed=packed,
                given=given, weight=weight or dtype, **kw)


def _muon(dtype, width, layers, master=False, nesterov=True, tight=False, **kw):
    return dict(op="muon", dtype=dtype, width=width, layers=layers, master=master,
                nesterov=nesterov, tight=tight, **kw)


def listed():
    return [
        # One new sample of each of 64 signals that arrive as they are measured: the
        # smallest call, its latency is what counts.
        _delta("bf16", 64, 1, 4, 1, 64, 64, False, name="delta_token"),
        # Training on 16 signals of up to 10,000 samples, ragged, in 32 bits.
        _delta("f32", 16, 10000, 2, 1, 32, 32, True, ragged=True, start=False, name="delta_signals"),
        # Training a wide encoder, two heads of values to a key, slices of one projection.
        _delta("bf16", 8, 4096, 16, 2, 128, 128, True, packed=True, start=False, gates="bf16",
               name="delta_train"),
        # Reading one very long recording: few heads in parallel, a long axis.
        _delta("bf16", 1, 131072, 4, 1, 128, 128, False, name="delta_long"),
        # One new sample's queries and keys.
        _qk("bf16", 64, 1, 4, 4, 64, 64, False, name="qk_token"),
        # Heads of an odd width over 28 x 28 inputs, partly rotated, in 32 bits.
        _qk("f32", 16, 784, 5, 3, 50, 24, True, neighbours=True, given=False, name="qk_odd"),
        # Training a wide encoder, slices of one projection.
        _qk("bf16", 8, 4096, 16, 4, 128, 128, True, packed=True, name="qk_train"),
        # A small encoder that gives theta (49 numbers): many small matrices.
        _muon("f32", 64, 8, name="muon_small"),
        # A large one, all in 32 bits.
        _muon("f32", 2048, 4, name="muon_large"),
        # A wide one in bf16, with master weights.
        _muon("bf16", 1280, 8, master=True, name="muon_master"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["delta", "qk", "muon"])
    dtype = rng.choice(["f32", "bf16"])
    if op == "delta":
        dk, dv = _log(rng, 8, 128), _log(rng, 8, 256)
        group = rng.choice([1, 1, 2, 3, 4])
        heads, batch = group * _log(rng, 1, 8), _log(rng, 1, 32)
        most = 3_000_000_000 // (batch * heads * max(dk, 32) * max(dv, 32))
        time = _log(rng, 1, max(1, min(16384, most)))
        return _delta(dtype, batch, time, heads, group, dk, dv, rng.random() < 0.6,
                      rng.random() < 0.4, rng.random() < 0.4, rng.random() < 0.5,
                      rng.choice([dtype, "f32"]))
    if op == "qk":
        width = _log(rng, 8, 256)
        key_heads = _log(rng, 1, 16)
        heads = key_heads * rng.choice([1, 1, 2, 4])
        batch = _log(rng, 1, 32)
        time = _log(rng, 1, max(1, min(16384, 48_000_000 // (batch * (heads + key_heads) * width))))
        turned = rng.choice([width // 2 * 2, width // 2 * 2, width // 4 * 2, 0])
        return _qk(dtype, batch, time, heads, key_heads, width, turned, rng.random() < 0.6,
                   rng.random() < 0.5, rng.random() < 0.5, rng.random() < 0.6,
                   rng.choice([dtype, "f32"]))
    width, layers = _log(rng, 16, 1400), rng.randint(1, 6)
    return _muon(dtype, width, layers, dtype == "bf16" and rng.random() < 0.6, rng.random() < 0.7,
                 rng.random() < 0.4)


# --------------------------------------------------------------------------
# inputs
# --------------------------------------------------------------------------

def _sizes(c):
    """The encoder's matrices: per layer the projection to the delta rule's inputs and the
    one back; then the head that gives theta."""
    w = c["width"]
    return [(3 * w, w), (w, w)] * c["layers"] + [(49, w)]


def _offsets(sizes, step):
    """Where each tensor begins in one buffer, at multiples of `step`; and the whole."""
    at, offs = 0, []
    for s in sizes:
        offs.append(at)
        at += -(-math.prod(s) // step) * step
    return offs, at


def _views(flat, offs, sizes):
    return [flat[o:o + math.prod(s)].view(s) for o, s in zip(offs, sizes)]


def _prepare_muon(c, gen):
    sizes = _sizes(c)
    dt = TYPES[c["dtype"]]
    offs, total = _offsets(sizes, 1 if c["tight"] else 256)
    live = torch.zeros(total, device=DEV, dtype=torch.bool)
    for v in _views(live, offs, sizes):
        v.fill_(True)

    def normal():
        return torch.randn(total, device=DEV, generator=gen) * live

    master, grad, mom = normal() * 0.02, normal() * 1e-3, normal() * 3e-4
    # gradients are far from orthogonal: a few directions hold most of them
    for g, m, s in zip(_views(grad, offs, sizes), _views(mom, offs, sizes), sizes):
        left = torch.randn(s[0], 3, device=DEV, generator=gen)
        right = torch.randn(3, s[1], device=DEV, generator=gen)
        g += left @ right * 2e-3
        m += left @ right * 1e-3
    st = {"case": c, "sizes": sizes, "param": master.to(dt), "grad": grad.to(dt), "momentum": mom}
    st["params"], st["grads"] = _views(st["param"], offs, sizes), _views(st["grad"], offs, sizes)
    st["momenta"] = _views(mom, offs, sizes)
    if c["master"]:
        st["master"], st["masters"] = master, _views(master, offs, sizes)
    return st


def _lengths(st, gen, B, T):
    low = max(1, T // 4)
    lengths = torch.randint(low, T + 1, (B,), device=DEV, generator=gen, dtype=torch.int32)
    lengths[0] = T
    if B >= 8:
        lengths[B // 2] = 0   # a signal that is missing
    st["lengths"] = lengths
    return torch.arange(T, device=DEV)[None, :] >= lengths[:, None]


def _slices(parts, dt, packed, train):
    """[B, T, H, D] each, of type dt: slices of one tensor, or each its own."""
    if packed:
        B, T = parts[0].shape[:2]
        whole = torch.cat([p.reshape(B, T, -1) for p in parts], -1).to(dt)
        out, at = [], 0
        for p in parts:
            n = p.shape[2] * p.shape[3]
            out.append(whole[..., at:at + n].unflatten(-1, p.shape[2:]))
            at += n
    else:
        out = [p.to(dt) for p in parts]
    return [p.detach().requires_grad_(train) for p in out]


def prepare(case, seed):
    c = dict(case)
    gen = torch.Generator(device=DEV).manual_seed(int(seed))

    def normal(*shape):
        return torch.randn(*shape, device=DEV, generator=gen)

    if c["op"] == "muon":
        return _prepare_muon(c, gen)
    dt = TYPES[c["dtype"]]
    train = c["train"]
    st = {"case": c}
    B, T, H = c["batch"], c["time"], c["heads"]
    if c["op"] == "qk":
        K, D = c["key_heads"], c["width"]
        size = torch.exp(0.5 * normal(B, T, 1, 1))
        st["q"], st["k"] = _slices([normal(B, T, H, D) * size, normal(B, T, K, D) * size], dt,
                                   c["packed"], train)
        for name in ("q_weight", "k_weight"):
            st[name] = (1 + 0.1 * normal(D)).to(TYPES[c["weight"]]).requires_grad_(train)
        if c["turned"]:
            st["freqs"] = BASE ** (-torch.arange(0, c["turned"], 2, device=DEV) / c["turned"])
        if c["given"]:
            begin = torch.randint(0, 1 << 20, (B, 1), device=DEV, generator=gen)
            st["positions"] = begin + torch.arange(T, device=DEV)
        if train:
            st["dq"], st["dk"] = normal(B, T, H, D).to(dt), normal(B, T, K, D).to(dt)
        return st
    K, dk, dv = H // c["group"], c["dk"], c["dv"]
    # queries and keys of length 1, the keys near each other as those of a signal are
    shared = normal(B, 1, K, dk)
    q, k = normal(B, T, K, dk), normal(B, T, K, dk) + 0.5 * shared
    q, k = (t / t.norm(dim=-1, keepdim=True) for t in (q, k))
    v = normal(B, T, H, dv)
    # states that remember from 2 samples to some hundreds, by head
    keep = 6 * torch.rand(H, device=DEV, generator=gen)
    gate = -torch.nn.functional.softplus(-(normal(B, T, H) + keep))
    beta = torch.sigmoid(normal(B, T, H))
    if c["ragged"]:
        # what lies behind a signal's end is nobody's
        pad = _lengths(st, gen, B, T)
        for t in (q, k, v):
            t.masked_fill_(pad[..., None, None], float("nan"))
        for t in (gate, beta):
            t.masked_fill_(pad[..., None], float("nan"))
    st["q"], st["k"], st["v"] = _slices([q, k, v], dt, c["packed"], train)
    st["decay"] = gate.to(TYPES[c["gates"]]).requires_grad_(train)
    st["beta"] = beta.to(TYPES[c["gates"]]).requires_grad_(train)
    if c["start"]:
        st["h0"] = (0.5 * normal(B, H, dk, dv)).requires_grad_(train)
    if train:
        st["do"] = normal(B, T, H, dv).to(dt)
        st["dh"] = normal(B, H, dk, dv)
    return st


# --------------------------------------------------------------------------
# one pass
# --------------------------------------------------------------------------

def run(st):
    op = st["case"]["op"]
    if op == "muon":
        if own:
            _own_muon(st)
        else:
            _plain_muon(st)
        return {k: st[k] for k in ("param", "master", "momentum") if k in st}
    if op == "qk":
        return _own_qk(st) if own else _plain_qk(st)
    return _own_delta(st) if own else _plain_delta(st)


def _own_muon(st):
    _cpab().muon_step(st["params"], st["grads"], st["momenta"], nesterov=st["case"]["nesterov"],
                      masters=st.get("masters"), **MUON)


def _own_qk(st):
    c = st["case"]
    args = dict(neighbours=c["neighbours"], eps=EPS)
    if c["turned"]:   # positions go with frequencies: without these nothing turns
        args.update(freqs=st["freqs"], positions=st.get("positions"))
    given = [st[k] for k in ("q", "k", "q_weight", "k_weight")]
    if not c["train"]:
        with torch.no_grad():
            q, k = _cpab().qk_norm(*given, **args)
        return {"q": q, "k": k}
    q, k = _cpab().qk_norm(*given, **args)
    grads = torch.autograd.grad((q, k), given, (st["dq"], st["dk"]))
    return dict({"q": q, "k": k}, **dict(zip(("grad_q", "grad_k", "grad_q_weight", "grad_k_weight"),
                                             grads)))


def _own_delta(st):
    c = st["case"]
    names = [k for k in ("q", "k", "v", "decay", "beta", "h0") if k in st]
    given = [st[k] for k in names]
    if not c["train"]:
        with torch.no_grad():
            o, h = _cpab().gated_delta_rule(*given, lengths=st.get("lengths"))
        return {"o": o, "h": h}
    o, h = _cpab().gated_delta_rule(*given, lengths=st.get("lengths"))
    grads = torch.autograd.grad((o, h), given, (st["do"], st["dh"]))
    return dict({"o": o, "h": h}, **{"grad_" + k: v for k, v in zip(names, grads)})


# --------------------------------------------------------------------------
# the plain forms
# --------------------------------------------------------------------------

def _plain_muon(st):
    c = st["case"]
    mu, (a, b, cc) = MUON["momentum"], MUON["ns_coefficients"]
    values = st["masters"] if c["master"] else st["params"]
    # the matrices of one shape together
    for shape in sorted(set(st["sizes"])):
        at = [i for i, s in enumerate(st["sizes"]) if s == shape]
        g = torch.stack([st["grads"][i] for i in at]).float()
        m = torch.stack([st["momenta"][i] for i in at])
        m = mu * m + (1 - mu) * g
        x = mu * m + (1 - mu) * g if c["nesterov"] else m
        tall = shape[0] > shape[1]
        if tall:
            x = x.transpose(1, 2).contiguous()
        x = x / x.square().sum((1, 2), keepdim=True).sqrt().clamp(min=MUON["eps"])
        for _ in range(MUON["ns_steps"]):
            s = x @ x.transpose(1, 2).contiguous()
            x = a * x + (b * s + cc * (s @ s)) @ x
        if tall:
            x = x.transpose(1, 2)
        rate = MUON["lr"] * math.sqrt(max(1.0, shape[0] / shape[1]))
        w = torch.stack([values[i] for i in at]).float()
        w = w * (1 - MUON["lr"] * MUON["weight_decay"]) - rate * x
        for k, i in enumerate(at):
            st["momenta"][i].copy_(m[k])
            st["params"][i].copy_(w[k])
            if c["master"]:
                st["masters"][i].copy_(w[k])


def _pairs(x, turned, neighbours):
    """The two halves of each rotated pair."""
    if neighbours:
        return x[..., 0:turned:2], x[..., 1:turned:2]
    return x[..., :turned // 2], x[..., turned // 2:turned]


def _joined(a, b, rest, neighbours):
    whole = torch.stack([a, b], -1).flatten(-2) if neighbours else torch.cat([a, b], -1)
    return torch.cat([whole, rest], -1)


def _plain_qk(st):
    c = st["case"]
    R, side = c["turned"], c["neighbours"]
    with torch.no_grad():
        out = {}
        T = c["time"]
        if R:
            at = st["positions"] if c["given"] else torch.arange(T, device=DEV)[None]
            angle = at.double()[..., None] * st["freqs"].double()
            cos, sin = angle.cos().float()[:, :, None], angle.sin().float()[:, :, None]
        for name in ("q", "k"):
            x, w = st[name].float(), st[name + "_weight"].float()
            s = torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS)
            n = x * s
            y = n * w
            if R:
                a, b = _pairs(y, R, side)
                y = _joined(a * cos - b * sin, b * cos + a * sin, y[..., R:], side)
            out[name] = y.to(st[name].dtype)
            if c["train"]:
                dy = st["d" + name].float()
                if R:
                    a, b = _pairs(dy, R, side)
                    dy = _joined(a * cos + b * sin, b * cos - a * sin, dy[..., R:], side)
                u = dy * w
                out["grad_" + name] = (s * (u - n * (u * n).mean(-1, keepdim=True))).to(st[name].dtype)
                out["grad_" + name + "_weight"] = (dy * n).sum((0, 1, 2)).to(st[name + "_weight"].dtype)
        return out


CHUNK = 64


def _inverse(m):
    """Inverses of unit lower triangular matrices: the blocks on the diagonal double, and
    the block below joins two of them."""
    n = m.shape[-1]
    out = torch.eye(n, device=m.device, dtype=m.dtype).expand_as(m).clone()
    half = 1
    while half < n:
        blocks = m.unflatten(-1, (-1, 2 * half)).unflatten(-3, (-1, 2 * half))
        done = out.unflatten(-1, (-1, 2 * half)).unflatten(-3, (-1, 2 * half))
        below = torch.diagonal(blocks[..., half:, :, :half], 0, -4, -2).movedim(-1, -3)
        first = torch.diagonal(done[..., :half, :, :half], 0, -4, -2).movedim(-1, -3)
        second = torch.diagonal(done[..., half:, :, half:], 0, -4, -2).movedim(-1, -3)
        join = -(second.contiguous() @ below.contiguous() @ first.contiguous())
        torch.diagonal(done[..., half:, :, :half], 0, -4, -2).copy_(join.movedim(-3, -1))
        half *= 2
    return out


def _chunks(t, H, n, live):
    """[B, T, heads, D] to [B H, n, CHUNK, D] in 32 bits, zeros where nothing lives."""
    t = torch.where(live, t.float(), torch.zeros((), device=t.device))
    t = torch.nn.functional.pad(t, (0, 0, 0, 0, 0, n * CHUNK - t.shape[1]))
    t = t.repeat_interleave(H // t.shape[2], 2)
    return t.permute(0, 2, 1, 3).reshape(-1, n, CHUNK, t.shape[3])


def _tokens(t, B, T):
    """[B H, n, CHUNK, D] back to [B, T, H, D]."""
    t = t.reshape(B, -1, t.shape[1] * CHUNK, t.shape[3])[:, :, :T]
    return t.transpose(1, 2)


def _plain_step(st):
    """One sample of each row: the definition itself."""
    c = st["case"]
    with torch.no_grad():
        H = c["heads"]
        q, k = (st[x][:, 0].float().repeat_interleave(c["group"], 1) for x in ("q", "k"))
        v, decay, beta = (st[x][:, 0].float() for x in ("v", "decay", "beta"))
        if "lengths" in st:
            live = (st["lengths"] > 0)[:, None]
            q, k, v = (t.masked_fill(~live[..., None], 0) for t in (q, k, v))
            decay, beta = decay.masked_fill(~live, 0), beta.masked_fill(~live, 0)
        if "h0" in st:
            S = st["h0"] * decay.exp()[..., None, None]
        else:
            S = torch.zeros(c["batch"], H, c["dk"], c["dv"], device=DEV)
        u = beta[..., None] * (v - (S * k[..., None]).sum(2))
        S = S + k[..., None] * u[:, :, None]
        o = (S * (q * c["dk"] ** -0.5)[..., None]).sum(2)
        return {"o": o[:, None].to(st["q"].dtype), "h": S}


def _plain_delta(st):
    c = st["case"]
    if c["time"] == 1 and not c["train"]:
        return _plain_step(st)
    with torch.no_grad():
        B, T, H, dk, dv = (c[k] for k in ("batch", "time", "heads", "dk", "dv"))
        n = -(-T // CHUNK)
        scale = dk ** -0.5
        live = torch.ones(B, T, device=DEV, dtype=torch.bool)
        if "lengths" in st:
            live = torch.arange(T, device=DEV)[None] < st["lengths"][:, None]
        live = live[..., None, None]
        q, k, v = (_chunks(st[x], H, n, live) for x in ("q", "k", "v"))
        g, beta = (_chunks(st[x][..., None], H, n, live) for x in ("decay", "beta"))
        # between the samples of a chunk the decays' logarithms add up, in 64 bits
        G = g.double().cumsum(-2)
        low = torch.ones(CHUNK, CHUNK, device=DEV, dtype=torch.bool).tril()
        gap = (G - G.transpose(-1, -2)).masked_fill(~low, -math.inf)
        D = gap.exp().float()
        since, until = G.exp().float(), (G[..., -1:, :] - G).exp().float()
        total = since[..., -1:, :]
        kt = k.transpose(-1, -2).contiguous()
        kk = (D * (k @ kt)).tril(-1)
        P = scale * D * (q @ kt)
        inv = _inverse(kk * beta.transpose(-1, -2) + torch.eye(CHUNK, device=DEV))
        kg, kh, qg = k * since, k * until, q * (scale * since)
        W, X0, khb = inv @ kg, inv @ v, (kh * beta).transpose(-1, -2).contiguous()
        S = torch.zeros(B * H, n + 1, dk, dv, device=DEV)
        if "h0" in st:
            S[:, 0] = st["h0"].reshape(B * H, dk, dv)
        X = torch.empty(B * H, n, CHUNK, dv, device=DEV)
        for i in range(n):
            torch.baddbmm(X0[:, i], W[:, i], S[:, i], alpha=-1, out=X[:, i])
            S[:, i + 1] = torch.baddbmm(total[:, i] * S[:, i], khb[:, i], X[:, i])
        U = beta * X
        o = qg @ S[:, :-1] + P @ U
        dt, gt = st["q"].dtype, st["decay"].dtype
        out = {"o": _tokens(o, B, T).to(dt), "h": S[:, n].reshape(B, H, dk, dv).clone()}
        if not c["train"]:
            return out
        do = _chunks(st["do"], H, n, live)
        dS = torch.empty(B * H, n + 1, dk, dv, device=DEV)
        dS[:, n] = st["dh"].reshape(B * H, dk, dv)
        dU = P.transpose(-1, -2).contiguous() @ do
        Z = torch.empty_like(X)
        back = inv.transpose(-1, -2) * beta.transpose(-1, -2)
        add, kgt = qg.transpose(-1, -2).contiguous() @ do, kg.transpose(-1, -2).contiguous()
        for i in reversed(range(n)):
            dU[:, i] = torch.baddbmm(dU[:, i], kh[:, i], dS[:, i + 1])
            torch.bmm(back[:, i], dU[:, i], out=Z[:, i])
            dS[:, i] = torch.baddbmm(add[:, i] + total[:, i] * dS[:, i + 1], kgt[:, i], Z[:, i], alpha=-1)
        E = dU - kk.transpose(-1, -2).contiguous() @ Z
        dbeta = (X * E).sum(-1, keepdim=True)
        dP = scale * D * (do @ U.transpose(-1, -2).contiguous())
        M = -D.tril(-1) * beta.transpose(-1, -2) * (Z @ X.transpose(-1, -2).contiguous())
        before = S[:, :-1].transpose(-1, -2).contiguous()
        dq = scale * since * (do @ before) + dP @ k
        dkey = (dP.transpose(-1, -2).contiguous() @ q - since * (Z @ before)
                + until * (U @ dS[:, 1:].transpose(-1, -2).contiguous())
                + (M + M.transpose(-1, -2)) @ k)
        dG = (do.double() * o - Z.double() * v).sum(-1, keepdim=True)
        dG[..., -1, 0] += (S[:, 1:].double() * dS[:, 1:]).sum((-1, -2))
        dg = dG.flip(-2).cumsum(-2).flip(-2).float()

        def shared(t):   # the gradients of a key's value heads together
            return _tokens(t, B, T).reshape(B, T, -1, c["group"], dk).sum(3)

        zero = torch.zeros((), device=DEV)
        out["grad_q"], out["grad_k"] = shared(dq).to(dt), shared(dkey).to(dt)
        out["grad_v"] = _tokens(Z, B, T).to(dt)
        out["grad_decay"] = torch.where(live, _tokens(dg, B, T), zero)[..., 0].to(gt)
        out["grad_beta"] = torch.where(live, _tokens(dbeta, B, T), zero)[..., 0].to(gt)
        if "h0" in st:
            out["grad_h0"] = dS[:, 0].reshape(B, H, dk, dv).clone()
        return out


# --------------------------------------------------------------------------
# the same in 64 bits, from the definitions
# --------------------------------------------------------------------------

def _exact_muon(st):
    c = st["case"]
    mu, (a, b, cc) = MUON["momentum"], MUON["ns_coefficients"]
    out = {k: st[k].double() for k in ("param", "master", "momentum") if k in st}

    def place(name, part):
        at = (part.data_ptr() - st[name].data_ptr()) // st[name].element_size()
        return out[name][at:at + part.numel()].view(part.shape)

    for i, p in enumerate(st["params"]):
        g = st["grads"][i].double()
        m = place("momentum", st["momenta"][i])
        m += (1 - mu) * (g - m)
        x = g + mu * (m - g) if c["nesterov"] else m.clone()
        x /= max(float((x * x).sum()) ** 0.5, MUON["eps"])
        wide = x.shape[0] <= x.shape[1]
        for _ in range(MUON["ns_steps"]):
            # the same polynomial of the singular values, from the shorter side
            s = torch.mm(x, x.t()) if wide else torch.mm(x.t(), x)
            p2 = b * s + cc * torch.mm(s, s)
            x = a * x + (torch.mm(p2, x) if wide else torch.mm(x, p2))
        rows, cols = x.shape
        w = place("master", st["masters"][i]) if c["master"] else place("param", p)
        w -= MUON["lr"] * (MUON["weight_decay"] * w + max(1.0, rows / cols) ** 0.5 * x)
        if c["master"]:
            place("param", p).copy_(w)
    return out


def _exact_qk(st):
    c = st["case"]
    B, T, R = c["batch"], c["time"], c["turned"]
    i = torch.arange(R // 2, device=DEV)
    first, second = (2 * i, 2 * i + 1) if c["neighbours"] else (i, i + R // 2)
    if R:
        at = st["positions"] if c["given"] else torch.arange(T, device=DEV).expand(B, T)
        turn = torch.exp(1j * (at[:, :, None].double() * st["freqs"].double()))[:, :, None, :]
    out = {}
    for name in ("q", "k"):
        x, w = st[name].detach().double(), st[name + "_weight"].detach().double()
        D = x.shape[-1]
        root = ((x * x).sum(-1, keepdim=True) / D + EPS).sqrt()
        y = x / root * w
        if R:
            z = torch.complex(y[..., first], y[..., second]) * turn
            y[..., first], y[..., second] = z.real, z.imag
        out[name] = y
        if c["train"]:
            dy = st["d" + name].double()
            if R:
                z = torch.complex(dy[..., first], dy[..., second]) * turn.conj()
                dy[..., first], dy[..., second] = z.real, z.imag
            out["grad_" + name + "_weight"] = (dy * x / root).sum((0, 1, 2))
            u = dy * w
            out["grad_" + name] = u / root - x * (u * x).sum(-1, keepdim=True) / D / root ** 3
    return out


def _exact_delta(st):
    """Sample by sample; the backward from states that are computed again, some samples at
    a time."""
    c = st["case"]
    B, T, H, dk, dv = (c[k] for k in ("batch", "time", "heads", "dk", "dv"))
    N, group, scale = B * H, c["group"], dk ** -0.5
    dead = None
    if "lengths" in st:
        dead = torch.arange(T, device=DEV)[:, None] >= st["lengths"][None, :]

    def by_time(t, heads):
        """[T, B H, D], zeros behind a row's end."""
        t = t.detach().transpose(0, 1)
        if dead is not None:
            t = t.masked_fill(dead.view(T, B, *[1] * (t.dim() - 2)), 0)
        if heads != H:
            t = t[:, :, :, None].expand(-1, -1, -1, H // heads, -1)
        return t.reshape(T, N, -1).double()

    q, k = (by_time(st[x], H // group) for x in ("q", "k"))
    v, decay, beta = (by_time(st[x], H) for x in ("v", "decay", "beta"))
    a = decay.exp()
    S = torch.zeros(N, dk, dv, device=DEV, dtype=torch.float64)
    if "h0" in st:
        S = st["h0"].detach().double().reshape(N, dk, dv)

    def step(S, t):
        """(the state decayed, what the key misses, the state after)"""
        old = S * a[t][..., None]
        miss = v[t] - torch.bmm(k[t][:, None], old)[:, 0]
        return old, miss, torch.baddbmm(old, k[t][..., None], (beta[t] * miss)[:, None])

    span = 64
    kept, o = [], torch.empty(T, N, dv, device=DEV, dtype=torch.float64)
    for t in range(T):
        if t % span == 0:
            kept.append(S)
        S = step(S, t)[2]
        o[t] = torch.bmm(q[t][:, None], S)[:, 0] * scale

    def rows(t, tail):
        return t.view(T, B, H, *tail).transpose(0, 1)

    out = {"o": rows(o, (dv,)), "h": S.view(B, H, dk, dv)}
    if not c["train"]:
        return out
    do = by_time(st["do"], H)
    L = st["dh"].double().reshape(N, dk, dv)
    gq, gk, gv = torch.empty_like(q), torch.empty_like(k), torch.empty_like(v)
    ga, gb = torch.empty_like(a), torch.empty_like(a)
    for s in reversed(range(0, T, span)):
        S, seen = kept[s // span], []
        for t in range(s, min(T, s + span)):
            before = S
            old, miss, S = step(S, t)
            seen.append((before, old, miss, S))
        for t in reversed(range(s, min(T, s + span))):
            before, old, miss, after = seen.pop()
            gq[t] = torch.bmm(after, do[t][..., None])[..., 0] * scale
            L = torch.baddbmm(L, q[t][..., None], do[t][:, None], alpha=scale)
            du = torch.bmm(k[t][:, None], L)[:, 0]
            gb[t] = (du * miss).sum(-1, keepdim=True)
            gv[t] = beta[t] * du
            gk[t] = (torch.bmm(L, (beta[t] * miss)[..., None]) - torch.bmm(old, gv[t][..., None]))[..., 0]
            L = torch.baddbmm(L, k[t][..., None], gv[t][:, None], alpha=-1)
            ga[t] = a[t] * (L * before).sum((1, 2))[:, None]
            L = L * a[t][..., None]
    if dead is not None:
        ga.view(T, B, H).masked_fill_(dead[..., None], 0)
    for name, g, d in (("q", gq, dk), ("k", gk, dk)):
        out["grad_" + name] = rows(g, (d,)).reshape(B, T, H // group, group, d).sum(3)
    out["grad_v"] = rows(gv, (dv,))
    out["grad_decay"], out["grad_beta"] = rows(ga, ()), rows(gb, ())
    if "h0" in st:
        out["grad_h0"] = L.view(B, H, dk, dv)
    return out


def exact(case, seed):
    st = prepare(case, seed)
    return {"muon": _exact_muon, "qk": _exact_qk, "delta": _exact_delta}[case["op"]](st)


# --------------------------------------------------------------------------
# work
# --------------------------------------------------------------------------

def work(case):
    """Bytes: every input read once, every output written once.  Operations: a
    multiplication, an addition or a call of exp, a division or a root counts as one;
    a symmetric product counts its half."""
    c = case
    e = 4 if c["dtype"] == "f32" else 2
    if c["op"] == "muon":
        sizes = _sizes(c)
        n = sum(math.prod(s) for s in sizes)
        each = e + 8 + (e + 8 if c["master"] else 2 * e)   # g, momentum, parameter (and master)
        flops = 12.0 * n
        for r, k in sizes:
            m, w = float(min(r, k)), float(max(r, k))
            flops += MUON["ns_steps"] * (3 * m * m * w + m ** 3)
        return {"bytes": float(n) * each, "flops": flops}
    tokens = float(c["batch"]) * c["time"]
    if c["op"] == "qk":
        n = tokens * (c["heads"] + c["key_heads"]) * c["width"]
        at = tokens * 8 if c["given"] and c["turned"] else 0
        return {"bytes": n * e * (2 + (3 if c["train"] else 0)) + at,
                "flops": n * (8 + (16 if c["train"] else 0))}
    H, K, dk, dv = c["heads"], c["heads"] // c["group"], c["dk"], c["dv"]
    values = e * (2 * K * dk + 2 * H * dv)                  # q, k, v and o
    gates = (4 if c["gates"] == "f32" else 2) * 2 * H
    state = c["batch"] * H * dk * dv * 4.0
    bytes_ = tokens * (values + gates) + state * (1 + c["start"])
    flops = tokens * H * dk * dv * 6
    if c["train"]:
        # q, k, v and do again, their gradients; the gates and theirs; the states' gradients
        bytes_ += tokens * (e * (4 * K * dk + 3 * H * dv) + 2 * gates) + state * (1 + 2 * c["start"])
        flops += tokens * H * dk * dv * 12
    return {"bytes": bytes_, "flops": flops}
