"""The operators over heads in plain float64 torch on the CPU, written from their
definitions."""
import torch

U = 2.0 ** -24          # half a unit in the last place of a 32-bit float
UNIT = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}


def f64(t):
    return None if t is None else t.detach().double().cpu()


def pairs(R, neighbours):
    """Indices of the first and the second of each pair."""
    i = torch.arange(R // 2)
    return (2 * i, 2 * i + 1) if neighbours else (i, i + R // 2)


def turned(x, freqs, positions, neighbours, sign=1.0):
    """x [B, T, H, D] with its first 2 len(freqs) values turned."""
    if freqs is None:
        return x
    B, T = x.shape[:2]
    p = torch.arange(T, dtype=torch.float64).expand(B, T) if positions is None else positions.expand(B, T)
    angle = sign * p[:, :, None, None] * freqs
    a, b = pairs(2 * len(freqs), neighbours)
    y = x.clone()
    y[..., a] = x[..., a] * angle.cos() - x[..., b] * angle.sin()
    y[..., b] = x[..., b] * angle.cos() + x[..., a] * angle.sin()
    return y


def norm(x, w, eps):
    return x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * w


def qk_norm(q, k, qw, kw, freqs=None, positions=None, neighbours=False, eps=1e-6):
    return tuple(turned(norm(x, w, eps), freqs, positions, neighbours) for x, w in ((q, qw), (k, kw)))


def delta_rule(q, k, v, decay, beta, h0=None, lengths=None, scale=None):
    """(o, h), sample by sample."""
    B, T, H, dv = v.shape
    dk = q.shape[-1]
    scale = dk ** -0.5 if scale is None else scale
    q, k = (t.repeat_interleave(H // t.shape[2], 2) for t in (q, k))
    S = torch.zeros(B, H, dk, dv, dtype=torch.float64) if h0 is None else h0
    n = torch.full((B,), T) if lengths is None else lengths.long().clamp(0, T)
    out = []
    for t in range(T):
        live = (t < n)[:, None]
        old = S * torch.exp(decay[:, t])[..., None, None]
        miss = v[:, t] - (old * k[:, t, :, :, None]).sum(2)
        new = old + k[:, t, :, :, None] * (beta[:, t, :, None] * miss)[:, :, None]
        S = torch.where(live[..., None, None], new, S)
        o = scale * (S * q[:, t, :, :, None]).sum(2)
        out.append(torch.where(live[..., None], o, torch.zeros_like(o)))
    o = torch.stack(out, 1) if T else torch.zeros(B, 0, H, dv, dtype=torch.float64)
    return o, S


def muon(p, g, m, lr, wd, mu, nesterov, coefficients, eps, steps, rate):
    """(p, m) after a step."""
    m = mu * m + (1 - mu) * g
    x = mu * m + (1 - mu) * g if nesterov else m
    x = x / max(float(x.norm()), eps)
    a, b, c = coefficients
    for _ in range(steps):
        if x.shape[0] <= x.shape[1]:
            s = x @ x.T
            x = a * x + (b * s + c * s @ s) @ x
        else:
            s = x.T @ x
            x = a * x + x @ (b * s + c * s @ s)
    return p * (1 - lr * wd) - rate * x, m


def delta_rule_grads(q, k, v, decay, beta, h0, lengths, scale, do, dh):
    """(gradients by name, sizes): the definition's gradients, sample by sample backwards,
    and the largest norms that what they are sums of reach."""
    B, T, H, dv = v.shape
    dk, K = q.shape[-1], q.shape[2]
    scale = dk ** -0.5 if scale is None else scale
    qh, kh = (t.repeat_interleave(H // K, 2) for t in (q, k))
    S = torch.zeros(B, H, dk, dv, dtype=torch.float64) if h0 is None else h0
    n = torch.full((B,), T) if lengths is None else lengths.long().clamp(0, T)
    seen = []
    for t in range(T):
        live = (t < n).double()[:, None]
        a = torch.where(live > 0, decay[:, t].exp(), torch.ones(()).double())
        b = torch.where(live > 0, beta[:, t], torch.zeros(()).double())
        kt = torch.where(live[..., None] > 0, kh[:, t], torch.zeros(()).double())
        old = S * a[..., None, None]
        miss = torch.where(live[..., None] > 0, v[:, t], torch.zeros(()).double()) - (old * kt[..., None]).sum(2)
        seen.append((S, old, a, b, kt, miss, live))
        S = old + kt[..., None] * (b[..., None] * miss)[:, :, None]
    size = {"S": 0.0, "L": 0.0, "x": 0.0, "e": 0.0}
    L = dh.clone()
    g = {"q": torch.zeros(B, T, H, dk).double(), "k": torch.zeros(B, T, H, dk).double(), "v": torch.zeros_like(v),
         "decay": torch.zeros_like(decay), "beta": torch.zeros_like(beta)}
    after = S

    def largest(name, t):
        if t.numel():
            size[name] = max(size[name], float(t.abs().max()))
    for t in reversed(range(T)):
        S, old, a, b, kt, miss, live = seen[t]
        qt = torch.where(live[..., None] > 0, qh[:, t], torch.zeros(()).double())
        ot = torch.where(live[..., None] > 0, do[:, t], torch.zeros(()).double())
        g["q"][:, t] = scale * (after * ot[:, :, None]).sum(3)
        L = L + scale * qt[..., None] * ot[:, :, None]
        du = (L * kt[..., None]).sum(2)
        largest("L", L.norm(dim=(2, 3)))
        largest("S", after.norm(dim=(2, 3)))
        largest("x", miss.norm(dim=2))
        largest("e", du.norm(dim=2))
        g["beta"][:, t] = (du * miss).sum(2)
        g["v"][:, t] = b[..., None] * du
        g["k"][:, t] = (L * (b[..., None] * miss)[:, :, None]).sum(3) - (old * g["v"][:, t][:, :, None]).sum(3)
        L = L - kt[..., None] * g["v"][:, t][:, :, None]
        g["decay"][:, t] = torch.where(live > 0, (L * old).sum((2, 3)), torch.zeros(()).double())
        L = L * a[..., None, None]
        after = S
    largest("S", S.norm(dim=(2, 3)))
    largest("L", L.norm(dim=(2, 3)))
    for name in ("q", "k"):
        g[name] = g[name].view(B, T, K, H // K, dk).sum(3)
    g["h0"] = L
    return g, size
