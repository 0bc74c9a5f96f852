"""The operators around the transform in plain float64 torch on the CPU, written from
their definitions, and error bounds for 32-bit arithmetic."""
import numpy as np
import torch

U = 2.0 ** -24          # half a unit in the last place of a 32-bit float
UNIT = {torch.float32: U, torch.bfloat16: 2.0 ** -8}


def f64(t):
    return None if t is None else t.detach().double().cpu()


def recurrence(x, f, g=None, h0=None, lengths=None):
    """(y, h, all states [B, T + 1, C]), sample by sample."""
    B, T, C = x.shape
    h = torch.zeros(B, C, dtype=torch.float64) if h0 is None else h0
    states, ys = [h], []
    n = torch.full((B,), T) if lengths is None else lengths.long().clamp(0, T)
    for t in range(T):
        live = (t < n)[:, None]
        a = torch.sigmoid(f[:, t])
        new = a * h + torch.sigmoid(-f[:, t]) * x[:, t]
        h = torch.where(live, new, h)
        y = h if g is None else h * g[:, t] * torch.sigmoid(g[:, t])
        ys.append(torch.where(live, y, torch.zeros_like(y)))
        states.append(h)
    y = torch.stack(ys, 1) if T else torch.zeros(B, 0, C, dtype=torch.float64)
    return y, h, torch.stack(states, 1)


def padding_zeroed(t, lengths):
    """t with what lies behind each row's end as zeros (a NaN there would reach the
    64-bit gradients through 0 * NaN)."""
    if t is None or lengths is None:
        return t
    T = t.shape[1]
    live = torch.arange(T)[None, :] < lengths.long().clamp(0, T)[:, None]
    return torch.where(live[..., None], t, torch.zeros_like(t))


def recurrence_grads(x, f, g, h0, lengths, dy, dh):
    """The definition's gradients by float64 autograd: dict of arrays."""
    given = {k: v.clone().requires_grad_() for k, v in
             (("x", x), ("f", f), ("g", g), ("h0", h0)) if v is not None}
    y, h, _ = recurrence(given["x"], given["f"], given.get("g"), given.get("h0"), lengths)
    loss = (h * dh).sum() + (y * dy).sum()
    return dict(zip(given, torch.autograd.grad(loss, list(given.values()), allow_unused=True)))


def recurrence_memory(f, T):
    """Samples over which a rounding of a gate adds up: 1 / (1 - a) at most, and T."""
    if T == 0:
        return 1.0
    return min(float(T), 1.0 + float(torch.exp(f.max().clamp(max=60.0))))


def rms_norm(x, w, residual=None, eps=1e-6):
    r = x if residual is None else x + residual
    s = 1.0 / torch.sqrt((r * r).mean(-1, keepdim=True) + eps)
    return r * s * w, r, s


def rms_norm_grads(x, w, residual, eps, dy, dres):
    given = [t.clone().requires_grad_() for t in (x, w, residual) if t is not None]
    y, r, _ = rms_norm(given[0], given[1], given[2] if residual is not None else None, eps)
    loss = (y * dy).sum() + ((r * dres).sum() if dres is not None else 0.0)
    return torch.autograd.grad(loss, given)


def mix(z):
    z = z.astype(np.uint32)
    z ^= z >> np.uint32(16)
    z *= np.uint32(0x9E3779B1)
    z ^= z >> np.uint32(15)
    z *= np.uint32(0xB504F333)
    z ^= z >> np.uint32(16)
    return z


def random_bits(n, seed, step, ordinal):
    with np.errstate(over="ignore"):
        key = mix(np.array([(seed ^ (step * 0x9E3779B1)) & 0xFFFFFFFF], np.uint32)) + np.uint32(ordinal)
        return mix((np.arange(n, dtype=np.uint64) & 0xFFFFFFFF).astype(np.uint32) + mix(key))


def mx_scale(x):
    """Scale of each 32 values: the least power of two (from 2^-127) with
    max |finite x| <= 448 scale, by trying them."""
    pad = np.zeros(-len(x) % 32)
    top = np.where(np.isfinite(x), np.abs(x), 0.0)
    top = np.concatenate([top, pad]).reshape(-1, 32).max(1) if len(x) else np.zeros(0)
    powers = 2.0 ** np.arange(-127, 128)
    return powers[np.searchsorted(448 * powers, top, side="left")]


def mx_round(x, bits16, least=False):
    """(values in units of the scale, scales) of x [n] float64 rounded at random."""
    scale = mx_scale(x)
    a = np.abs(x) / np.repeat(scale, 32)[:len(x)]
    with np.errstate(divide="ignore", invalid="ignore"):
        e = np.floor(np.log2(np.maximum(a, 2.0 ** -6)))
        step = 2.0 ** (e - 3)
        z = np.floor(a / step + bits16 / 65536.0) * step
    if least:
        z = np.where(x > 0, np.maximum(z, 2.0 ** -9), z)
    return np.copysign(np.where(np.isfinite(x), z, np.nan), x), scale


def mx_values(codes, scales):
    """float64 values of float8_e4m3fn codes with float8_e8m0fnu scales."""
    s = 2.0 ** (scales.view(torch.uint8).cpu().numpy().astype(np.float64) - 127)
    c = codes.float().cpu().numpy().astype(np.float64)
    return c * np.repeat(s, 32)[:len(c)]


def adamw(p, g, m, v, step, lr, betas, eps, wd):
    b1, b2 = betas
    m = b1 * m + (1 - b1) * g
    v = b2 * v + (1 - b2) * g * g
    update = lr * (m / (1 - b1 ** step)) / (np.sqrt(v / (1 - b2 ** step)) + eps)
    return p - lr * wd * p - update, m, v
