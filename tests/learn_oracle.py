"""The learned-filter operators and the AdamW step in float64, step by step, with the bounds that the tests hold float32 kernels to.

Every function takes float64 CPU tensors.  `Bound`s: half a step of the stored type relative to the value, plus 2^-24 times a count of
roundings times the same expression over absolute values (what those roundings can move)."""
import torch

EPS32 = 2.0 ** -24          # half a step of float32


def half(dtype):
    return torch.finfo(dtype).eps / 2


def silu(v):
    return v * torch.sigmoid(v)


def conv(x, w, bias=None, state=None, lengths=None, act=False):
    """y, last: causal_conv on [B, T, D]."""
    B, T, D = x.shape
    W = w.shape[1]
    state = x.new_zeros(B, W - 1, D) if state is None else state
    ys, lasts = [], []
    for b in range(B):
        n = T if lengths is None else min(max(int(lengths[b]), 0), T)
        line = torch.cat((state[b], x[b, :n]))
        v = sum(line[k:k + n] * w[:, k] for k in range(W))
        v = v if bias is None else v + bias
        y = silu(v) if act else v
        ys.append(torch.cat((y, x.new_zeros(T - n, D))))
        lasts.append(line[n:])
    return torch.stack(ys), torch.stack(lasts)


def scan(u, delta, A, Bm, Cm, D=None, z=None, delta_bias=None, softplus=False, state=None, lengths=None):
    """y, last: selective_scan; B, C [B, T, G, N]."""
    B, T, nD = u.shape
    G = Bm.shape[2]
    group = torch.arange(nD) // (nD // G)
    raw = delta if delta_bias is None else delta + delta_bias
    dl = torch.nn.functional.softplus(raw, threshold=1e9) if softplus else raw
    h = u.new_zeros(B, nD, A.shape[1]) if state is None else state
    n = torch.full((B,), T) if lengths is None else lengths.clamp(0, T)
    ys = []
    for t in range(T):
        on = (t < n)[:, None]
        new = torch.exp(dl[:, t, :, None] * A) * h + (dl[:, t] * u[:, t])[..., None] * Bm[:, t, group]
        h = torch.where(on[..., None], new, h)
        y = (h * Cm[:, t, group]).sum(-1)
        y = y if D is None else y + D * u[:, t]
        y = y if z is None else y * silu(z[:, t])
        ys.append(torch.where(on, y, torch.zeros_like(y)))
    return torch.stack(ys, 1), h


def scan_size(u, delta, A, Bm, Cm, D=None, z=None, delta_bias=None, softplus=False, state=None, lengths=None):
    """The scan of absolute values (the step sizes and decays themselves are positive): what relative roundings act on.  Each step's
    decay is charged for the rounding of its exponent, which is relative to 1 + |dl A|."""
    raw = delta if delta_bias is None else delta + delta_bias
    dl = torch.nn.functional.softplus(raw, threshold=1e9) if softplus else raw
    ab = lambda t: None if t is None else t.abs()  # noqa: E731
    gate = None if z is None else ab(silu(z))
    y, h = scan(ab(u), ab(dl), A, ab(Bm), ab(Cm), ab(D), None, None, False, ab(state), lengths)
    return (y if gate is None else y * gate), h


def adamw(p, g, m, v, step, lr, betas, eps, weight_decay):
    b1, b2 = betas
    m = b1 * m + (1 - b1) * g
    v = b2 * v + (1 - b2) * g * g
    return p * (1 - lr * weight_decay) - lr * (m / (1 - b1 ** step)) / (torch.sqrt(v / (1 - b2 ** step)) + eps), m, v


def pack8(x, root=False):
    """(e4m3 values, scales) of blocks of 256 of a float64 vector whose length is a multiple of 256."""
    x = x.reshape(-1, 256)
    top = x.abs().amax(1, keepdim=True)
    unit = torch.where(top < 1e-30, torch.ones_like(top), top / 448)
    r = torch.where(top < 1e-30, torch.zeros_like(x), x / unit)
    step = torch.exp2(torch.floor(torch.log2(r.abs().clamp(min=2.0 ** -6))) - 3)
    code = torch.round(r / step) * step
    if root:
        code = torch.where((code == 0) & (r > 0), torch.full_like(code, 2.0 ** -9), code)
    return code.reshape(-1), torch.where(top < 1e-30, torch.zeros_like(top), top / 448).reshape(-1)
