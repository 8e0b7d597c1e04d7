"""lqg_amd.belief.ssm: the short causal convolution and the selective state-space scan, against float64 step by step."""
import gc

import pytest
import torch

import learn_oracle as O
from lqg_amd import options
from lqg_amd._abi import LqgHipError
from lqg_amd.belief import ssm

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
gpu = pytest.mark.gpu


def rnd(gen, *shape, dtype=F32, scale=1.0, dev="cuda"):
    return (torch.randn(*shape, generator=gen) * scale).to(dtype).to(dev)


def d64(t):
    return None if t is None else t.detach().double().cpu()


def within(got, ref, bound, what=""):
    got, err = d64(got), (d64(got) - ref).abs()
    worst = float((err / bound.clamp(min=1e-300)).max()) if got.numel() else 0.0
    assert torch.isfinite(got).all() and worst <= 1.0, f"{what}: {worst:.2f} of the bound"


# ------------------------------------------------------------------------------------------------ refusals (no GPU)

def _conv_inputs():
    return torch.zeros(2, 5, 6), torch.zeros(6, 4)


def test_conv_refuses():
    x, w = _conv_inputs()
    for bad, msg in (
            (lambda: ssm.causal_conv(x[0], w), "x: a tensor of 3 dimensions"),
            (lambda: ssm.causal_conv(x.double(), w), "x: float32, bfloat16 or float16"),
            (lambda: ssm.causal_conv(x, torch.zeros(6, 9)), "weight: shape"),
            (lambda: ssm.causal_conv(x, torch.zeros(5, 4)), "weight: shape"),
            (lambda: ssm.causal_conv(x, torch.zeros(6, 0)), "weight: shape"),
            (lambda: ssm.causal_conv(x, w.double()), "weight: float32"),
            (lambda: ssm.causal_conv(x, w, torch.zeros(5)), "bias: shape"),
            (lambda: ssm.causal_conv(x, w, state=torch.zeros(2, 4, 6)), "state: "),
            (lambda: ssm.causal_conv(x, w, state=torch.zeros(2, 3, 6, dtype=BF16)), "state: "),
            (lambda: ssm.causal_conv(x, w, lengths=torch.tensor([1.0, 2.0])), "lengths: "),
            (lambda: ssm.causal_conv(x, w, lengths=torch.tensor([1, 2, 3])), "lengths: "),
            (lambda: ssm.causal_conv(x, w), "no CPU fallback"),
            (lambda: ssm.causal_conv_step(x, torch.zeros(2, 3, 6), w), "x: a tensor of 2 dimensions"),
            (lambda: ssm.causal_conv_step(x[:, 0], None, w), "state: "),
            (lambda: ssm.causal_conv_step(x[:, 0], torch.zeros(3, 2, 6).transpose(0, 1), w), "state: a contiguous"),
            (lambda: ssm.causal_conv_step(x[:, 0], torch.zeros(1, 3, 6).expand(2, 3, 6), w), "state: a contiguous"),
            (lambda: ssm.causal_conv_step(x[:, 0].requires_grad_(), torch.zeros(2, 3, 6), w), "no gradient"),
            (lambda: ssm.causal_conv_step(x[:, 0], torch.zeros(2, 3, 6), w), "no CPU fallback")):
        with pytest.raises(LqgHipError, match=msg.replace("(", r"\(")):
            bad()
    both = torch.zeros(2, 3, 6)
    with pytest.raises(LqgHipError, match="shares memory"):
        ssm.causal_conv_step(both[:, 0], both, w)


def _scan_inputs(T=5, N=4, G=None):
    u = torch.zeros(2, T, 6)
    m = torch.zeros(2, T, N) if G is None else torch.zeros(2, T, G, N)
    return dict(u=u, delta=u.clone(), A=torch.zeros(6, N), B=m, C=m.clone())


def test_scan_refuses():
    i = _scan_inputs()
    for change, msg in (
            (dict(u=i["u"].double()), "u: float32"), (dict(u=i["u"][0]), "u: a tensor of 3 dimensions"),
            (dict(delta=i["u"].to(BF16)), "delta: torch.bfloat16 on cpu"), (dict(delta=torch.zeros(2, 5, 7)), "delta: the shape of u"),
            (dict(z=torch.zeros(2, 4, 6)), "z: the shape of u"), (dict(A=torch.zeros(5, 4)), "A: shape"),
            (dict(A=torch.zeros(6, 65)), "A: shape"), (dict(A=torch.zeros(6, 4).double()), "A: float32"),
            (dict(B=torch.zeros(2, 5, 3)), "B: shape"), (dict(B=torch.zeros(2, 5, 4, 4)), "B: shape"),
            (dict(B=torch.zeros(2, 5, 2, 4)), "the same groups"), (dict(C=torch.zeros(2, 4, 4)), "C: shape"),
            (dict(D=torch.zeros(5)), "D: shape"), (dict(delta_bias=torch.zeros(7)), "delta_bias: shape"),
            (dict(state=torch.zeros(2, 6, 4, dtype=BF16)), "state: "), (dict(state=torch.zeros(2, 6, 3)), "state: "),
            (dict(lengths=torch.zeros(2)), "lengths: "), ({}, "no CPU fallback")):
        with pytest.raises(LqgHipError, match=msg):
            ssm.selective_scan(**{**i, **change})
    s = {k: (v[:, 0] if v.dim() == 3 else v) for k, v in i.items()}
    st = torch.zeros(2, 6, 4)
    for change, msg in ((dict(state=None), "state: "), (dict(state=torch.zeros(2, 4, 6).transpose(1, 2)), "contiguous"),
                        (dict(u=s["u"].clone().requires_grad_()), "no gradient"), (dict(u=i["u"]), "u: a tensor of 2"),
                        (dict(state=st), "no CPU fallback")):
        with pytest.raises(LqgHipError, match=msg):
            ssm.selective_scan_step(**{**s, "state": st, **change})


# ------------------------------------------------------------------------------------------------ convolution

CONV = [  # B, T, D, W, dtype, silu, bias, state, lengths
    (1, 1, 1, 1, F32, False, False, False, None), (1, 1, 3, 4, F32, True, True, False, None),
    (2, 2, 65, 4, F32, True, True, True, (2, 1)), (3, 37, 130, 3, F32, False, True, True, (0, 37, 20)),
    (2, 129, 257, 4, BF16, True, True, True, None), (2, 300, 64, 2, F16, True, False, False, (300, 129)),
    (1, 33, 300, 8, F32, True, True, True, (31,)), (5, 5, 70, 7, BF16, False, True, True, (5, 4, 3, 1, 0)),
    (2, 64, 33, 5, F16, True, True, True, None), (2, 40, 20, 6, F32, True, False, True, (1000, -5)),
    (300, 9, 16, 4, F32, True, True, True, None),
]


def conv_case(B, T, D, W, dtype, act, bias, state, lengths, seed=0):
    g = torch.Generator().manual_seed(seed + T * 131 + D)
    wide = rnd(g, B, T, D + 3, dtype=dtype)
    return dict(x=wide[..., 1:D + 1], weight=rnd(g, D, W, dtype=dtype, scale=0.5), bias=rnd(g, D, dtype=F32) if bias else None,
                state=rnd(g, B, W - 1, D, dtype=dtype) if state else None,
                lengths=torch.tensor(lengths, device="cuda") if lengths is not None else None), act, rnd(g, B, T, D, dtype=dtype), \
        rnd(g, B, W - 1, D, dtype=dtype)


def conv_bound(i, act, dtype, y):
    """W + 1 fused roundings of the sum; silu turns a relative error of v into one of y times at most 1.1 + |v| and adds 4 ulp and the
    rounding of its exponent (2 |v|)."""
    W = i["weight"].shape[1]
    n = None if i["lengths"] is None else i["lengths"].cpu()
    absd = lambda t: None if t is None else d64(t).abs()  # noqa: E731
    S, _ = O.conv(absd(i["x"]), absd(i["weight"]), absd(i["bias"]), absd(i["state"]), n)
    return O.half(dtype) * y.abs() + O.EPS32 * ((W + 1) * 1.1 + (4 + 4 * S if act else 0) + 1) * S + 1e-37 + (2.0 ** -25 if dtype == F16 else 0)


@gpu
@pytest.mark.parametrize("case", CONV, ids=str)
def test_conv_forward_and_state(case):
    i, act, _, _ = conv_case(*case)
    n = None if i["lengths"] is None else i["lengths"].cpu()
    y, last = ssm.causal_conv(**i, silu=act, return_state=True)
    ref, rlast = O.conv(d64(i["x"]), d64(i["weight"]), d64(i["bias"]), d64(i["state"]), n, act)
    within(y, ref, conv_bound(i, act, case[4], ref), "y")
    assert torch.equal(d64(last), rlast)
    assert torch.equal(ssm.causal_conv(**i, silu=act), y)


@gpu
@pytest.mark.parametrize("case", CONV, ids=str)
def test_conv_gradients(case):
    i, act, dy, dlast = conv_case(*case)
    n = None if i["lengths"] is None else i["lengths"].cpu()
    names = [k for k in ("x", "weight", "bias", "state") if i[k] is not None]
    leaves = {k: i[k].detach().requires_grad_() for k in names}
    y, last = ssm.causal_conv(**{**i, **leaves}, silu=act, return_state=True)
    got = torch.autograd.grad((y, last), list(leaves.values()), (dy, dlast))
    dl = {k: d64(i[k]).requires_grad_() for k in names}
    ry, rl = O.conv(*(dl.get(k) for k in ("x", "weight", "bias", "state")), n, act)
    ref = torch.autograd.grad((ry, rl), list(dl.values()), (d64(dy), d64(dlast)))
    # the same sums over absolute values; act' <= 1.1 and its own error is below 8 + 8 S ulp of 1 + S, S = sum |w x|
    ab = {k: d64(i[k]).abs().requires_grad_() for k in names}
    ay, al = O.conv(*(ab.get(k) for k in ("x", "weight", "bias", "state")), n, False)
    big = float(ay.detach().max()) if act else 0.0
    size = torch.autograd.grad((ay, al), list(ab.values()), (d64(dy).abs() * (1.1 if act else 1.0), d64(dlast).abs()))
    W = i["weight"].shape[1]
    terms = 2 * W + 4 + (8 + 8 * big) * (1 + big)
    for k, a, r, s in zip(names, got, ref, size):
        dt = i[k].dtype
        # (sums over a lane's 128 steps are sequential in float; the sums of those are in double)
        m = terms + (128 if k in ("weight", "bias") else 0)
        within(a, r, O.half(dt) * r.abs() + O.EPS32 * m * s + 1e-37 + (2.0 ** -25 if dt == F16 else 0), k)


@gpu
def test_conv_gradient_against_differences():
    g = torch.Generator().manual_seed(3)
    x, w, b, st = rnd(g, 2, 7, 5), rnd(g, 5, 4, scale=0.5), rnd(g, 5), rnd(g, 2, 3, 5)
    dy = rnd(g, 2, 7, 5)
    f = lambda *a: float((d64(ssm.causal_conv(a[0], a[1], a[2], state=a[3], silu=True)) * d64(dy)).sum())  # noqa: E731
    ins = [t.clone().requires_grad_() for t in (x, w, b, st)]
    grads = torch.autograd.grad(ssm.causal_conv(ins[0], ins[1], ins[2], state=ins[3], silu=True), ins, dy)
    for j, t in enumerate((x, w, b, st)):
        v = rnd(g, *t.shape)
        h = 2.0 ** -6
        up, dn = [[a + s * h * v if k == j else a for k, a in enumerate((x, w, b, st))] for s in (1, -1)]
        est, want = (f(*up) - f(*dn)) / (2 * h), float((grads[j] * v).sum())
        # rounding: |f| of some 100 terms at 2^-24 over h = 1e-3 at most; truncation h^2 / 6 times third derivatives of order 10^2
        assert abs(est - want) < 2e-2 + 1e-2 * abs(want), (j, est, want)


@gpu
@pytest.mark.parametrize("dtype", (F32, BF16))
def test_conv_steps_continue_a_prompt(dtype):
    g = torch.Generator().manual_seed(5)
    x, w, b = rnd(g, 3, 12, 70, dtype=dtype), rnd(g, 70, 4, dtype=dtype), rnd(g, 70, dtype=dtype)
    whole, last = ssm.causal_conv(x, w, b, silu=True, return_state=True)
    y, st = ssm.causal_conv(x[:, :7], w, b, silu=True, return_state=True)
    assert torch.equal(y, whole[:, :7])
    y2, st2 = ssm.causal_conv(x[:, 7:], w, b, state=st, silu=True, return_state=True)
    assert torch.equal(y2, whole[:, 7:]) and torch.equal(st2, last)
    for t in range(7, 12):
        before = st._version
        assert torch.equal(ssm.causal_conv_step(x[:, t], st, w, b, silu=True), whole[:, t])
        assert st._version > before
    assert torch.equal(st, last)


@gpu
def test_padding_is_never_used():
    """NaN and infinities behind a trial's end reach nothing."""
    g = torch.Generator().manual_seed(6)
    n = torch.tensor([5, 0, 19], device="cuda", dtype=torch.int32)
    pad = (torch.arange(20, device="cuda") >= n[:, None])[..., None]
    x, w = rnd(g, 3, 20, 66), rnd(g, 66, 4)
    for junk in (float("nan"), float("inf"), -3.4e38):
        leaves = [torch.where(pad, junk, x).requires_grad_(), w.clone().requires_grad_()]
        clean = [torch.where(pad, 0.0, x).requires_grad_(), w.clone().requires_grad_()]
        dy = rnd(g, 3, 20, 66)
        a = ssm.causal_conv(*leaves, lengths=n, silu=True, return_state=True)
        b = ssm.causal_conv(*clean, lengths=n, silu=True, return_state=True)
        ga = torch.autograd.grad(a[0], leaves, torch.where(pad, junk, dy))
        gb = torch.autograd.grad(b[0], clean, torch.where(pad, 0.0, dy))
        for p, q in zip((*a, *ga), (*b, *gb)):
            assert torch.equal(p, q)
    i, kw = scan_case(3, 20, 66, 6, 2, F32, gate=True, softplus=True, state=True, skip=True, bias=True, lengths=(5, 0, 19))
    seqs = ("u", "delta", "B", "C", "z")
    for junk in (float("nan"), float("inf"), -3.4e38):
        outs = []
        for fill in (junk, 0.0):
            v = {k: (torch.where(pad if t.dim() == 3 else pad[..., None], fill, t) if k in seqs else t).detach().requires_grad_()
                 for k, t in i.items() if t is not None and k != "lengths"}
            y, last = ssm.selective_scan(**v, lengths=n, return_state=True, **kw)
            grads = torch.autograd.grad((y, last), list(v.values()), (torch.where(pad, fill, i["u"]), i["state"]))
            outs.append((y, last, *grads))
        for p, q in zip(*outs):
            assert torch.equal(p, q)


# ------------------------------------------------------------------------------------------------ scan

SCAN = [  # B, T, D, N, G, dtype, gate, softplus, state, D skip, delta bias, lengths
    (1, 1, 1, 1, 1, F32, False, False, False, False, False, None), (1, 1, 5, 16, 1, F32, True, True, True, True, True, None),
    (2, 17, 65, 16, 1, F32, True, True, False, True, True, None), (3, 33, 130, 6, 2, F32, False, True, True, True, True, (0, 33, 16)),
    (2, 40, 96, 13, 3, BF16, True, True, True, False, True, (40, 23)), (1, 16, 64, 20, 1, F32, True, True, True, True, False, None),
    (2, 19, 70, 40, 1, F32, True, True, True, True, True, (19, 9)), (1, 50, 200, 64, 2, F16, True, True, False, True, True, None),
    (2, 100, 64, 4, 1, F32, False, False, True, False, False, (99, 100)), (4, 35, 63, 8, 1, F16, True, True, True, True, True, (35, 1, 0, 17)),
    (2, 31, 33, 2, 33, F32, True, True, True, True, True, None), (2, 150, 80, 16, 1, BF16, True, True, True, True, True, (150, 77)),
    (70, 3, 8, 5, 2, F32, True, True, True, True, True, None),
    # long enough for the loops over whole tiles, each shape of a workgroup
    (2, 200, 40, 16, 1, F32, True, True, True, True, True, (200, 131)), (2, 150, 72, 20, 3, F32, True, True, True, True, True, (97, 150)),
    (3, 130, 33, 6, 1, BF16, False, True, True, True, True, (130, 128, 5)), (1, 90, 70, 40, 2, F16, True, True, False, True, True, None),
    (2, 176, 40, 3, 2, F32, True, True, True, True, True, None), (1, 128, 64, 13, 1, F32, False, True, False, False, True, None),
]
KEYS = ("gate", "softplus", "state", "skip", "bias", "lengths")


def scan_case(B, T, D, N, G, dtype, gate=False, softplus=False, state=False, skip=False, bias=False, lengths=None, seed=0):
    g = torch.Generator().manual_seed(seed + T * 131 + D * 7 + N)
    wide, proj = rnd(g, B, T, 2 * D + 1, dtype=dtype), rnd(g, B, T, 2 * G * N + 1, dtype=dtype)
    delta = rnd(g, B, T, D, dtype=dtype, scale=0.5)
    if not softplus:
        delta = (delta.abs() * 0.3).to(dtype)
    i = dict(u=wide[..., 1:D + 1], delta=delta, A=-torch.rand(D, N, generator=g).cuda() * 2,
             B=proj[..., :G * N].unflatten(-1, (G, N)), C=proj[..., G * N:2 * G * N].unflatten(-1, (G, N)),
             D=rnd(g, D) if skip else None, z=wide[..., D + 1:] if gate else None, delta_bias=rnd(g, D) - 2 if bias else None,
             state=rnd(g, B, D, N) if state else None,
             lengths=torch.tensor(lengths, device="cuda", dtype=torch.int32) if lengths is not None else None)
    return i, dict(softplus=softplus)


ORDER = ("u", "delta", "A", "B", "C", "D", "z", "delta_bias")


def scan_ref(i, kw):
    n = None if i["lengths"] is None else i["lengths"].cpu().long()
    args = [d64(i[k]) for k in ORDER]
    y, h = O.scan(*args, kw["softplus"], d64(i["state"]), n)
    sy, sh = O.scan_size(*args, kw["softplus"], d64(i["state"]), n)
    raw = args[1] if i["delta_bias"] is None else args[1] + args[7]
    dl = torch.nn.functional.softplus(raw) if kw["softplus"] else raw
    # per step: decay 3 roundings + its exponent's (dl 12 ulp, product 2) times |dl A|; input term 16; addition 1
    per = 20 + 14 * float((dl.abs().max() * args[2].abs().max()))
    return y, h, sy, sh, per


def scan_bounds(i, kw, dtype):
    y, h, sy, sh, per = scan_ref(i, kw)
    T, N = i["u"].shape[1], i["A"].shape[1]
    gate = 12 if i["z"] is not None else 0
    zmax = float(d64(i["z"]).abs().max()) if gate else 0.0
    k = per * T + N + 4 + gate + 4 * zmax
    return y, h, O.half(dtype) * y.abs() + O.EPS32 * k * sy + 1e-37 + (2.0 ** -25 if dtype == F16 else 0), O.EPS32 * per * T * sh + 1e-37


@gpu
@pytest.mark.parametrize("chunks", (0, 1, 3, 64))
@pytest.mark.parametrize("case", SCAN, ids=str)
def test_scan_forward_and_state(case, chunks):
    i, kw = scan_case(*case[:6], **dict(zip(KEYS, case[6:])))
    y, h, by, bh = scan_bounds(i, kw, case[5])
    with options.override(SELSCAN_CHUNKS=chunks):
        got, last = ssm.selective_scan(**i, **kw, return_state=True)
    within(got, y, by, "y")
    within(last, h, bh, "state")


@gpu
@pytest.mark.parametrize("chunks", (0, 1, 3, 64))
@pytest.mark.parametrize("case", SCAN, ids=str)
def test_scan_gradients(case, chunks):
    i, kw = scan_case(*case[:6], **dict(zip(KEYS, case[6:])))
    dtype, names = case[5], [k for k in (*ORDER, "state") if i[k] is not None]
    g = torch.Generator().manual_seed(11)
    dy, dlast = rnd(g, *i["u"].shape, dtype=dtype), rnd(g, *i["u"].shape[::2], i["A"].shape[1])
    leaves = {k: i[k].detach().requires_grad_() for k in names}
    with options.override(SELSCAN_CHUNKS=chunks):
        y, last = ssm.selective_scan(**{**i, **leaves}, **kw, return_state=True)
        got = torch.autograd.grad((y, last), list(leaves.values()), (dy, dlast))
    n = None if i["lengths"] is None else i["lengths"].cpu().long()
    up = {k: d64(i[k]).requires_grad_() for k in names}
    ry, rl = O.scan(*(up.get(k) for k in ORDER), kw["softplus"], up.get("state"), n)
    ref = torch.autograd.grad((ry, rl), list(up.values()), (d64(dy), d64(dlast)))
    # The sizes that roundings act on: the gradients of the scan of absolute values, with step sizes as they are, for |dy silu(z)|.
    raw = d64(i["delta"]) + (0 if i["delta_bias"] is None else d64(i["delta_bias"]))
    dl = torch.nn.functional.softplus(raw) if kw["softplus"] else raw
    ab = {k: d64(i[k]).abs().requires_grad_() for k in ("u", "B", "C", "D", "state") if i[k] is not None}
    step, decay = dl.clone().requires_grad_(), (-d64(i["A"]).abs()).requires_grad_()
    ay, al = O.scan(ab["u"], step, decay, ab["B"], ab["C"], ab.get("D"), None, None, False, ab.get("state"), n)
    gate = 1.0 if i["z"] is None else O.silu(d64(i["z"])).abs()
    w = d64(dy).abs() * gate
    asked = [*ab.values(), step, decay]
    size = dict(zip([*ab, "step", "A"], torch.autograd.grad((ay, al), asked, (w, d64(dlast).abs()))))
    # d/d step of the decays is negative where that of the inputs is positive: sum their magnitudes, (input term) - (decay term)
    through = size["u"] - (w * ab["D"].detach() if "D" in ab else 0)
    size["step"] = size["step"].abs() + 2 * through.clamp(min=0) * ab["u"].detach() / dl.abs().clamp(min=1e-30)
    size["delta"] = size["step"]
    lead = (size["step"] if n is None else size["step"] * (torch.arange(dl.shape[1])[None] < n[:, None])[..., None])
    size["delta_bias"] = lead.sum((0, 1))
    size["A"] = size["A"].abs()
    if i["z"] is not None:
        z = d64(i["z"])
        sg = torch.sigmoid(z)
        size["z"] = d64(dy).abs() * ay.detach() * (sg * (1 + z.abs() * (1 - sg)))
    T, N = i["u"].shape[1], i["A"].shape[1]
    zmax = 0.0 if i["z"] is None else float(d64(i["z"]).abs().max())
    per = 24 + 14 * float(dl.abs().max() * d64(i["A"]).abs().max())
    k_ = 2 * per * T + 2 * N + 24 + 8 * zmax + i["u"].shape[2]
    for k, a, r in zip(names, got, ref):
        dt = a.dtype
        within(a, r, O.half(dt) * r.abs() + O.EPS32 * k_ * size[k] + 1e-37 + (2.0 ** -25 if dt == F16 else 0), k)
        # the bounds above are wide where T is: what most elements show is far less (a factor of 8 over all of them)
        wide = O.EPS32 * k_ * float(size[k].norm()) / 8 + O.half(dt) * float(r.norm()) + 1e-30
        assert float((d64(a) - r).norm()) <= wide + (2.0 ** -25 * r.numel() ** 0.5 if dt == F16 else 0), k


@gpu
def test_scan_gradient_against_differences():
    i, kw = scan_case(2, 9, 6, 4, 2, F32, gate=True, softplus=True, state=True, skip=True, bias=True)
    names = [*ORDER, "state"]
    g = torch.Generator().manual_seed(2)
    dy, dlast = rnd(g, 2, 9, 6), rnd(g, 2, 6, 4)

    def f(v):
        y, last = ssm.selective_scan(**v, **kw, lengths=None, return_state=True)
        return float((d64(y) * d64(dy)).sum() + (d64(last) * d64(dlast)).sum())

    base = {k: i[k].detach().clone() for k in names}
    leaves = {k: v.clone().requires_grad_() for k, v in base.items()}
    y, last = ssm.selective_scan(**leaves, **kw, return_state=True)
    grads = dict(zip(names, torch.autograd.grad((y, last), list(leaves.values()), (dy, dlast))))
    for k in names:
        v, h = rnd(g, *base[k].shape), 2.0 ** -6
        est = (f({**base, k: base[k] + h * v}) - f({**base, k: base[k] - h * v})) / (2 * h)
        want = float((grads[k] * v).sum())
        assert abs(est - want) < 2e-2 + 1e-2 * abs(want), (k, est, want)


@gpu
@pytest.mark.parametrize("dtype,N,G", ((F32, 16, 1), (BF16, 16, 1), (F32, 1, 1), (F16, 6, 2), (F32, 13, 1), (F32, 20, 3), (BF16, 64, 1)))
def test_scan_steps_continue_a_prompt(dtype, N, G):
    T, at, D = 24, 17, 66
    i, kw = scan_case(3, T, D, N, G, dtype, gate=True, softplus=True, state=True, skip=True, bias=True)
    y, h, by, bh = scan_bounds(i, kw, dtype)
    cut = lambda s: {k: (v[:, s] if k in ("u", "delta", "B", "C", "z") else v) for k, v in i.items() if k != "lengths"}  # noqa: E731
    with torch.no_grad():
        first, st = ssm.selective_scan(**cut(slice(0, at)), **kw, return_state=True)
        within(first, y[:, :at], by[:, :at])
        st = st.clone()
        for t in range(at, T):
            before = st._version
            out = ssm.selective_scan_step(**{**cut(t), "state": st}, **kw)
            within(out, y[:, t], by[:, t], t)
            assert st._version > before
    within(st, h, bh, "state")


@gpu
def test_scan_parameters_in_narrow_types():
    i, kw = scan_case(2, 20, 40, 8, 1, BF16, softplus=True, skip=True, bias=True)
    narrow = {k: i[k].to(BF16) for k in ("A", "D", "delta_bias")}
    wide = {k: t.float() for k, t in narrow.items()}
    leaves = {k: t.requires_grad_() for k, t in narrow.items()}
    a, b = ssm.selective_scan(**{**i, **leaves}, **kw), ssm.selective_scan(**{**i, **wide}, **kw)
    assert torch.equal(a.detach(), b)
    for t, g in zip(leaves.values(), torch.autograd.grad(a, list(leaves.values()), torch.ones_like(a))):
        assert g.dtype == BF16 and g.shape == t.shape and torch.isfinite(g).all()


@gpu
@pytest.mark.parametrize("shape", ((0, 5, 6), (2, 0, 6), (2, 5, 0)))
def test_empty_calls(shape):
    B, T, D = shape
    x = torch.zeros(shape, device="cuda").requires_grad_()
    w, st = torch.ones(D, 3, device="cuda").requires_grad_(), torch.ones(B, 2, D, device="cuda").requires_grad_()
    y, last = ssm.causal_conv(x, w, state=st, return_state=True)
    assert y.shape == shape and torch.equal(last, st)
    for t, g in zip((x, w, st), torch.autograd.grad(y.sum() + last.sum(), (x, w, st))):
        assert g.shape == t.shape
    A, h = -torch.ones(D, 4, device="cuda").requires_grad_(), torch.ones(B, D, 4, device="cuda").requires_grad_()
    m = torch.ones(B, T, 4, device="cuda")
    if D == 0:
        return
    y, last = ssm.selective_scan(x, x, A, m, m, state=h, return_state=True)
    assert y.shape == shape and torch.equal(last, h)
    assert torch.autograd.grad(y.sum() + last.sum(), (x, A, h))[2].shape == h.shape


@gpu
def test_orders_and_broadcasts():
    """Channel-first inputs, an expanded trial axis and one shared map give what their contiguous copies give, gradients included."""
    i, kw = scan_case(3, 21, 40, 8, 1, F32, gate=True, softplus=True, skip=True, bias=True)
    g = torch.Generator().manual_seed(8)
    u = rnd(g, 1, 21, 40)
    delta = rnd(g, 3, 40, 21).transpose(1, 2)
    Bm = rnd(g, 1, 21, 1, 8)
    dy = rnd(g, 3, 40, 21).transpose(1, 2)
    outs = []
    for copy in (False, True):
        leaf = [t.detach().clone(memory_format=torch.preserve_format).requires_grad_() for t in (u, delta, Bm)]
        a = [leaf[0].expand(3, -1, -1), leaf[1], leaf[2].expand(3, -1, -1, -1)]
        a = [t.contiguous() for t in a] if copy else a
        y = ssm.selective_scan(**{**i, "u": a[0], "delta": a[1], "B": a[2]}, **kw)
        x = ssm.causal_conv(a[1], i["A"][:, :4].contiguous(), silu=True)
        outs.append((y, x, *torch.autograd.grad((y, x), leaf, (dy, dy.contiguous() if copy else dy))))
    for p, q in zip(*outs):
        assert torch.equal(p, q)


@gpu
def test_many_trials_and_runs_alike():
    """More trials than a grid's second axis holds; the same call twice gives the same bits (no atomics)."""
    B = 70000
    g = torch.Generator().manual_seed(9)
    u, m = rnd(g, B, 2, 3), rnd(g, B, 2, 2)
    A = -torch.rand(3, 2, generator=g).cuda()
    outs = []
    for _ in range(2):
        leaf = [t.clone().requires_grad_() for t in (u, A, m)]
        y = ssm.selective_scan(leaf[0], u.abs() * 0.1, leaf[1], leaf[2], m)
        outs.append((y, *torch.autograd.grad(y, leaf, u)))
    for p, q in zip(*outs):
        assert torch.equal(p, q)
    pick = [0, 1, 65535, 65536, B - 1]
    ref, _ = O.scan(d64(u[pick]), d64(u[pick]).abs() * 0.1, d64(A), d64(m[pick])[:, :, None], d64(m[pick])[:, :, None])
    assert float((d64(outs[0][0][pick]) - ref).abs().max()) < 2.0 ** -24 * 64 * float(ref.abs().max())


@gpu
def test_streams_and_graphs():
    """A forward and backward pass on another stream, and captured and replayed with eager work between the replays."""
    i, kw = scan_case(2, 40, 70, 16, 1, F32, gate=True, softplus=True, state=True, skip=True, bias=True)
    w = i["A"][:, :4].contiguous()
    names = [k for k in (*ORDER, "state") if i[k] is not None]

    def both(v):
        x = ssm.causal_conv(v["u"], w, silu=True)
        y, last = ssm.selective_scan(**{**v, "u": x}, **kw, return_state=True)
        return (y, last, *torch.autograd.grad((y, last), [v[k] for k in names], (i["u"], i["state"])))

    def leaves(scale=1.0):
        return {k: (None if t is None else (t * scale).detach().requires_grad_() if t.is_floating_point() else t) for k, t in i.items()}

    want = both(leaves())
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = both(leaves())
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    static = leaves()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        both(static)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = both(static)
    for scale in (1.0, 0.5, 1.0, 0.25):
        with torch.no_grad():
            for k, t in static.items():
                if t is not None:
                    t.copy_(i[k] * scale)
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(out, both(leaves(scale))):
            assert torch.equal(a, b)


@gpu
def test_captured_steps():
    i, kw = scan_case(3, 2, 70, 16, 1, F32, gate=True, softplus=True, skip=True, bias=True)
    one = {k: (v[:, 0].contiguous() if k in ("u", "delta", "B", "C", "z") else v) for k, v in i.items() if k not in ("lengths", "state")}
    w = i["A"][:, :4].contiguous()
    with torch.no_grad():
        cs, hs = torch.zeros(3, 3, 70, device="cuda"), torch.zeros(3, 70, 16, device="cuda")
        graph = torch.cuda.CUDAGraph()
        ssm.causal_conv_step(one["u"], cs.clone(), w, silu=True)
        with torch.cuda.graph(graph):
            y = ssm.selective_scan_step(**{**one, "u": ssm.causal_conv_step(one["u"], cs, w, silu=True)}, state=hs, **kw)
        ec, eh = torch.zeros_like(cs), torch.zeros_like(hs)
        for _ in range(4):
            graph.replay()
            want = ssm.selective_scan_step(**{**one, "u": ssm.causal_conv_step(one["u"], ec, w, silu=True)}, state=eh, **kw)
            torch.cuda.synchronize()
            assert torch.equal(y, want) and torch.equal(cs, ec) and torch.equal(hs, eh)


@gpu
def test_extremes():
    """Step sizes at the softplus' ends, decays that underflow, and infinities that stay in their own channel."""
    raw = torch.tensor([-100.0, -30.0, -7.0, -1e-3, 0.0, 1e-3, 7.0, 30.0, 1e4], device="cuda")
    D = raw.numel()
    u, one = torch.ones(1, 1, D, device="cuda"), torch.ones(1, 1, 1, device="cuda")
    y = ssm.selective_scan(u, raw.view(1, 1, D), torch.zeros(D, 1, device="cuda"), one, one, softplus=True)
    ref = torch.nn.functional.softplus(d64(raw), threshold=1e9)
    # exponential of a rounded exponent (|x| ulp), reciprocal and series: below 16 + 2 |x| half steps while x > -80 (subnormals flush)
    err = (d64(y)[0, 0] - ref).abs()
    assert (err <= 2.0 ** -24 * (16 + 2 * d64(raw).abs().clamp(max=100)) * ref + 1e-37).all(), err / ref
    A = torch.full((4, 1), -1e30, device="cuda")
    u = torch.tensor([1.0, float("inf"), float("nan"), 2.0], device="cuda").view(1, 1, 4).expand(1, 20, 4)
    y = ssm.selective_scan(u, torch.full_like(u, 0.5), A, one.expand(1, 20, 1), one.expand(1, 20, 1))
    assert torch.equal(y[0, :, 0], torch.full((20,), 0.5, device="cuda")) and torch.equal(y[0, :, 3], torch.ones(20, device="cuda"))
    assert not torch.isfinite(y[0, :, 1:3]).any()


@gpu
def test_far_apart_steps():
    """Time strides at and beyond what the kernels address without a copy."""
    A = -torch.rand(8, 4, device="cuda")
    for stride in ((1 << 22) - 1, 1 << 22):
        base = torch.empty(18 * stride, dtype=BF16, device="cuda")
        u = base.as_strided((1, 18, 8), (18 * stride, stride, 1))
        u.copy_(torch.randn(1, 18, 8, device="cuda"))
        m = u[..., :4]
        flat = u.contiguous()
        outs = []
        for v, k in ((u, m), (flat, m.contiguous())):
            # (a leaf for each use: of one leaf autograd would add the uses' bfloat16 gradients, in an order that a copy's node changes)
            x, dl, z, xc = (t.detach().requires_grad_() for t in (v, v.abs() * 0.3, v, v))
            y = ssm.selective_scan(x, dl, A, k, k, z=z)
            c = ssm.causal_conv(xc, A, silu=True)
            outs.append((y, c, *torch.autograd.grad((y, c), (x, dl, z, xc), (flat, flat))))
        for p, q in zip(*outs):
            assert torch.equal(p, q)


@gpu
def test_offsets_beyond_32_bits():
    """More than 2^31 elements: the last rows are those of the same channels alone."""
    T, D = 70000, 32768
    u = torch.randn(1, T, D, dtype=BF16, device="cuda")
    few = slice(D - 40, D)
    A, m = -torch.rand(D, 1, device="cuda"), torch.randn(1, T, 1, dtype=BF16, device="cuda")
    w = torch.randn(D, 3, dtype=BF16, device="cuda")
    last = torch.tensor([T - 3], device="cuda", dtype=torch.int32)
    with options.override(SELSCAN_CHUNKS=1):
        y, h = ssm.selective_scan(u, u, A, m, m, softplus=True, lengths=last, return_state=True)
        v = u[..., few].contiguous()
        y2, h2 = ssm.selective_scan(v, v, A[few].contiguous(), m, m, softplus=True, lengths=last, return_state=True)
    assert torch.equal(y[..., few], y2) and torch.equal(h[:, few], h2)
    del y
    c, s = ssm.causal_conv(u, w, silu=True, lengths=last, return_state=True)
    c2, s2 = ssm.causal_conv(v, w[few].contiguous(), silu=True, lengths=last, return_state=True)
    assert torch.equal(c[..., few], c2) and torch.equal(s[..., few], s2)


@gpu
def test_inference_mode_and_refused_gradients():
    i, kw = scan_case(2, 3, 8, 4, 1, F32, softplus=True)
    with torch.inference_mode():
        y, h = ssm.selective_scan(**i, **kw, return_state=True)
        one = {k: (v[:, 0] if k in ("u", "delta", "B", "C") else v) for k, v in i.items() if k in ("u", "delta", "A", "B", "C")}
        ssm.selective_scan_step(**one, state=h, **kw)
        x, s = ssm.causal_conv(i["u"], i["A"], return_state=True)
        ssm.causal_conv_step(i["u"][:, 0], s, i["A"])
    assert torch.isfinite(h).all() and torch.isfinite(s).all()
    u = i["u"].detach().requires_grad_()
    g, = torch.autograd.grad(ssm.selective_scan(**{**i, "u": u}, **kw).sum(), u, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(g.sum(), u)              # once differentiable
    st = torch.zeros(2, 8, 4, device="cuda")
    y = ssm.selective_scan(**{**i, "u": u, "state": st}, **kw)
    with torch.no_grad():
        ssm.selective_scan_step(**one, state=st, **kw)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()


@gpu
def test_gradient_sums_of_many_trials_and_wide_rows():
    """Sums over trials where rows are many and so are columns."""
    B, D, N = 257, 262144, 16
    g = torch.Generator(device="cuda").manual_seed(3)
    u = torch.randn(B, 1, D, dtype=BF16, device="cuda", generator=g)
    m = torch.randn(B, 1, N, dtype=BF16, device="cuda", generator=g)
    A, skip = -torch.rand(D, N, device="cuda", generator=g), torch.randn(D, device="cuda", generator=g)
    h = torch.randn(B, D, N, device="cuda", generator=g)
    A.requires_grad_(), skip.requires_grad_()
    delta = u.abs() * 0.25
    dA, dD = torch.autograd.grad(ssm.selective_scan(u, delta, A, m, m, skip, state=h).float().sum(), (A, skip))
    # one step: dA = sum_b C dl exp(dl A) h, dD = sum_b u; relative to the terms' magnitudes each is a few roundings to float
    for few in (slice(0, 500), slice(D - 500, D)):
        dl, C = d64(delta[:, 0, few]), d64(m[:, 0])
        terms = C[:, None, :] * dl[..., None] * torch.exp(dl[..., None] * d64(A[few].detach())) * d64(h[:, few])
        assert float((d64(dA[few]) - terms.sum(0)).abs().max() / terms.abs().sum(0).max()) < 16 * 2.0 ** -24
        x = d64(u[:, 0, few])
        assert float((d64(dD[few]) - x.sum(0)).abs().max() / x.abs().sum(0).max()) < 16 * 2.0 ** -24


def test_a_single_step_has_no_time_stride():
    from lqg_amd import _learn
    x = torch.zeros(4, 8).as_strided((4, 1, 8), (8, 1 << 23, 1))
    assert _learn.seq(ssm._sequence(x, "x", 3))[2] == 0


@gpu
def test_single_steps_far_apart():
    """One step of trials that are laid out time first: its time stride, beyond what a tile addresses, is not used."""
    i, kw = scan_case(3, 1, 8, 4, 1, F32, softplus=True)
    far = {k: (t.as_strided(t.shape, (t.stride(0), 1 << 23, *t.stride()[2:])) if k in ("u", "delta", "B", "C") else t) for k, t in i.items()}
    leaf = lambda v: {k: (t.detach().requires_grad_() if k == "u" else t) for k, t in v.items()}  # noqa: E731
    a, b = leaf(i), leaf(far)
    b["u"] = far["u"].detach().requires_grad_()
    ya, yb = ssm.selective_scan(**a, **kw), ssm.selective_scan(**b, **kw)
    assert torch.equal(ya, yb)
    for p, q in zip(torch.autograd.grad(ya, a["u"], i["u"]), torch.autograd.grad(yb, b["u"], far["u"])):
        assert torch.equal(p, q)
    assert torch.equal(ssm.causal_conv(i["u"], i["A"]), ssm.causal_conv(far["u"], i["A"]))


@gpu
def test_capture_beside_a_living_eager_graph_is_refused():
    i, kw = scan_case(2, 5, 8, 4, 1, F32, softplus=True)
    A = i["A"].detach().requires_grad_()
    calls = {"selective_scan": lambda: ssm.selective_scan(**{**i, "A": A}, **kw), "causal_conv": lambda: ssm.causal_conv(i["u"], A)}
    for name, call in calls.items():
        alive = call()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = call()                               # (a forward pass alone may be captured)
            with pytest.raises(LqgHipError, match=name + ".*drop that call's outputs"):
                torch.autograd.grad(y, A, i["u"])
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, alive)
        want, = torch.autograd.grad(alive, A, i["u"])
        del alive, y
        gc.collect()                                 # (what the error's traceback held)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got, = torch.autograd.grad(call(), A, i["u"])
        for _ in range(3):
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(got, want)


def selscan_spaces(B, T, D, N, chunks=0):
    """Bytes of workspace forward and backward, of a call described by its sizes alone."""
    from lqg_amd import _learn
    p = _learn.SELSCAN.pack(_learn.T_F32, 1, B, T, D, N, 1, *(6 * _learn.NO_SEQ), *(3 * _learn.NO_PARAM), 0, 0, 0, 0, chunks, 0)
    lib = _learn.load()
    return lib.lqg_selscan_workspace(p), lib.lqg_selscan_grad_workspace(p)


def test_the_time_axis_is_cut_where_waves_are_few():
    for B, T, D, N, forward, backward in ((1, 2048, 2048, 16, True, True), (8, 2048, 2048, 16, False, False), (4, 2048, 2048, 16, False, True),
                                          (1, 64, 2048, 16, False, False), (1, 16384, 1024, 4, True, True), (1, 100000, 32, 64, True, True)):
        ws, gws = selscan_spaces(B, T, D, N)
        _, gws1 = selscan_spaces(B, T, D, N, 1)
        assert (ws > 0) is forward and (gws > gws1) is backward, (B, T, D, N)
        # a carry for each state and a sum of step sizes for each channel of a piece, 64 at most
        assert ws % (4 * B * (N + 1) * D) == 0 and ws // (4 * B * (N + 1) * D) in range(0, 65)


LONG = [(1, 2100, 40, 16, 1, F32, True, True, True, True, True, None), (2, 1700, 33, 6, 1, BF16, True, True, True, False, True, (1700, 600)),
        (1, 1500, 64, 3, 2, F32, False, True, False, True, True, (1333,)), (2, 1300, 40, 24, 1, F32, True, True, True, True, True, (200, 1290)),
        (1, 900, 33, 50, 1, F16, True, True, True, True, True, None)]


@gpu
@pytest.mark.parametrize("case", LONG, ids=str)
def test_scan_cut_by_the_rule(case):
    assert min(selscan_spaces(*case[:4])) > 0
    test_scan_forward_and_state(case, 0)
    test_scan_gradients(case, 0)


@gpu
@pytest.mark.parametrize("channels", (16, 32))
@pytest.mark.parametrize("case", SCAN + LONG, ids=str)
def test_scan_workgroups_of_either_width(case, channels):
    """Both widths of a workgroup, uncut and cut, whichever the rule would take."""
    with options.override(SELSCAN_CHANNELS=channels):
        for chunks in (1, 3):
            test_scan_forward_and_state(case, chunks)
        test_scan_gradients(case, 0)


@gpu
@pytest.mark.parametrize("channels", (16, 32))
@pytest.mark.parametrize("case", SCAN + LONG, ids=str)
def test_gradients_of_workgroups_of_either_width(case, channels):
    with options.override(SELSCAN_CHANNELS=channels):
        for chunks in (1, 3):
            test_scan_gradients(case, chunks)


def test_bytes_of_checkpoints():
    from lqg_amd import _learn
    lib = _learn.load()
    for N in range(1, 65):
        for B, T, D in ((1, 1, 1), (3, 16, 5), (2, 17, 7), (5, 1067, 771)):
            p = _learn.SELSCAN.pack(_learn.T_F32, 1, B, T, D, N, 1, *(6 * _learn.NO_SEQ), *(3 * _learn.NO_PARAM), 0, 0, 0, 0, 0, 0)
            assert ssm._checkpoint_bytes(B, T, D, N) == lib.lqg_selscan_checkpoint_bytes(p)


@gpu
@pytest.mark.parametrize("N", (33, 50, 64))
def test_wide_states_with_and_without_checkpoints(N):
    """Beyond 32 states a call that needs no gradient may use other workgroups than one that does: both within the bounds."""
    case = (2, 300, 40, N, 1, F32, True, True, True, True, True, (300, 171))
    i, kw = scan_case(*case[:6], **dict(zip(KEYS, case[6:])))
    y, h, by, bh = scan_bounds(i, kw, F32)
    for channels in (0, 16, 32):
        for chunks in (0, 1, 3):
            with options.override(SELSCAN_CHANNELS=channels, SELSCAN_CHUNKS=chunks):
                for grads in (False, True):
                    got, last = ssm.selective_scan(**{**i, "u": i["u"].detach().requires_grad_(grads)}, **kw, return_state=True)
                    within(got.detach(), y, by, "y")
                    within(last.detach(), h, bh, "state")


@gpu
def test_gradients_beyond_32_bits():
    """More than 2^31 elements: the gradients of the last channels are those of the same channels alone."""
    T, D = 70000, 32768
    u = torch.randn(1, T, D, dtype=BF16, device="cuda")
    few = slice(D - 40, D)
    A, m = -torch.rand(D, 1, device="cuda"), torch.randn(1, T, 1, dtype=BF16, device="cuda")
    w = torch.randn(D, 3, dtype=BF16, device="cuda")
    last = torch.tensor([T - 3], device="cuda", dtype=torch.int32)

    def scan(x, a):
        leaves = [t.detach().requires_grad_() for t in (x, x, a)]
        y = ssm.selective_scan(*leaves, m, m, softplus=True, lengths=last)
        return torch.autograd.grad(y, leaves, x)

    v = u[..., few].contiguous()
    for channels in (16, 32):
        with options.override(SELSCAN_CHUNKS=1, SELSCAN_CHANNELS=channels):
            whole, part = scan(u, A), scan(v, A[few].contiguous())
        assert torch.equal(whole[0][..., few], part[0]) and torch.equal(whole[1][..., few], part[1]) and torch.equal(whole[2][few], part[2])
        del whole
    dx = []
    for x, k in ((u, w), (v, w[few].contiguous())):
        x = x.detach().requires_grad_()
        dx.append(torch.autograd.grad(ssm.causal_conv(x, k, silu=True, lengths=last), x, x.detach())[0])
    assert torch.equal(dx[0][..., few], dx[1])
