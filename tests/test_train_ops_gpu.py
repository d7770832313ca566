"""GPU parity of the training-step operators (layer norm with its backward pass, the gated
linear recurrence, the distillation loss from top logits) against their definitions in float64.

Tolerances are bounds, not fits: half a step of the output's type relative to the value, plus
the float32 roundings of the formula, each at most 2^-24 of the magnitudes that meet in it
(summed along the recurrence where there is one).
"""
import math

import pytest
import torch

import delta_phase_b200 as dp
from delta_phase_b200 import _capi
from delta_phase_b200.kernels import gated_scan, gated_scan_step, layer_norm

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
U = 2.0 ** -24  # half a step of float32
# smallest half step of float16 (its subnormals); the others' are far below every tolerance here
TINY = {F32: 0.0, BF16: 0.0, F16: 2.0 ** -25}


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def randn(g, *shape, dtype=F32, std=1.0, mean=0.0):
    return (torch.randn(*shape, generator=g, device="cuda") * std + mean).to(dtype)


def check(got, ref, extra, what=""):
    """|got - ref| <= half a step of got's type + extra (a float or a tensor), NaN where ref is."""
    r = ref.double()
    bad_ref = ~torch.isfinite(r)
    assert torch.equal(torch.isnan(got), torch.isnan(r)), what
    err = (got.double() - r).abs()
    lim = r.abs() * (torch.finfo(got.dtype).eps / 2) + extra + TINY[got.dtype]
    over = (err > lim * 1.0000001) & ~bad_ref
    assert not bool(over.any()), (what, float((err / lim.clamp(min=1e-300))[over].max()), int(over.sum()))


# ---------------------------------------------------------------- layer norm
def ln_ref(x, w, b, eps, res=None):
    s = x.double() if res is None else x.double() + res.double()
    m = s.mean(-1, keepdim=True)
    r = 1 / ((s - m).square().mean(-1, keepdim=True) + eps).sqrt()
    n = (s - m) * r
    y = n
    if w is not None:
        y = y * w.double()
    if b is not None:
        y = y + b.double()
    return s, n, r, y


def ln_case(rows, d, dtype, residual, seed, out_dtype=None, mean=0.3, wdt=F32, affine=True):
    g = gen(seed)
    x = randn(g, rows, d, dtype=dtype, mean=mean).requires_grad_(True)
    w = randn(g, d, std=0.2, mean=1.0, dtype=wdt).requires_grad_(True) if affine else None
    b = randn(g, d, std=0.2, dtype=wdt).requires_grad_(True) if affine else None
    res = randn(g, rows, d, std=2.0).requires_grad_(True) if residual else None
    out = layer_norm(x, w, b, 1e-5, residual=res, out_dtype=out_dtype)
    y, s = out if residual else (out, None)
    dy = randn(g, *y.shape, dtype=y.dtype)
    ds = randn(g, *y.shape) if residual else None
    ins = [t for t in (x, w, b, res) if t is not None]
    grads = torch.autograd.grad((y, s) if residual else y, ins, (dy, ds) if residual else dy)
    grads = dict(zip([n for n, t in zip("xwbr", (x, w, b, res)) if t is not None], grads))
    s64, n, r, y64 = ln_ref(x.detach(), None if w is None else w.detach(), None if b is None else b.detach(), 1e-5,
                            None if res is None else res.detach())
    # n: a mean of d values (at most 32 added one after another, then a tree of depth <= 12)
    # off by 44 U of the largest, the centred value and 1/sigma by a few U
    big = s64.abs().amax(-1, keepdim=True)
    en = 48 * U * big * r + 64 * U * n.abs()
    wa = 1.0 if w is None else w.detach().double().abs()
    assert y.dtype == (out_dtype or dtype)
    check(y, y64, en * wa + 4 * U * y64.abs(), "y")
    if residual:
        check(s, s64, 0.0, "s")
    dy64 = dy.double()
    gv = dy64 * (1.0 if w is None else w.detach().double())
    c1, c2 = gv.mean(-1, keepdim=True), (gv * n).mean(-1, keepdim=True)
    dx = r * (gv - c1 - n * c2) + (0 if ds is None else ds.double())
    # the two means carry 44 U of the mean magnitudes, n its own error twice
    mag = gv.abs() + gv.abs().mean(-1, keepdim=True) + n.abs() * (gv * n).abs().mean(-1, keepdim=True)
    ex = r * (64 * U * mag + en * (c2.abs() + gv.abs().mean(-1, keepdim=True) * n.abs().amax(-1, keepdim=True))) + \
        en * r * gv.abs().mean(-1, keepdim=True) + 4 * U * dx.abs()
    check(grads["x"], dx, ex, "dx")
    if residual:
        check(grads["r"], dx, ex, "dres")
    if affine:
        # sums over the rows: each product off by n's error, the sum by (rows per chain + 32 + tree) U
        chain = rows / 256 + 64
        check(grads["w"], (dy64 * n).sum(0), (dy64.abs() * en).sum(0) + chain * U * (dy64 * n).abs().sum(0), "dw")
        check(grads["b"], dy64.sum(0), chain * U * dy64.abs().sum(0), "db")
    return x, y, grads


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("rows,d", [(1, 1), (1, 8), (3, 7), (5, 64), (2, 255), (17, 256), (33, 513), (7, 1000),
                                    (300, 512), (130, 1024), (9, 1029), (4, 2048), (3, 4095), (2, 8192), (2, 8195),
                                    (3, 16384)])
def test_layer_norm_forward_backward(rows, d, dtype, residual):
    ln_case(rows, d, dtype, residual, seed=rows * 31 + d)


@pytest.mark.parametrize("rows,d,dtype", [(5000, 512, BF16), (4099, 1001, F16), (20000, 64, F32), (2500, 2048, BF16),
                                          (700, 8192, F32)])
def test_layer_norm_many_rows(rows, d, dtype):
    """More rows than one pass of the grid: the weight gradients cross blocks."""
    ln_case(rows, d, dtype, True, seed=5)


@pytest.mark.parametrize("dtype,out_dtype", [(F32, BF16), (BF16, F32), (F16, BF16), (F32, F16)])
def test_layer_norm_types(dtype, out_dtype):
    ln_case(37, 320, dtype, False, 3, out_dtype=out_dtype)
    ln_case(37, 320, dtype, True, 4, out_dtype=out_dtype, wdt=BF16)
    ln_case(37, 321, dtype, False, 4, affine=False)


def test_layer_norm_matches_the_inference_kernel():
    """The same rows as dp_layernorm, the operator's form without a backward pass."""
    g = gen(1)
    x, res, w, b = randn(g, 64, 512, dtype=BF16), randn(g, 64, 512), randn(g, 512), randn(g, 512)
    y0, s0 = torch.empty(64, 512, device="cuda", dtype=BF16), torch.empty(64, 512, device="cuda")
    _capi.layernorm(x, w, b, 1e-5, y0, residual=res, sum_out=s0)
    y, s = layer_norm(x, w, b, 1e-5, residual=res)
    assert torch.equal(s, s0)
    _, n, _, y64 = ln_ref(x, w, b, 1e-5, res)
    # each is half a bf16 step and 100 U of n off the value
    assert float(((y.double() - y0.double()).abs() - 2.0 ** -7 * y64.abs() - 400 * U * (n * w).abs()).max()) < 1e-5


def test_layer_norm_layouts():
    g = gen(2)
    base = randn(g, 6, 40, 2 * 96)
    w, b = randn(g, 96), randn(g, 96)
    views = [base[..., :96], base[..., 1:97], base.transpose(0, 1)[..., 96:], base[:, ::3, :96],
             base[0, 0, :96], base[:0, :, :96]]
    flat = randn(g, 6 * 96 + 1)[1:].view(6, 96)  # contiguous, 4 bytes off a 16-byte boundary
    for x in views + [flat, flat.to(BF16)[1:], randn(g, 5, 1, 96).expand(5, 4, 96)]:
        y = layer_norm(x, w, b)
        assert y.shape == x.shape
        if x.numel():
            s, n, r, ref = ln_ref(x, w, b, 1e-5)
            en = 48 * U * s.abs().amax(-1, keepdim=True) * r + 64 * U * n.abs()
            check(y, ref, en * w.double().abs() + 4 * U * ref.abs())
    x = randn(g, 4, 96, 10).transpose(1, 2).requires_grad_(True)
    dy = randn(g, 1, 1, 96).expand(4, 10, 96)
    gx, = torch.autograd.grad(layer_norm(x, w, b), x, dy)
    xc = x.detach().contiguous().requires_grad_(True)
    gc, = torch.autograd.grad(layer_norm(xc, w, b), xc, dy.contiguous())
    assert torch.equal(gx, gc)


def test_layer_norm_no_rows_and_partial_gradients():
    w = torch.ones(24, device="cuda", requires_grad=True)
    b = torch.zeros(24, device="cuda", requires_grad=True)
    x = torch.zeros(0, 24, device="cuda", requires_grad=True)
    y = layer_norm(x, w, b)
    gx, gw, gb = torch.autograd.grad(y, (x, w, b), torch.zeros_like(y))
    assert gx.shape == (0, 24) and not gw.any() and not gb.any()
    g = gen(3)
    x, res = randn(g, 9, 24).requires_grad_(True), randn(g, 9, 24).requires_grad_(True)
    full = torch.autograd.grad(layer_norm(x, w, b, residual=res)[0].square().sum(), (x, res, w, b))
    for i, t in enumerate((x, res, w, b)):
        one, = torch.autograd.grad(layer_norm(x, w, b, residual=res)[0].square().sum(), t)
        assert torch.equal(one, full[i])
    y, s = layer_norm(x, w, b, residual=res)
    ds = randn(g, 9, 24)
    gx, gr, gw = torch.autograd.grad(s, (x, res, w), ds, allow_unused=True)
    assert torch.equal(gx, ds) and torch.equal(gr, ds) and not gw.any()
    layer_norm(x.detach(), w, None).sum().backward()
    assert w.grad is not None


def test_layer_norm_special_values():
    g = gen(4)
    x = randn(g, 6, 200)
    x[0] = 3.0                      # no variance: n = 0
    x[1, 7] = math.nan
    x[2, 7] = math.inf
    x[3] = torch.finfo(F32).tiny    # below eps by far
    y = layer_norm(x)
    assert not y[0].any() and bool(y[1].isnan().all()) and bool(y[2].isnan().all()) and not y[3].any()
    check(y[4:], ln_ref(x[4:], None, None, 1e-5)[3], 1e-5)
    far = randn(g, 40, 512, mean=1000.0)  # a mean far from 0: statistics in two passes
    n = ln_ref(far, None, None, 1e-5)[1]
    check(layer_norm(far), n, 48 * U * 1010 + 64 * U * n.abs())


def test_layer_norm_repeats_bit_for_bit():
    for _ in range(2):
        _, y1, g1 = ln_case(3000, 384, BF16, True, 8)
        _, y2, g2 = ln_case(3000, 384, BF16, True, 8)
        assert torch.equal(y1, y2) and all(torch.equal(g1[k], g2[k]) for k in g1)


# ---------------------------------------------------------------- gated recurrence
def scan_ref(x, gate, h0, mode, dout=None, dfin=None, du=16 * U):
    """Definition in float64, token by token, with a bound on the float32 error beside every value."""
    x, gate = x.double(), gate.double()
    B, L, D = x.shape
    a = torch.sigmoid(gate) if mode == "sigmoid" else torch.exp(gate)
    d = torch.sigmoid(-gate) if mode == "sigmoid" else -torch.expm1(gate)
    u = d * x if mode == "sigmoid" else x
    h = torch.zeros(B, D, dtype=torch.float64, device=x.device) if h0 is None else h0.double()
    e = torch.zeros_like(h)
    hs, es, before, ebefore = [], [], [], []
    for t in range(L):
        before.append(h)
        ebefore.append(e)
        e = a[:, t] * e + du * (h.abs() + u[:, t].abs())
        h = a[:, t] * h + u[:, t]
        hs.append(h)
        es.append(e)
    stack = lambda v: torch.stack(v, 1) if v else torch.zeros_like(x)  # noqa: E731
    out = {"out": (stack(hs), stack(es)), "fin": (h, e)}
    if dout is None:
        return out
    q = torch.zeros_like(h) if dfin is None else dfin.double()
    eq = torch.zeros_like(q)
    px, ex, pg, eg = [], [], [], []
    for t in range(L - 1, -1, -1):
        p = dout[:, t].double() + q
        ep = eq + du * (dout[:, t].double().abs() + q.abs())
        q, eq = a[:, t] * p, a[:, t] * ep + du * p.abs()
        if mode == "sigmoid":
            diff, k = before[t] - x[:, t], d[:, t]
            ediff = ebefore[t] + du * (before[t].abs() + x[:, t].abs())
        else:
            diff, k, ediff = before[t], 1.0, ebefore[t]
        px.append(p * k)
        ex.append(ep * k + du * (p * k).abs())
        pg.append(q * k * diff)
        eg.append(k * (eq * diff.abs() + q.abs() * ediff) + 2 * du * (q * k * diff).abs())
    out["dx"] = (stack(px[::-1]), stack(ex[::-1]))
    out["dgate"] = (stack(pg[::-1]), stack(eg[::-1]))
    out["dh0"] = (q, eq)
    return out


def scan_inputs(B, L, D, dtype, mode, seed, resets=True):
    g = gen(seed)
    x = randn(g, B, L, D, dtype=dtype)
    raw = randn(g, B, L, D) + torch.rand(D, generator=g, device="cuda") * 8 - 6
    gate = -raw if mode == "sigmoid" else -torch.nn.functional.softplus(raw)
    if resets and L > 2:
        gate[:, L // 2] = -math.inf
        gate[:1, 0] = -math.inf
    return x, gate.to(dtype), randn(g, B, D), randn(g, B, L, D, dtype=dtype), randn(g, B, D)


# 16-bit gates: 1 - exp(gate) is within 2^-18 = 64 U of its value (the hardware exponential's
# 2^-22 of 1, where 1 - a is at least 1/16)
DU = {F32: 16 * U, BF16: 80 * U, F16: 80 * U}


def scan_case(x, gate, h0, dout, dfin, mode):
    leaves = [t.detach().requires_grad_(True) for t in (x, gate)]
    h = None if h0 is None else h0.detach().requires_grad_(True)
    out, fin = gated_scan(*leaves, h, gate_mode=mode)
    assert out.dtype == x.dtype and fin.dtype == F32 and out.shape == x.shape
    ins = leaves + ([] if h is None else [h])
    grads = torch.autograd.grad((out, fin), ins, (dout, dfin))
    with torch.no_grad():
        out2, fin2 = gated_scan(x, gate, h0, gate_mode=mode)
    assert torch.equal(out, out2) and torch.equal(fin, fin2)
    ref = scan_ref(x, gate, h0, mode, dout, dfin, DU[x.dtype])
    got = {"out": out, "fin": fin, "dx": grads[0], "dgate": grads[1]}
    if h is not None:
        got["dh0"] = grads[2]
    for k, v in got.items():
        check(v.detach(), ref[k][0], ref[k][1], (k, mode, tuple(x.shape)))
    return got


@pytest.mark.parametrize("mode", ["decay", "sigmoid"])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("B,L,D", [(1, 1, 1), (2, 1, 64), (1, 2, 3), (3, 15, 32), (2, 16, 33), (1, 17, 64),
                                   (2, 127, 66), (1, 128, 130), (2, 129, 31), (1, 257, 64), (1, 600, 96),
                                   (2, 2047, 40), (1, 2048, 64), (1, 2049, 34), (1, 4500, 65)])
def test_scan_forward_backward(B, L, D, dtype, mode):
    x, gate, h0, dout, dfin = scan_inputs(B, L, D, dtype, mode, B + L + D)
    scan_case(x, gate, h0, dout, dfin, mode)


@pytest.mark.parametrize("mode", ["decay", "sigmoid"])
def test_scan_many_channels(mode):
    """More chains than the GPU holds at once, no initial state."""
    x, gate, _, dout, dfin = scan_inputs(48, 200, 512, BF16, mode, 1)
    scan_case(x, gate, None, dout, dfin, mode)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_scan_long_memory(dtype):
    """Constant gates that keep 1 - 2^-13 of the state: the digits of 1 - a decide."""
    g = gen(9)
    x = randn(g, 1, 9000, 32, dtype=dtype, mean=1.0)
    gate = torch.full((1, 9000, 32), -2.0 ** -13, device="cuda", dtype=dtype)
    scan_case(x, gate, None, randn(g, 1, 9000, 32, dtype=dtype), randn(g, 1, 32), "decay")


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_scan_dropped_state_leaves_nothing(dtype):
    """After a gate of -inf the outputs are bit for bit those of a sequence that starts there,
    at every place of the cut against the tiles, however large the dropped state was."""
    g = gen(10)
    L = 700
    for cut in (1, 5, 16, 100, 128, 300, 512, 699):
        x = randn(g, 1, L, 64, dtype=dtype)
        gate = -torch.rand(1, L, 64, generator=g, device="cuda").to(dtype)
        gate[:, cut] = -math.inf
        big = torch.full((1, 64), 1e30, device="cuda")
        out, fin = gated_scan(x, gate, big)
        ref = scan_ref(x[:, cut:], gate[:, cut:], None, "decay", du=DU[dtype])
        check(out[:, cut:], *ref["out"], what=cut)
        check(fin, *ref["fin"], what=cut)


def test_scan_layouts():
    """Slices of one projection, transposed and broadcast inputs, odd storage offsets."""
    g = gen(11)
    for dtype in (F32, BF16):
        proj = randn(g, 3, 50, 2 * 48 + 1, dtype=dtype)
        a, b = proj[..., :48], proj[..., 48:96]
        for x, gate in ((a, b), (b, proj[..., 1:49]), (proj[..., :47], proj[..., 49:96]),
                        (a.transpose(0, 1), b.transpose(0, 1)), (a[:, ::2], b[:, 1::2]),
                        (a[:1].expand(3, 50, 48), b), (randn(g, 3, 48, 50, dtype=dtype).transpose(1, 2), b)):
            h0 = randn(g, x.shape[2], x.shape[0]).t()
            dout = randn(g, *x.shape, dtype=dtype)
            scan_case(x, gate, h0, dout, randn(g, x.shape[0], x.shape[2]), "sigmoid")
    x = randn(g, 2, 30, 16).requires_grad_(True)
    out, fin = gated_scan(x, torch.zeros(2, 30, 16, device="cuda"))
    dx, = torch.autograd.grad(out.sum(), x)  # an expanded gradient, without one for the state
    assert torch.equal(dx, torch.arange(30, 0, -1, device="cuda", dtype=F32)[None, :, None].expand_as(dx))


def test_scan_empty_and_initial_state_kept():
    h0 = torch.randn(2, 8, device="cuda")
    keep = h0.clone()
    x = torch.zeros(2, 0, 8, device="cuda")
    out, fin = gated_scan(x, x, h0)
    assert out.shape == (2, 0, 8) and torch.equal(fin, h0) and fin.data_ptr() != h0.data_ptr()
    assert not gated_scan(x, x)[1].any()
    h = h0.clone().requires_grad_(True)
    _, fin = gated_scan(x, x, h)
    dh, = torch.autograd.grad(fin, h, keep)
    assert torch.equal(dh, keep)
    assert gated_scan(x[:0], x[:0])[0].shape == (0, 0, 8)
    gated_scan(torch.ones(2, 5, 8, device="cuda"), torch.zeros(2, 5, 8, device="cuda"), h0)
    assert torch.equal(h0, keep)


@pytest.mark.parametrize("mode", ["decay", "sigmoid"])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_scan_steps_continue_a_sequence(dtype, mode):
    """A prefix by gated_scan, then tokens by gated_scan_step in place: the sequence's outputs."""
    x, gate, h0, _, _ = scan_inputs(3, 40, 37, dtype, mode, 12)
    ref = scan_ref(x, gate, h0, mode, du=DU[dtype])
    _, h = gated_scan(x[:, :30], gate[:, :30], h0, gate_mode=mode)
    for t in range(30, 40):
        out, h2 = gated_scan_step(h, x[:, t], gate[:, t], gate_mode=mode, state_out=h)
        assert h2 is h
        check(out, ref["out"][0][:, t], ref["out"][1][:, t])
    check(h, *ref["fin"])
    keep = h.clone()
    o = torch.empty(3, 64, device="cuda", dtype=dtype)[:, :37]
    out, h3 = gated_scan_step(h, x[:, 0], gate[:, 0], gate_mode=mode, out=o)
    assert out is o and torch.equal(h, keep) and h3.data_ptr() != h.data_ptr()


def test_scan_special_values():
    """An infinity or a NaN stays in its channel and from its token on (an infinite state is documented
    to become NaN: h - d h, where the definition has a h)."""
    g = gen(13)
    x, gate = randn(g, 1, 300, 64), -torch.rand(1, 300, 64, generator=g, device="cuda") - 0.1
    clean, _ = gated_scan(x, gate)
    x[0, 140, 3] = math.nan
    x[0, 200, 5] = math.inf
    gate[0, 10, 7] = math.nan
    out, _ = gated_scan(x, gate)
    assert bool(out[0, 140:, 3].isnan().all()) and not bool(torch.isfinite(out[0, 200:, 5]).any())
    assert bool(out[0, 10:, 7].isnan().all())
    ok = torch.ones_like(clean, dtype=torch.bool)
    ok[0, 140:, 3] = ok[0, 200:, 5] = ok[0, 10:, 7] = False
    assert torch.equal(out[ok], clean[ok])


def test_scan_gradients_against_differences():
    g = gen(14)
    for mode in ("decay", "sigmoid"):
        x, gate, h0, dout, dfin = scan_inputs(1, 150, 4, F32, mode, 14, resets=False)
        leaves = [t.requires_grad_(True) for t in (x, gate, h0)]
        out, fin = gated_scan(*leaves, gate_mode=mode)
        grads = torch.autograd.grad((out, fin), leaves, (dout, dfin))

        def f(*v):
            r = scan_ref(*v, mode)
            return float((r["out"][0] * dout.double()).sum() + (r["fin"][0] * dfin.double()).sum())

        base = [t.detach().double() for t in leaves]
        for i, gr in enumerate(grads):
            v = torch.randn(base[i].shape, generator=g, device="cuda", dtype=torch.float64)
            e = 1e-5
            diff = (f(*[b + e * v if j == i else b for j, b in enumerate(base)]) -
                    f(*[b - e * v if j == i else b for j, b in enumerate(base)])) / (2 * e)
            dot = (gr.double() * v).abs().sum()
            # a difference in 64 bits is good to e^2 and 1e-16 / e of the terms; the gradient to 1e-5
            assert abs(float((gr.double() * v).sum()) - diff) < 1e-5 * float(dot) + 1e-6


# ---------------------------------------------------------------- distillation
def distill_ref(z, index, teacher, tau, weight, grad=None):
    V = z.shape[-1]
    z, teacher = z.double(), teacher.double()
    ok = (index >= 0) & (index < V) & (teacher != -math.inf)
    some = ok.any(-1)
    t = torch.where(ok, teacher / tau, -math.inf)
    t = torch.where(some[..., None], t, 0.0)
    p = torch.softmax(t, -1) * ok
    logp = torch.log_softmax(t, -1)
    logq = torch.log_softmax(z / tau, -1)
    lq = logq.gather(-1, index.long().clamp(0, V - 1))
    terms = torch.where(p > 0, p * (logp - lq), 0.0)
    w = torch.ones(z.shape[:-1], dtype=torch.float64, device=z.device) if weight is None else weight.double()
    on = some & (w != 0)
    loss = torch.where(on, w * tau * tau * terms.sum(-1), 0.0)
    # float32 errors: exponentials within 2 + 1.2 |x| steps, sums of at most 64 + 16 in a row
    x = z / tau - (z / tau).amax(-1, keepdim=True)
    q = logq.exp()
    e_exp = 2 * U * (3 + 1.2 * x.abs().clamp(max=200))
    e_lse = (q * e_exp).sum(-1) + 96 * U
    mag = torch.where(p > 0, p * (logp.abs() + lq.abs() + 4), 0.0).sum(-1)
    xk = (t - t.amax(-1, keepdim=True)).abs().clamp(max=200)
    e_p = p * (2 * U * (3 + 1.2 * xk) + 96 * U)
    e_ent = (e_p * (logp - lq).abs().nan_to_num(0, 0, 0)).sum(-1)
    e_loss = torch.where(on, w.abs() * tau * tau * (e_lse + 16 * U * mag + e_ent), 0.0)
    c = w * tau * (1.0 if grad is None else grad.double())
    pd = torch.zeros_like(z).scatter_add_(-1, index.long().clamp(0, V - 1), p)
    epd = torch.zeros_like(z).scatter_add_(-1, index.long().clamp(0, V - 1), e_p)
    on2 = (on & (c != 0))[..., None]
    dz = torch.where(on2, c[..., None] * (q - pd), 0.0)
    # an exponential below 2^-126, the smallest normal float32, counts as 0: with the sum of all
    # at least 1 (the maximum's own) q and p are then off by less than 2^-126 each
    e_dz = torch.where(on2, c.abs()[..., None] * (q * (e_exp + e_lse[..., None] + 8 * U) + epd + 8 * U * pd +
                                                  2 * 2.0 ** -126), 0.0)
    return loss, e_loss, dz, e_dz


def distill_inputs(N, V, K, dtype, seed, tdt=F32, idt=torch.int64):
    g = gen(seed)
    z = randn(g, N, V, dtype=dtype, std=3.0)
    index = torch.randint(0, V, (N, K), generator=g, device="cuda", dtype=idt)
    teacher = randn(g, N, K, std=2.0, mean=3.0, dtype=tdt)
    weight = torch.rand(N, generator=g, device="cuda") + 0.5
    if N > 2:
        weight[1] = 0.0
        index[2] = -1
        index[0, K // 2:] = torch.where(torch.arange(K // 2, K, device="cuda") % 2 == 0, V, -1).to(idt)
    return z, index, teacher, weight


def distill_case(z, index, teacher, tau, weight):
    loss, dz = dp.distill_loss_and_grad(z, index, teacher, tau, weight)
    rl, el, rd, ed = distill_ref(z, index, teacher, tau, weight)
    assert loss.dtype == F32 and dz.dtype == z.dtype and dz.is_contiguous()
    check(loss, rl, el, "loss")
    check(dz, rd, ed, "dz")
    g = torch.rand(loss.shape, generator=gen(1), device="cuda")
    leaf = z.detach().requires_grad_(True)
    loss2 = dp.distill_loss(leaf, index, teacher, tau, weight)
    check(loss2, rl, el, "loss alone")
    with torch.no_grad():
        assert torch.equal(dp.distill_loss(z, index, teacher, tau, weight), loss2)
    dz2, = torch.autograd.grad(loss2, leaf, g)
    _, _, rd, ed = distill_ref(z, index, teacher, tau, weight, g)
    check(dz2, rd, ed, "dz autograd")
    return loss, dz


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("N,V,K", [(1, 1, 1), (3, 2, 1), (4, 7, 3), (5, 64, 8), (3, 255, 255), (6, 1000, 16),
                                   (4, 4099, 33), (3, 8191, 64), (700, 257, 5), (2, 32768, 64), (400, 9001, 20),
                                   (3, 40007, 100), (5, 131072, 7), (3, 100003, 1024)])
def test_distill_loss_and_gradient(N, V, K, dtype):
    z, index, teacher, weight = distill_inputs(N, V, K, dtype, N + V + K)
    distill_case(z, index, teacher, 2.0, weight)


@pytest.mark.parametrize("dtype,V", [(F32, 262136), (BF16, 524272)])
def test_distill_widest_rows(dtype, V):
    z, index, teacher, weight = distill_inputs(3, V, 16, dtype, 2)
    distill_case(z, index, teacher, 1.0, weight)


@pytest.mark.parametrize("tau", [0.25, 1.0, 7.5])
def test_distill_types_and_temperatures(tau):
    for tdt in (F32, BF16, F16):
        for idt in (torch.int32, torch.int64):
            z, index, teacher, _ = distill_inputs(6, 301, 9, BF16, 3, tdt, idt)
            distill_case(z, index, teacher, tau, None)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("tau", [2.0 ** -9, 2.0 ** -20, 2.0 ** -24, 2.0 ** -28, 2.0 ** -31, 2.0 ** -60, 2.0 ** -90, 2.0 ** 40])
def test_distill_extreme_temperatures(tau, dtype):
    # powers of two, so that the kernel's float32 temperature is the definition's; the quotients
    # logit / tau reach from 2^-40 to past the float32 range
    for V in (7, 301, 9001, 131072):
        z, index, teacher, weight = distill_inputs(4, V, 5, dtype, V)
        distill_case(z, index, teacher, tau, weight)


def test_distill_repeated_indices():
    z, index, teacher, weight = distill_inputs(8, 500, 12, F32, 4)
    index[3] = 17
    index[4, ::3] = 499
    index[5, 1] = index[5, 0]
    distill_case(z, index, teacher, 1.5, weight)


def test_distill_masked_values():
    """Student logits masked by -inf or the type's lowest value, teacher entries by -inf; NaN in
    rows and entries that do not count; a row that its teacher leaves empty."""
    for dtype in (F32, BF16, F16):
        z, index, teacher, weight = distill_inputs(8, 700, 6, dtype, 5)
        low = torch.finfo(dtype).min
        z[3, 100:] = -math.inf
        index[3] = torch.arange(6, device="cuda")
        z[4, 100:] = low
        index[4] = torch.arange(10, 16, device="cuda")
        z[5] = low                      # all of them: the uniform distribution
        teacher[6, 2:] = -math.inf
        teacher[7] = torch.finfo(F32).min
        z[1] = math.nan                 # weight 0
        z[2] = math.nan                 # no entries
        teacher[0, 3:] = math.nan       # index out of range
        teacher[3, 0] = -math.inf
        distill_case(z, index, teacher.clone(), 2.0, weight)
        t2 = teacher.clone()
        t2[4] = -math.inf
        loss, dz = distill_case(z, index, t2, 2.0, weight)
        for r in (1, 2, 4):
            assert float(loss[r]) == 0.0 and not dz[r].any()
        z[3, 5] = math.nan              # one that counts
        loss, dz = dp.distill_loss_and_grad(z, index, teacher, 2.0, weight)
        assert bool(loss[3].isnan()) and bool(dz[3].isnan().all()) and not bool(loss[[0, 4, 5, 6, 7]].isnan().any())


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("N,V,K", [(300, 1101, 70), (310, 3001, 300), (297, 8192, 1), (300, 40007, 3), (500, 2081, 1024)])
def test_distill_many_rows(N, V, K, dtype):
    z, index, teacher, weight = distill_inputs(N, V, K, dtype, 31)
    distill_case(z, index, teacher, 1.5, weight)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("V", [700, 4003, 20000])
def test_distill_masked_values_in_many_rows(V, dtype):
    """The masks of the test above where the loss alone and the backward pass have their own
    kernels; values that rise or fall along the row, so that the running maximum moves always or
    never; a NaN and an infinity that count."""
    z, index, teacher, weight = distill_inputs(320, V, 6, dtype, 32)
    low = torch.finfo(dtype).min
    z[3, 100:] = -math.inf
    index[3] = torch.arange(6, device="cuda")
    z[4, 100:] = low
    z[5] = low
    z[6, :-1] = -math.inf
    index[6] = V - 1
    z[7] = torch.linspace(-20, 20, V, device="cuda").to(dtype)
    z[8] = torch.linspace(20, -20, V, device="cuda").to(dtype)
    teacher[9, 2:] = -math.inf
    teacher[10] = torch.finfo(F32).min
    z[1] = math.nan                 # weight 0
    z[2] = math.nan                 # no entries
    index[3:5, 5] = index[3:5, 0]
    index[4] = index[4] % 100
    distill_case(z, index, teacher, 2.0, weight)
    z[11, V // 2] = math.nan
    z[12, V // 3] = math.inf
    z[13] = -math.inf
    z[14, 0] = math.nan             # with V on an odd grid a single element before the vectors
    leaf = z.requires_grad_(True)
    loss = dp.distill_loss(leaf, index, teacher, 2.0, weight)
    dz, = torch.autograd.grad(loss.sum(), leaf)
    bad = torch.zeros(320, dtype=torch.bool, device="cuda")
    bad[11:15] = True
    assert torch.equal(loss.isnan(), bad) and torch.equal(dz.isnan().any(-1), bad)
    assert bool(dz[11].isnan().all()) and bool(dz[13].isnan().all()) and bool(dz[14].isnan().all())


def test_distill_entry_with_no_student_probability():
    """p > 0 where q = 0: the loss is infinite, as defined, the gradient finite."""
    z, index, teacher, weight = distill_inputs(3, 300, 4, F32, 6)
    index[0] = torch.tensor([5, 6, 7, 8], device="cuda")
    z[0, 5] = -math.inf
    loss, dz = dp.distill_loss_and_grad(z, index, teacher, 1.0, weight)
    assert float(loss[0]) == math.inf and bool(dz.isfinite().all())
    _, _, rd, ed = distill_ref(z, index, teacher, 1.0, weight)
    check(dz, rd, ed)


def test_distill_zero_upstream_gradient_hides_the_row():
    z, index, teacher, _ = distill_inputs(4, 200, 4, BF16, 7)
    index[2] = 3
    z[3] = math.nan
    leaf = z.requires_grad_(True)
    loss = dp.distill_loss(leaf, index, teacher)
    g = torch.tensor([1.0, 2.0, 0.5, 0.0], device="cuda")
    dz, = torch.autograd.grad(loss, leaf, g)
    assert not dz[3].any() and bool(dz[:3].isfinite().all())


def test_distill_layouts():
    """The shifted logits of a language model, transposed rows, odd storage offsets and row
    strides, four leading dimensions, one row."""
    g = gen(8)
    for dtype in (F32, BF16):
        for V in (96, 101):
            z = randn(g, 3, 9, V, dtype=dtype, std=2.0)
            off = randn(g, 3 * 8 * V + 3, dtype=dtype)[3:].view(3, 8, V)
            wide = randn(g, 3, 8, V + 5, dtype=dtype)
            perm = randn(g, 3, V, 8, dtype=dtype).transpose(1, 2)
            for x in (z[:, :-1], z[:, 1:], off, wide[..., 2:V + 2], perm, z.transpose(0, 1)[:8], z[0, 0],
                      z[:2, :4].reshape(2, 2, 2, V), z[:, ::4], z[:1, :1].expand(3, 4, V), z[:0], z[:, :0]):
                index = torch.randint(0, V, (*x.shape[:-1], 5), generator=g, device="cuda")
                teacher = randn(g, *x.shape[:-1], 5)
                w = torch.rand(x.shape[:-1], generator=g, device="cuda")
                loss, dz = distill_case(x, index, teacher, 2.0, w)
                assert loss.shape == x.shape[:-1] and dz.shape == x.shape


def test_distill_constants_are_refused_as_leaves():
    z, index, teacher, weight = distill_inputs(3, 50, 4, F32, 9)
    with pytest.raises(ValueError, match="constants"):
        dp.distill_loss(z.requires_grad_(True), index, teacher.requires_grad_(True))


def test_distill_gradient_against_differences():
    z, index, teacher, weight = distill_inputs(4, 60, 5, F32, 10)
    _, dz = dp.distill_loss_and_grad(z, index, teacher, 1.5, weight)
    g = gen(11)
    v = torch.randn(z.shape, generator=g, device="cuda", dtype=torch.float64)
    e = 1e-5
    f = lambda x: float(distill_ref(x, index, teacher, 1.5, weight)[0].sum())  # noqa: E731
    diff = (f(z.double() + e * v) - f(z.double() - e * v)) / (2 * e)
    assert abs(float((dz.double() * v).sum()) - diff) < 1e-5 * float((dz.double() * v).abs().sum()) + 1e-6


# ---------------------------------------------------------------- together, streams, graphs
def test_student_step_of_all_operators():
    """norm -> gates -> recurrence -> norm with residual -> head -> distillation, against the
    same chain of definitions in float64 under autograd."""
    B, L, d, V, K = 2, 70, 48, 203, 6
    g = gen(20)
    p32 = {n: randn(g, *s, std=sd).requires_grad_(True) for n, s, sd in
           (("x", (B, L, d), 1.0), ("w1", (d,), 1.0), ("b1", (d,), 0.1), ("wx", (d, d), 0.2), ("wg", (d, d), 0.2),
            ("w2", (d,), 1.0), ("b2", (d,), 0.1), ("head", (V, d), 0.2), ("h0", (B, d), 1.0))}
    index = torch.randint(0, V, (B, L, K), generator=g, device="cuda")
    teacher = randn(g, B, L, K, std=2.0)
    weight = (torch.rand(B, L, generator=g, device="cuda") > 0.2).float() / (B * L)

    def chain(p, norm, norm_res, scan, loss):
        n = norm(p["x"], p["w1"], p["b1"])
        h, _ = scan(n @ p["wx"], n @ p["wg"], p["h0"])
        y, s = norm_res(h, p["w2"], p["b2"], p["x"])
        return loss((y + s) @ p["head"].t()).sum()

    torch.backends.cuda.matmul.allow_tf32 = False
    got = chain(p32, layer_norm, lambda h, w, b, r: layer_norm(h, w, b, residual=r),
                lambda x, gt, h0: gated_scan(x, gt, h0, gate_mode="sigmoid"),
                lambda z: dp.distill_loss(z, index, teacher, 2.0, weight))
    grads = torch.autograd.grad(got, list(p32.values()))
    p64 = {n: t.detach().double().requires_grad_(True) for n, t in p32.items()}

    def scan64(x, gate, h0):
        a, h, hs = torch.sigmoid(gate), h0, []
        for t in range(L):
            h = a[:, t] * h + (1 - a[:, t]) * x[:, t]
            hs.append(h)
        return torch.stack(hs, 1), h

    def loss64(z):
        pk = torch.softmax(teacher.double() / 2.0, -1)
        lq = torch.log_softmax(z / 2.0, -1).gather(-1, index)
        return weight.double() * 4.0 * (pk * (pk.log() - lq)).sum(-1)

    ref = chain(p64, lambda x, w, b: ln_ref(x, w, b, 1e-5)[3], lambda h, w, b, r: ln_ref(h, w, b, 1e-5, r)[3::-3],
                scan64, loss64)
    refg = torch.autograd.grad(ref, list(p64.values()))
    # float32 products of width 48 and 203 and recurrences of 70 tokens: 1e-5 is 170 U
    assert abs(float(got.detach()) - float(ref.detach())) < 1e-5 * abs(float(ref.detach()))
    for n, a, b in zip(p32, grads, refg):
        assert float((a.double() - b).norm() / b.norm()) < 1e-5, n


def test_model_distill_step():
    """DeltaPhaseModel.distill_step: the loss and parameter gradients of distill_loss through
    the same model, on top of gradients that are there; padding tokens count nothing."""
    torch.manual_seed(0)
    cfg = dp.DeltaPhaseConfig(dim=32, emb_dim=16, n_layers=2, n_heads=2, vocab_size=97, chunk_size=8, num_banks=2)
    model = dp.DeltaPhaseModel(cfg).cuda()
    ids = torch.randint(0, 97, (2, 24), device="cuda")
    index = torch.randint(0, 97, (2, 24, 4), device="cuda")
    teacher = torch.randn(2, 24, 4, device="cuda")
    names, params = zip(*[(n, p) for n, p in model.named_parameters() if p.requires_grad])
    for weight in (None, (torch.rand(2, 24, device="cuda") > 0.3).float()):
        w = torch.full((2, 24), 1 / 48, device="cuda") if weight is None else weight
        ref = dp.distill_loss(model(ids), index, teacher, 2.0, w).sum()
        want = torch.autograd.grad(ref, params, allow_unused=True)
        for p in params:
            p.grad = None
        loss = model.distill_step(ids, index, teacher, 2.0, weight)
        assert not loss.requires_grad and abs(float(loss) - float(ref.detach())) <= 1e-6 * abs(float(ref.detach()))
        once = [None if p.grad is None else p.grad.clone() for p in params]
        model.distill_step(ids, index, teacher, 2.0, weight)
        for n, p, a, b in zip(names, params, once, want):
            assert (a is None) == (b is None), n
            if a is None:
                continue
            # the logits repeat bit for bit, and so do the head's products and norm_f below the
            # tied embedding; further down the blocks' backward adds in no fixed order, there
            # one token of the 48 left out or counted twice (2e-2) has to show
            tol = 1e-6 if n.startswith(("norm_f", "head_proj")) else 5e-3
            assert float((a - b).norm()) <= tol * float(b.norm()) + 1e-9, n
            assert float((p.grad - 2 * a).norm()) <= tol * float(a.norm()) + 1e-9, n


def test_model_distill_step_gradient_is_the_kernels(monkeypatch):
    """What distill_step sends backwards from the logits is the kernel's gradient, bit for bit,
    and it accumulates."""
    model = dp.DeltaPhaseModel(dp.DeltaPhaseConfig(dim=16, emb_dim=8, n_layers=1, n_heads=2, vocab_size=300)).cuda()
    z, index, teacher, weight = distill_inputs(12, 300, 5, BF16, 21)
    leaf = z.view(2, 6, 300).clone().requires_grad_(True)
    monkeypatch.setattr(model, "forward", lambda ids, states=None: leaf * 1.0)
    args = torch.zeros(2, 6, dtype=torch.long, device="cuda"), index.view(2, 6, 5), teacher.view(2, 6, 5), 1.5
    loss, dz = dp.distill_loss_and_grad(z, index, teacher, 1.5, weight)
    got = model.distill_step(*args, weight=weight.view(2, 6))
    assert torch.equal(got, loss.sum()) and torch.equal(leaf.grad, dz.view(2, 6, 300))
    model.distill_step(*args, weight=weight.view(2, 6))
    assert torch.equal(leaf.grad, 2 * dz.view(2, 6, 300))


def _pass(x, gate, res, w, b, z, index, teacher, h):
    """One pass through every kernel, on plain tensors."""
    y, s = layer_norm(x, w, b, residual=res)
    out, fin = gated_scan(x, gate, h, gate_mode="sigmoid")
    o1, h1 = gated_scan_step(fin, x[:, 0], gate[:, 0])
    loss, dz = dp.distill_loss_and_grad(z, index, teacher, 2.0)
    return [y, s, out, fin, o1, h1, loss, dz]


def _pass_inputs(seed):
    g = gen(seed)
    z, index, teacher, _ = distill_inputs(40, 300, 8, BF16, seed)
    return [randn(g, 4, 300, 64, dtype=BF16), randn(g, 4, 300, 64, dtype=BF16), randn(g, 4, 300, 64), randn(g, 64),
            randn(g, 64), z, index, teacher, randn(g, 4, 64)]


def test_captured_forward_replays_with_new_inputs():
    ins = _pass_inputs(30)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side), torch.no_grad():
        _pass(*ins)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.no_grad(), torch.cuda.graph(graph):
        outs = _pass(*ins)
    for seed in (31, 32):
        new = _pass_inputs(seed)
        for a, b in zip(ins, new):
            a.copy_(b)
        graph.replay()
        with torch.no_grad():
            want = _pass(*new)
        assert all(torch.equal(a, b) for a, b in zip(outs, want))


def test_captured_training_step_replays():
    """Forward and backward captured together, with leaves that no eager graph refers to; two
    graphs captured one after the other are replayed in turn."""
    def make(seed):
        g = gen(seed)
        x = randn(g, 300, 64, dtype=BF16).requires_grad_(True)
        w = randn(g, 64).requires_grad_(True)
        xs = randn(g, 2, 200, 32).requires_grad_(True)
        gs = randn(g, 2, 200, 32).requires_grad_(True)
        z, index, teacher, weight = distill_inputs(30, 120, 4, F32, seed)
        return [x, w, xs, gs, z.requires_grad_(True), index, teacher, weight]

    def step(x, w, xs, gs, z, index, teacher, weight):
        y = layer_norm(x, w)
        out, fin = gated_scan(xs, gs, gate_mode="sigmoid")
        loss = dp.distill_loss(z, index, teacher, 2.0, weight)
        return torch.autograd.grad((y, out, fin, loss), (x, w, xs, gs, z),
                                   tuple(torch.ones_like(t) for t in (y, out, fin, loss)))

    graphs = []
    for seed in (40, 41):
        ins = make(seed)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            for _ in range(2):
                step(*make(seed + 10))
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            grads = step(*ins)
        graphs.append((graph, ins, grads))
    for _ in range(2):
        for k, (graph, ins, grads) in enumerate(graphs):
            graph.replay()
        torch.cuda.synchronize()
        for k, (graph, ins, grads) in enumerate(graphs):
            want = step(*make(40 + k))
            assert all(torch.equal(a, b) for a, b in zip(grads, want)), k


def test_two_streams_at_once():
    """Independent passes on two streams share nothing."""
    a, b = _pass_inputs(50), _pass_inputs(51)
    with torch.no_grad():
        want = _pass(*a), _pass(*b)
        torch.cuda.synchronize()
        s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
        for _ in range(3):
            with torch.cuda.stream(s1):
                ga = _pass(*a)
            with torch.cuda.stream(s2):
                gb = _pass(*b)
        torch.cuda.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(ga, want[0]))
    assert all(torch.equal(x, y) for x, y in zip(gb, want[1]))


def test_without_autograd_and_in_inference_mode():
    """The same results without a graph; nothing requires grad."""
    ins = _pass_inputs(70)
    with torch.no_grad():
        want = _pass(*ins)
    with torch.inference_mode():
        got = _pass(*ins)
    assert all(torch.equal(a, b) and not b.requires_grad for a, b in zip(want, got))


def test_second_derivatives_are_refused():
    x = torch.randn(4, 6, 8, device="cuda", requires_grad=True)
    idx, t = torch.zeros(4, 6, 2, dtype=torch.long, device="cuda"), torch.zeros(4, 6, 2, device="cuda")
    for f in (lambda: layer_norm(x), lambda: gated_scan(x, torch.zeros_like(x))[0], lambda: dp.distill_loss(x, idx, t)):
        g, = torch.autograd.grad(f().square().sum(), x, create_graph=True)
        with pytest.raises(RuntimeError, match="once_differentiable"):
            g.sum().backward()


def test_other_stream_than_the_default():
    """Forward and backward on a side stream, with work of the default stream still pending."""
    ins = _pass_inputs(71)
    leaf = ins[0].clone().requires_grad_(True)
    ref, = torch.autograd.grad(gated_scan(leaf, ins[1], gate_mode="sigmoid")[0].float().square().sum(), leaf)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    big = torch.randn(4096, 4096, device="cuda")
    for _ in range(5):
        big = big @ big * 1e-3
    with torch.cuda.stream(side):
        got, = torch.autograd.grad(gated_scan(leaf, ins[1], gate_mode="sigmoid")[0].float().square().sum(), leaf)
    torch.cuda.synchronize()
    assert torch.equal(got, ref)


def test_saved_inputs_changed_in_place_are_noticed():
    x = torch.randn(4, 5, 8, device="cuda", requires_grad=True)
    y = x * 1.0
    out, _ = gated_scan(y, torch.zeros_like(y))
    y.mul_(2.0)
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        out.sum().backward()


# ---------------------------------------------------------------- sizes past 32 bits
def test_layer_norm_offsets_past_32_bits():
    rows, d = (1 << 31) // 1024 + 5000, 1024
    x = torch.empty(rows, d, device="cuda", dtype=BF16).normal_(generator=gen(60)).requires_grad_(True)
    w = torch.ones(d, device="cuda", requires_grad=True)
    y = layer_norm(x, w)
    dx, dw = torch.autograd.grad(y, (x, w), y.detach())
    tail = x.detach()[-300:].clone().requires_grad_(True)
    yt = layer_norm(tail, w)
    dxt, = torch.autograd.grad(yt, tail, yt.detach())
    assert torch.equal(y[-300:], yt) and torch.equal(dx[-300:], dxt)
    # dw = sum of y^2 over the rows where w = 1: d on average over the columns
    assert abs(float(dw.mean()) / rows - 1) < 1e-2


def test_scan_offsets_past_32_bits():
    """2.2e9 elements: the end of the sequence from the state before it, forward and backward."""
    B, L, D, cut = 1, (1 << 31) // 4096 + 20000, 4096, 4096
    x = torch.empty(B, L, D, device="cuda", dtype=BF16).normal_(generator=gen(61))
    gate = torch.full((1, 1, D), -0.05, device="cuda", dtype=BF16).expand(B, L, D)
    leaf = x.requires_grad_(True)
    out, fin = gated_scan(leaf, gate)
    dx, = torch.autograd.grad((out, fin), leaf, (leaf.detach(), fin.detach()))
    with torch.no_grad():
        _, before = gated_scan(x[:, :-cut], gate[:, :-cut])
    tail = x.detach()[:, -cut:].clone().requires_grad_(True)
    out_t, fin_t = gated_scan(tail, gate[:, -cut:], before)
    dx_t, = torch.autograd.grad((out_t, fin_t), tail, (tail.detach(), fin_t.detach()))
    # both round nearly the same values: each by half a bf16 step, 2^-8 of the value, together 2^-7
    # (the larger of the two, hence the second term); the recurrences add 80 U x 20 tokens x 30 = 3e-3
    for a, b in ((out[:, -cut:], out_t), (dx[:, -cut:], dx_t)):
        err = (a.float() - b.float()).abs()
        assert bool((err <= 2.0 ** -7 * b.float().abs() + 4e-3).all())
    assert float((fin.detach() - fin_t.detach()).abs().max()) < 4e-3


def test_distill_offsets_past_32_bits():
    N, V, K = (1 << 31) // 32768 + 700, 32768, 8
    z = torch.empty(N, V, device="cuda", dtype=BF16).normal_(generator=gen(62))
    index = torch.randint(0, V, (N, K), generator=gen(63), device="cuda")
    teacher = torch.randn(N, K, generator=gen(64), device="cuda")
    loss, dz = dp.distill_loss_and_grad(z, index, teacher)
    rl, el, rd, ed = distill_ref(z[-64:], index[-64:], teacher[-64:], 1.0, None)
    check(loss[-64:], rl, el, "loss")
    check(dz[-64:], rd, ed, "dz")
