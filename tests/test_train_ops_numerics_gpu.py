"""GPU numerics of the training-step operators where their values span many orders of magnitude:
masked logits and teacher entries, gates that keep almost all or almost nothing of the state.

Definitions and bounds as in test_train_ops_gpu.py: half a step of the output's type plus the
float32 roundings of the formula."""
import math

import pytest
import torch

import delta_phase_b200 as dp
from delta_phase_b200 import _capi
from delta_phase_b200.kernels import gated_scan, gated_scan_step
from test_train_ops_gpu import BF16, F16, F32, U, check, distill_case, distill_inputs, distill_ref

pytestmark = pytest.mark.gpu

# one warp a row, few rows (a cluster a row), many rows (a block a row)
ROWS = [(4, 700), (4, 9001), (5, 131072), (320, 4003), (320, 32768)]


# ---------------------------------------------------------------- distillation
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("N,V", ROWS)
@pytest.mark.parametrize("K", [64, 100, 700])
def test_distill_teacher_entries_masked_by_the_lowest_value(N, V, K, dtype):
    """All entries of a warp (32 in a row) at the type's lowest value, at either end, and all of a
    row's but one: they have the probability 0."""
    z, index, teacher, weight = distill_inputs(N, V, K, dtype, N + V + K, tdt=dtype)
    low = torch.finfo(dtype).min
    teacher[0, 32:] = low
    teacher[3, :-32] = low
    teacher[-1, 1:] = low
    index[0] = torch.arange(K, device="cuda")
    distill_case(z, index, teacher, 2.0, weight)


@pytest.mark.parametrize("dtype,masks", [(F32, (-1e9, -1e30, "low")), (BF16, (-1e9, "low")), (F16, (-6e4, "low"))])
@pytest.mark.parametrize("N,V", ROWS)
def test_distill_parts_of_the_row_masked_by_large_values(N, V, dtype, masks):
    """A stretch of the vocabulary masked by a large negative number, at its start, its end and in
    steps: the loss keeps the digits of the logits that are left."""
    for mask in masks:
        z, index, teacher, weight = distill_inputs(N, V, 40, dtype, N + V)
        value = torch.finfo(dtype).min if mask == "low" else mask
        half = V // 2
        z[0, :half] = value
        z[-1, half:] = value
        z[3] = torch.where(torch.arange(V, device="cuda") // 256 % 2 == 0, value, z[3])
        index[0] = half + torch.arange(40, device="cuda")
        index[-1] = torch.arange(40, device="cuda")
        index[3] = 256 + torch.arange(40, device="cuda")
        distill_case(z, index, teacher, 2.0, weight)


@pytest.mark.parametrize("N,V", ROWS)
def test_distill_entries_of_no_probability_at_masked_logits(N, V):
    """Entries so far below the teacher's best that their probability is 0 even in 64 bits count
    nothing, in whichever warp they are, also where the student's logit is masked by -inf."""
    z, index, teacher, weight = distill_inputs(N, V, 90, F32, N + V)
    index[3] = torch.arange(90, device="cuda")
    teacher[3, 40:] = -1e4
    z[3, 40:90] = -math.inf
    index[0] = torch.arange(90, device="cuda")
    teacher[0, :50] = -1e5
    z[0, :50] = -math.inf
    distill_case(z, index, teacher, 1.0, weight)


@pytest.mark.parametrize("N,V", ROWS)
def test_distill_likely_entries_at_the_lowest_logit(N, V):
    """Two entries that the teacher finds likely lie at logits masked by the type's lowest value:
    the loss is p 3.4e38, which float32 holds."""
    z, index, teacher, _ = distill_inputs(N, V, 5, F32, N + V)
    index[3] = torch.arange(5, device="cuda")
    z[3, :2] = torch.finfo(F32).min
    teacher[3] = 0.0
    loss, _ = distill_case(z, index, teacher, 1.0, None)
    assert 1e38 < float(loss[3]) < math.inf


@pytest.mark.parametrize("as_tensor", [False, True])
def test_model_distill_step_keeps_float16_gradients_in_range(as_tensor, monkeypatch):
    """The mean over many tokens puts most of float16 logits' gradients below the type's range; with a
    loss scale they reach the parameters, and the loss comes back without it."""
    V, B, L, K, scale = 4000, 4, 512, 8, 2.0 ** 20
    model = dp.DeltaPhaseModel(dp.DeltaPhaseConfig(dim=16, emb_dim=8, n_layers=1, n_heads=2, vocab_size=V)).cuda()
    z, index, teacher, _ = distill_inputs(B * L, V, K, F16, 3)
    leaf = z.view(B, L, V).clone().requires_grad_(True)
    monkeypatch.setattr(model, "forward", lambda ids, states=None: leaf * 1.0)
    args = torch.zeros(B, L, dtype=torch.long, device="cuda"), index.view(B, L, K), teacher.view(B, L, K), 1.5
    plain = model.distill_step(*args)
    tiny = float((leaf.grad == 0).double().mean())
    leaf.grad = None
    s = torch.amp.GradScaler("cuda", init_scale=scale).scale(torch.ones((), device="cuda")) if as_tensor else scale
    loss = model.distill_step(*args, loss_scale=s)
    w = torch.full((B * L,), scale / (B * L), device="cuda")
    rl, el, rd, ed = distill_ref(z, index, teacher, 1.5, w)
    check(leaf.grad.view(B * L, V), rd, ed, "dz")
    lost = (leaf.grad.view(B * L, V) == 0) & (rd.abs() > 2.0 ** -24)
    assert tiny > 0.5 and not bool(lost.any())
    # a sum of 2048 float32 losses: 64 roundings at most in a row, and the two products
    assert abs(float(loss) - float(rl.sum()) / scale) <= (float(el.sum()) + 70 * U * float(rl.abs().sum())) / scale
    assert abs(float(loss) - float(plain)) <= 140 * U * float(rl.abs().sum()) / scale + 2 * float(el.sum()) / scale
    # a weight of fewer bits takes the scale in float32
    mask = torch.ones(B, L, device="cuda", dtype=F16)
    assert math.isfinite(float(model.distill_step(*args, weight=mask / (B * L), loss_scale=s)))


# ---------------------------------------------------------------- gated recurrence, open gates
def constant_gate(gate, mode):
    """a and 1 - a of a gate in float64, and a as float32 holds it: the digits of 1 - a lost."""
    a, d = (1 / (1 + math.exp(-gate)), 1 / (1 + math.exp(gate))) if mode == "sigmoid" else \
        (math.exp(gate), -math.expm1(gate))
    return a, d, float(torch.tensor(a, dtype=F32))


@pytest.mark.parametrize("D", [8, 37])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("gate", [16.0, 16.25, 17.0])
def test_scan_open_gates_hold_the_fixed_point(gate, dtype, D):
    """x = 1 and h0 = 1: the state is 1 for ever."""
    L = 1 << 18
    x = torch.ones(1, L, D, device="cuda", dtype=dtype)
    g = torch.full((1, L, D), gate, device="cuda", dtype=dtype)
    out, fin = gated_scan(x, g, torch.ones(1, D, device="cuda"), gate_mode="sigmoid")
    # two roundings of the state a tile of tokens, and a tile's tokens one after another
    lim = (2 * L / _capi.scan_tile() + 2 * _capi.scan_tile()) * U
    assert float((fin - 1).abs().max()) <= lim
    assert float((out.double() - 1).abs().max()) <= lim + torch.finfo(dtype).eps / 2
    # a rounded to float32 would show: the state would run to (1 - a) / (1 - a32)
    a, d, a32 = constant_gate(gate, "sigmoid")
    assert gate != 16.25 or abs(d / (1 - a32) - 1) * -math.expm1(-L * d) > lim


@pytest.mark.parametrize("D", [8, 37])
@pytest.mark.parametrize("dtype,gate,mode", [(F32, -1.3e-6, "decay"), (BF16, -1.3e-6, "decay"), (F16, -2.0 ** -19, "decay"),
                                             (F32, 14.1, "sigmoid"), (BF16, 14.0, "sigmoid"), (F16, 14.1, "sigmoid")])
def test_scan_open_gates_decay_as_defined(dtype, gate, mode, D):
    """x = 0: h_L = a^L h0, and with dL/dh_L = 1 the gradients a^L of h0 and (1 - a) a^L or a^L h0 of
    every gate, forward and backward through the maps of 2048 tiles."""
    L = 1 << 18
    gates = torch.full((1, L, D), gate, device="cuda", dtype=dtype).requires_grad_(True)
    x = torch.zeros(1, L, D, device="cuda", dtype=dtype).requires_grad_(True)
    h0 = torch.full((1, D), 1.5, device="cuda").requires_grad_(True)
    _, fin = gated_scan(x, gates, h0, gate_mode=mode)
    _, dg, dh = torch.autograd.grad(fin, (x, gates, h0), torch.ones_like(fin))
    a, d, a32 = constant_gate(float(gates[0, 0, 0].detach()), mode)
    rest = math.exp(L * (math.log1p(-d)))
    # relative: two roundings a tile, a tile's tokens one after another, 1 - a within 8 U of itself
    rel = (2 * L / _capi.scan_tile() + 2 * _capi.scan_tile() + 8 * L * d) * U
    check(fin.detach(), torch.full_like(fin, 1.5 * rest, dtype=torch.float64), 1.5 * rest * rel, "h_L")
    check(dh, torch.full_like(dh, rest, dtype=torch.float64), rest * rel, "dh0")
    each = 1.5 * rest * (d if mode == "sigmoid" else 1.0)
    check(dg, torch.full_like(dg, each, dtype=torch.float64), 2 * each * rel, "dgate")
    # with a rounded to float32 the first two would fail (-2^-19 loses next to nothing that way)
    assert gate == -2.0 ** -19 or abs(a32 ** L / rest - 1) > rel


@pytest.mark.parametrize("D", [8, 37])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("gate", [16.0, 16.25, 17.0])
def test_scan_open_gates_hold_the_fixed_point_for_a_million_tokens(gate, dtype, D):
    """What a tile adds to a state at its fixed point is 0 but for the roundings of its own small terms,
    so the state does not collect a rounding a tile."""
    L = 1 << 20
    x = torch.ones(1, L, D, device="cuda", dtype=dtype)
    g = torch.full((1, L, D), gate, device="cuda", dtype=dtype)
    _, fin = gated_scan(x, g, torch.ones(1, D, device="cuda"), gate_mode="sigmoid")
    # n + H of a tile: both 128 d within 128 roundings; the state runs to -H / n at most
    assert float((fin - 1).abs().max()) <= 2 * _capi.scan_tile() * U


# ---------------------------------------------------------------- gated recurrence, closed gates
def a_of(gate, mode):
    g = gate.double()
    return torch.sigmoid(g) if mode == "sigmoid" else torch.exp(g)


@pytest.mark.parametrize("mode", ["decay", "sigmoid"])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("cuts", [(0,), (5,), (127,), (128,), (699,), (20, 25), (100, 300), (3, 130, 690)])
def test_scan_closed_gates_keep_the_digits_of_a(cuts, dtype, mode):
    """Gates of -1 to -40 at some tokens, open ones elsewhere, no input: what is left of the state, and
    the gradients of the gates and of the initial state, to the digits of their own value."""
    L, D = 700, 79
    closed = -torch.linspace(1, 40, D, device="cuda").to(dtype) / len(cuts)
    closed = closed.to(dtype)
    open_ = math.inf if mode == "sigmoid" else 0.0
    gate = torch.full((1, L, D), open_, device="cuda", dtype=dtype)
    for t in cuts:
        gate[:, t] = closed
    x = torch.zeros(1, L, D, device="cuda", dtype=dtype).requires_grad_(True)
    h0 = torch.linspace(0.5, 3.0, D, device="cuda")[None].requires_grad_(True)
    leaf = gate.clone().requires_grad_(True)
    out, fin = gated_scan(x, leaf, h0, gate_mode=mode)
    _, dg, dh = torch.autograd.grad(fin, (x, leaf, h0), torch.ones_like(fin))
    a = a_of(closed, mode)[None]
    # relative: exp within 4 U (8 U and 2 |gate| U from the hardware exponential), the factor cut to
    # 23 bits 2 U, a product and a state 2 U each; the open tokens change nothing
    rel = (24 * len(cuts) + 2 * len(cuts) * closed.double().abs()[None]) * U
    left = h0.detach().double()
    start = 0
    for t in cuts:
        if t > start:
            check(out[:, start:t].detach(), left[:, None].expand(1, t - start, D), (rel * left)[:, None], t)
        left, start = left * a, t
    check(out[:, start:].detach(), left[:, None].expand(1, L - start, D), (rel * left)[:, None], "out")
    check(fin.detach(), left, rel * left, "h_L")
    check(dh, left / h0.detach().double(), rel * left / h0.detach().double(), "dh0")
    for t in cuts:
        want = left * (torch.sigmoid(-closed.double()) if mode == "sigmoid" else 1.0)
        check(dg[:, t], want, 2 * rel * want, "dgate")


@pytest.mark.parametrize("mode", ["decay", "sigmoid"])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_scan_closed_gates_against_a_large_state(dtype, mode):
    """A state far larger than the inputs, then a closed gate: out is a h + u to its own digits."""
    D = 64
    x = torch.linspace(0.25, 1.0, D, device="cuda").to(dtype).expand(1, 300, D)
    for at in (0, 7, 128, 200):
        for g in (-8.0, -20.0, -30.0, -math.inf):
            gate = torch.full((1, 300, D), math.inf if mode == "sigmoid" else 0.0, device="cuda", dtype=dtype)
            gate[:, at] = g
            xs = x.clone()
            xs[:, :at] = 0
            h0 = torch.full((1, D), 1e6, device="cuda")
            out, _ = gated_scan(xs, gate, h0, gate_mode=mode)
            a = float(a_of(torch.tensor(g), mode))
            u = xs[0, at].double() * (float(torch.sigmoid(-torch.tensor(g).double())) if mode == "sigmoid" else 1.0)
            want = a * 1e6 + u
            check(out[0, at], want, (32 + 2 * min(abs(g), 100)) * U * want, (at, g))
            o, h = gated_scan_step(h0, xs[:, at], gate[:, at], gate_mode=mode)
            check(o[0], want, 32 * U * want, (at, g))
            check(h[0], want, 32 * U * want, (at, g))


@pytest.mark.parametrize("D", [64, 33])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("gate", [math.inf, 1000.0, 200.0])
def test_scan_gates_that_let_nothing_in(gate, dtype, D):
    """sigmoid = 1 in float32, and 1 - sigmoid below its range: the state stays, bit for bit, and x has
    no part in it and no gradient."""
    x = torch.linspace(-1e4, 1e4, 300 * D, device="cuda").view(1, 300, D).to(dtype).requires_grad_(True)
    g = torch.full((1, 300, D), gate, device="cuda", dtype=dtype)
    for h0 in (torch.zeros(1, D, device="cuda"), torch.linspace(-3, 3, D, device="cuda")[None]):
        out, fin = gated_scan(x, g, h0, gate_mode="sigmoid")
        assert torch.equal(fin, h0) and torch.equal(out, h0[:, None].expand(1, 300, D).to(dtype))
        dx, = torch.autograd.grad((out, fin), x, (torch.ones_like(out), fin.detach()))
        assert not dx.any()


@pytest.mark.parametrize("mode", ["decay", "sigmoid"])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_scan_gates_on_both_sides_of_a_half(dtype, mode):
    """Gates around the one where the factor changes its form; in decay mode growth, too."""
    D, L = 66, 40
    mid = 0.0 if mode == "sigmoid" else -math.log(2.0)
    gate = (torch.linspace(-0.02, 0.02, D, device="cuda") + mid).to(dtype).expand(1, L, D).clone()
    x = torch.zeros(1, L, D, device="cuda", dtype=dtype)
    h0 = torch.ones(1, D, device="cuda")
    _, fin = gated_scan(x, gate, h0, gate_mode=mode)
    want = a_of(gate[:, 0], mode) ** L
    check(fin, want, want * L * 96 * U)  # 16-bit gates: 1 - a within 64 U
    if mode == "decay":
        for lo, hi, n in ((1e-5, 1e-3, 4000), (0.1, 3.0, 12)):
            gate = torch.linspace(lo, hi, D, device="cuda").to(dtype).expand(1, n, D)
            x = torch.zeros(1, n, D, device="cuda", dtype=dtype)
            _, fin = gated_scan(x, gate, h0)
            want = torch.exp(n * gate[:, 0].double())
            # 2 U a tile or token and 8 U (64 U from the hardware exponential) of each n, or of a
            rel = (4 * n / 16 + 32 + n * 96 * gate[:, 0].double().expm1()) * U
            check(fin, want, want * rel)


def test_scan_step_in_place_is_noticed_by_autograd():
    """A state that a graph has saved and the step then overwrites."""
    x = torch.randn(2, 30, 16, device="cuda", requires_grad=True)
    gate = -torch.rand(2, 30, 16, device="cuda")
    for name in ("state_out", "out"):
        _, h = gated_scan(x, gate)
        loss = h.square().sum()  # saves h
        with torch.no_grad():
            gated_scan_step(h, x[:, 0], gate[:, 0], **{name: h})
        with pytest.raises(RuntimeError, match="modified by an inplace"):
            loss.backward()
    with torch.inference_mode():
        h = torch.zeros(2, 16, device="cuda")
        gated_scan_step(h, x[:, 0], gate[:, 0], state_out=h)


# ---------------------------------------------------------------- gated recurrence, layouts
def test_scan_tokens_far_apart():
    """Tokens further apart than the kernels' 32 bits of bytes, and one token whose stride moves nothing."""
    far = (1 << 28) + 8
    gen = torch.Generator(device="cuda").manual_seed(3)
    for shape, stride in (((1, 2, 8), (8, far, 1)), ((3, 1, 8), (8, far, 1))):
        plain = torch.randn(shape, generator=gen, device="cuda").to(BF16)
        x = torch.empty_strided(shape, stride, dtype=BF16, device="cuda")
        x.copy_(plain)
        gate = -plain.abs()
        ref_leaf, leaf = plain.clone().requires_grad_(True), x.requires_grad_(True)
        ref, rf = gated_scan(ref_leaf, gate)
        out, fin = gated_scan(leaf, gate)
        assert torch.equal(out, ref) and torch.equal(fin, rf)
        dout = torch.empty_strided(shape, stride, dtype=BF16, device="cuda").copy_(plain)
        assert torch.equal(torch.autograd.grad(out, leaf, dout)[0], torch.autograd.grad(ref, ref_leaf, plain)[0])
