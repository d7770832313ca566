"""What is measured of the training-step operators: the layer norm with the residual add and
its backward pass, the gated linear recurrence with its backward pass and its single-token
step, and the distillation loss from a teacher's top logits with its gradient.

``run`` makes either the plain form (elementary torch operations in 32 bits, rounded once at
the end) or, where ``own`` is true, the calls that a user makes of this package.  Sizes come
from this repository's configurations and benchmark: model width 512 and 1024, vocabulary
32768, sequences of 2048 and 32768 tokens, 65536 rows of width 1024; the odd ones are generic.
"""
import math

import torch

own = False

_DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
_BYTES = {"f32": 4, "bf16": 2, "f16": 2}
_EPS = 1e-5


# ------------------------------------------------------------------ cases
def listed():
    return [
        # a fine-tuning step on a handful of tokens at the default model width: latency counts
        {"name": "norm_few_rows", "op": "norm", "rows": 64, "d": 512, "dtype": "f32", "residual": False},
        # norm2 of one block of the default model: 8 sequences of 2048 tokens, bf16 branch
        # added to the float32 residual stream
        {"name": "norm_block", "op": "norm", "rows": 16384, "d": 512, "dtype": "bf16", "residual": True},
        # a ragged batch, a width that is no multiple of a warp's loads
        {"name": "norm_odd", "op": "norm", "rows": 4099, "d": 1001, "dtype": "f16", "residual": False},
        # the largest activations the benchmark runs (65536 rows of width 1024)
        {"name": "norm_large", "op": "norm", "rows": 65536, "d": 1024, "dtype": "bf16", "residual": True},
        # one decode token for each of 16 sequences
        {"name": "scan_step", "op": "step", "B": 16, "D": 1024, "dtype": "bf16", "mode": "sigmoid"},
        # training at the default model's width and sequence length, float32
        {"name": "scan_train", "op": "scan", "B": 8, "L": 2048, "D": 512, "dtype": "f32", "mode": "sigmoid"},
        # a ragged batch of short sequences, odd width
        {"name": "scan_odd", "op": "scan", "B": 3, "L": 1237, "D": 333, "dtype": "f16", "mode": "decay"},
        # training on long sequences: few rows, so the sequence itself has to be split
        {"name": "scan_long", "op": "scan", "B": 2, "L": 32768, "D": 1024, "dtype": "bf16", "mode": "decay"},
        # evaluation of one decode batch against a teacher's 8 best tokens: latency counts
        {"name": "distill_eval", "op": "distill", "N": 16, "V": 32768, "K": 8, "dtype": "bf16", "how": "loss"},
        # one training sequence of the default model, loss and gradient in one call
        {"name": "distill_sequence", "op": "distill", "N": 2048, "V": 32768, "K": 64, "dtype": "bf16", "how": "grad"},
        # odd vocabulary and row count, through autograd
        {"name": "distill_odd", "op": "distill", "N": 509, "V": 50021, "K": 33, "dtype": "f32", "how": "train"},
        # the default model's training batch: 8 sequences of 2048 tokens
        {"name": "distill_batch", "op": "distill", "N": 16384, "V": 32768, "K": 64, "dtype": "bf16", "how": "grad"},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    dtype = rng.choice(["f32", "bf16", "f16"])
    op = rng.choice(["norm", "norm", "scan", "scan", "step", "distill", "distill"])
    if op == "norm":
        d = _log_int(rng, 64, 8192)
        if rng.random() < 0.5:
            d = max(64, d // 64 * 64)
        rows = _log_int(rng, 1, max(1, min(65536, 2 ** 25 // d)))
        return {"op": op, "rows": rows, "d": d, "dtype": dtype, "residual": rng.random() < 0.5}
    if op == "step":
        return {"op": op, "B": _log_int(rng, 1, 512), "D": _log_int(rng, 16, 4096), "dtype": dtype,
                "mode": rng.choice(["sigmoid", "decay"])}
    if op == "scan":
        D = _log_int(rng, 16, 2048)
        if rng.random() < 0.5:
            D = max(16, D // 16 * 16)
        L = _log_int(rng, 1, min(32768, 2 ** 25 // D))
        B = _log_int(rng, 1, max(1, min(64, 2 ** 25 // (D * L))))
        return {"op": op, "B": B, "L": L, "D": D, "dtype": dtype, "mode": rng.choice(["sigmoid", "decay"])}
    V = _log_int(rng, 256, 131072)
    if rng.random() < 0.5:
        V = V // 64 * 64
    N = _log_int(rng, 1, min(16384, 2 ** 27 // V))
    return {"op": op, "N": N, "V": V, "K": _log_int(rng, 1, min(256, V)), "dtype": dtype,
            "how": rng.choice(["loss", "grad", "train"])}


# ------------------------------------------------------------------ inputs
def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed) * 2654435761 % (1 << 62) + 17)
    dt = _DTYPES[case["dtype"]]

    def normal(*shape, dtype=torch.float32, mean=0.0, std=1.0):
        return (torch.randn(*shape, generator=g, device="cuda") * std + mean).to(dtype)

    def uniform(*shape, lo=0.0, hi=1.0):
        return torch.rand(*shape, generator=g, device="cuda") * (hi - lo) + lo

    st = dict(case)
    if case["op"] == "norm":
        rows, d = case["rows"], case["d"]
        st["x"] = normal(rows, d, dtype=dt, mean=0.1).requires_grad_(True)
        st["w"] = normal(d, mean=1.0, std=0.1).requires_grad_(True)
        st["b"] = normal(d, std=0.1).requires_grad_(True)
        st["dy"] = normal(rows, d, dtype=dt)
        if case["residual"]:  # the float32 residual stream and the gradient that reaches it
            st["res"] = normal(rows, d, std=2.0).requires_grad_(True)
            st["ds"] = normal(rows, d)
        return st
    if case["op"] in ("scan", "step"):
        B, D = case["B"], case["D"]
        shape = (B, D) if case["op"] == "step" else (B, case["L"], D)
        x = normal(*shape, dtype=dt)
        # each channel has a time scale of its own, from a few tokens to some hundreds
        offset = uniform(D, lo=-6.0, hi=1.0)
        raw = normal(*shape) + offset
        if case["mode"] == "sigmoid":
            gate = -raw  # forget-gate logits: a = sigmoid(gate)
        else:
            gate = -torch.nn.functional.softplus(raw)  # log a
            if case["op"] == "scan" and case["L"] > 1:  # packed documents: the state is dropped
                cut = torch.rand(B, case["L"], generator=g, device="cuda") < 1.0 / 1024
                gate[cut] = -math.inf
        gate = gate.to(dt)
        state = normal(B, D)
        if case["op"] == "step":
            return st | {"x": x, "gate": gate, "state": state}
        return st | {"x": x.requires_grad_(True), "gate": gate.requires_grad_(True),
                     "state": state.requires_grad_(True), "dout": normal(*shape, dtype=dt), "dfin": normal(B, D)}
    N, V, K = case["N"], case["V"], case["K"]
    z = normal(N, V, dtype=dt, std=2.0)
    index = torch.randint(0, V, (N, K), generator=g, device="cuda")
    teacher = normal(N, K, std=2.0, mean=4.0).sort(-1, descending=True).values
    # some rows have fewer entries than K, a few none at all; padding rows have weight zero
    kept = torch.randint(0, K + 1, (N, 1), generator=g, device="cuda")
    short = torch.rand(N, 1, generator=g, device="cuda") < 0.1
    index = torch.where(short & (torch.arange(K, device="cuda") >= kept), -1, index)
    weight = uniform(N, lo=0.5, hi=1.5) * (torch.rand(N, generator=g, device="cuda") > 0.05)
    if case["how"] == "train":
        z.requires_grad_(True)
    return st | {"z": z, "index": index, "teacher": teacher, "weight": weight, "tau": 2.0,
                 "dloss": uniform(N, lo=0.5, hi=1.5)}


# ------------------------------------------------------------------ plain forms
def _plain_norm(s):
    x, w = s["x"].float(), s["w"]
    if s["residual"]:
        x = x + s["res"]
    mean = x.mean(-1, keepdim=True)
    rstd = torch.rsqrt((x - mean).square().mean(-1, keepdim=True) + _EPS)
    xh = (x - mean) * rstd
    y = xh * w + s["b"]
    dy = s["dy"].float()
    wdy = w * dy
    dx = (wdy - wdy.mean(-1, keepdim=True) - xh * (wdy * xh).mean(-1, keepdim=True)) * rstd
    out = {"y": y.to(s["x"].dtype), "dw": (dy * xh).sum(0), "db": dy.sum(0)}
    if s["residual"]:
        dx = dx + s["ds"]
        out |= {"s": x, "dres": dx}
    return out | {"dx": dx.to(s["x"].dtype)}


def _drop_and_input(s):
    """1 - a_t (kept, not a_t: a close to 1 has lost the digits of 1 - a) and what a_t h_{t-1} is added to."""
    x, gate = s["x"].float(), s["gate"].float()
    if s["mode"] == "sigmoid":
        drop = torch.sigmoid(-gate)
        return drop, drop * x
    return -torch.expm1(gate), x


def _plain_scan(drop, u):
    """h_t = (1 - drop_t) h_{t-1} + u_t along dim 1 from zero, by doubling the span of each partial result."""
    h, d, span = u, drop, 1
    while span < u.shape[1]:
        late = d[:, span:]
        h = torch.cat((h[:, :span], h[:, span:] + (h[:, :-span] - late * h[:, :-span])), 1)
        d = torch.cat((d[:, :span], late + (d[:, :-span] - late * d[:, :-span])), 1)
        span *= 2
    return h


def _plain_recurrence(s):
    x, gate, h0 = s["x"].float(), s["gate"].float(), s["state"]
    drop, u = _drop_and_input(s)
    u = torch.cat((u[:, :1] + (h0 - drop[:, 0] * h0)[:, None], u[:, 1:]), 1)
    h = _plain_scan(drop, u)
    before = torch.cat((h0[:, None], h[:, :-1]), 1)
    # the gradient of h runs the same recurrence backwards: p_t = dout_t + a_{t+1} p_{t+1}
    dout = s["dout"].float()
    dout = torch.cat((dout[:, :-1], dout[:, -1:] + s["dfin"][:, None]), 1)
    next_drop = torch.cat((drop[:, 1:], torch.zeros_like(drop[:, :1])), 1)
    p = _plain_scan(next_drop.flip(1), dout.flip(1)).flip(1)
    if s["mode"] == "sigmoid":
        dx, dgate = p * drop, p * (drop * torch.sigmoid(gate)) * (before - x)
    else:
        dx, dgate = p, p * torch.exp(gate) * before
    dt = s["x"].dtype
    return {"out": h.to(dt), "fin": h[:, -1], "dx": dx.to(dt), "dgate": dgate.to(dt),
            "dstate": p[:, 0] - drop[:, 0] * p[:, 0]}


def _plain_step(s):
    drop, u = _drop_and_input(s)
    h = s["state"] - drop * s["state"] + u
    return {"out": h.to(s["x"].dtype), "state": h}


def _plain_distill(s):
    z, tau, index = s["z"].float() / s["tau"], s["tau"], s["index"]
    on = index >= 0
    safe = index.clamp(min=0)
    t = (s["teacher"] / tau).masked_fill(~on, -math.inf)
    t = t - t.amax(-1, keepdim=True).clamp(min=-1e30)
    e = t.exp()
    total = e.sum(-1, keepdim=True).clamp(min=1e-30)  # a row without entries: p = 0
    p = e / total
    logp = (t - total.log()).masked_fill(~on, 0.0)
    zmax = z.amax(-1, keepdim=True)
    ez = (z - zmax).exp()
    zsum = ez.sum(-1, keepdim=True)
    logq = z.gather(1, safe) - zmax - zsum.log()
    scale = s["weight"] * tau * tau
    out = {"loss": scale * (p * (logp - logq)).sum(-1)}
    if s["how"] == "loss":
        return out
    c = s["weight"] * tau * on.any(-1)
    if s["how"] == "train":
        c = c * s["dloss"]
    dz = (ez / zsum).scatter_add_(1, safe, -p) * c[:, None]
    return out | {"dz": dz.to(s["z"].dtype)}


def run(state):
    s = state
    if own:
        import delta_phase_b200 as dp

        if s["op"] == "norm":
            if s["residual"]:
                y, total = dp.layer_norm(s["x"], s["w"], s["b"], _EPS, residual=s["res"])
                dx, dres, dw, db = torch.autograd.grad((y, total), (s["x"], s["res"], s["w"], s["b"]),
                                                       (s["dy"], s["ds"]))
                return {"y": y, "s": total, "dx": dx, "dres": dres, "dw": dw, "db": db}
            y = dp.layer_norm(s["x"], s["w"], s["b"], _EPS)
            dx, dw, db = torch.autograd.grad(y, (s["x"], s["w"], s["b"]), s["dy"])
            return {"y": y, "dx": dx, "dw": dw, "db": db}
        if s["op"] == "step":
            out, h = dp.gated_scan_step(s["state"], s["x"], s["gate"], gate_mode=s["mode"])
            return {"out": out, "state": h}
        if s["op"] == "scan":
            out, fin = dp.gated_scan(s["x"], s["gate"], s["state"], gate_mode=s["mode"])
            dx, dgate, dstate = torch.autograd.grad((out, fin), (s["x"], s["gate"], s["state"]),
                                                    (s["dout"], s["dfin"]))
            return {"out": out, "fin": fin, "dx": dx, "dgate": dgate, "dstate": dstate}
        args = (s["z"], s["index"], s["teacher"], s["tau"], s["weight"])
        if s["how"] == "grad":
            loss, dz = dp.distill_loss_and_grad(*args)
            return {"loss": loss, "dz": dz}
        loss = dp.distill_loss(*args)
        if s["how"] == "loss":
            return {"loss": loss}
        return {"loss": loss, "dz": torch.autograd.grad(loss, s["z"], s["dloss"])[0]}
    with torch.no_grad():
        if s["op"] == "norm":
            return _plain_norm(s)
        if s["op"] == "step":
            return _plain_step(s)
        if s["op"] == "scan":
            return _plain_recurrence(s)
        return _plain_distill(s)


# ------------------------------------------------------------------ what a pass cannot do without
def work(case):
    e = _BYTES[case["dtype"]]
    if case["op"] == "norm":
        n, d = case["rows"] * case["d"], case["d"]
        # x, dy, y, dx; with a residual also res, ds, s, dres in float32; w, b, dw, db
        return {"bytes": 4 * n * e + (16 * n if case["residual"] else 0) + 16 * d, "flops": 18 * n}
    if case["op"] == "step":
        n = case["B"] * case["D"]
        return {"bytes": 3 * n * e + 8 * n, "flops": 6 * n}
    if case["op"] == "scan":
        n = case["B"] * case["L"] * case["D"]
        # x, gate, dout, out, dx, dgate; the states and their gradients in float32
        return {"bytes": 6 * n * e + 16 * case["B"] * case["D"], "flops": 20 * n}
    n, k = case["N"] * case["V"], case["N"] * case["K"]
    passes = 1 if case["how"] == "loss" else 2
    return {"bytes": passes * n * e + 12 * k + 8 * case["N"], "flops": (3 + 3 * (passes - 1)) * n}


# ------------------------------------------------------------------ the definitions in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        return {"norm": _exact_norm, "step": _exact_step, "scan": _exact_scan, "distill": _exact_distill}[case["op"]](s)


def _exact_norm(s):
    d = s["d"]
    out = {}
    v = s["x"].detach().double()
    if s["residual"]:
        v += s["res"].detach().double()
        out["s"] = v
    w, dy = s["w"].detach().double(), s["dy"].double()
    m = v.sum(1) / d
    c = v - m[:, None]
    sigma = ((c * c).sum(1) / d + _EPS).sqrt()
    n = c / sigma[:, None]
    out["y"] = n * w + s["b"].detach().double()
    out["dw"] = torch.einsum("nd,nd->d", dy, n)
    out["db"] = dy.sum(0)
    # the Jacobian of c / sigma: (I - 1/d - n n^T / d) / sigma
    g = dy * w
    dx = (g - (g.sum(1) / d)[:, None] - n * (torch.einsum("nd,nd->n", g, n) / d)[:, None]) / sigma[:, None]
    if s["residual"]:
        dx += s["ds"].double()
        out["dres"] = dx
    out["dx"] = dx
    return out


def _exact_gate(s):
    gate = s["gate"].detach().double()
    if s["mode"] == "sigmoid":
        keep = 1 / (1 + torch.exp(-gate))
        return keep, 1 / (1 + torch.exp(gate))
    return torch.exp(gate), torch.ones_like(gate)


def _exact_step(s):
    keep, take = _exact_gate(s)
    h = keep * s["state"].double() + take * s["x"].double()
    return {"out": h, "state": h}


def _exact_scan(s):
    keep, take = (t.transpose(0, 1).contiguous() for t in _exact_gate(s))
    x = s["x"].detach().double().transpose(0, 1).contiguous()
    dout = s["dout"].double().transpose(0, 1).contiguous()
    L = x.shape[0]
    h = torch.empty(L + 1, *x.shape[1:], dtype=torch.float64, device=x.device)
    h[0] = s["state"].detach()
    put = take * x
    for t in range(L):
        torch.addcmul(put[t], keep[t], h[t], out=h[t + 1])
    p = torch.empty_like(dout)
    carry = s["dfin"].double()
    for t in range(L - 1, -1, -1):
        torch.add(dout[t], carry, out=p[t])
        carry = p[t] * keep[t]
    dgate = p * keep * h[:-1]
    if s["mode"] == "sigmoid":
        dgate = p * keep * take * (h[:-1] - x)
    out = {"out": h[1:], "dx": p * take, "dgate": dgate}
    return {k: v.transpose(0, 1).contiguous() for k, v in out.items()} | {"fin": h[L].clone(), "dstate": carry}


def _exact_distill(s):
    N, V = s["z"].shape
    tau, index, teacher = s["tau"], s["index"], s["teacher"].double()
    loss = torch.zeros(N, dtype=torch.float64, device="cuda")
    dz = None if s["how"] == "loss" else torch.empty(N, V, dtype=torch.float64, device="cuda")
    for lo in range(0, N, 1024):
        r = slice(lo, lo + 1024)
        logq = torch.log_softmax(s["z"].detach()[r].double() / tau, 1)
        p = torch.zeros_like(logq)
        on = (index[r] >= 0).double()
        some = on.sum(1).clamp(max=1)
        pk = torch.softmax(torch.where(on > 0, teacher[r] / tau, -1e300), 1) * on
        loss[r] = (torch.xlogy(pk, pk) - pk * logq.gather(1, index[r].clamp(min=0))).sum(1)
        if dz is not None:
            p.scatter_add_(1, index[r].clamp(min=0), pk)
            dz[r] = logq.exp() * some[:, None] - p
    w = s["weight"].double()
    loss *= w * tau * tau
    if dz is None:
        return {"loss": loss}
    if s["how"] == "train":
        w = w * s["dloss"].double()
    dz *= (w * tau)[:, None]
    return {"loss": loss, "dz": dz}
