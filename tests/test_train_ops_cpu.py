"""Refusals of the training-step operators (layer norm, gated recurrence, distillation loss):
the C entry points check their arguments before they touch a device, the Python entry points
before they launch.  No GPU needed."""
import ctypes
import importlib

import pytest
import torch

import delta_phase_b200 as dp
from delta_phase_b200 import _capi

P = 1 << 20  # an address that is never read: these calls are refused, or have nothing to do


def _strides(n):
    return (ctypes.c_int64 * n)(*([0] * n))


def test_layernorm_fwd_arguments():
    f = _capi.lib().dp_layernorm_fwd

    def call(x=P, xd=0, res=None, s=None, y=P, yd=0, mean=P, rstd=P, rows=4, d=8):
        return f(x, xd, res, None, None, 1e-5, s, y, yd, mean, rstd, rows, d, None)

    assert call(rows=-1) == 1 and call(d=0) == 1 and call(xd=7) == 1 and call(yd=-1) == 1
    assert call(x=None) == 1 and call(y=None) == 1 and call(mean=None) == 1 and call(rstd=None) == 1
    assert call(res=P) == 1 and call(s=P) == 1  # residual and sum_out come together
    assert call(rows=1 << 31) == 2 and call(d=(1 << 30) + 1) == 2
    assert call(rows=0, x=None) == 0


def test_layernorm_bwd_arguments():
    L = _capi.lib()

    def call(s=P, sd=0, dy=P, dyd=0, dx=P, dxd=0, gw=P, rows=4, d=8, ws=P, nbytes=None):
        n = L.dp_layernorm_bwd_workspace_size(rows, d) if nbytes is None else nbytes
        return L.dp_layernorm_bwd(s, sd, dy, dyd, None, P, P, None, dx, dxd, None, gw, None, rows, d, ws, n, None)

    assert call(rows=-1) == 1 and call(d=0) == 1 and call(sd=3) == 1 and call(dyd=3) == 1 and call(dxd=3) == 1
    assert call(s=None) == 1 and call(dy=None) == 1
    assert call(ws=None) == 6 and call(nbytes=3) == 6 and call(ws=P + 4) == 3
    assert call(rows=1 << 31) == 2 and call(d=(1 << 30) + 1) == 2
    assert L.dp_layernorm_bwd_workspace_size(0, 8) == 0
    for rows, d in ((1, 1), (5, 257), (1 << 20, 8192), (3, 9000)):
        assert L.dp_layernorm_bwd_workspace_size(rows, d) >= 8 * d


def test_scan_arguments():
    L = _capi.lib()
    st = _strides(6)
    assert L.dp_scan_tile() >= 1

    def fwd(x=P, dt=0, mode=0, h0=None, out=P, hL=P, B=1, T=4, D=8):
        return L.dp_scan_fwd(x, P, dt, mode, h0, out, hL, None, B, T, D, st, None)

    assert fwd(B=-1) == 1 and fwd(T=-1) == 1 and fwd(D=0) == 1 and fwd(dt=5) == 1 and fwd(mode=2) == 1
    assert fwd(x=None) == 1 and fwd(out=None) == 1 and fwd(hL=None) == 1 and fwd(h0=P) == 1
    assert fwd(B=0, x=None) == 0
    assert fwd(T=(1 << 30) + 1) == 2

    far = _strides(6)
    far[1] = (1 << 28) + 1  # tokens further apart than the kernels' 32 bits of bytes
    assert L.dp_scan_fwd(P, P, 0, 0, None, P, P, None, 1, 4, 8, far, None) == 2
    assert L.dp_scan_bwd(P, P, P, 0, 0, P, None, P, P, None, 1, 4, 8, far, None) == 2

    def bwd(x=P, dt=0, mode=0, saved=P, dx=P, B=1, T=4, D=8):
        return L.dp_scan_bwd(x, P, P, dt, mode, saved, None, dx, P, None, B, T, D, st, None)

    assert bwd(B=-1) == 1 and bwd(D=0) == 1 and bwd(dt=5) == 1 and bwd(mode=-1) == 1
    assert bwd(x=None) == 1 and bwd(saved=None) == 1 and bwd(dx=None) == 1
    assert bwd(T=(1 << 30) + 1) == 2
    assert bwd(B=0, x=None) == 0 and bwd(T=0, x=None) == 0

    def step(h=P, x=P, dt=0, mode=0, B=1, D=8):
        return L.dp_scan_step(h, P, x, P, dt, mode, P, B, D, _strides(3), None)

    assert step(B=-1) == 1 and step(D=0) == 1 and step(dt=9) == 1 and step(mode=3) == 1
    assert step(h=None) == 1 and step(x=None) == 1 and step(B=0, h=None) == 0


def test_distill_arguments():
    L = _capi.lib()

    def fwd(z=P, zd=0, ib=8, td=0, tau=1.0, loss=P, stats=None, dz=2 * P, B=1, T=2, V=100, K=4):
        return L.dp_distill(z, zd, P, ib, P, td, None, tau, loss, stats, dz, B, T, V, K, _strides(2), None)

    def bwd(z=P, zd=0, ib=8, td=0, tau=1.0, stats=P, dz=2 * P, B=1, T=2, V=100, K=4):
        return L.dp_distill_bwd(z, zd, P, ib, P, td, None, stats, None, tau, dz, B, T, V, K, _strides(2), None)

    for call in (fwd, bwd):
        assert call(B=-1) == 1 and call(T=-1) == 1 and call(V=0) == 1 and call(K=0) == 1
        assert call(zd=4) == 1 and call(td=4) == 1 and call(ib=2) == 1
        for tau in (0.0, -1.0, float("nan"), float("inf")):
            assert call(tau=tau) == 1
        assert call(z=None) == 1 and call(dz=P) == 1 and call(stats=P + 4) == 3
        assert call(K=1025) == 2 and call(V=1 << 18) == 2 and call(zd=1, V=1 << 19) == 2
        assert call(B=1 << 14, T=1 << 14) == 2
        assert call(B=0, z=None) == 0 and call(T=0, z=None) == 0
    assert fwd(loss=None) == 1 and bwd(stats=None) == 1 and bwd(dz=None) == 1


def test_python_refusals():
    z = torch.zeros
    x, g = z(2, 3, 8), z(2, 3, 8)
    with pytest.raises(RuntimeError):
        dp.layer_norm(x)
    with pytest.raises(ValueError):
        dp.layer_norm(z(()))
    with pytest.raises(ValueError):
        dp.layer_norm(x, weight=z(7))
    with pytest.raises(ValueError):
        dp.layer_norm(x, bias=z(8, 1))
    with pytest.raises(TypeError):
        dp.layer_norm(x.double())
    with pytest.raises(TypeError):
        dp.layer_norm(x, out_dtype=torch.float64)
    with pytest.raises(TypeError):
        dp.layer_norm(x, residual=x.bfloat16())
    with pytest.raises(ValueError):
        dp.layer_norm(x, residual=z(3, 8))
    with pytest.raises(RuntimeError):
        dp.gated_scan(x, g)
    with pytest.raises(ValueError):
        dp.gated_scan(x, g, gate_mode="tanh")
    with pytest.raises(ValueError):
        dp.gated_scan(x, g[:1])
    with pytest.raises(ValueError):
        dp.gated_scan(x[0], g[0])
    with pytest.raises(TypeError):
        dp.gated_scan(x, g.bfloat16())
    with pytest.raises(TypeError):
        dp.gated_scan(x.double(), g.double())
    with pytest.raises(ValueError):
        dp.gated_scan(x, g, z(2, 3))
    with pytest.raises(TypeError):
        dp.gated_scan(x, g, z(2, 8).half())
    with pytest.raises(ValueError):
        dp.gated_scan_step(z(2, 8), x, g)
    with pytest.raises(RuntimeError):
        dp.gated_scan_step(z(2, 8), x[:, 0], g[:, 0])
    logits, idx, t = z(2, 3, 50), z(2, 3, 4, dtype=torch.long), z(2, 3, 4)
    with pytest.raises(RuntimeError):
        dp.distill_loss(logits, idx, t)
    with pytest.raises(ValueError):
        dp.distill_loss(logits, idx[:1], t[:1])
    with pytest.raises(ValueError):
        dp.distill_loss(logits, idx, t[..., :3])
    with pytest.raises(TypeError):
        dp.distill_loss(logits, idx.float(), t)
    with pytest.raises(TypeError):
        dp.distill_loss(logits.double(), idx, t)
    with pytest.raises(ValueError):
        dp.distill_loss(logits, idx, t, weight=z(2))
    for tau in (0.0, -1.0, float("nan"), float("inf")):
        with pytest.raises(ValueError):
            dp.distill_loss(logits, idx, t, tau)
    with pytest.raises(TypeError):
        dp.distill_loss(logits, idx, t, torch.tensor(1.0))
    with pytest.raises(RuntimeError):
        dp.distill_loss_and_grad(logits, idx, t)
    model = dp.DeltaPhaseModel(dp.DeltaPhaseConfig(dim=16, emb_dim=8, n_layers=1, n_heads=2, vocab_size=32))
    with torch.no_grad(), pytest.raises(RuntimeError, match="gradients enabled"):
        model.distill_step(torch.zeros(1, 4, dtype=torch.long), idx[:1], t[:1])


def test_sizes_past_the_c_interface_are_refused():
    # the entry points take 32-bit sizes; one value, expanded, stands for the large tensors
    one, n = torch.zeros(1), (1 << 32) + 8
    idx = torch.zeros(1, dtype=torch.int32)
    with pytest.raises(ValueError, match="2\\*\\*30"):
        dp.layer_norm(one.expand(2, n))
    for shape in ((1, n, 1), (n, 1, 1), (1, 1, n)):
        with pytest.raises(ValueError, match="2\\*\\*30"):
            dp.gated_scan(one.expand(shape), one.expand(shape))
    for shape in ((n, 1), (1, n)):
        with pytest.raises(ValueError, match="2\\*\\*30"):
            dp.gated_scan_step(one.expand(shape), one.expand(shape), one.expand(shape))
    for lead, V, K in (((1, n), 1, 1), ((n, 1), 1, 1), ((1, 1), n, 1), ((1, 1), 1, n), ((n,), 1, 1), ((1 << 16, 1, 1 << 16), 1, 1)):
        with pytest.raises(ValueError, match="2\\*\\*30"):
            dp.distill_loss(one.expand(*lead, V), idx.expand(*lead, K), one.expand(*lead, K))


@pytest.mark.parametrize("scale", [0.0, -1.0, float("nan"), float("inf"), torch.ones(2)])
def test_distill_step_refuses_loss_scales(scale):
    model = dp.DeltaPhaseModel(dp.DeltaPhaseConfig(dim=16, emb_dim=8, n_layers=1, n_heads=2, vocab_size=32))
    idx = torch.zeros(1, 4, 2, dtype=torch.long)
    with pytest.raises(ValueError, match="loss_scale"):
        model.distill_step(torch.zeros(1, 4, dtype=torch.long), idx, idx.float(), loss_scale=scale)


def test_step_output_rows_must_not_share_memory():
    z = torch.zeros
    with pytest.raises(ValueError, match="out"):
        dp.gated_scan_step(z(2, 8), z(2, 8), z(2, 8), out=z(1, 8).expand(2, 8))


def test_scan_sequences_reach_the_kernels_within_their_strides():
    seq = importlib.import_module("delta_phase_b200.kernels.gated_scan")._seq
    far = (1 << 28) + 8
    for shape, stride in (((1, 2, 8), (8, far, 1)), ((3, 1, 8), (8, far, 1)), ((1, 1, 8), (far, far, 1)),
                          ((2, 5, 8), (40, 8, 1)), ((2, 5, 8), (8, 16, 1)), ((2, 5, 1), (40, 8, 7)),
                          ((2, 0, 8), (8, far, 1))):
        x = torch.empty_strided(shape, stride, dtype=torch.bfloat16)
        if x.numel():
            x[:] = torch.arange(x.numel(), dtype=torch.bfloat16).view(shape)
        s = seq(x)
        assert s.shape == x.shape and s.stride(1) <= 1 << 28 and torch.equal(s, x)
        assert (s.data_ptr() == x.data_ptr()) == (stride[1] != far or shape[1] != 2)


def test_step_outputs_must_not_overlap_other_tensors():
    """dp_scan_step refuses outputs that overlap another tensor, except element for element, before it
    touches a device; addresses that are never read, 4 rows of 8 values."""
    f = _capi.lib().dp_scan_step
    B, D = 4, 8

    def refused(h=1 << 20, h2=2 << 20, x=3 << 20, gate=4 << 20, out=5 << 20, dt=0, strides=(8, 8, 8), B=B):
        rc = f(h, h2, x, gate, dt, 0, out, B, D, (ctypes.c_int64 * 3)(*strides), None)
        assert rc in (1, 4)  # 4: launched, without a device here
        assert (rc == 1) == (b"overlaps" in _capi.lib().dp_last_error())
        return rc == 1

    P, row = 1 << 20, 32
    if torch.cuda.is_available():
        pytest.skip("calls that are not refused would run")
    assert not refused() and not refused(h2=P) and not refused(out=3 << 20) and not refused(out=4 << 20)
    assert refused(h2=P + 4) and refused(h2=P - row) and refused(h2=P + 3 * row) and not refused(h2=P + 4 * row)
    assert refused(h2=(3 << 20) + row) and refused(out=P + 8) and refused(out=(2 << 20) - 4)
    assert refused(out=P, dt=1)  # 16-bit outputs on a float32 state
    # slices of the rows of one buffer: x | gate | out, 24 values a row, then out one value too far left
    for dt, e in ((0, 4), (1, 2)):
        assert not refused(x=3 << 20, gate=(3 << 20) + 8 * e, out=(3 << 20) + 16 * e, dt=dt, strides=(24, 24, 24))
        assert refused(x=3 << 20, gate=(3 << 20) + 8 * e, out=(3 << 20) + 15 * e, dt=dt, strides=(24, 24, 24))
        assert refused(x=3 << 20, out=(3 << 20) + 17 * e, dt=dt, strides=(24, 8, 24))
    assert refused(x=3 << 20, out=3 << 20, strides=(0, 8, 8)) and refused(x=3 << 20, out=3 << 20, strides=(16, 8, 8))
    assert not refused(x=3 << 20, out=3 << 20, strides=(0, 8, 8), B=1)


def test_distill_more_blocks_than_a_launch_holds():
    """Rows that are few enough, but so wide that the gradient from the sums takes 64 blocks for each."""
    L, P2 = _capi.lib(), 2 * P
    for rows in ((1 << 26) - 1, 1 << 25):
        rc = L.dp_distill_bwd(P, 0, P, 8, P, 0, None, P, None, 1.0, P2, 1, rows, 262136, 4, _strides(2), None)
        assert rc == 2 and b"too many rows" in L.dp_last_error()
