"""GPU numerics of the training-step operators where their values span many orders of magnitude:
masked logits and teacher entries, gates that keep almost all or almost nothing of the state.

Definitions and bounds as in test_train_ops_gpu.py: half a step of the output's type plus the
float32 roundings of the formula."""
import math

import pytest
import torch

import delta_phase_b200 as dp
from test_train_ops_gpu import BF16, F16, F32, distill_case, distill_inputs

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
