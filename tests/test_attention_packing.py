"""Results and gradients of a sequence do not depend on what it is packed with, nor on slots of cu_seqlens that hold nothing: the bits are the same as
long as its rows fall on the same places of their tiles (runs of 128 rows) and nothing is dealt over workgroups."""

import pytest
import torch

from tests.test_attention import BF, DEV, F32, check, inputs, reference, step

gpu = pytest.mark.gpu


@gpu
@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("D", [64, 128, 40, 75, 200])
@pytest.mark.parametrize("rows", [2, 5, 31])
def test_short_sequences_behind_a_long_one(rows, D, dtype):
    """By themselves (an average length below 32) and behind one of 8192 rows (above): the two bf16 pieces in which short sequences hold ds are theirs
    wherever they lie, so the bound on its rounding is h^2 = 2^-16 in both."""
    H, long, T = 16, 8192, 128 // rows * rows
    print(f"varlen_attention {T // rows} sequences of {rows} behind {long} rows, heads of {D} {dtype}", flush=True)
    leaves, dout = inputs(long + T, H, H, D, dtype, seed=rows + D)
    cu = torch.arange(0, T + 1, rows, dtype=torch.int32, device=DEV)
    behind = torch.cat([torch.zeros(1, dtype=torch.int32, device=DEV), cu + long])
    alone = [t.detach()[long:].clone().requires_grad_() for t in leaves]
    want, got = step(alone, dout[long:].clone(), cu), step(leaves, dout, behind)
    for name, x, y in zip(("out", "dq", "dk", "dv"), got, want):
        assert torch.equal(x[long:], y), name
    val, off = reference(*alone, dout[long:], cu.tolist(), D**-0.5, dtype, ds_rounding=2.0**-16 if dtype == BF else None)
    check(want, val, off, dtype)


@gpu
@pytest.mark.parametrize("dtype", [BF, F32])
def test_slots_that_hold_nothing(dtype):
    """A caller who captures a step for up to 256 sequences pads cu_seqlens with its last entry."""
    T, H, D = 4096, 32, 64
    print(f"varlen_attention with empty slots {dtype}", flush=True)
    leaves, dout = inputs(T, H, H, D, dtype, seed=3)
    want = step(leaves, dout, torch.tensor([0, T], dtype=torch.int32, device=DEV))
    got = step(leaves, dout, torch.tensor([0] + [T] * 256, dtype=torch.int32, device=DEV))
    for name, x, y in zip(("out", "dq", "dk", "dv"), got, want):
        assert torch.equal(x, y), name
