"""The scale's range: scores enter the bf16 backward over scale log2(e), which has to stay a number for every row."""

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

from tests.test_attention import BF, DEV, F32, check, inputs, reference, step
from torchllmtuner_amd import _lib, ops


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF, F32])
def test_the_least_scale(dtype):
    print(f"varlen_attention at a scale of 2^-100 {dtype}", flush=True)
    leaves, dout = inputs(300, 4, 2, 64, dtype, seed=5)
    got = step(leaves, dout, torch.tensor([0, 200, 300], dtype=torch.int32, device=DEV), 2.0**-100)
    check(got, *reference(*leaves, dout, [0, 200, 300], 2.0**-100, dtype), dtype)


@pytest.mark.parametrize("scale", [2.0**-101, 1e-38, 1e-45, 1e-300, 2.0**101, 3e38, 1e300])
def test_scales_out_of_range_are_refused(scale):
    with FakeTensorMode():
        q, k = (torch.empty(10, n, 64, dtype=BF, device="cuda") for n in (8, 2))
        cu = torch.empty(3, dtype=torch.int32, device="cuda")
        with pytest.raises(ValueError, match="from 2\\^-100 to 2\\^100"):
            ops.varlen_attention(q, k, k, cu, scale=scale)
        for s in (2.0**-100, 2.0**100):
            assert ops.varlen_attention(q, k, k, cu, scale=s).shape == q.shape
    lib, p = _lib.load(), 0x1000  # (never dereferenced)
    forward = lib.mi355_varlen_attention_fwd(p, 512, 64, p, 128, 64, p, 128, 64, 1, p, 2, min(scale, 3.4e38), p, p, p, p, 10, 8, 2, 64, None)
    assert forward == -1 and b"from 2^-100 to 2^100" in lib.mi355_moe_last_error()
    backward = lib.mi355_varlen_attention_bwd(p, p, 512, 64, p, 128, 64, p, 128, 64, p, p, p, 1, p, 2, min(scale, 3.4e38), p, p, p, p, 10, 8, 2, 64, None)
    assert backward == -1 and b"from 2^-100 to 2^100" in lib.mi355_moe_last_error()
