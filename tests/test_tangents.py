"""Forward-mode derivatives: the operators have backward formulas only, so a tangent is refused, with and without requires_grad; a call
below Autograd would lose it without a word.  On fake tensors: the refusal stands in front of any kernel."""

import pytest
import torch
import torch.autograd.forward_ad as fw
from torch._subclasses.fake_tensor import FakeTensorMode

from torchllmtuner_amd import kernel_registry, ops

O = torch.ops.mi355_moe


def t(*shape, dtype=torch.float32):
    return torch.empty(shape, dtype=dtype, device="cuda")


def calls():
    """name -> (the inputs that may carry a tangent, the call)"""
    ints = dict(dtype=torch.int32)
    q, k, w, pos, freq, cu = t(5, 4, 64), t(5, 2, 64), t(64), t(5, **ints), t(32), t(2, **ints)
    x, gate, logits, weights = t(8, 128), t(4, 128), t(8, 4), t(8, 2)
    w1, w2, rows = t(4, 256, 128), t(4, 128, 256), t(16, 128)
    plan = (t(5, **ints), t(4, **ints), t(6, **ints), t(6, **ints), t(1, **ints))
    ros = t(16, **ints)
    return {
        "rotary": ((q, k, freq), lambda q, k, f: kernel_registry.rotary(q, k, pos, f)),
        "qk_norm_rotary_fwd": ((q, k, w, w, freq),
                               lambda q, k, a, b, f: kernel_registry.qk_norm_rotary(q, k, a, b, pos, f, 1e-6)),
        "varlen_attention_fwd": ((q, k, k), lambda q, k, v: kernel_registry.varlen_attention(q, k, v, cu)),
        "rms_norm_fwd": ((x, t(128)), lambda x, w: kernel_registry.rms_norm(x, w, 1e-6)),
        "router_gate_fwd": ((x, gate, t(4)), lambda x, w, b: O.router_gate_fwd(x, w, b)),
        "router_select_fwd": ((logits,), lambda l: O.router_select_fwd(l, None, 2, 1, True, 1.0, 0, 0, 0, True, True)),
        "router_select_cutoff_fwd": ((logits,), lambda l: O.router_select_cutoff_fwd(l, t(4), 2, 0, True, 1.0)),
        "balance_loss_fwd": ((logits,), lambda l: O.balance_loss_fwd(l, t(8, 4, dtype=torch.bool), None)),
        "rows_experts_combine_fwd": ((x, weights, w1, w1, w2), lambda x, s, a, b, c: O.rows_experts_combine_fwd(
            x, s, a, b, c, ros, ros, plan[4], *plan, 2, 16, False)),
        "gather_experts_combine_fwd": ((x, weights, w1, w1, w2), lambda x, s, a, b, c: O.gather_experts_combine_fwd(
            x, s, a, b, c, ros, ros, ros, *plan, 2, 16, False, True)),
        "permute_rows_fwd": ((x,), None), "combine_fwd": ((rows, weights), None), "grouped_linear_fwd": ((rows, w1), None),
        "moe_block": ((x, gate, None, w1, w1, w2), None),
        "grouped_swiglu_fwd": ((rows, w1, w1, w2), None),
    }


def by_schema(name, given):
    """A call of an operator by its schema: the given tensors for its floating arguments in order, something that fits for the rest."""
    args, left = [], list(given)
    for a in getattr(O, name).default._schema.arguments:
        kind = str(a.type)
        if kind == "Tensor" or (kind == "Optional[Tensor]" and name == "moe_block" and a.name == "gate_bias"):
            args.append(left.pop(0) if left else t(8, dtype=torch.int32))
        else:
            args.append({"int": 1, "bool": False, "float": 1.0}.get(kind))
    return getattr(O, name)(*args)


with FakeTensorMode():
    NAMES = list(calls())


@pytest.mark.parametrize("requires_grad", [False, True])
@pytest.mark.parametrize("name", NAMES)
def test_a_tangent_is_refused(name, requires_grad):
    with FakeTensorMode(), fw.dual_level():
        inputs, call = calls()[name]
        call = call or (lambda *given: by_schema(name, given))
        for i, x in enumerate(inputs):
            if x is None:
                continue
            given = [y.clone().requires_grad_() if requires_grad and y is not None and y.ndim > 1 else y for y in inputs]
            given[i] = fw.make_dual(given[i], torch.ones_like(x))
            with pytest.raises(NotImplementedError, match=f"{name} has no forward-mode derivative"):
                call(*given)


def test_functional_jvp_is_refused():
    with FakeTensorMode():
        q, k, cu = t(5, 4, 64), t(5, 2, 64), t(2, dtype=torch.int32)
        with pytest.raises(NotImplementedError, match="no forward-mode derivative"):
            torch.func.jvp(lambda q: ops.varlen_attention(q, k, k, cu), (q,), (torch.ones_like(q),))
        # and nothing is refused where no tangent is
        with fw.dual_level():
            assert ops.varlen_attention(q, k, k, cu).shape == q.shape
