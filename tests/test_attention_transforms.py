"""The attention half's operators under torch's transforms: vmap and batched gradients give what a loop gives, functional gradients raise."""

import pytest
import torch

from torchllmtuner_amd import ops

DEV = "cuda:0"
T, H, G, D, N = 37, 4, 2, 64, 3


def operators(device):
    cu, positions = torch.tensor([0, 20, 35], dtype=torch.int32, device=device), torch.arange(T, device=device)
    inv_freq, weight = ops.rotary_frequencies(D)[0].to(device), torch.linspace(0.5, 1.5, D, device=device)
    return {
        "rotary": lambda q, k, v: ops.rotary(q, k, positions, inv_freq),
        "qk_norm_rotary": lambda q, k, v: ops.qk_norm_rotary(q, k, weight, weight, positions, inv_freq, 1e-6),
        "varlen_attention": lambda q, k, v: (ops.varlen_attention(q, k, v, cu),),
    }


@pytest.mark.gpu
@pytest.mark.parametrize("name", ["rotary", "qk_norm_rotary", "varlen_attention"])
def test_vmap_and_batched_gradients_are_loops(name):
    print(f"{name} under vmap", flush=True)
    gen = torch.Generator(device=DEV).manual_seed(1)
    q, k, v = (torch.randn(N, T, n, D, device=DEV, generator=gen) for n in (H, G, G))
    run = operators(DEV)[name]
    for got, want in zip(torch.func.vmap(run)(q, k, v), zip(*(run(q[i], k[i], v[i]) for i in range(N)))):
        assert torch.equal(got, torch.stack(want))
    leaves = [x[0].clone().requires_grad_() for x in (q, k, v)]
    out = run(*leaves)
    grads = [torch.randn(N, *o.shape, device=DEV, generator=gen) for o in out]
    used = leaves if name == "varlen_attention" else leaves[:2]
    got = torch.autograd.grad(out, used, grads, is_grads_batched=True, retain_graph=True)
    want = [torch.autograd.grad(out, used, [g[i] for g in grads], retain_graph=True) for i in range(N)]
    for x, each in zip(got, zip(*want)):
        assert torch.equal(x, torch.stack(each))


@pytest.mark.gpu
@pytest.mark.parametrize("name", ["rotary", "qk_norm_rotary", "varlen_attention"])
def test_functional_gradients_raise(name):
    q, k, v = (torch.ones(T, n, D, device=DEV) for n in (H, G, G))
    with pytest.raises(RuntimeError, match="functorch"):
        torch.func.grad(lambda q: operators(DEV)[name](q, k, v)[0].sum())(q)
