"""Rotary positions of queries and keys, alone and behind the norm of every head, against the formulas in fp64.

Tolerances, all for arithmetic in fp32 (unit u = 2^-24, half a step of fp32) with one rounding to the storage type:

* turned pair (a, b): cosine and sine are good to 2 units each in the last place (4 u) times the factor's rounding (u), their
  angle to pi u (half a turn at most, rounded once, in turns), the products and the sum to 3 u more: below 16 u of
  f hypot(a, b) in all.
* norm: a sum of squares is at most 16 additions in a lane and 6 across lanes, halved by the root, then a division, a root and
  two products: below 24 u of the value.
* dx = r (gw - xh mean(gw xh)): the same 40 u on gw, 24 u of additions on the mean, 64 u of both terms' sizes.
* dw: additions in one order or another of tokens x heads terms: u of the sum of their sizes a term, and 64 u as above.
* rounding to bf16: 2^-8 of the value.
"""

import math

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

from torchllmtuner_amd import _lib, kernel_registry, ops

DEV = "cuda:0"
U = 2.0**-24
BF, F32 = torch.bfloat16, torch.float32
HALF_STEP = {BF: 2.0**-8, F32: 2.0**-24}
gpu = pytest.mark.gpu


# ---- the formulas in fp64 ------------------------------------------------------------------------


def turn(x, angle, factor, interleaved):
    """x (T, heads, D) fp64, angle (T, pairs) fp64."""
    n = angle.shape[1]
    c, s = (factor * angle.cos())[:, None], (factor * angle.sin())[:, None]
    y = x.clone()
    one, two = (slice(0, 2 * n, 2), slice(1, 2 * n, 2)) if interleaved else (slice(0, n), slice(n, 2 * n))
    y[..., one] = x[..., one] * c - x[..., two] * s
    y[..., two] = x[..., two] * c + x[..., one] * s
    return y


def pair_size(x, n, factor, interleaved):
    """For every element the size of the pair that it is turned with, times the factor; of itself behind the pairs."""
    y = x.abs()
    one, two = (slice(0, 2 * n, 2), slice(1, 2 * n, 2)) if interleaved else (slice(0, n), slice(n, 2 * n))
    y[..., one] = y[..., two] = factor * torch.hypot(x[..., one], x[..., two])
    return y


def angles(positions, inv_freq):
    return positions.cpu().double().reshape(-1, 1) * inv_freq.cpu().double()


def normed(x, w, eps):
    r = 1.0 / torch.sqrt(x.pow(2).mean(-1, keepdim=True) + eps)
    return x * r * w, r


def close(got, want, slack, dtype, what):
    got, want = got.detach().cpu().double(), want.double()
    over = (got - want).abs() - slack - HALF_STEP[dtype] * (want.abs() + slack) - 1e-38
    assert not got.isnan().any() and over.max() <= 0, f"{what}: {over.max():.3g} beyond the bound"


def inputs(T, H, G, D, dtype, seed, fused=False, weights=False):
    gen = torch.Generator().manual_seed(seed)
    rows = torch.randn(T, H + 2 * G, D, generator=gen).to(dtype)
    grads = [torch.randn(T, n, D, generator=gen).to(dtype) for n in (H, G)]
    w = [(1 + 0.2 * torch.randn(D, generator=gen)).to(dtype) for _ in range(2)]
    if fused:
        dev = rows.to(DEV)
        q, k = dev[:, :H], dev[:, H:H + G]
    else:
        q, k = rows[:, :H].contiguous().to(DEV), rows[:, H:H + G].contiguous().to(DEV)
    return q, k, (w if weights else None), grads


# (tokens, heads, key heads, head size, turned elements)
SHAPES = [
    (1, 1, 1, 2, 2),
    (1, 32, 4, 128, 128),
    (3, 32, 4, 128, 64),
    (37, 5, 5, 80, 40),
    (130, 12, 3, 96, 48),
    (257, 3, 1, 64, 64),
    (19, 2, 2, 33, 32),
    (11, 2, 1, 75, 50),
    (9, 7, 2, 100, 100),
    (5, 3, 3, 36, 20),
    (4, 2, 1, 512, 512),
    (6, 1, 1, 511, 2),
    (5, 2, 2, 510, 510),
    (4500, 9, 2, 32, 32),
]


@gpu
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("T,H,G,D,R", SHAPES)
def test_rotary_matches_the_formula_in_both_directions(T, H, G, D, R, dtype, interleaved):
    print(f"rotary {T}x{H}+{G}x{D} turned {R} {dtype} interleaved={interleaved}", flush=True)
    fused = T % 2 == 1
    q, k, _, grads = inputs(T, H, G, D, dtype, seed=T + D, fused=fused)
    inv_freq, factor = ops.rotary_frequencies(R, 10000.0, device=DEV)[0], 1.25
    positions = (torch.arange(T, dtype=torch.int64 if H % 2 else torch.int32) + 1000).to(DEV)
    q.requires_grad_(), k.requires_grad_()
    out = kernel_registry.rotary(q, k, positions, inv_freq, interleaved=interleaved, attention_factor=factor)
    got = torch.autograd.grad(out, (q, k), [g.to(DEV) for g in grads])
    a = angles(positions, inv_freq)
    for x, y, g, dx in zip((q, k), out, grads, got):
        assert y.shape == x.shape and y.is_contiguous() and y.dtype == dtype
        x64, g64 = x.detach().cpu().double(), g.double()
        close(y, turn(x64, a, factor, interleaved), 16 * U * pair_size(x64, R // 2, factor, interleaved), dtype, "result")
        close(dx, turn(g64, -a, factor, interleaved), 16 * U * pair_size(g64, R // 2, factor, interleaved), dtype, "gradient")
        if R < D:  # elements behind the pairs are copied
            assert torch.equal(y[..., R:], x[..., R:]) and torch.equal(dx[..., R:].cpu(), g[..., R:])


@gpu
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("T,H,G,D,R", SHAPES)
def test_qk_norm_rotary_matches_the_formula_in_both_directions(T, H, G, D, R, dtype, interleaved):
    print(f"qk_norm_rotary {T}x{H}+{G}x{D} turned {R} {dtype} interleaved={interleaved}", flush=True)
    eps, factor = 1e-5, 0.75
    q, k, w, grads = inputs(T, H, G, D, dtype, seed=3 * T + D, fused=T % 2 == 0, weights=True)
    inv_freq = ops.rotary_frequencies(R, 500000.0, device=DEV)[0]
    positions = (torch.arange(T) * 7).to(DEV)
    leaves = [q.requires_grad_(), k.requires_grad_(), *(t.to(DEV).requires_grad_() for t in w)]
    out = kernel_registry.qk_norm_rotary(*leaves, positions, inv_freq, eps, interleaved=interleaved, attention_factor=factor)
    got = torch.autograd.grad(out, leaves, [g.to(DEV) for g in grads])
    a = angles(positions, inv_freq)
    for i in range(2):
        x, wi, g = leaves[i].detach().cpu().double(), w[i].double(), grads[i].double()
        n, r = normed(x, wi, eps)
        size = pair_size(n, R // 2, factor, interleaved)
        close(out[i], turn(n, a, factor, interleaved), 40 * U * size, dtype, "result")
        back = turn(g, -a, factor, interleaved)
        gw, xh = back * wi, x * r
        mean = (gw * xh).mean(-1, keepdim=True)
        turned = pair_size(g, R // 2, factor, interleaved)
        slack = 64 * U * r * (turned * wi.abs() + xh.abs() * (turned * wi.abs() * xh.abs()).mean(-1, keepdim=True))
        close(got[i], r * (gw - xh * mean), slack, dtype, "dx")
        terms = (turned * xh.abs()).sum((0, 1))
        close(got[2 + i], (back * xh).sum((0, 1)), (64 + T * leaves[i].shape[1]) * U * terms, dtype, "dw")


@gpu
def test_gradients_match_differences():
    """The kernels' gradients along a direction against central differences of the formula in fp64: step 1e-5, of which
    the third derivative's share is below 1e-9 and the fp64 noise below 1e-9 of sums of a few hundred terms of order 1; the kernels' own
    error is bounded as above, 64 u of some 500 terms of order 1 to 10."""
    T, H, G, D, R, eps, factor = 7, 4, 2, 24, 16, 1e-5, 1.5
    q, k, w, grads = inputs(T, H, G, D, F32, seed=5, weights=True)
    inv_freq = ops.rotary_frequencies(R, 100.0, device=DEV)[0]
    positions = torch.arange(T, device=DEV) + 3
    leaves = [q.requires_grad_(), k.requires_grad_(), *(t.to(DEV).requires_grad_() for t in w)]
    a = angles(positions, inv_freq)
    gen = torch.Generator().manual_seed(6)
    way = [torch.randn(t.shape, generator=gen, dtype=torch.float64) for t in leaves]
    base = [t.detach().cpu().double() for t in leaves]
    for norm in (False, True):
        def value(step):
            at = [b + step * d for b, d in zip(base, way)]
            ys = [normed(at[i], at[2 + i], eps)[0] if norm else at[i] for i in range(2)]
            return sum((turn(y, a, factor, False) * g.double()).sum() for y, g in zip(ys, grads))

        if norm:
            out = ops.qk_norm_rotary(*leaves, positions, inv_freq, eps, attention_factor=factor)
        else:
            out = ops.rotary(*leaves[:2], positions, inv_freq, attention_factor=factor)
        n = 4 if norm else 2
        got = torch.autograd.grad(out, leaves[:n], [g.to(DEV) for g in grads])
        along = sum((g.cpu().double() * d).sum() for g, d in zip(got, way))
        assert abs(along - (value(1e-5) - value(-1e-5)) / 2e-5) < 64 * U * 5000 + 1e-6


@gpu
@pytest.mark.parametrize("base,start", [(10000.0, 10**6), (1000000.0, 2**29 - 40), (10000.0, -(2**29) + 3)])
def test_far_positions_are_as_good_as_near_ones(base, start):
    """Products of a position below 2^29 and an fp32 frequency are exact in fp64; the formula here takes the sine of them."""
    T, H, G, D = 33, 4, 1, 128
    print(f"rotary from position {start}", flush=True)
    q, k, _, _ = inputs(T, H, G, D, F32, seed=11)
    inv_freq = ops.rotary_frequencies(D, base, device=DEV)[0]
    positions = torch.arange(T, device=DEV) + start
    for x, y in zip((q, k), ops.rotary(q, k, positions, inv_freq)):
        x64 = x.cpu().double()
        # (the reference's own angle is off by up to 2^-53 of 2^29)
        close(y, turn(x64, angles(positions, inv_freq), 1.0, False), (16 * U + 2.0**-23) * pair_size(x64, D // 2, 1.0, False),
              F32, "result")


@gpu
def test_layouts_streams_and_graphs_give_the_same_bits():
    T, H, G, D, R, eps = 66, 6, 2, 64, 64, 1e-6
    q, k, w, grads = inputs(T, H, G, D, BF, seed=21, weights=True)
    grads = [g.to(DEV) for g in grads]
    inv_freq = ops.rotary_frequencies(R, device=DEV)[0]
    positions = torch.arange(T, device=DEV)
    leaves = [q.requires_grad_(), k.requires_grad_(), *(t.to(DEV).requires_grad_() for t in w)]

    def step(ls, pos, gs, interleaved=True):
        out = ops.qk_norm_rotary(*ls, pos, inv_freq, eps, interleaved=interleaved)
        turned = ops.rotary(*out, pos, inv_freq, interleaved=interleaved, attention_factor=2.0)
        return [t.detach() for t in (*out, *turned)] + list(torch.autograd.grad(turned, ls, gs))

    want = step(leaves, positions, grads)
    # (batch, sequence, heads, size); heads in front of the tokens; off 16 bytes; every other element
    batch = [t.detach().unflatten(0, (2, 33)).requires_grad_() for t in leaves[:2]] + leaves[2:]
    got = step(batch, positions.view(2, 33), [g.unflatten(0, (2, 33)) for g in grads])
    assert all(torch.equal(a.reshape(b.shape), b) for a, b in zip(got, want))
    heads_first = [t.detach().transpose(0, 1).contiguous().transpose(0, 1).requires_grad_() for t in leaves[:2]] + leaves[2:]
    assert all(torch.equal(a, b) for a, b in zip(step(heads_first, positions, grads), want))
    off = []
    for t in leaves[:2]:
        flat = torch.empty(t.numel() + 1, dtype=BF, device=DEV)
        flat[1:] = t.detach().flatten()
        off.append(flat[1:].view(t.shape).requires_grad_())
    for a, b in zip(step(off + leaves[2:], positions, grads), want):  # (other pieces: sums in another order)
        torch.testing.assert_close(a, b, rtol=2**-6, atol=2**-6)
    apart = [t.detach().repeat_interleave(2, -1)[..., ::2].requires_grad_() for t in leaves[:2]] + leaves[2:]
    assert all(torch.equal(a, b) for a, b in zip(step(apart, positions, grads), want))
    # another stream
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step(leaves, positions, grads)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    # a captured step, replayed over changed inputs with eager work between the replays
    fresh = [t.detach().clone().requires_grad_() for t in leaves]
    del got, batch, heads_first, off, apart
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(fresh, positions, grads)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step(fresh, positions, grads)
    for turn_ in range(3):
        with torch.no_grad():
            for t in fresh:
                t.mul_(0.5)
        graph.replay()
        torch.cuda.synchronize()
        eager = step([t.detach().clone().requires_grad_() for t in fresh], positions, grads)
        assert all(torch.equal(a, b) for a, b in zip(captured, eager)), turn_


@gpu
def test_values_that_are_not_finite_stay_with_their_pair_or_head():
    T, H, G, D, R = 3, 2, 1, 64, 32
    q, k, w, _ = inputs(T, H, G, D, BF, seed=31, weights=True)
    q[1, 0, 5], q[2, 1, 40] = math.inf, math.nan
    inv_freq = ops.rotary_frequencies(R, device=DEV)[0]
    positions = torch.arange(T, device=DEV)
    y, _ = ops.rotary(q, k, positions, inv_freq)
    bad = ~y.isfinite()
    assert bad[1, 0, 5] and bad[1, 0, 5 + R // 2] and bad[2, 1, 40] and bad.sum() == 3
    y, yk = ops.qk_norm_rotary(q, k, *(t.to(DEV) for t in w), positions, inv_freq, 1e-6)
    bad = y.isnan()
    assert bad[2, 1].all() and bad[0].logical_not().all() and bad[1, 1].logical_not().all() and yk.isfinite().all()


@gpu
def test_no_tokens_and_unused_results():
    inv_freq = ops.rotary_frequencies(8, device=DEV)[0]
    q, k, w = torch.empty(0, 4, 16, device=DEV), torch.empty(0, 2, 16, device=DEV), torch.ones(16, device=DEV)
    pos = torch.empty(0, dtype=torch.int32, device=DEV)
    assert [t.shape for t in ops.rotary(q, k, pos, inv_freq)] == [q.shape, k.shape]
    leaves = [t.requires_grad_() for t in (q, k, w.clone(), w.clone())]
    out = ops.qk_norm_rotary(*leaves, pos, inv_freq, 1e-6)
    got = torch.autograd.grad(out, leaves, [torch.empty_like(t) for t in out])
    assert not got[2].any() and not got[3].any()
    # one result alone is differentiated: the gradients of the other's inputs are zeros or absent, its own are as ever
    q, k, w, grads = inputs(5, 2, 1, 16, F32, seed=1, weights=True)
    leaves = [q.requires_grad_(), k.requires_grad_(), *(t.to(DEV).requires_grad_() for t in w)]
    pos = torch.arange(5, device=DEV)
    both = torch.autograd.grad(ops.qk_norm_rotary(*leaves, pos, inv_freq, 1e-6), leaves, [g.to(DEV) for g in grads])
    one = torch.autograd.grad(ops.qk_norm_rotary(*leaves, pos, inv_freq, 1e-6)[0], leaves, grads[0].to(DEV), allow_unused=True)
    assert torch.equal(one[0], both[0]) and torch.equal(one[2], both[2]) and one[1] is None and one[3] is None
    turned = torch.autograd.grad(ops.rotary(*leaves[:2], pos, inv_freq)[1], leaves[:2], grads[1].to(DEV), allow_unused=True)
    assert turned[0] is None or not turned[0].any()
    # only the weights, only the heads
    part = [q.detach(), k.detach(), *leaves[2:]]
    got = torch.autograd.grad(ops.qk_norm_rotary(*part, pos, inv_freq, 1e-6), part[2:], [g.to(DEV) for g in grads])
    assert torch.equal(got[0], both[2]) and torch.equal(got[1], both[3])


# ---- without a GPU ---------------------------------------------------------------------------------


def test_frequencies_against_their_formulas():
    R, base, factor, context = 64, 10000.0, 8.0, 4096
    plain = [base ** (-2 * i / R) for i in range(R // 2)]

    def same(got, want):
        torch.testing.assert_close(got, torch.tensor(want, dtype=torch.float64).float(), rtol=2**-23, atol=0)

    freq, f = ops.rotary_frequencies(R, base)
    same(freq, plain)
    assert f == 1.0 and freq.dtype == F32
    same(ops.rotary_frequencies(R, base, scaling="linear", factor=factor)[0], [x / factor for x in plain])
    ntk = ops.rotary_frequencies(R, base, scaling="ntk", factor=factor)[0]
    same(ntk[:1], plain[:1])  # the fastest pair stays, the slowest is interpolated in full
    torch.testing.assert_close(ntk[-1].item(), plain[-1] / factor, rtol=1e-6, atol=0)
    yarn, f = ops.rotary_frequencies(R, base, scaling="yarn", factor=factor, original_context=context)
    assert f == pytest.approx(0.1 * math.log(factor) + 1)
    for x, p in zip(yarn.tolist(), plain):
        turns = context * p / (2 * math.pi)
        assert p / factor * (1 - 1e-6) <= x <= p * (1 + 1e-6)
        if turns > 40:
            assert x == pytest.approx(p, rel=1e-6)
        if turns < 0.7:
            assert x == pytest.approx(p / factor, rel=1e-6)
    llama = ops.rotary_frequencies(R, base, scaling="llama3", factor=factor, original_context=context)[0]
    for x, p in zip(llama.tolist(), plain):
        wavelength = 2 * math.pi / p
        if wavelength < context / 4:
            want = p
        elif wavelength > context:
            want = p / factor
        else:
            smooth = (context / wavelength - 1) / 3
            want = (1 - smooth) * p / factor + smooth * p
        assert x == pytest.approx(want, rel=1e-6)


@pytest.mark.parametrize("kwargs,message", [
    (dict(rotary_dim=7), "positive even"), (dict(rotary_dim=0), "positive even"),
    (dict(rotary_dim=8, base=1.0), "above 1"), (dict(rotary_dim=8, base=math.inf), "finite"),
    (dict(rotary_dim=8, scaling="cubic"), "Unknown rotary scaling"),
    (dict(rotary_dim=8, scaling="linear", factor=0.5), "at least 1"),
    (dict(rotary_dim=8, scaling="yarn", factor=2.0), "needs original_context"),
    (dict(rotary_dim=8, scaling="yarn", factor=2.0, original_context=64, beta_fast=1.0), "beta_fast > beta_slow"),
    (dict(rotary_dim=8, scaling="llama3", factor=2.0, original_context=64, high_freq_factor=1.0), "high_freq_factor"),
])
def test_frequencies_refuse(kwargs, message):
    with pytest.raises(ValueError, match=message):
        ops.rotary_frequencies(**kwargs)


def test_operators_are_registered_for_the_gpu_only():
    for name, function in (("rotary", kernel_registry.rotary_mi355), ("qk_norm_rotary", kernel_registry.qk_norm_rotary_mi355)):
        assert kernel_registry.get_kernel(name, "cuda") is function
        assert set(kernel_registry._KERNEL_REGISTRY[name]) == {"cuda"}
    q, w, pos, freq = torch.ones(2, 1, 4), torch.ones(4), torch.arange(2), torch.ones(2)
    with pytest.raises(KeyError, match="not available"):
        kernel_registry.rotary(q, q, pos, freq)
    with pytest.raises(KeyError, match="not available"):
        kernel_registry.qk_norm_rotary(q, q, w, w, pos, freq, 1e-6)
    with pytest.raises(NotImplementedError, match="no torch-math backend"):
        kernel_registry.rotary(q, q, pos, freq, use_eager=True)
    with pytest.raises(NotImplementedError, match="no torch-math backend"):
        kernel_registry.qk_norm_rotary(q, q, w, w, pos, freq, 1e-6, use_eager=True)
    with pytest.raises(RuntimeError, match="no CPU implementation"):
        ops.rotary(q, q, pos, freq)


def test_operators_refuse_what_does_not_fit_and_propagate_shapes():
    with FakeTensorMode():
        def t(*shape, dtype=F32):
            return torch.empty(shape, dtype=dtype, device="cuda")

        q, k, w, pos, freq = t(2, 3, 8, 64), t(2, 3, 2, 64), t(64), t(2, 3, dtype=torch.int32), t(32)

        def refused(error, message, *, norm_only=False, **change):
            a = dict(q=q, k=k, q_weight=w, k_weight=w, positions=pos, inv_freq=freq, epsilon=1e-6, attention_factor=1.0)
            a.update(change)
            with pytest.raises(error, match=message):
                ops.qk_norm_rotary(**a)
            if not norm_only:
                with pytest.raises(error, match=message):
                    ops.rotary(a["q"], a["k"], a["positions"], a["inv_freq"], attention_factor=a["attention_factor"])

        refused(ValueError, "agree in all but the heads", k=t(2, 3, 2, 32))
        refused(ValueError, "agree in all but the heads", k=t(2, 4, 2, 64))
        refused(ValueError, "agree in all but the heads", q=t(8, 64), k=t(2, 64))
        refused(TypeError, "share a dtype", k=k.to(BF))
        refused(TypeError, "float32 and bfloat16", q=q.half(), k=k.half())
        refused(TypeError, "float32 and bfloat16", q=q.double(), k=k.double())
        refused(ValueError, "2 to 512", q=t(2, 3, 8, 514), k=t(2, 3, 2, 514))
        refused(ValueError, "2 to 512", q=t(2, 3, 0, 64))
        refused(TypeError, "positions must be int32 or int64", positions=t(2, 3))
        refused(ValueError, "must match the tokens", positions=t(6, dtype=torch.int32))
        refused(TypeError, "inv_freq must be a 1-D float32", inv_freq=t(32, dtype=BF))
        refused(TypeError, "inv_freq must be a 1-D float32", inv_freq=t(1, 32))
        refused(ValueError, "no gradient for inv_freq", inv_freq=t(32).requires_grad_())
        refused(ValueError, "frequencies turn", inv_freq=t(33))
        refused(ValueError, "frequencies turn", inv_freq=t(0))
        refused(ValueError, "must be finite", attention_factor=math.inf)
        refused(ValueError, "must be finite", attention_factor=math.nan)
        refused(TypeError, "norm weights", norm_only=True, q_weight=w.to(BF))
        refused(ValueError, "norm weights must be", norm_only=True, k_weight=t(32))
        refused(ValueError, "finite and nonnegative", norm_only=True, epsilon=-1.0)
        refused(ValueError, "finite and nonnegative", norm_only=True, epsilon=math.nan)
        q.requires_grad_(), w.requires_grad_()
        out = ops.qk_norm_rotary(q, k, w, w, pos, freq, 1e-6)
        assert [o.shape for o in out] == [q.shape, k.shape] and out[0].requires_grad
        assert [o.shape for o in ops.rotary(*out, pos, freq)] == [q.shape, k.shape]
        back = torch.ops.mi355_moe.qk_norm_rotary_bwd(out[0].detach(), None, q, k, w, w, pos, freq, 1e-6, False, 1.0, True, False)
        assert [o.shape for o in back] == [q.shape, k.shape, (0,), (0,)]


def test_c_entry_points_refuse_before_any_launch():
    lib, p = _lib.load(), 0x1000  # (never dereferenced)

    def rotary(T=4, H=2, G=1, D=64, pairs=32, dtype=1, factor=1.0, q=p):
        return lib.mi355_rotary(q, H * D, D, p, G * D, D, dtype, p, 0, p, pairs, factor, 0, 0, p, p, T, H, G, D, None)

    def text(rc, needle):
        assert rc == -1 and needle in lib.mi355_moe_last_error(), (rc, lib.mi355_moe_last_error())

    text(rotary(dtype=2), b"neither fp32 nor bf16")
    text(rotary(D=513), b"head size 513")
    text(rotary(D=1, pairs=1), b"head size 1 ")
    text(rotary(pairs=33), b"turn more elements")
    text(rotary(pairs=0), b"turn more elements")
    text(rotary(T=-1), b"bad shape")
    text(rotary(H=0), b"bad shape")
    text(rotary(factor=math.inf), b"attention factor")
    text(rotary(q=None), b"null pointer")
    assert rotary(T=0) == 0
    norm = lib.mi355_qk_norm_rotary_fwd
    text(norm(p, 128, 64, p, 64, 64, p, p, 1, p, 0, p, 32, 1.0, 0, -1.0, p, p, 4, 2, 1, 64, None), b"epsilon")
    text(norm(p, 128, 64, p, 64, 64, None, p, 1, p, 0, p, 32, 1.0, 0, 1e-6, p, p, 4, 2, 1, 64, None), b"null pointer")
    back = lib.mi355_qk_norm_rotary_bwd
    text(back(p, p, p, 128, 64, p, 64, 64, p, p, 1, p, 0, p, 32, 1.0, 0, 1e-6, p, p, p, p, None, 4, 2, 1, 64, None), b"workspace")
    assert lib.mi355_qk_norm_rotary_bwd_workspace_bytes(64) >= 2 * 64 * 4
