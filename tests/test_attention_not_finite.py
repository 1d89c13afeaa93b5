"""Attention over values that are not finite: which results they reach, and what they cost.

What is finite is compared with the formulas in fp64 within the bounds of tests/test_attention.py; a sum is not finite if, and only if, it has a
visible term that is not.  Such values have to stay cheap: a step whose activations overflowed is one that a trainer wants to see and skip.
"""

import math

import pytest
import torch

from tests.test_attention import BF, DEV, F32, HALF_STEP, TINY, U, bounds_of, inputs, step
from torchllmtuner_amd import ops

gpu = pytest.mark.gpu


def visible_sum(w, x, seen):
    """sum_j w_rj x_j over the seen (r, j); NaN where one of those is not finite."""
    total = torch.where(seen & w.isfinite(), w, 0.0) @ x.nan_to_num(0.0, 0.0, 0.0)
    bad = (seen & ~w.isfinite()).any(1, keepdim=True) | ((seen.double() @ (~x.isfinite()).double()) > 0)
    return total.masked_fill(bad, math.nan)


def reference(q, k, v, dout, cu, dtype):
    """Values and bounds as in tests/test_attention.py, of visible terms only."""
    q, k, v, dout = (t.detach().cpu().double() for t in (q, k, v, dout))
    T, H, D = q.shape
    group, scale = H // k.shape[1], D**-0.5
    h = 2.0**-8 if dtype == BF else 0.0
    kept = HALF_STEP[dtype] if dtype == F32 else HALF_STEP[dtype] ** 2
    val = [torch.zeros_like(t) for t in (q, q, k, v)]
    off = [torch.zeros_like(t) for t in (q, q, k, v)]
    for a, b in zip(cu, cu[1:]):
        n = b - a
        if n == 0:
            continue
        seen = torch.ones(n, n, dtype=torch.bool).tril()
        for head in range(H):
            g = head // group
            Q, K, V, G = q[a:b, head], k[a:b, g], v[a:b, g], dout[a:b, head]
            s = (Q @ K.T * scale).masked_fill(~seen, -math.inf)
            # (a score of -inf is exact, and its weight zero)
            size = (scale * (Q.abs() @ K.abs().T)).masked_fill(~seen | ~s.isfinite(), 0)
            p = torch.softmax(s, 1)
            e = 2 * ((D + 4) * U * size).amax(1, keepdim=True) + (2 * n + 32) * U
            out, out_off = visible_sum(p, V, seen), visible_sum(p * (e + h + n * U) + TINY, V.abs(), seen)
            val[0][a:b, head], off[0][a:b, head] = out, out_off
            e = e + 4 * U * torch.logsumexp(s, 1, keepdim=True).abs()
            N = n * group
            val[3][a:b, g] += visible_sum(p.T, G, seen.T)
            off[3][a:b, g] += visible_sum((p * (e + h + N * U) + TINY).T, G.abs(), seen.T)
            dp, delta = G @ V.T, (G * out).sum(1, keepdim=True)
            e_delta = (G.abs() * (kept * (out.abs() + out_off) + out_off)).sum(1, keepdim=True) + 2 * D * U * (G.abs() * out.abs()).sum(1, keepdim=True)
            e_dp = D * U * (G.abs() @ V.abs().T)
            ds = p * (dp - delta)
            ds[0] = 0.0  # (one visible key: no gradient through the score, whatever it is)
            e_ds = TINY * (1 + dp.abs() + delta.abs()) + p * ((dp.abs() + delta.abs() + e_dp + e_delta) * (e + h + 4 * U) + e_dp + e_delta) * (1 + h)
            e_ds[0] = 0.0
            val[1][a:b, head] = scale * visible_sum(ds, K, seen)
            off[1][a:b, head] = scale * visible_sum(e_ds + (n + 4) * U * ds.abs(), K.abs(), seen)
            val[2][a:b, g] += scale * visible_sum(ds.T, Q, seen.T)
            off[2][a:b, g] += scale * visible_sum((e_ds + (N + 4) * U * ds.abs()).T, Q.abs(), seen.T)
    return val, off


@gpu
@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("lengths,behind,H,G,D", [
    ([20, 30, 250, 60], 6, 4, 2, 64),
    ([300, 5, 1, 130], 0, 3, 1, 128),
    ([150, 40], 3, 2, 2, 75),
    ([170, 90], 1, 2, 1, 200),
    ([1100], 20, 2, 1, 64),      # keys (queries) dealt over workgroups
    ([2, 900, 300], 0, 2, 2, 128),
])
def test_reach_what_sees_them_and_nothing_else(lengths, behind, H, G, D, dtype):
    cu, T = bounds_of(lengths, behind)
    print(f"varlen_attention not finite {lengths}+{behind} heads {H}/{G} of {D} {dtype}", flush=True)
    at = torch.tensor(cu, dtype=torch.int32, device=DEV)
    gen = torch.Generator().manual_seed(T)
    for which in range(4):
        for value in (math.nan, math.inf, -math.inf):
            for many in (1, 4):
                leaves, dout = inputs(T, H, G, D, dtype, seed=T + D)
                spoilt = [t.detach().clone() for t in (*leaves, dout)]
                x = spoilt[which]
                for _ in range(many):
                    r, head, d = (int(torch.randint(n, (1,), generator=gen)) for n in x.shape)
                    x[r, head, d] = value
                if behind:
                    x[cu[-1]:] = value
                got = step([t.requires_grad_() for t in spoilt[:3]], spoilt[3], at)
                val, off = reference(*spoilt, cu, dtype)
                for y, want, bound, name in zip(got, val, off, ("out", "dq", "dk", "dv")):
                    y = y.detach().cpu().double()
                    what = f"{name} with {many} of {value} in {'q k v dout'.split()[which]}"
                    ok = want.isfinite()
                    if name in ("dq", "dk"):  # an infinite result times a gradient of zero, or two of different signs: not finite either way, but not by this rule
                        assert not (y.isfinite() & ~ok).any() or value != value, what
                    assert torch.equal(y.isfinite() | ~ok, torch.ones_like(ok)), f"{what}: {(ok & ~y.isfinite()).sum()} spoilt that see nothing"
                    if value != value:
                        assert torch.equal(y.isfinite(), ok), f"{what}: {(~ok & y.isfinite()).sum()} not spoilt"
                    over = ((y - want).abs() - bound - HALF_STEP[dtype] * (want.abs() + bound) - 256 * TINY)[ok]
                    assert over.numel() == 0 or over.max() <= 0, f"{what}: {over.max():.3g} beyond the bound"


def spoil(tensors, pattern, T, first_end, last_end):
    for x in tensors if pattern in ("everything", "rows behind", "the next sequence") else []:
        x[dict(everything=slice(0, T)).get(pattern, slice(last_end, T) if pattern == "rows behind" else slice(first_end, last_end))] = math.nan
    q, k, v, dout = tensors
    if pattern in ("values", "gradients"):
        (v if pattern == "values" else dout).fill_(math.nan)
    if pattern == "infinite values":
        v.mul_(math.inf)
    if pattern == "one early key":
        k[3, 0, 0] = math.nan
    if pattern == "one early value":
        v[3, 0, 0] = math.nan
    if pattern == "one query":
        q[T // 3, 0, 0] = math.nan
    if pattern == "the second half's values":
        v[first_end // 2:] = math.nan


PATTERNS = ["everything", "values", "infinite values", "gradients", "one early key", "one early value", "one query", "the second half's values",
            "rows behind", "the next sequence"]


@gpu
@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("pattern", PATTERNS)
def test_cost_no_more_than_a_few_steps(pattern, dtype):
    """A step over such values takes at most 25 times one over finite ones: formed key by key, each row over all its keys, it took 50 to
    several hundred times as long, and more the longer the sequences."""
    T, H, G, D, first_end, last_end = 4096, 8, 2, 128, 3000, 4000
    print(f"varlen_attention step with {pattern} NaN {dtype}", flush=True)
    cu = torch.tensor([0, first_end, last_end], dtype=torch.int32, device=DEV)
    tensors = [torch.randn(T, n, D, device=DEV).to(dtype) for n in (H, G, G, H)]

    def least(leaves, dout):
        times = []
        for _ in range(4):
            a, b = (torch.cuda.Event(enable_timing=True) for _ in "ab")
            a.record()
            torch.autograd.grad(ops.varlen_attention(*leaves, cu), leaves, dout)
            b.record()
            torch.cuda.synchronize()
            times.append(a.elapsed_time(b))
        return min(times)

    plain = least([t.clone().requires_grad_() for t in tensors[:3]], tensors[3])
    spoil(tensors, pattern, T, first_end, last_end)
    spoilt = least([t.requires_grad_() for t in tensors[:3]], tensors[3])
    print(f"{plain:.3f} -> {spoilt:.3f} ms, {spoilt / plain:.1f} times", flush=True)
    assert spoilt < 25 * plain
