"""Causal attention over packed sequences against the formulas in fp64, element by element within derived bounds.

Arithmetic is fp32 (u = 2^-24, half a step) on the stored inputs; with bf16 storage the weights p and the ds of the backward may
be rounded to bf16 in front of their products and results are rounded to bf16 (half a step h = 2^-8 of the value).  With n visible
keys, in natural units:

* a score is a sum of D products: off by D u |scale| sum |q k|; its scaling, the row maximum and lse by 4 u of their sizes.  E = the
  largest of that over a row's keys.
* a weight: exp of it, over a sum of n such: off by e = 2 E + (2 n + 32) u of the weight; from lse (backward) 4 u |lse| more.
* a result: sum p |v| (e + h + n u).
* dp off by D u sum |do v|; delta = do . o by sum |do| (r |o| + the result's bound), of o as stored: fp32, r = u; bf16 and
  what its rounding took, in bf16 as well, r = h^2; and 2 D u sum |do o|.
* a weight below 2^-126, the least normal number of fp32, may come out as zero: exp2 has no others.  TINY = 2^-126 of absolute error
  a weight, which a ds takes times |dp| + |delta|, and the products' results and the stored ones once more each.
* ds = p (dp - delta): p ((|dp| + |delta|) (e + h + 4 u) + both errors), then sums of N terms add N u of their sizes.
"""

import math

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

from torchllmtuner_amd import _lib, kernel_registry, ops

DEV = "cuda:0"
U = 2.0**-24
TINY = 2.0**-126
BF, F32 = torch.bfloat16, torch.float32
HALF_STEP = {BF: 2.0**-8, F32: 2.0**-24}
gpu = pytest.mark.gpu


def reference(q, k, v, dout, cu, scale, dtype, ds_rounding=None):
    """fp64 values and bounds of out, dq, dk, dv (before the storage rounding), on the CPU."""
    q, k, v, dout = (t.detach().cpu().double() for t in (q, k, v, dout))
    T, H, D = q.shape
    group = H // k.shape[1]
    h = 2.0**-8 if dtype == BF else 0.0
    store = HALF_STEP[dtype]
    h_ds = h if ds_rounding is None else ds_rounding
    val = [torch.zeros_like(t) for t in (q, q, k, v)]
    off = [torch.zeros_like(t) for t in (q, q, k, v)]
    for a, b in zip(cu, cu[1:]):
        n = b - a
        if n <= 0:
            continue
        seen = torch.ones(n, n, dtype=torch.bool).tril()
        for head in range(H):
            g = head // group
            Q, K, V, G = q[a:b, head], k[a:b, g], v[a:b, g], dout[a:b, head]
            s = (Q @ K.T * scale).masked_fill(~seen, -math.inf)
            size = scale * (Q.abs() @ K.abs().T)
            lse = torch.logsumexp(s, 1, keepdim=True)
            p = torch.exp(s - lse)
            E = ((D + 4) * U * size).masked_fill(~seen, 0).amax(1, keepdim=True)
            e = 2 * E + (2 * n + 32) * U
            out = p @ V
            dout_bound = (p * (e + h + n * U) + TINY) @ V.abs()
            val[0][a:b, head], off[0][a:b, head] = out, dout_bound
            e = e + 4 * U * lse.abs()
            N = n * group
            val[3][a:b, g] += p.T @ G
            off[3][a:b, g] += (p * (e + h + N * U) + TINY * seen).T @ G.abs()
            dp, delta = G @ V.T, (G * out).sum(1, keepdim=True)
            kept = store if dtype == F32 else store * store
            e_delta = (G.abs() * (kept * (out.abs() + dout_bound) + dout_bound)).sum(1, keepdim=True)
            e_delta = e_delta + 2 * D * U * (G.abs() * out.abs()).sum(1, keepdim=True)
            e_dp = D * U * (G.abs() @ V.abs().T)
            ds = p * (dp - delta)
            e_ds = TINY * seen * (1 + dp.abs() + delta.abs()) + p * ((dp.abs() + delta.abs() + e_dp + e_delta) * (e + h_ds + 4 * U) + e_dp + e_delta) * (1 + h_ds)
            val[1][a:b, head] = scale * (ds @ K)
            off[1][a:b, head] = scale * ((e_ds + (n + 4) * U * ds.abs()) @ K.abs())
            val[2][a:b, g] += scale * (ds.T @ Q)
            off[2][a:b, g] += scale * ((e_ds + (N + 4) * U * ds.abs()).T @ Q.abs())
    return val, off


def inputs(T, H, G, D, dtype, seed, fused=False, size=1.0):
    gen = torch.Generator().manual_seed(seed)
    rows = (size * torch.randn(T, H + 2 * G, D, generator=gen)).to(dtype).to(DEV)
    dout = torch.randn(T, H, D, generator=gen).to(dtype).to(DEV)
    q, k, v = rows[:, :H], rows[:, H:H + G], rows[:, H + G:]
    if not fused:
        q, k, v = q.contiguous(), k.contiguous(), v.contiguous()
    return [t.detach().requires_grad_() for t in (q, k, v)], dout


def bounds_of(lengths, behind=0):
    cu = [0]
    for n in lengths:
        cu.append(cu[-1] + n)
    return cu, cu[-1] + behind


def check(got, val, off, dtype, names=("out", "dq", "dk", "dv")):
    for x, want, bound, name in zip(got, val, off, names):
        x = x.detach().cpu().double()
        assert not x.isnan().any(), name
        over = (x - want).abs() - bound - HALF_STEP[dtype] * (want.abs() + bound) - 256 * TINY
        worst = over.flatten().argmax().item()
        assert over.max() <= 0, (f"{name}: {over.max():.3g} beyond the bound, {x.flatten()[worst]:.6g} for "
                                 f"{want.flatten()[worst]:.6g}, element {worst} of {tuple(x.shape)}")


def step(leaves, dout, cu, scale=None):
    out = kernel_registry.varlen_attention(*leaves, cu, scale=scale)
    return [out.detach(), *torch.autograd.grad(out, leaves, dout)]


# (lengths, rows behind, heads, key heads, head size)
CASES = [
    ([1], 0, 1, 1, 64),
    ([1, 1, 1], 2, 4, 2, 128),
    ([0, 2, 0, 0, 5, 0], 0, 2, 1, 32),
    ([33], 0, 3, 3, 128),
    ([64], 0, 2, 1, 64),
    ([65, 63], 0, 2, 2, 128),
    ([127, 1, 129], 3, 4, 1, 128),
    ([300], 0, 8, 2, 64),
    ([31, 200, 7, 90], 17, 5, 1, 96),
    ([130, 0, 260], 1, 2, 1, 80),
    ([97, 100], 0, 6, 3, 112),
    ([75, 50], 0, 2, 2, 8),
    ([40, 85], 5, 2, 1, 160),
    ([70, 66], 0, 2, 1, 192),
    ([140], 9, 2, 2, 256),
    ([30, 70], 0, 3, 1, 33),
    ([45], 2, 2, 1, 1),
    ([90, 20], 0, 1, 1, 127),
    ([3] * 60, 4, 2, 2, 64),
    ([513], 0, 4, 4, 128),
    ([400, 380], 0, 2, 1, 128),
    ([200, 90], 3, 4, 2, 75),    # heads that are no whole number of 16 bytes, copied into padded rows
    ([260], 0, 3, 1, 150),
    ([0, 301, 2], 1, 2, 2, 33),
    ([250], 0, 2, 1, 201),
    ([300], 5, 2, 1, 1),
    ([2, 0, 3] * 50, 1, 2, 1, 64),        # more boundaries than a wave has lanes ...
    ([0] * 200 + [40] + [0] * 100 + [9] * 30, 0, 2, 2, 64),
    ([1, 0, 2] * 1400, 3, 1, 1, 32),      # ... and than lanes times lanes
    ([600, 520], 7, 8, 8, 64),   # long on average and more tiles than the card holds at once: sorted by their work
    ([512, 3, 1100], 0, 16, 4, 40),
]


@gpu
@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("lengths,behind,H,G,D", CASES)
def test_attention_matches_the_formula_in_both_directions(lengths, behind, H, G, D, dtype):
    cu, T = bounds_of(lengths, behind)
    print(f"varlen_attention {lengths}+{behind} heads {H}/{G} of {D} {dtype}", flush=True)
    leaves, dout = inputs(T, H, G, D, dtype, seed=T + D, fused=T % 2 == 0)
    got = step(leaves, dout, torch.tensor(cu, dtype=torch.int32, device=DEV))
    for x, like in zip(got, (leaves[0], *leaves)):
        assert x.shape == like.shape and x.dtype == dtype and x.is_contiguous()
    val, off = reference(*leaves, dout, cu, D**-0.5, dtype)
    check(got, val, off, dtype)
    if behind:  # rows in no sequence: zeros, not merely small
        assert not any(x[cu[-1]:].any() for x in got)


@gpu
@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("lengths,behind,H,G,D", [
    ([520], 0, 2, 1, 64),          # long on average and few tiles: their keys (queries) dealt over two, four, eight workgroups
    ([1030], 5, 1, 1, 128),
    ([2100], 0, 1, 1, 40),
    ([2048], 0, 2, 2, 33),
    ([1, 2200], 0, 4, 2, 64),      # rows that not every share has a key of
    ([1500, 0, 1700, 40], 3, 1, 1, 96),
    ([2300], 0, 3, 1, 200),
    ([2, 1040], 0, 1, 1, 75),
    ([1100, 960], 2, 8, 2, 64),    # in fp32 sorted by their work as well
    ([3000, 1100], 0, 10, 2, 128),  # and in bf16
])
def test_keys_dealt_over_workgroups(lengths, behind, H, G, D, dtype):
    test_attention_matches_the_formula_in_both_directions(lengths, behind, H, G, D, dtype)


@gpu
@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("value", [math.nan, -math.inf])
def test_values_in_masked_places_with_keys_dealt_over_workgroups(value, dtype):
    T, at = 1100, 700
    cu = torch.tensor([0, T], dtype=torch.int32, device=DEV)
    print(f"varlen_attention with {value} at {at} of {T} {dtype}", flush=True)
    leaves, dout = inputs(T, 2, 1, 64, dtype, seed=21)
    val, off = reference(*leaves, dout, [0, T], 64**-0.5, dtype)
    for which in range(4):
        spoilt = [t.detach().clone() for t in (*leaves, dout)]
        spoilt[which][at, 0, :3] = value
        got = step([t.requires_grad_() for t in spoilt[:3]], spoilt[3], cu)
        above, below = slice(0, at), slice(at + 1, T)
        check([got[0][above]], [val[0][above]], [off[0][above]], dtype)  # rows that do not see it
        if which in (0, 3):  # and the gradients of keys that it does not see
            check([x[below] for x in got], [w[below] for w in val], [o[below] for o in off], dtype)
        else:
            check([got[1][above]], [val[1][above]], [off[1][above]], dtype)


@gpu
@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("D", [64, 96, 75, 200])
def test_rows_that_see_one_key_or_two(D, dtype):
    """A row that sees one key has the weight 1: its result is the value, its gradients through the score exactly zero.  Sequences of two rows: what
    rounding takes from ds weighs most there, and the bound on it (h of ds) is u for the kernels of short sequences up to 128
    elements, which hold ds in two pieces: h^2 below u."""
    print(f"varlen_attention of one and two rows {D} {dtype}", flush=True)
    T, H, G = 150, 4, 2
    leaves, dout = inputs(T, H, G, D, dtype, seed=17)
    got = step(leaves, dout, torch.arange(T + 1, dtype=torch.int32, device=DEV))
    v, g = (t.detach().cpu().double() for t in (leaves[2], dout))
    # (its weight w = exp2 of what rounding left of score and maximum is not quite 1: w v / w, three roundings of v, of which none is left in bf16)
    v = v.repeat_interleave(2, 1)
    assert ((got[0].cpu().double() - v).abs() <= (0.0 if dtype == BF else 3 * U) * v.abs()).all()
    assert not got[1].any() and not got[2].any()
    want = g.unflatten(1, (G, H // G)).sum(2)
    close = (got[3].cpu().double() - want).abs() - (4 * U * g.abs().unflatten(1, (G, H // G)).sum(2) + HALF_STEP[dtype] * want.abs())
    assert close.max() <= 2.0**-30
    cu = list(range(0, T + 1, 2))
    got = step(leaves, dout, torch.tensor(cu, dtype=torch.int32, device=DEV))
    val, off = reference(*leaves, dout, cu, D**-0.5, dtype, ds_rounding=None if D > 128 or dtype == F32 else 2.0**-16)
    check(got, val, off, dtype)


@gpu
@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("size,scale", [(1.0, 0.01), (4.0, None), (12.0, 0.5)])
def test_attention_over_flat_and_peaked_scores(size, scale, dtype):
    cu, T = bounds_of([150, 60])
    print(f"varlen_attention size {size} scale {scale} {dtype}", flush=True)
    leaves, dout = inputs(T, 4, 2, 64, dtype, seed=3, size=size)
    got = step(leaves, dout, torch.tensor(cu, dtype=torch.int32, device=DEV), scale)
    check(got, *reference(*leaves, dout, cu, scale or 64**-0.5, dtype), dtype)


@gpu
def test_gradients_match_differences():
    """Along a direction, against central differences of the formula in fp64 (step 1e-5: fp64 noise and the third derivative
    below 1e-8 of the sum's size); the kernel's share is bounded element by element as above."""
    cu, T = bounds_of([37, 22], 2)
    leaves, dout = inputs(T, 4, 2, 24, F32, seed=8)
    got = step(leaves, dout, torch.tensor(cu, dtype=torch.int32, device=DEV))[1:]
    gen = torch.Generator().manual_seed(9)
    way = [torch.randn(t.shape, generator=gen, dtype=torch.float64) for t in leaves]
    base = [t.detach().cpu().double() for t in leaves]

    def value(t):
        q, k, v = (b + t * d for b, d in zip(base, way))
        total = 0.0
        for a, b in zip(cu, cu[1:]):
            seen = torch.ones(b - a, b - a, dtype=torch.bool).tril()
            for h in range(4):
                s = (q[a:b, h] @ k[a:b, h // 2].T * 24**-0.5).masked_fill(~seen, -math.inf)
                total = total + ((s.softmax(1) @ v[a:b, h // 2]) * dout[a:b, h].cpu().double()).sum()
        return total

    along = sum((g.cpu().double() * d).sum() for g, d in zip(got, way))
    _, off = reference(*leaves, dout, cu, 24**-0.5, F32)
    bound = sum(((o + U * g.cpu().double().abs()) * d.abs()).sum() for o, g, d in zip(off[1:], got, way))
    assert abs(along - (value(1e-5) - value(-1e-5)) / 2e-5) < bound + 1e-6


@gpu
@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("D", [64, 128, 40, 160, 35])
@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf])
def test_values_in_masked_places_reach_no_row(value, D, dtype):
    """A sequence whose inputs are spoilt, and the rows behind the last sequence, leave the others' results as they were bit for bit; in a
    sequence, what comes before a spoilt row is its own, too."""
    cu, T = bounds_of([20, 30, 90 if D > 35 else 250], 6)
    print(f"varlen_attention with {value} {D} {dtype}", flush=True)
    leaves, dout = inputs(T, 4, 2, D, dtype, seed=12)
    at = torch.tensor(cu, dtype=torch.int32, device=DEV)
    want = step(leaves, dout, at)
    val, off = reference(*leaves, dout, cu, D**-0.5, dtype)
    for which in range(4):
        spoilt = [t.detach().clone() for t in (*leaves, dout)]
        spoilt[which][33, 0, :3] = value  # in the second sequence
        spoilt[which][cu[-1]:] = value    # in none
        got = step([t.requires_grad_() for t in spoilt[:3]], spoilt[3], at)
        clean = torch.ones(T, dtype=torch.bool)
        clean[20:50] = False
        for x, y in zip(got, want):
            x, y = x[clean], y[clean]
            assert x.isfinite().all()
            torch.testing.assert_close(x, y, rtol=2**-5, atol=2**-5)
        # (formed again key by key where a tile was spoilt: within the same bounds, though not of the same bits)
        check([x[clean.to(DEV)] for x in got], [w[clean] for w in val], [o[clean] for o in off], dtype)
        assert not any(x[cu[-1]:].any() for x in got)
        # causality within the spoilt sequence: results above the row are as they were, gradients of keys behind it too
        above, below = slice(20, 33), slice(34, 50)
        check([got[0][above]], [val[0][above]], [off[0][above]], dtype)
        if which in (0, 3):
            check([x[below] for x in got], [w[below] for w in val], [o[below] for o in off], dtype)
            assert got[0 if which == 0 else 1][33, 0].isnan().any()
        else:
            check([got[1][above]], [val[1][above]], [off[1][above]], dtype)


@gpu
@pytest.mark.parametrize("dtype", [BF, F32])
def test_layouts_give_the_same_bits(dtype):
    T, H, G, D = 150, 6, 2, 64
    cu = torch.tensor([0, 70, 149], dtype=torch.int32, device=DEV)
    leaves, dout = inputs(T, H, G, D, dtype, seed=2)
    want = step(leaves, dout, cu)

    def same(other, g=dout):
        return all(torch.equal(a, b) for a, b in zip(step([t.detach().requires_grad_() for t in other], g, cu), want))

    fused = torch.cat(leaves, 1).detach()
    assert same([fused[:, :H], fused[:, H:H + G], fused[:, H + G:]])
    assert same([t.detach().transpose(0, 1).contiguous().transpose(0, 1) for t in leaves])  # heads in front
    assert same([t.detach().repeat_interleave(2, -1)[..., ::2] for t in leaves])            # every other element
    assert same(leaves, dout.repeat_interleave(2, 0)[::2])
    off = []
    for t in leaves:
        flat = torch.empty(t.numel() + 1, dtype=dtype, device=DEV)
        flat[1:] = t.detach().flatten()
        off.append(flat[1:].view(t.shape))
    for a, b in zip(step([t.requires_grad_() for t in off], dout, cu), want):
        torch.testing.assert_close(a, b, rtol=2**-6, atol=2**-6)
    # one key head for all, by a stride of zero: its gradient is the sum
    one = [leaves[0], *(t.detach()[:, :1] for t in leaves[1:])]
    a = step([t.detach().requires_grad_() for t in one], dout, cu)
    wide = [one[0].detach().requires_grad_(), *(t.expand(T, 3, D).detach().requires_grad_() for t in one[1:])]
    b = step(wide, dout, cu)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    for x, y in zip(a[2:], b[2:]):  # (three sums rounded to the storage type, then added)
        torch.testing.assert_close(x.double(), y.double().sum(1, keepdim=True), rtol=2**-6, atol=2**-4 if dtype == BF else 2**-18)


@gpu
@pytest.mark.parametrize("times,dtype", [(1, BF), (12, BF), (12, F32)])  # (12: keys dealt over workgroups)
def test_streams_and_graphs_over_other_lengths_give_the_same_bits(times, dtype):
    T, H, G, D = 200 * times, 4, 2, 128
    print(f"varlen_attention captured, {T} rows {dtype}", flush=True)
    leaves, dout = inputs(T, H, G, D, dtype, seed=4)
    lengths = [[0, 120, 190], [0, 3, 200], [0, 0, 64], [0, 200, 200], [0, 77, 78]]
    cus = [torch.tensor([times * n for n in c], dtype=torch.int32, device=DEV) for c in lengths]
    want = [step(leaves, dout, c) for c in cus]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step(leaves, dout, cus[0])
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want[0]))
    # a captured step, replayed over other lengths, with eager work between the replays; two graphs alive at once
    fresh = [t.detach().clone().requires_grad_() for t in leaves]
    graphs = []
    for _ in range(2):
        cu = cus[0].clone()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step(fresh, dout, cu)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            captured = step(fresh, dout, cu)
        graphs.append((graph, cu, captured))
    for i in range(len(cus)):
        for j, (graph, cu, captured) in enumerate(graphs):
            cu.copy_(cus[(i + j) % len(cus)])
            graph.replay()
        torch.cuda.synchronize()
        eager = step(leaves, dout, cus[i])
        assert all(torch.equal(a, b) for a, b in zip(eager, want[i]))
        for j, (graph, cu, captured) in enumerate(graphs):
            assert all(torch.equal(a, b) for a, b in zip(captured, want[(i + j) % len(cus)])), (i, j)


@gpu
@pytest.mark.parametrize("dtype,D", [(BF, 64), (BF, 33), (F32, 64)])
def test_rows_beyond_32_bit_offsets(dtype, D):
    """Heads that are views of rows so long that the last ones begin past 4 GiB: the same bits as of dense copies."""
    T = 700_000
    print(f"varlen_attention of rows 8 KiB apart, {T} of them, {dtype} {D}", flush=True)
    wide = torch.empty(T, 4096 if dtype == BF else 2048, dtype=dtype, device=DEV)
    assert wide.numel() * wide.element_size() > 5 << 30
    wide[:, -4 * D:].normal_(generator=torch.Generator(device=DEV).manual_seed(3))
    heads = [wide[:, -4 * D:-2 * D].view(T, 2, D), wide[:, -2 * D:-D].view(T, 1, D), wide[:, -D:].view(T, 1, D)]
    cu = torch.arange(0, T + 1, 100, dtype=torch.int32, device=DEV)
    dout = torch.randn(T, 2, D, dtype=dtype, device=DEV)
    far = step([t.detach().requires_grad_() for t in heads], dout, cu)
    near = step([t.detach().contiguous().requires_grad_() for t in heads], dout, cu)
    assert all(torch.equal(a, b) for a, b in zip(far, near))
    last = slice(T - 100, T)  # and the last sequence against the formula
    val, off = reference(*(t[last] for t in heads), dout[last], [0, 100], D**-0.5, dtype)
    check([t[last] for t in far], val, off, dtype)


@gpu
def test_two_calls_at_once_and_a_traced_one_give_the_same_bits():
    cu = torch.tensor([0, 700, 1500], dtype=torch.int32, device=DEV)
    inv_freq = ops.rotary_frequencies(64, device=DEV)[0]
    positions = torch.arange(1500, device=DEV)
    weight = torch.ones(64, dtype=BF, device=DEV)

    def layer(q, k, v):
        q, k = ops.qk_norm_rotary(q, k, weight, weight, positions, inv_freq, 1e-6)
        q, k = ops.rotary(q, k, positions, inv_freq, interleaved=True)
        return ops.varlen_attention(q, k, v, cu)

    sets = [inputs(1500, 8, 2, 64, BF, seed=s) for s in (1, 2)]

    def whole(leaves, dout, f=layer):
        out = f(*leaves)
        return [out.detach(), *torch.autograd.grad(out, leaves, dout)]

    want = [whole(*s) for s in sets]
    streams = [torch.cuda.Stream() for _ in sets]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    got = []
    for s, (leaves, dout) in zip(streams, sets):
        with torch.cuda.stream(s):
            got.append([whole(leaves, dout) for _ in range(3)])
    torch.cuda.synchronize()
    for runs, w in zip(got, want):
        assert all(torch.equal(a, b) for run in runs for a, b in zip(run, w))
    traced = torch.compile(layer, backend="aot_eager", fullgraph=True)
    assert all(torch.equal(a, b) for a, b in zip(whole(*sets[0], traced), want[0]))


@gpu
def test_bounds_out_of_order_stay_inside_the_tensors():
    """Entries that no caller should pass: results mean nothing, but every look-up stays inside (the sequence of a row always contains
    it) and rows keep to what a call with sound bounds writes."""
    T = 130
    leaves, dout = inputs(T, 2, 1, 64, BF, seed=6)
    for cu in ([0, 100, 50, 130], [5, 60], [-7, 40, 1000], [0, 2**31 - 1], [90, 90, 3], [7]):
        print(f"varlen_attention bounds {cu}", flush=True)
        got = step(leaves, dout, torch.tensor(cu, dtype=torch.int32, device=DEV))
        assert all(x.isfinite().all() for x in got)
    got = step(leaves, dout, torch.tensor([5, 60], dtype=torch.int32, device=DEV))
    assert not any(x[:5].any() or x[60:].any() for x in got)  # rows in front of the first sequence are in none


@gpu
def test_no_tokens_and_only_some_gradients():
    cu = torch.zeros(3, dtype=torch.int32, device=DEV)
    leaves, dout = inputs(0, 4, 2, 64, BF, seed=1)
    assert [x.shape for x in step(leaves, dout, cu)] == [(0, 4, 64), (0, 4, 64), (0, 2, 64), (0, 2, 64)]
    cu = torch.tensor([0, 50], dtype=torch.int32, device=DEV)
    leaves, dout = inputs(50, 4, 2, 64, BF, seed=1)
    want = step(leaves, dout, cu)
    for i in range(3):
        part = [t if j == i else t.detach() for j, t in enumerate(leaves)]
        out = ops.varlen_attention(*part, cu)
        assert torch.equal(torch.autograd.grad(out, part[i], dout)[0], want[1 + i])
    with torch.no_grad():
        assert torch.equal(ops.varlen_attention(*leaves, cu), want[0])
    # a gradient in another dtype, as autocast hands it on
    assert torch.equal(torch.ops.mi355_moe.varlen_attention_bwd(
        dout.float(), *(t.detach() for t in leaves), *torch.ops.mi355_moe.varlen_attention_fwd(
            *(t.detach() for t in leaves), cu, 64**-0.5, True), cu, 64**-0.5)[0], want[1])


@gpu
def test_a_derivative_of_the_backward_is_refused():
    (q, k, v), dout = inputs(40, 4, 2, 64, BF, seed=5)
    cu = torch.tensor([0, 40], dtype=torch.int32, device=DEV)
    weights = [torch.ones(64, dtype=BF, device=DEV, requires_grad=True) for _ in "qk"]
    positions, inv_freq = torch.arange(40, device=DEV), ops.rotary_frequencies(64, device=DEV)[0]
    runs = {
        "varlen_attention_bwd": (lambda: ops.varlen_attention(q, k, v, cu), dout, (q, k, v)),
        "qk_norm_rotary_bwd": (lambda: ops.qk_norm_rotary(q, k, *weights, positions, inv_freq, 1e-6)[0], torch.ones_like(q), (q, weights[0])),
    }
    for name, (run, grad, leaves) in runs.items():
        plain = torch.autograd.grad(run(), leaves, grad)
        assert not any(g.requires_grad for g in plain)
        kept = torch.autograd.grad(run(), leaves, grad, create_graph=True)  # by itself no error
        assert all(torch.equal(a, b) for a, b in zip(plain, kept))
        with pytest.raises(RuntimeError, match=f"{name} is not implemented"):
            torch.autograd.grad(kept[0], leaves[0], torch.ones_like(kept[0]))
    # a rotation is linear: its backward has one
    g = torch.ones_like(q, requires_grad=True)
    dq, = torch.autograd.grad(ops.rotary(q, k, positions, inv_freq)[0], q, g, create_graph=True)
    again, = torch.autograd.grad(dq, g, dout)
    assert torch.equal(again, ops.rotary(dout, k.detach(), positions, inv_freq)[0])


@gpu
@pytest.mark.parametrize("dtype", [BF, F32])
def test_the_attention_half_of_a_layer(dtype):
    """Norms and rotation, then attention, over packed sequences whose positions start over: against the same in fp64 with
    autograd.  The kernels' own bounds hold by themselves; here the chain's, by relative L2: bf16 rounds q and k, then p, out, ds and
    the gradients, each by at most 2^-8 of the value (rms half that), some eight roundings on the longest way; fp32 in the same way
    2^-24 times a few hundred additions."""
    H, G, D, eps = 8, 2, 64, 1e-6
    cu, T = bounds_of([100, 28, 60], 3)
    print(f"norm, rotation, attention {dtype}", flush=True)
    leaves, dout = inputs(T, H, G, D, dtype, seed=41, fused=True)
    gen = torch.Generator().manual_seed(42)
    w = [(1 + 0.1 * torch.randn(D, generator=gen)).to(dtype).to(DEV).requires_grad_() for _ in range(2)]
    inv_freq, factor = ops.rotary_frequencies(D, 1e4, scaling="yarn", factor=4.0, original_context=64, device=DEV)
    positions = torch.cat([torch.arange(b - a) for a, b in zip(cu, [*cu[1:], T])]).to(DEV)
    at = torch.tensor(cu, dtype=torch.int32, device=DEV)
    turned = kernel_registry.qk_norm_rotary(leaves[0], leaves[1], *w, positions, inv_freq, eps, attention_factor=factor)
    out = kernel_registry.varlen_attention(*turned, leaves[2], at)
    got = [out, *torch.autograd.grad(out, [*leaves, *w], dout)]

    exact = [t.detach().cpu().double().requires_grad_() for t in (*leaves, *w)]
    angle = positions.cpu().double()[:, None] * inv_freq.cpu().double()
    c, s = factor * angle.cos()[:, None], factor * angle.sin()[:, None]
    qk = []
    for x, wi in zip(exact[:2], exact[3:]):
        y = x / (x.pow(2).mean(-1, keepdim=True) + eps).sqrt() * wi
        u, v = y.chunk(2, -1)
        qk.append(torch.cat([u * c - v * s, v * c + u * s], -1))
    rows = []
    for a, b in zip(cu, cu[1:]):
        seen = torch.ones(b - a, b - a, dtype=torch.bool).tril()
        heads = [((qk[0][a:b, h] @ qk[1][a:b, h // 4].T * D**-0.5).masked_fill(~seen, -math.inf).softmax(1)
                  @ exact[2][a:b, h // 4]) for h in range(H)]
        rows.append(torch.stack(heads, 1))
    rows.append(torch.zeros(T - cu[-1], H, D, dtype=torch.float64))
    want = torch.cat(rows)
    want = [want, *torch.autograd.grad(want, exact, dout.cpu().double())]
    for x, y in zip(got, want):
        err = (x.detach().cpu().double() - y.detach()).norm() / y.detach().norm()
        assert err < (8 * 2.0**-8 if dtype == BF else 300 * 2.0**-24), err


# ---- without a GPU ---------------------------------------------------------------------------------


def test_operator_is_registered_for_the_gpu_only():
    assert kernel_registry.get_kernel("varlen_attention", "cuda") is kernel_registry.varlen_attention_mi355
    assert set(kernel_registry._KERNEL_REGISTRY["varlen_attention"]) == {"cuda"}
    q, cu = torch.ones(2, 1, 4), torch.tensor([0, 2], dtype=torch.int32)
    with pytest.raises(KeyError, match="not available"):
        kernel_registry.varlen_attention(q, q, q, cu)
    with pytest.raises(NotImplementedError, match="no torch-math backend"):
        kernel_registry.varlen_attention(q, q, q, cu, use_eager=True)
    with pytest.raises(RuntimeError, match="no CPU implementation"):
        ops.varlen_attention(q, q, q, cu)


def test_operator_refuses_what_does_not_fit_and_propagates_shapes():
    with FakeTensorMode():
        def t(*shape, dtype=BF):
            return torch.empty(shape, dtype=dtype, device="cuda")

        q, k, cu = t(10, 8, 64), t(10, 2, 64), t(3, dtype=torch.int32)

        def refused(error, message, **change):
            a = dict(q=q, k=k, v=k, cu_seqlens=cu, scale=None)
            a.update(change)
            with pytest.raises(error, match=message):
                ops.varlen_attention(**a)

        refused(ValueError, "agree in tokens and size", k=t(9, 2, 64))
        refused(ValueError, "agree in tokens and size", v=t(10, 2, 32))
        refused(ValueError, "agree in tokens and size", v=t(10, 1, 64))
        refused(ValueError, "agree in tokens and size", q=t(1, 10, 8, 64))
        refused(ValueError, "agree in tokens and size", q=t(10, 8, 32))
        refused(TypeError, "share a dtype", v=k.float())
        refused(TypeError, "float32 and bfloat16", q=q.half(), k=k.half(), v=k.half())
        refused(TypeError, "float32 and bfloat16", q=q.double(), k=k.double(), v=k.double())
        refused(ValueError, "no multiple", q=t(10, 5, 64))
        refused(ValueError, "no multiple", k=t(10, 0, 64), v=t(10, 0, 64))
        refused(ValueError, "1 to 256", q=t(10, 8, 257), k=t(10, 2, 257), v=t(10, 2, 257))
        refused(ValueError, "cu_seqlens", cu_seqlens=t(3, dtype=torch.int64))
        refused(ValueError, "cu_seqlens", cu_seqlens=t(0, dtype=torch.int32))
        refused(ValueError, "cu_seqlens", cu_seqlens=t(1, 3, dtype=torch.int32))
        for scale in (0.0, -1.0, math.inf, math.nan):
            refused(ValueError, "finite and positive", scale=scale)
        q.requires_grad_()
        out = ops.varlen_attention(q, k, k, cu)
        assert out.shape == q.shape and out.dtype == BF and out.requires_grad
        out, lse, rest = torch.ops.mi355_moe.varlen_attention_fwd(q.detach(), k, k, cu, 0.1, True)
        assert lse.shape == (8, 10) and lse.dtype == F32 and rest.shape == q.shape
        assert torch.ops.mi355_moe.varlen_attention_fwd(q.detach(), k, k, cu, 0.1, False)[2].shape == (0,)
        assert [x.shape for x in torch.ops.mi355_moe.varlen_attention_bwd(out, q.detach(), k, k, out, lse, rest, cu, 0.1)] == [
            q.shape, k.shape, k.shape]


def test_c_entry_points_refuse_before_any_launch():
    lib, p = _lib.load(), 0x1000  # (never dereferenced)

    def forward(T=4, H=4, G=2, D=64, dtype=1, scale=0.1, cu=p, sequences=1, k=p, k_token=None, workspace=p):
        return lib.mi355_varlen_attention_fwd(p, H * D, D, k, k_token or G * D, D, p, G * D, D, dtype, cu, sequences, scale, p, p, p,
                                              workspace, T, H, G, D, None)

    def backward(T=4, H=4, G=2, D=64, workspace=p):
        return lib.mi355_varlen_attention_bwd(p, p, H * D, D, p, G * D, D, p, G * D, D, p, p, p, 1, p, 1, 0.1, p, p, p, workspace, T, H,
                                              G, D, None)

    def text(rc, needle):
        assert rc == -1 and needle in lib.mi355_moe_last_error(), (rc, lib.mi355_moe_last_error())

    text(forward(dtype=2), b"neither fp32 nor bf16")
    text(forward(D=257), b"head size 257")
    text(forward(D=0), b"head size 0")
    text(forward(H=3), b"no multiple")
    text(forward(T=1 << 30), b"bad shape")
    text(forward(T=-1), b"bad shape")
    text(forward(sequences=-1), b"bad shape")
    text(forward(scale=0.0), b"finite and positive")
    text(forward(scale=math.nan), b"finite and positive")
    text(forward(cu=None), b"null pointer")
    text(forward(k=p + 2), b"whole pieces of 16 bytes")
    text(forward(k_token=2 * 64 + 4), b"whole pieces of 16 bytes")
    text(forward(k_token=1 << 22), b"whole pieces of 16 bytes")
    text(forward(D=65, workspace=None), b"workspace required")
    text(forward(workspace=p + 4), b"16-byte")
    text(forward(H=65536, G=1), b"no multiple")
    text(forward(H=32768, G=1, D=128), b"too many")
    text(forward(T=1 << 25, H=64, G=1, D=8, sequences=0), b"too many")
    assert forward(T=0) == 0
    text(backward(H=3), b"no multiple")
    text(backward(workspace=None), b"null pointer")
    text(backward(workspace=p + 8), b"16-byte")
    assert backward(T=0) == 0
    assert lib.mi355_varlen_attention_bwd_workspace_bytes(100, 4, 2, 64, 1) >= 4 * 4 * 100
    assert lib.mi355_varlen_attention_bwd_workspace_bytes(0, 4, 2, 64, 1) == 0
    assert lib.mi355_varlen_attention_fwd_workspace_bytes(100, 4, 2, 64, 1, 1) == 0
    assert lib.mi355_varlen_attention_fwd_workspace_bytes(100, 4, 2, 65, 1, 1) >= 2 * 100 * 8 * 72
