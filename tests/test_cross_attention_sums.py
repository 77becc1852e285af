"""ops.cross_attention where its sums are hard to form: keys that take no part beside weights that are small, values at the ends of
bf16's range, infinities, key masks of any length; every row held to a bound of its own.

Roundings.  To bf16 a value is off by half a step, 2^-8 of it at most and 0.0017 of it in the mean square (2^-8 / sqrt 3 times the mean
of 1 / m^2 over a mantissa m, 0.54, to the half).  The kernels round the weights (sum and norm have the rounded ones alike) and the result.
A row's error has then, per element d, the mean square 0.0017^2 (sum_i w_i^2 (v_id - o_d)^2 + o_d^2), w_i the weights of sum one.  `row_bound`
asks for four times the root of its sum over the row's elements (32 at least; a row of one weight: 2^-8 each, 2.3 times).
fp32 sums: an addition is off by 2^-24 of the sum at most; a lane adds Nk / 8 pairs of weights: Nk 2^-27.
"""
import math

import pytest
import torch

from test_cross_attention import PLANS, heads, inputs, oracle

STEP = 0.0017


def row_bound(q, k, v, want, keep, exp2_domain=False):
    """[n, H] for the rows q [n, H, D] of one member whose keys are k, v [Nk, Hk, D] where keep [Nk]."""
    bound = torch.zeros(q.shape[:2], dtype=torch.float64, device=q.device)
    H, D = q.shape[1:]
    for h in range(H):
        kk, vv = k[keep, h // (H // k.shape[1])].double(), v[keep, h // (H // k.shape[1])].double()
        w = torch.softmax(q[:, h].double() @ kk.T * (math.log(2) if exp2_domain else D ** -0.5), -1)
        o, w2 = want[:, h], w.square()
        spread = w2 @ vv.square() - 2 * (w2 @ vv) * o + w2.sum(-1, keepdim=True) * o.square()
        bound[:, h] = 4 * STEP * (spread + o.square()).sum(-1).clamp_min(0).sqrt() + (k.shape[0] * 2.0 ** -27 + 2.0 ** -12) * o.norm(dim=-1)
    return bound


def level_inputs(Nq, D, Nk, level, cuda, seed):
    """q (prescaled) and k whose logits, base 2, are all `level` within about 0.05."""
    g = torch.Generator().manual_seed(seed)
    small = (0.05 / math.sqrt(D)) ** 0.5
    q, k = torch.randn(1, Nq, 1, D, generator=g) * small, torch.randn(1, Nk, 1, D, generator=g) * small
    q[..., 0], k[..., 0] = -4.0, -level / 4.0
    return q.bfloat16().to(cuda), k.bfloat16().to(cuda), g


@pytest.mark.gpu
@pytest.mark.parametrize("D", [32, 64, 128])
@pytest.mark.parametrize("Nq,Nk", [(1, 300), (1, 8000), (1, 60000), (20, 8000), (60, 60000), (600, 8000), (9000, 300), (9000, 8000), (9000, 60000), (400000, 8000), (400000, 60000),
                                   (70000, 77), (70000, 250), (70000, 500)])
@pytest.mark.parametrize("masked", ["tenth", "most", "lanes"])
def test_small_weights_beside_keys_that_take_no_part(pkg, cuda, D, Nq, Nk, masked):
    """All logits far below zero, and one value at every key that takes part: the result is that value, whatever the weights, unless the
    sums of weights are off by half of bf16's smallest relative step, 1 / 510.  (fp32 allows for Nk 2^-27 + 2^-12 < 1 / 1400, and as much
    again in the sums of the products.)"""
    for level in (-7.0, -10.0, -12.5):
        q, k, g = level_inputs(Nq, D, Nk, level, cuda, Nq + Nk)
        if masked == "lanes":  # keys that always meet the same lanes
            mask = (torch.arange(Nk) % 16 >= 4)[None]
        else:
            mask = torch.rand(1, Nk, generator=g) >= (0.1 if masked == "tenth" else 0.6)
        v = (torch.randn(1, 1, 1, D, generator=g).bfloat16() + torch.zeros(1, Nk, 1, D, dtype=torch.bfloat16)).to(cuda)
        want = v[:, :1].expand(1, Nq, 1, D).clone()
        mask = mask.to(cuda)
        v[~mask], k[~mask] = math.nan, math.inf
        got = pkg.ops.cross_attention(q, k, v, key_mask=mask, q_prescaled=True)
        wrong = (got != want).flatten(1).sum().item()
        assert wrong == 0, (level, wrong, float((got.double() / want.double()).mean()))


@pytest.mark.gpu
@pytest.mark.parametrize("D", [32, 64, 128])
@pytest.mark.parametrize("Nq,Nk", [(1, 8000), (50, 3000), (600, 8000), (9000, 500), (70000, 77)])
@pytest.mark.parametrize("level", [-3.0, -10.0])
def test_rows_under_masks(pkg, cuda, D, Nq, Nk, level):
    """Values that differ from key to key, every row by its own bound."""
    q, k, g = level_inputs(Nq, D, Nk, level, cuda, Nk)
    v = torch.randn(1, Nk, 1, D, generator=g).bfloat16().to(cuda)
    mask = (torch.rand(1, Nk, generator=g) >= 0.4).to(cuda)
    v[~mask], k[~mask] = math.nan, math.inf
    some = sorted({n for n in [0, 15, 63, 64, 127, 128, Nq - 1] + torch.randint(0, Nq, (40,), generator=g).tolist() if n < Nq})
    got = pkg.ops.cross_attention(q, k, v, key_mask=mask, q_prescaled=True)[:, some]
    want = oracle(q[:, some], k, v, mask=mask, exp2_domain=True)
    off = (got.double() - want)[0].norm(dim=-1)
    assert bool((off <= row_bound(q[0, some], k[0], v[0], want[0], mask[0], True)).all())


# sizes for every kernel: few rows, whole and in parts; many rows; keys that stay; a prefix in one and apart
FORMS = PLANS + [(1, 1, 2, 1, 64, 300, 0), (1, 1, 2, 2, 64, 20000, 0), (1, 3000, 8, 8, 64, 1000, 0), (2, 16000, 4, 4, 64, 700, 0)]


def form_inputs(B, Nq, H, Hk, D, Nk, Np, cuda, seed):
    (q, k, v), g = inputs(B, Nq, H, Hk, D, Nk, cuda, seed)
    prefix = tuple(heads((Np, Hk, D), "rows", g, cuda) for _ in range(2)) if Np else None
    some = sorted({n for n in [0, 16, 63, 130, Nq - 1] + torch.randint(0, Nq, (8,), generator=g).tolist() if n < Nq})
    return q, k, v, prefix, some, g


def whole_bound(q, k, v, prefix, want):
    """`row_bound` for every member, all keys taking part."""
    def of(b):
        kk, vv = (t[b] if prefix is None else torch.cat([p, t[b]]) for p, t in zip(prefix or (None, None), (k, v)))
        return row_bound(q[b], kk, vv, want[b], torch.ones(len(kk), dtype=torch.bool, device=q.device))
    return torch.stack([of(b) for b in range(len(q))])


@pytest.mark.gpu
@pytest.mark.parametrize("B,Nq,H,Hk,D,Nk,Np", FORMS)
@pytest.mark.parametrize("power", [70, 120])
def test_large_finite_values(pkg, cuda, B, Nq, H, Hk, D, Nk, Np, power):
    """The weighted mean of values is no larger than the largest, whatever the weights sum up to: 2^120 and the largest that bf16 holds."""
    q, k, v, prefix, some, _ = form_inputs(B, Nq, H, Hk, D, Nk, Np, cuda, 40 + Nq)
    for t in [v] + ([prefix[1]] if Np else []):
        t.mul_(2.0 ** power)
    got = pkg.ops.cross_attention(q, k, v, prefix=prefix)
    assert bool(torch.isfinite(got).all())
    want = oracle(q[:, some], k, v, prefix=prefix)
    assert bool(((got[:, some].double() - want).norm(dim=-1) <= whole_bound(q[:, some], k, v, prefix, want)).all())
    # one value at every key, the largest of either sign: it comes back
    most = torch.finfo(torch.bfloat16).max
    for t in [v] + ([prefix[1]] if Np else []):
        t.fill_(most)
        t[..., 1::2] = -most
    got = pkg.ops.cross_attention(q, k, v, prefix=prefix)
    assert bool((got[..., 0::2] == most).all()) and bool((got[..., 1::2] == -most).all())


@pytest.mark.gpu
@pytest.mark.parametrize("B,Nq,H,Hk,D,Nk,Np", FORMS)
def test_infinite_values_that_take_part(pkg, cuda, B, Nq, H, Hk, D, Nk, Np):
    """An infinity in a value is that element of every row of its heads in the result, for few rows and for many; infinities of both signs
    leave no number; the other elements are as without them.  (Logits: standard normal, no weight is below 2^-40 of the largest.)"""
    q, k, v, prefix, some, g = form_inputs(B, Nq, H, Hk, D, Nk, Np, cuda, 60 + Nq)
    key, b, hk, group = Nk // 2, B - 1, Hk - 1, H // Hk
    rows = slice(hk * group, (hk + 1) * group)
    want = oracle(q[:, some], k, v, prefix=prefix)
    bound = whole_bound(q[:, some], k, v, prefix, want)
    v[b, key, hk, 3] = math.inf
    v[b, key, hk, 9] = -math.inf
    v[b, key, hk, 12], v[b, (key + 20) % Nk, hk, 12] = math.inf, -math.inf
    if Np:
        prefix[1][Np - 2, hk, 20] = -math.inf
    got = pkg.ops.cross_attention(q, k, v, prefix=prefix)
    assert bool((got[b, :, rows, 3] == math.inf).all()) and bool((got[b, :, rows, 9] == -math.inf).all())
    both = got[b, :, rows, 12]  # (of ten keys the one twenty further on is the same, and holds the second alone)
    assert bool((both.isnan() if 20 % Nk else both == -math.inf).all())
    special = torch.zeros(got.shape, dtype=torch.bool, device=cuda)
    special[b, :, rows, 3] = special[b, :, rows, 9] = special[b, :, rows, 12] = True
    if Np:
        assert bool((got[:, :, rows, 20] == -math.inf).all())
        special[:, :, rows, 20] = True
    assert torch.equal(special, ~torch.isfinite(got))
    got, want = (torch.where(special[:, some], 0.0, t.double()) for t in (got[:, some], want))
    assert bool(((got - want).norm(dim=-1) <= bound).all())


def sizes(pkg, B, Nq, H, Hk, D, Nk, Np=0, masked=False, lengths=False, prescaled=False):
    """What the C call is told of a call's sizes, with addresses that are never read."""
    at, row, krow = 1 << 20, H * D, Hk * D
    return pkg.ops.CROSS_ATTENTION.pack(at, at, at, at if Np else 0, at if Np else 0, at, at if lengths else 0, at if masked else 0, B, Nq, H, D, B, Nk, Hk, Np,
                                        B if lengths else 0, B if masked else 0, Nq * row, row, D, 1, Nk * krow, krow, D, 1, Nk * krow, krow, D, 1,
                                        krow, D, 1, krow, D, 1, Nk if masked else 0, prescaled, D ** -0.5)


@pytest.mark.parametrize("B,Nq,H,Hk,D,Nk,Np", [(1, 1036800, 16, 16, 64, 129600, 0), (1, 1036800, 16, 16, 64, 1036800, 0), (4, 64800, 8, 8, 128, 500, 259200),
                                               (1, 1036800, 24, 24, 64, 1100000, 0), (2, 3, 4, 4, 64, 900000, 0), (1, 300, 8, 2, 32, 70000, 70000)])
def test_a_mask_needs_no_workspace_of_its_own(pkg, B, Nq, H, Hk, D, Nk, Np):
    need = pkg._lib.lib().aeris_cross_attention_workspace_bytes
    plain, masked = (need(sizes(pkg, B, Nq, H, Hk, D, Nk, Np, masked=m)) for m in (False, True))
    assert masked == plain
    if Nq > 1000:
        assert plain == 0


@pytest.mark.gpu
@pytest.mark.parametrize("B,Nq,H,Hk,D,Nk,Np", [(1, 200000, 1, 1, 32, 66000, 0), (1, 200000, 1, 1, 64, 66000, 0), (1, 200000, 1, 1, 128, 66000, 0), (2, 3, 4, 4, 64, 300000, 0),
                                               (2, 64800, 2, 1, 64, 300, 70001), (3, 40, 2, 2, 128, 70001, 129), (8, 1, 1, 1, 32, 65, 70000)])
def test_masks_of_any_length(pkg, cuda, B, Nq, H, Hk, D, Nk, Np):
    """More than 65 536 keys under a mask, with rows that fill the chip and with few; masks in rows that start anywhere; whole chunks, and
    all of a member's keys, masked; a prefix, which no mask covers, ahead of them."""
    q, k, v, prefix, some, g = form_inputs(B, Nq, H, Hk, D, Nk, Np, cuda, 80 + Nq)
    mask = torch.rand(B, Nk, generator=g) < 0.5
    mask[0, Nk // 3:Nk // 3 + min(Nk // 2, 5000)] = False
    if B > 1:
        mask[-1] = False
    buf = torch.ones(B * (Nk + 13) + 7, dtype=torch.bool)
    buf[7:].view(B, Nk + 13)[:, :Nk] = mask
    k[~mask.to(cuda)], v[~mask.to(cuda)] = math.nan, math.inf
    mask = buf.to(cuda)[7:].view(B, Nk + 13)[:, :Nk]
    some = some[:6]
    got = pkg.ops.cross_attention(q, k, v, key_mask=mask, prefix=prefix)[:, some]
    want = oracle(q[:, some], k, v, mask=mask, prefix=prefix)
    keep = torch.cat([torch.ones(B, Np, dtype=torch.bool, device=cuda), mask], 1)
    for b in range(B):
        kk, vv = (t[b] if prefix is None else torch.cat([p, t[b]]) for p, t in zip(prefix or (None, None), (k, v)))
        off = (got[b].double() - want[b]).norm(dim=-1)
        assert bool((off <= row_bound(q[b, some], kk, vv, want[b], keep[b])).all()), b


@pytest.mark.gpu
@pytest.mark.parametrize("D", [32, 64, 128])
@pytest.mark.parametrize("B,Nq,H,Hk,Nk,layout", [
    (1, 1, 1, 1, 2, "rows"), (2, 3, 4, 2, 63, "planes"), (3, 33, 2, 2, 65, "rows"), (1, 128, 3, 3, 127, "planes"), (2, 129, 2, 1, 129, "fused"),
    (1, 300, 12, 3, 200, "rows"), (2, 5, 8, 2, 1111, "planes"), (1, 130, 1, 1, 5000, "fused"), (1, 1025, 3, 3, 257, "planes"), (1, 2500, 16, 16, 77, "rows"),
    (2, 16001, 4, 4, 77, "planes"), (1, 4000, 8, 8, 700, "rows")])
def test_every_row(pkg, cuda, D, B, Nq, H, Hk, Nk, layout):
    """No row of a call hides behind the others' norm."""
    (q, k, v), _ = inputs(B, Nq, H, Hk, D, Nk, cuda, 200 * D + Nq, layout)
    got, want = pkg.ops.cross_attention(q, k, v), oracle(q, k, v)
    assert bool(((got.double() - want).norm(dim=-1) <= whole_bound(q, k, v, None, want)).all())


@pytest.mark.gpu
@pytest.mark.parametrize("D", [32, 64, 128])
@pytest.mark.parametrize("Nq", [9, 40, 150, 3000])
def test_every_row_of_a_call_with_a_loud_one(pkg, cuda, D, Nq):
    """A row, and ten keys, far beyond the range of exp2: that row and all others, each by its own bound.  The fp32 sum of a logit is off by D 2^-24 of the
    sum of its products' sizes at most, the scale by 2^-23 of the logit: e_i.  Weights w_i exp(d_i) with |d_i| <= e_i give a row that is off by
    |sum_i w_i (exp(d_i) - 1) (v_i - o)| / sum_i w_i exp(d_i) <= exp(max e) sum_i w_i (exp(e_i) - 1) |v_i - o|."""
    (q, k, v), _ = inputs(1, Nq, 1, 1, D, 6000, cuda, 2)
    q[0, Nq // 2] *= 200
    k[0, 4500:4510] *= 30
    got, want = pkg.ops.cross_attention(q, k, v), oracle(q, k, v)
    bound = whole_bound(q, k, v, None, want)[0, :, 0]
    qq, kk, vv, o = q[0, :, 0].double(), k[0, :, 0].double(), v[0, :, 0].double(), want[0, :, 0]
    s = qq @ kk.T * D ** -0.5
    e = qq.abs() @ kk.abs().T * D ** -0.5 * D * 2.0 ** -24 + s.abs() * 2.0 ** -23
    w = torch.softmax(s, -1)
    bound = bound + e.amax(-1).exp() * (w * e.expm1() * torch.cdist(o, vv)).sum(-1)
    assert bool(((got[0, :, 0].double() - o).norm(dim=-1) <= bound).all())


@pytest.mark.gpu
def test_graphs_on_streams_of_their_own(pkg, cuda):
    """Two captured calls whose sums go through scratch memory, replayed beside each other and beside eager calls of a third stream."""
    ops, calls = pkg.ops, []
    for i, (B, Nq, H, D, Nk) in enumerate([(2, 3, 4, 64, 90000), (1, 9, 4, 128, 60000), (4, 1, 8, 64, 70000)]):
        (q, k, v), _ = inputs(B, Nq, H, H, D, Nk, cuda, 90 + i)
        assert pkg._lib.lib().aeris_cross_attention_workspace_bytes(sizes(pkg, B, Nq, H, H, D, Nk)) > 0
        calls.append(((q, k, v), ops.cross_attention(q, k, v).clone()))
    torch.cuda.synchronize()
    graphs, outs, streams = [], [], [torch.cuda.Stream() for _ in range(3)]
    for (args, _), stream in zip(calls[:2], streams):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            outs.append(ops.cross_attention(*args))
        graphs.append(graph)
    for _ in range(4):
        for out in outs:
            out.fill_(5.0)
        torch.cuda.synchronize()
        eager = []
        for _ in range(5):
            for graph, stream in zip(graphs, streams):
                with torch.cuda.stream(stream):
                    graph.replay()
            with torch.cuda.stream(streams[2]):
                eager.append(ops.cross_attention(*calls[2][0]))
        torch.cuda.synchronize()
        assert all(torch.equal(out, want) for out, (_, want) in zip(outs, calls)) and all(torch.equal(t, calls[2][1]) for t in eager)


def test_a_capture_has_scratch_memory_of_its_own(pkg, monkeypatch):
    """... and leaves the eager calls' as it is."""
    ops, cpu = pkg.ops, torch.device("cpu")
    shared = torch.empty(4096, dtype=torch.uint8)
    monkeypatch.setattr(ops, "_WORKSPACE", {("cross_attention", cpu, torch.uint8): shared})
    monkeypatch.setattr(ops, "_WS_OWNER", {("cross_attention", cpu, torch.uint8): (7, None)})
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda index: 7, raising=False)
    monkeypatch.setattr(torch._C, "_cuda_isCurrentStreamCapturing", lambda: False, raising=False)
    assert ops._workspace_ptr("cross_attention", 100, cpu) == shared.data_ptr()
    monkeypatch.setattr(torch._C, "_cuda_isCurrentStreamCapturing", lambda: True, raising=False)
    assert ops._workspace_ptr("cross_attention", 100, cpu) != shared.data_ptr()
    assert ops._WORKSPACE == {("cross_attention", cpu, torch.uint8): shared}
