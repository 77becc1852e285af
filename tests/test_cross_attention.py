"""ops.cross_attention against softmax attention in 64 bits, and its refusals.

Tolerance, for standard normal q, k, v and scale D^-0.5: a rounding to bf16 is off by up to 2^-8 of the value, 0.0017 of it in the mean square
(uniform over the step, over a mantissa's range).  Three take part: of P (the weights of the sum and of the norm alike: 0.0017 of the result),
of q times the factor (logits of variance one are off by 0.0017, and so are the weights), of the result.  Together sqrt(3) 0.0017 = 0.0029 of
the 2-norm; fp32 sums add less than 1e-5.  Few values scatter around that: 2 x 0.0029 is asked of every member's output.
With one key the weight is one whatever P was rounded to: the result is v, to 2^-8 plus the reciprocal's 2^-22.
"""
import math

import pytest
import torch

REL = 2 * math.sqrt(3) * 0.0017


def oracle(q, k, v, lengths=None, mask=None, prefix=None, scale=None, exp2_domain=False):
    """[B, Nq, H, D] in 64 bits, one member and head at a time, over the keys that take part alone."""
    B, Nq, H, D = q.shape
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    for b in range(B):
        bk = b if k.shape[0] > 1 else 0
        n = k.shape[1]
        if lengths is not None:
            n = min(max(int(lengths[b if lengths.numel() > 1 else 0]), 0), n)
        keep = torch.arange(n, device=q.device)
        if mask is not None:
            keep = keep[mask[b if mask.shape[0] > 1 else 0, :n].bool()]
        for h in range(H):
            hk = h // (H // k.shape[2])
            kk, vv = k[bk, keep, hk].double(), v[bk, keep, hk].double()
            if prefix is not None:
                kk, vv = torch.cat([prefix[0][:, hk].double(), kk]), torch.cat([prefix[1][:, hk].double(), vv])
            if kk.shape[0]:
                s = q[b, :, h].double() @ kk.T * (math.log(2) if exp2_domain else D ** -0.5 if scale is None else scale)
                out[b, :, h] = torch.softmax(s, -1) @ vv
    return out


def check(got, want, rel=REL):
    assert got.dtype == torch.bfloat16 and got.is_contiguous() and got.shape == want.shape
    assert bool(torch.isfinite(got).all())
    for b in range(want.shape[0]):
        norm = float(want[b].norm())
        off = float((got[b].double() - want[b]).norm())
        assert off <= rel * norm, (b, off / max(norm, 1e-300))


def heads(shape, layout, g, device, dtype=torch.bfloat16):
    *lead, n, h, d = shape
    x = torch.randn(*lead, n, 2 * h if layout == "fused" else h, d, generator=g).to(dtype).to(device)
    if layout == "planes":
        return x.transpose(-3, -2).contiguous().transpose(-3, -2)
    return x[..., :h, :]


def inputs(B, Nq, H, Hk, D, Nk, cuda, seed, layout="rows", kv_batch=None):
    g = torch.Generator().manual_seed(seed)
    kv = (B if kv_batch is None else kv_batch, Nk, Hk, D)
    return (heads((B, Nq, H, D), layout, g, cuda), heads(kv, layout, g, cuda), heads(kv, layout, g, cuda)), g


@pytest.mark.gpu
@pytest.mark.parametrize("D", [32, 64, 128])
@pytest.mark.parametrize("B,Nq,H,Hk,Nk,layout", [
    (1, 1, 1, 1, 2, "rows"), (2, 3, 4, 2, 63, "planes"), (1, 31, 6, 1, 64, "fused"), (3, 33, 2, 2, 65, "rows"), (1, 128, 3, 3, 127, "planes"),
    (2, 129, 2, 1, 129, "fused"), (1, 300, 12, 3, 200, "rows"), (1, 1, 2, 2, 3000, "rows"), (2, 5, 8, 2, 1111, "planes"), (1, 130, 1, 1, 5000, "fused"),
    (1, 1024, 3, 3, 257, "planes"), (1, 2500, 16, 16, 77, "rows")])
def test_values(pkg, cuda, D, B, Nq, H, Hk, Nk, layout):
    (q, k, v), _ = inputs(B, Nq, H, Hk, D, Nk, cuda, 100 * D + Nq, layout)
    check(pkg.ops.cross_attention(q, k, v), oracle(q, k, v))


@pytest.mark.gpu
@pytest.mark.parametrize("D", [32, 64, 128])
@pytest.mark.parametrize("Nq", [1, 40, 200])
def test_one_key_is_its_value(pkg, cuda, D, Nq):
    (q, k, v), _ = inputs(2, Nq, 2, 1, D, 70, cuda, 5)
    lengths = torch.tensor([1, 70], dtype=torch.int32, device=cuda)
    mask = torch.ones(2, 70, dtype=torch.bool, device=cuda)
    mask[1] = False
    mask[1, 66] = True
    got = pkg.ops.cross_attention(q, k, v, lengths=lengths, key_mask=mask)
    for b, key in ((0, 0), (1, 66)):
        want = v[b, key, 0].double()
        assert bool(((got[b].double() - want).abs() <= (2.0 ** -8 + 2.0 ** -20) * want.abs()).all())


@pytest.mark.gpu
@pytest.mark.parametrize("D,Nq,Nk", [(64, 1, 300), (64, 37, 1500), (128, 1, 9000), (32, 260, 500), (128, 260, 130), (64, 3, 64)])
@pytest.mark.parametrize("mask_batch", [0, 1, 5])
def test_lengths_and_masks(pkg, cuda, D, Nq, Nk, mask_batch):
    """Members of different lengths, one of none and one of more than there are; what takes no part holds NaN and infinities."""
    B = 5
    (q, k, v), g = inputs(B, Nq, 4, 2, D, Nk, cuda, Nk + Nq, "fused")
    lengths = torch.tensor([Nk, 0, Nk + 1000, 1, Nk * 2 // 3], dtype=torch.int32)
    mask = None
    dead = torch.arange(Nk)[None] >= lengths[:, None]
    if mask_batch:
        mask = torch.rand(mask_batch, Nk, generator=g) < 0.5
        mask[:, :min(Nk, 64 if Nq > 30 else 7)] = False  # a first chunk, or the start of it, that nobody sees
        dead = dead | ~mask
        mask = mask.to(cuda)
        if mask_batch == 1:
            mask = mask.to(torch.uint8) * 200
    dead, lengths = dead.to(cuda), lengths.to(cuda)
    k[dead], v[dead] = math.nan, math.inf
    got = pkg.ops.cross_attention(q, k, v, lengths=lengths, key_mask=mask)
    check(got, oracle(q, k, v, lengths, mask))
    assert bool((got[1] == 0).all())


@pytest.mark.gpu
@pytest.mark.parametrize("Nq", [1, 200])
def test_nothing_to_attend_to(pkg, cuda, Nq):
    """No keys at all, a mask that leaves none, negative lengths: zeros."""
    (q, k, v), _ = inputs(2, Nq, 2, 2, 64, 100, cuda, 1)
    nan = torch.full_like(k, math.nan)
    none = torch.zeros(1, 100, dtype=torch.bool, device=cuda)
    for kw in (dict(key_mask=none), dict(lengths=torch.tensor([-5, 0], dtype=torch.int32, device=cuda))):
        assert bool((pkg.ops.cross_attention(q, nan, nan, **kw) == 0).all())
    assert bool((pkg.ops.cross_attention(q, k[:, :0], v[:, :0]) == 0).all())
    assert pkg.ops.cross_attention(q[:, :0], k, v).shape == (2, 0, 2, 64)


@pytest.mark.gpu
@pytest.mark.parametrize("D,B,Nq,H,Hk,Np,Nk", [(64, 5, 1, 4, 4, 700, 30), (128, 3, 9, 6, 2, 2000, 100), (32, 4, 2, 3, 1, 65, 1), (64, 2, 300, 2, 2, 129, 70),
                                               (128, 2, 130, 3, 3, 64, 64), (64, 7, 16, 8, 2, 5000, 500), (64, 1, 3, 2, 2, 900, 200), (128, 16, 1, 1, 1, 4096, 0),
                                               (64, 3, 128, 1, 1, 100, 0)])
@pytest.mark.parametrize("masked", [False, True])
def test_prefix(pkg, cuda, D, B, Nq, H, Hk, Np, Nk, masked):
    (q, k, v), g = inputs(B, Nq, H, Hk, D, Nk, cuda, Np + B, "planes")
    prefix = tuple(heads((Np, Hk, D), "fused" if Nq % 2 else "planes", g, cuda) for _ in range(2))
    lengths = mask = None
    if masked:
        lengths = torch.randint(0, Nk + 1, (B,), generator=g, dtype=torch.int32)
        lengths[-1] = 0
        mask = (torch.rand(B, Nk, generator=g) < 0.6).to(cuda)
        dead = (torch.arange(Nk)[None] >= lengths[:, None]).to(cuda) | ~mask
        k[dead], v[dead] = math.inf, math.nan
        lengths = lengths.to(cuda)
    got = pkg.ops.cross_attention(q, k, v, lengths=lengths, key_mask=mask, prefix=prefix)
    check(got, oracle(q, k, v, lengths, mask, prefix))
    # the same states as the first of each member's own: the same result up to the sums' order
    if not masked:
        rep = [torch.cat([p[None].expand(B, *p.shape), t], 1) for p, t in zip(prefix, (k, v))]
        check(pkg.ops.cross_attention(q, *rep), oracle(q, k, v, None, None, prefix))


@pytest.mark.gpu
@pytest.mark.parametrize("Nq,Nk", [(1, 4000), (9, 333), (128, 100), (500, 130)])
def test_states_of_batch_one_serve_every_member(pkg, cuda, Nq, Nk):
    (q, k, v), g = inputs(4, Nq, 4, 2, 64, Nk, cuda, Nk, kv_batch=1)
    mask = (torch.rand(1, Nk, generator=g) < 0.7).to(cuda)
    n = torch.tensor([Nk - 1], dtype=torch.int32, device=cuda)
    for kw in (dict(), dict(key_mask=mask), dict(lengths=n, key_mask=mask)):
        want = oracle(q, k, v, kw.get("lengths"), kw.get("key_mask"))
        check(pkg.ops.cross_attention(q, k, v, **kw), want)
        check(pkg.ops.cross_attention(q, k.expand(4, -1, -1, -1), v.expand(4, -1, -1, -1), **kw), want)
    lengths = torch.tensor([Nk, 5, 0, Nk // 2], dtype=torch.int32, device=cuda)  # one set of states, each member sees its start
    check(pkg.ops.cross_attention(q, k, v, lengths=lengths), oracle(q, k, v, lengths))


@pytest.mark.gpu
@pytest.mark.parametrize("D", [32, 64, 128])
@pytest.mark.parametrize("Nq,Nk", [(1, 2000), (40, 200), (200, 700)])
@pytest.mark.parametrize("size", [40.0, -1e4, 1e5])
def test_logits_beyond_the_range_of_exp2(pkg, cuda, D, Nq, Nk, size):
    """q as the kernel takes it (q_prescaled: nothing is rounded but P and the result); logits of hundreds, all of them far below zero
    (the weights then are those of the differences alone), and of 1e5 and more.  The fp32 sum of a logit is off by up to D / 2 x 2^-24 of the sum of its
    products' sizes: 2^-19 of 2e4 for "far below", 0.04, which a row's weights share but for the spread of the logits (a hundredth of their
    size); 1e5: weights of nought and one, where two keys come closest they differ by more than the sum's error in all but few rows."""
    (q, k, v), g = inputs(2, Nq, 2, 1, D, Nk, cuda, 17)
    if size < 0:  # logits about -1e4 (exp2 domain), spread of order one: q along one direction that all k share
        q = torch.randn(q.shape, generator=g).mul(0.1).to(cuda)
        q[..., 0] = -100.0
        k = torch.randn(k.shape, generator=g).mul(0.1).to(cuda)
        k[..., 0] = 100.0
        q, k = q.bfloat16(), k.bfloat16()
    else:
        q = (q.float() * (size / D ** 0.5)).bfloat16()
    got = pkg.ops.cross_attention(q, k, v, q_prescaled=True)
    want = oracle(q, k, v, exp2_domain=True)
    assert bool(torch.isfinite(got).all())
    rows = ((got.double() - want).norm(dim=-1) / want.norm(dim=-1)).flatten()
    assert float(rows.median()) <= REL
    if size < 1e5:
        check(got, want)


@pytest.mark.gpu
def test_one_loud_row_among_quiet_ones(pkg, cuda):
    """A row that leaves the range takes its workgroup through the running maximum: the others' results stay within the tolerance, and so
    do parts of a long key range of which one alone is loud."""
    (q, k, v), _ = inputs(1, 150, 1, 1, 64, 6000, cuda, 2)
    q[0, 77] *= 200
    k[0, 4500:4510] *= 30
    want = oracle(q, k, v)
    got = pkg.ops.cross_attention(q, k, v)
    rows = (got.double() - want)[0, :, 0].norm(dim=-1) / want[0, :, 0].norm(dim=-1)
    # (logits of a loud key have a deviation of 30, and an error of 0.0017 of that: 0.05 of a weight)
    assert float(rows.median()) <= 0.06 and bool(torch.isfinite(got).all())
    quiet = pkg.ops.cross_attention(q[:, :64], k[:, :4000], v[:, :4000])
    check(quiet, oracle(q[:, :64], k[:, :4000], v[:, :4000]))


@pytest.mark.gpu
@pytest.mark.parametrize("Nq,Nk", [(1, 100), (1, 8000), (200, 300)])
def test_nan_and_infinity_that_take_part(pkg, cuda, Nq, Nk):
    """NaN in a value reaches that element of every row of its head, and nothing else; in a query its row."""
    (q, k, v), _ = inputs(2, Nq, 2, 2, 64, Nk, cuda, 8)
    v[0, 60, 1, 5] = math.nan
    got = pkg.ops.cross_attention(q, k, v)
    bad = torch.zeros_like(got, dtype=torch.bool)
    bad[0, :, 1, 5] = True
    assert torch.equal(torch.isnan(got), bad)
    (q, k, v), _ = inputs(2, Nq, 2, 2, 64, Nk, cuda, 8)
    q[1, 0, 1, 7] = math.nan
    got = pkg.ops.cross_attention(q, k, v)
    assert bool(torch.isnan(got[1, 0, 1]).all())
    got[1, 0, 1] = 0
    assert bool(torch.isfinite(got).all())


@pytest.mark.gpu
@pytest.mark.parametrize("Nq,Nk", [(1, 3000), (16, 70), (140, 500)])
def test_scale_and_prescaled_queries(pkg, cuda, Nq, Nk):
    (q, k, v), _ = inputs(1, Nq, 2, 2, 64, Nk, cuda, 4)
    check(pkg.ops.cross_attention(q, k, v, scale=0.05), oracle(q, k, v, scale=0.05))
    pre, _ = pkg.ops.qk_norm_rope(q[0], normed=False, q_scale=0.125 * pkg.ops.LOG2E)
    check(pkg.ops.cross_attention(pre[None], k, v, q_prescaled=True), oracle(pre[None], k, v, exp2_domain=True), rel=2 * math.sqrt(2) * 0.0017)


@pytest.mark.gpu
def test_uniform_values_come_back(pkg, cuda):
    """The same value at every key is the result whatever the weights: P's rounding is in the sum and in the norm alike."""
    (q, k, _), _ = inputs(2, 70, 4, 2, 128, 4321, cuda, 6)
    v = torch.randn(2, 1, 2, 128, generator=torch.Generator().manual_seed(1)).bfloat16().to(cuda).expand(2, 4321, 2, 128)
    got = pkg.ops.cross_attention(q, k, v)
    want = v[:, :1].repeat_interleave(2, dim=2).double()
    assert bool(((got.double() - want).abs() <= (2.0 ** -8 + 2.0 ** -12) * want.abs()).all())


@pytest.mark.gpu
@pytest.mark.parametrize("Nq", [1, 200])
def test_offsets_beyond_32_bits(pkg, cuda, Nq):
    """Rows 2^23 - 8 elements apart: the last key lies 5 GB behind the first."""
    n, stride = 300, (1 << 23) - 8
    buf = torch.empty((n - 1) * stride + 128, dtype=torch.bfloat16, device=cuda)
    k = buf.as_strided((1, n, 1, 64), (0, stride, 64, 1))
    v = buf.as_strided((1, n, 1, 64), (0, stride, 64, 1), 64)
    g = torch.Generator().manual_seed(9)
    k.copy_(torch.randn(k.shape, generator=g))
    v.copy_(torch.randn(v.shape, generator=g))
    q = torch.randn(1, Nq, 2, 64, generator=g).bfloat16().to(cuda)
    check(pkg.ops.cross_attention(q, k, v), oracle(q, k, v))


@pytest.mark.gpu
@pytest.mark.parametrize("B,Nq,H,Hk,D,Nk,Np", [(1, 1, 2, 2, 64, 20000, 0), (3, 4, 4, 1, 128, 300, 3000), (1, 700, 3, 3, 64, 333, 0)])
def test_repeats_captures_and_streams(pkg, cuda, B, Nq, H, Hk, D, Nk, Np):
    """The same bits from call to call, from a captured graph replayed between eager calls of other sizes that use the same workspace, and
    on another stream; the output's neighbours stay as they were."""
    ops = pkg.ops
    (q, k, v), g = inputs(B, Nq, H, Hk, D, Nk, cuda, 12)
    prefix = tuple(heads((Np, Hk, D), "rows", g, cuda) for _ in range(2)) if Np else None
    want = ops.cross_attention(q, k, v, prefix=prefix).clone()
    check(want, oracle(q, k, v, None, None, prefix))
    buf = torch.full((want.numel() + 4096,), 3.0, dtype=torch.bfloat16, device=cuda)
    out = buf[2048:2048 + want.numel()].view(want.shape)
    assert ops.cross_attention(q, k, v, prefix=prefix, out=out) is out and torch.equal(out, want)
    assert bool((buf[:2048] == 3.0).all()) and bool((buf[2048 + want.numel():] == 3.0).all())
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        assert torch.equal(ops.cross_attention(q, k, v, prefix=prefix), want)
    side.synchronize()
    (q2, k2, v2), _ = inputs(2, 3, 4, 4, 128, 9000, cuda, 13)
    want2 = ops.cross_attention(q2, k2, v2).clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = ops.cross_attention(q, k, v, prefix=prefix)
    for _ in range(3):
        got.fill_(5.0)
        graph.replay()
        again = ops.cross_attention(q2, k2, v2)
        torch.cuda.synchronize()
        assert torch.equal(got, want) and torch.equal(again, want2)


@pytest.mark.gpu
def test_refusals_on_the_gpu(pkg, cuda):
    ops, z = pkg.ops, lambda *s, dtype=torch.bfloat16: torch.zeros(*s, dtype=dtype, device=cuda)  # noqa: E731
    q, kv = z(2, 5, 4, 64), z(2, 9, 2, 64)
    bad = [
        dict(q=z(2, 5, 4, 48), k=z(2, 9, 2, 48), v=z(2, 9, 2, 48)), dict(q=q.float()), dict(k=kv.float()), dict(k=z(2, 9, 3, 64), v=z(2, 9, 3, 64)),
        dict(k=z(3, 9, 2, 64), v=z(3, 9, 2, 64)), dict(v=z(2, 8, 2, 64)), dict(k=z(2, 9, 2, 32)), dict(q=z(5, 4, 64)), dict(k=z(2, 9, 2, 72)[..., 4:68]),
        dict(k=z(2, 9, 2, 68)[..., :64]), dict(q=z(2, 5, 64, 4).transpose(2, 3)), dict(lengths=z(2, dtype=torch.int64)), dict(lengths=z(3, dtype=torch.int32)),
        dict(lengths=z(4, dtype=torch.int32)[::2]), dict(key_mask=z(2, 8, dtype=torch.bool)), dict(key_mask=z(2, 9)), dict(key_mask=z(9, 2, dtype=torch.bool).T),
        dict(prefix=(z(3, 2, 64), z(4, 2, 64))), dict(prefix=(z(3, 4, 64), z(3, 4, 64))), dict(prefix=(z(3, 2, 64).float(), z(3, 2, 64))),
        dict(out=z(2, 5, 4, 32)), dict(out=z(2, 4, 5, 64).transpose(1, 2)), dict(out=q.float()), dict(scale=0.0), dict(scale=-1.0), dict(scale=math.nan),
        dict(q=q.cpu()), dict(k=kv.cpu()), dict(lengths=torch.zeros(2, dtype=torch.int32)),
        dict(k=z(2 * 9 * 64).as_strided((2, 9, 2, 64), (0, 1, 64, 1))),
    ]
    for kw in bad:
        with pytest.raises(RuntimeError):
            ops.cross_attention(**{"q": q, "k": kv, "v": kv, **kw})
    if torch.cuda.device_count() > 1:
        with pytest.raises(RuntimeError):
            ops.cross_attention(q.to("cuda:1"), kv.to("cuda:1"), kv.to("cuda:1"))


def test_refusals_without_a_gpu(pkg):
    L, at = pkg._lib, 1 << 20
    S = pkg.ops.CROSS_ATTENTION
    names = ("q k v pk pv out lengths mask B Nq heads D Bk Nk kv_heads Np n_lengths mask_batch qb qr qh qe kb kr kh ke vb vr vh ve pkr pkh pke pvr pvh pve "
             "ms pre scale").split()
    base = dict(zip(names, [at, at, at, 0, 0, at, 0, 0, 2, 5, 4, 64, 2, 9, 2, 0, 0, 0, 1280, 256, 64, 1, 1152, 128, 64, 1, 1152, 128, 64, 1, 0, 0, 0, 0, 0, 0, 0, 0,
                            0.125]))

    def call(ws=at, ws_bytes=1 << 40, **kw):
        a = S.pack(*{**base, **kw}.values())
        return L.lib().aeris_cross_attention_fwd(a, ws, ws_bytes, None)

    for kw in [dict(q=0), dict(k=0), dict(v=0), dict(out=0), dict(Np=4), dict(q=at + 8), dict(out=at + 2), dict(k=at + 4), dict(B=0), dict(Nq=0), dict(heads=0),
               dict(kv_heads=0), dict(heads=5), dict(Nk=-1), dict(Np=-1), dict(qr=4), dict(kb=-8), dict(vh=63), dict(qe=2), dict(ve=0),
               dict(Np=4, pk=at, pv=at, pkr=1, pke=1, pve=1), dict(Np=4, pk=at, pv=at), dict(Bk=3), dict(lengths=at, n_lengths=3), dict(lengths=at + 2, n_lengths=2),
               dict(mask=at, mask_batch=2, ms=-1), dict(mask=at, mask_batch=4), dict(scale=0.0), dict(scale=float("nan")), dict(scale=float("inf"))]:
        assert call(**kw) == L.EINVAL, kw
        assert "aeris_cross_attention_fwd" in L.last_error()
    for kw in [dict(D=48), dict(D=256), dict(kr=1 << 23), dict(vr=1 << 23), dict(Nq=1 << 30), dict(B=1 << 40, Bk=1), dict(Nk=1 << 31), dict(Np=1 << 31, pk=at, pv=at),
               dict(heads=1 << 17, kv_heads=1)]:
        assert call(**kw) == L.EUNSUPPORTED, kw
    assert L.lib().aeris_cross_attention_fwd(None, at, 0, None) == L.EINVAL
    # a long key range and few queries: parts of it are summed in a workspace, which has to be there
    long = dict(Nk=100000, kr=128, vr=128)
    need = L.lib().aeris_cross_attention_workspace_bytes(S.pack(*{**base, **long}.values()))
    assert need > 0
    for kw in (dict(ws=None), dict(ws_bytes=need - 1), dict(ws=at + 8)):
        assert call(**long, **kw) == L.EINVAL and "workspace" in L.last_error()
    assert L.lib().aeris_cross_attention_workspace_bytes(S.pack(*{**base, "B": 0}.values())) == 0
    assert S.size == 312
    t = torch.zeros(1, 1, 1, 64, dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match="GPU"):
        pkg.ops.cross_attention(t, t, t)


# (form, head size, rows) that the sizes below lead to: rows of a wave or workgroup, the keys whole or in parts
PLANS = [
    (1, 2, 1, 1, 32, 73, 0), (1, 2, 2, 1, 32, 74, 4588), (1, 1374, 3, 1, 32, 102, 1153), (1, 82, 2, 1, 32, 132, 14864), (1, 4508, 2, 1, 32, 252, 3293),
    (2, 175, 4, 4, 32, 105, 12953), (1, 1, 1, 1, 64, 74, 0), (1, 2, 1, 1, 64, 79, 4586), (1, 4130, 1, 1, 64, 119, 1308), (1, 105, 4, 4, 64, 92, 9906),
    (1, 4428, 2, 2, 64, 244, 1954), (1, 582, 3, 3, 64, 105, 15424), (1, 1, 1, 1, 128, 74, 0), (1, 1, 2, 1, 128, 75, 9702), (1, 4151, 1, 1, 128, 212, 0),
    (1, 296, 2, 1, 128, 159, 7899), (1, 8431, 1, 1, 128, 162, 868), (1, 604, 2, 1, 128, 75, 14617),  # the keys divided among waves: 16, 32, 64 rows
    (40, 68, 16, 8, 32, 197, 233), (40, 238, 8, 8, 64, 147, 0), (40, 600, 8, 8, 64, 147, 0), (40, 137, 8, 8, 128, 73, 0),         # keys that stay
    (1, 5482, 3, 3, 32, 150, 0), (1, 4134, 12, 4, 32, 90, 0), (1, 628, 4, 2, 32, 129, 13739), (1, 2735, 3, 1, 64, 104, 0), (5, 1637, 2, 1, 64, 161, 464),
    (5, 69, 9, 3, 64, 82, 12565), (5, 8613, 3, 1, 64, 108, 764), (1, 2065, 2, 1, 128, 85, 0), (2, 4129, 2, 1, 128, 82, 45), (2, 794, 1, 1, 128, 86, 15413),
    (64, 8300, 8, 8, 32, 330, 0),  # (65 row blocks for a wave)
    (64, 1, 4, 4, 32, 300, 0), (66, 3, 8, 4, 32, 90, 200), (24, 100, 6, 6, 64, 130, 100), (40, 30, 4, 1, 64, 500, 300), (9, 700, 2, 2, 64, 700, 0), (1, 1, 2, 1, 32, 70, 20000),
    (16, 1, 4, 4, 32, 995, 7255), (30, 65, 2, 2, 32, 124, 7057), (9, 65, 3, 3, 32, 527, 22632), (9, 2, 8, 8, 64, 1776, 3992), (30, 65, 1, 1, 64, 28, 14157),
    (16, 65, 2, 2, 64, 2023, 25529), (5, 1, 8, 8, 128, 1807, 3165), (16, 34, 1, 1, 128, 10, 22724), (30, 35, 3, 3, 128, 1494, 5251),
    (3, 72, 8, 8, 32, 22, 29633), (9, 65, 3, 3, 64, 30, 23859), (5, 73, 4, 4, 128, 60, 15456),  # the prefix once for all members
]


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["masked", "loud", "prescaled"])
@pytest.mark.parametrize("B,Nq,H,Hk,D,Nk,Np", PLANS)
def test_every_kernel(pkg, cuda, B, Nq, H, Hk, D, Nk, Np, kind):
    """Sizes for every kernel and every way to divide a call among workgroups; the queries at the ends of blocks and some between are checked."""
    (q, k, v), g = inputs(B, Nq, H, Hk, D, Nk, cuda, Nq + Nk + D, "rows" if Nq % 2 else "planes")
    prefix = tuple(heads((Np, Hk, D), "fused", g, cuda) for _ in range(2)) if Np else None
    lengths = mask = None
    kw = {}
    some = sorted({n for n in [0, 15, 16, 63, 64, 127, 128, 255, 256, Nq - 1] + torch.randint(0, Nq, (30,), generator=g).tolist() if n < Nq})
    if kind == "masked":
        lengths = torch.randint(0, Nk + 1, (B,), generator=g, dtype=torch.int32)
        lengths[0] = Nk - 3
        if B > 1:
            lengths[-1] = 0
        mask = torch.rand(B, Nk, generator=g) < 0.7
        dead = ((torch.arange(Nk)[None] >= lengths[:, None]) | ~mask).to(cuda)
        k[dead], v[dead] = math.nan, math.inf
        mask, lengths = mask.to(cuda), lengths.to(cuda)
    elif kind == "loud":  # a few queries whose logits need a maximum, among others that do not
        q[:, some[::5]] *= 40
    else:
        q.copy_((q.float() * (D ** -0.5 * pkg.ops.LOG2E)).bfloat16())
        kw = dict(q_prescaled=True)
    got = pkg.ops.cross_attention(q, k, v, lengths=lengths, key_mask=mask, prefix=prefix, **kw)
    assert bool(torch.isfinite(got).all())
    check(got[:, some].contiguous(), oracle(q[:, some], k, v, lengths, mask, prefix, exp2_domain=kind == "prescaled"))


@pytest.mark.gpu
@pytest.mark.parametrize("B,Nq,H,Hk,Nk", [(1, 1, 2, 1, 300), (1, 2, 1, 1, 4700), (1, 2735, 3, 1, 104), (40, 238, 8, 8, 147), (40, 600, 8, 8, 147)])
@pytest.mark.parametrize("level,power", [(6.0, 60), (-3.0, -100)])
def test_values_of_any_size(pkg, cuda, B, Nq, H, Hk, Nk, level, power):
    """Logits of 70 and -35 (base 2) all along with values of 2^60 and 2^-100: the result is the values' mean, weights times values do not fit fp32."""
    (q, k, v), _ = inputs(B, Nq, H, Hk, 64, Nk, cuda, 21)
    q.fill_(1.0)
    k.mul_(0.1).add_(level)
    v.mul_(2.0 ** power)
    some = sorted({n for n in (0, 1, 130, 777, Nq - 1) if n < Nq})
    check(pkg.ops.cross_attention(q, k, v)[:, some].contiguous(), oracle(q[:, some], k, v))


def test_grids_that_cannot_be_launched(pkg):
    L, at = pkg._lib, 1 << 20
    S = pkg.ops.CROSS_ATTENTION

    def call(B, Nq, heads, Nk, Np=0):
        kb = Nk * heads * 64
        a = S.pack(at, at, at, at, at, at, 0, 0, B, Nq, heads, 64, B, Nk, heads, Np, 0, 0, *([Nq * heads * 64, heads * 64, 64, 1] + [kb, heads * 64, 64, 1] * 2),
                   *([heads * 64, 64, 1] * 2), 0, 0, 0.125)
        return L.lib().aeris_cross_attention_fwd(a, at, 1 << 60, None)

    for args in [(1 << 24, 1, 1, 9), (1 << 29, 1, 1, 9), (1 << 20, 1, 16, 100), (1 << 26, 1, 1, 9, 100), (1 << 28, 1, 4, 1)]:
        # (the last has 2^28 * 4 = 2^30 rows, one more than the limit of rows lets through)
        assert call(*args) == L.EUNSUPPORTED and ("workgroups" in L.last_error() or "rows" in L.last_error()), args


@pytest.mark.gpu
def test_workspace_first_asked_for_under_a_capture(pkg, cuda):
    """The sums' buffer is made by the first call that needs it, which may be one that is captured; eager calls then go on with it."""
    ops = pkg.ops
    (q, k, v), _ = inputs(2, 3, 4, 4, 64, 9000, cuda, 14)
    want = oracle(q, k, v)
    check(ops.cross_attention(q[:, :, :, :], k[:, :100], v[:, :100]), oracle(q, k[:, :100], v[:, :100]))  # (one that needs none)
    for made in (ops._WORKSPACE, ops._WS_OWNER):
        for key in [key for key in made if key[0] == "cross_attention"]:
            ops._RETIRED.append(made.pop(key))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = ops.cross_attention(q, k, v)
    for _ in range(3):
        check(ops.cross_attention(q, k, v), want)
        got.fill_(5.0)
        graph.replay()
        torch.cuda.synchronize()
        check(got, want)


@pytest.mark.gpu
@pytest.mark.parametrize("Nq,D", [(1, 32), (40, 64), (3000, 64), (1500, 128), (60000, 32), (60000, 64)])
def test_masks_longer_than_a_workgroup_holds(pkg, cuda, Nq, D):
    """More chunks of keys than a workgroup has words for their mask: the keys are divided even where the rows alone fill the chip."""
    Nk = 70001
    (q, k, v), g = inputs(2, Nq, 2, 1, D, Nk, cuda, 31)
    mask = (torch.rand(2, Nk, generator=g) < 0.5).to(cuda)
    mask[1, :40000] = False
    lengths = torch.tensor([Nk, 65536], dtype=torch.int32, device=cuda)
    k[~mask], v[~mask] = math.nan, math.nan
    some = sorted({n for n in (0, 17, 63, 64, 128, 1000, Nq - 1) if n < Nq})
    got = pkg.ops.cross_attention(q, k, v, lengths=lengths, key_mask=mask)
    check(got[:, some].contiguous(), oracle(q[:, some], k, v, lengths, mask))


@pytest.mark.gpu
def test_one_set_of_states_with_a_mask_for_each_member(pkg, cuda):
    """Keys of batch 1 and lengths or masks of every member: members share what they read, not what they see."""
    (q, k, v), g = inputs(6, 130, 4, 2, 64, 700, cuda, 33, kv_batch=1)
    mask = (torch.rand(6, 700, generator=g) < 0.5).to(cuda)
    mask[2] = False
    lengths = torch.tensor([700, 0, 300, 1, 64, 65], dtype=torch.int32, device=cuda)
    for nq in (1, 7, 128, 130):
        for kw in (dict(key_mask=mask), dict(lengths=lengths), dict(lengths=lengths, key_mask=mask), dict(lengths=lengths, key_mask=mask[:1])):
            check(pkg.ops.cross_attention(q[:, :nq], k, v, **kw), oracle(q[:, :nq], k, v, kw.get("lengths"), kw.get("key_mask")))
