"""ops.qk_norm_rope against the formula in 64 bits, and its refusals.

Tolerance: an output is rounded once, by at most half a step (bf16 2^-8 of the value, f32 2^-24).  Ahead of that everything is fp32: the mean of
D <= 128 squares (partial sums of 8, then up to 4 levels: 12 roundings at most), the reciprocal root (2 units), the products with
factor, gain, cosine / sine and scale and one sum: 20 roundings of 2^-24 at most, of values up to the pair's length - below 2^-19 of it.
"""
import math

import pytest
import torch


def oracle(x, gain, table, positions, interleaved, normed, eps, scale):
    """-> (y, length of each element's pair) in 64 bits; x [T, H, D]."""
    y = x.double()
    if normed:
        y = y / (y.square().mean(-1, keepdim=True) + eps).sqrt()
    if gain is not None:
        y = y * gain.double()
    size = y.abs()
    if table is not None:
        T, R, P = x.shape[0], table.shape[1], table.shape[0]
        t = torch.arange(T, device=x.device)
        pos = positions.long()[t % positions.numel()] if positions is not None else t % P
        known = (pos >= 0) & (pos < P)
        row = table.double()[torch.where(known, pos, 0)][:, None]
        j = torch.arange(R // 2, device=x.device)
        ja, jb = (2 * j, 2 * j + 1) if interleaved else (j, j + R // 2)
        a, b, c, s = y[..., ja], y[..., jb], row[..., :R // 2], row[..., R // 2:]
        z = y.clone()
        z[..., ja], z[..., jb] = a * c - b * s, a * s + b * c
        y = torch.where(known[:, None, None], z, y)
        size = size.clone()
        size[..., ja] = size[..., jb] = torch.hypot(a, b)
    return y * scale, size * abs(scale)


def check(got, x, gain, table=None, positions=None, interleaved=False, normed=True, eps=1e-6, scale=1.0):
    want, size = oracle(x, gain, table, positions, interleaved, normed, eps, scale)
    half = torch.finfo(got.dtype).eps / 2
    off = (got.double() - want).abs()
    bound = half * want.abs() + 2.0 ** -19 * (1 + half) * size
    assert bool((off <= bound).all()), float((off / bound.clamp_min(1e-300)).max())


def table_for(P, R, device, g):
    a = torch.rand(P, R // 2, generator=g, dtype=torch.float64).mul(2 * math.pi)
    return torch.cat([a.cos(), a.sin()], 1).float().to(device)


@pytest.mark.gpu
@pytest.mark.parametrize("D,R,interleaved", [(32, 32, False), (32, 16, True), (64, 64, False), (64, 64, True), (64, 48, False), (64, 0, False),
                                             (128, 128, False), (128, 128, True), (128, 64, False), (128, 16, False), (128, 112, True)])
@pytest.mark.parametrize("T,H,Hk,layout", [(1, 1, 1, "rows"), (5, 3, 0, "rows"), (67, 5, 2, "fused"), (8200, 4, 4, "planes"), (3001, 7, 1, "planes")])
def test_values(pkg, cuda, D, R, interleaved, T, H, Hk, layout):
    g = torch.Generator().manual_seed(1000 * D + 10 * T + R)
    parts = H + Hk + (1 if layout == "fused" else 0)
    x = torch.randn(parts, T, D, generator=g).mul(torch.rand(parts, 1, 1, generator=g) * 3 + 0.1).bfloat16().to(cuda)
    if layout == "planes":
        q, k = x[:H].permute(1, 0, 2), x[H:H + Hk].permute(1, 0, 2)
    else:
        rows = x.permute(1, 0, 2).contiguous()
        q, k = rows[:, :H], rows[:, H:H + Hk]
    table = table_for(23, R, cuda, g) if R else None
    positions = torch.randint(0, 23, (max(1, T // 2),), generator=g, dtype=torch.int32).to(cuda) if R and T % 2 else None
    per_head, gain_dtype = T % 3 == 0, torch.float32 if H % 2 else torch.bfloat16
    q_gain = (1 + 0.3 * torch.randn((H, D) if per_head else (D,), generator=g)).to(gain_dtype).to(cuda)
    k_gain = (1 + 0.3 * torch.randn(D, generator=g)).to(gain_dtype).to(cuda) if Hk else None
    yq, yk = pkg.ops.qk_norm_rope(q, k if Hk else None, q_gain, k_gain, rotation=table, positions=positions, interleaved=interleaved, q_scale=0.18)
    assert yq.shape == q.shape and (layout != "planes" or yq.stride() == q.stride())
    check(yq, q, q_gain, table, positions, interleaved, scale=0.18)
    if Hk:
        check(yk, k, k_gain, table, positions, interleaved)
    else:
        assert yk is None


@pytest.mark.gpu
@pytest.mark.parametrize("x_dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("y_dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("normed", [True, False])
def test_types_and_given_outputs(pkg, cuda, x_dtype, y_dtype, normed):
    """Outputs in buffers of the caller's, whose other parts stay as they were; no gain; the norm left out."""
    g = torch.Generator().manual_seed(7)
    q, k = (torch.randn(333, 3, 64, generator=g).to(x_dtype).to(cuda) for _ in range(2))
    table = table_for(50, 64, cuda, g)
    buf = torch.full((335, 8, 64), 7.0, dtype=y_dtype, device=cuda)
    yq, yk = pkg.ops.qk_norm_rope(q, k, rotation=table, normed=normed, q_out=buf[1:334, 1:4], k_out=buf[1:334, 4:7])
    assert yq.data_ptr() == buf[1:, 1:].data_ptr() and yk.dtype == y_dtype
    check(yq, q, None, table, normed=normed)
    check(yk, k, None, table, normed=normed)
    untouched = torch.ones_like(buf, dtype=torch.bool)
    untouched[1:334, 1:7] = False
    assert bool((buf[untouched] == 7.0).all())


@pytest.mark.gpu
def test_in_place_on_head_planes(pkg, cuda):
    g = torch.Generator().manual_seed(3)
    planes = torch.randn(3 * 4, 500, 64, generator=g).bfloat16().to(cuda)
    before = planes.clone()
    q, k = planes[:4].permute(1, 0, 2), planes[4:8].permute(1, 0, 2)
    table, gain = table_for(36, 64, cuda, g), torch.ones(64, device=cuda)
    pkg.ops.qk_norm_rope(q, k, gain, gain, rotation=table, q_out=q, k_out=k)
    check(q, before[:4].permute(1, 0, 2), gain, table)
    check(k, before[4:8].permute(1, 0, 2), gain, table)
    assert torch.equal(planes[8:], before[8:])


@pytest.mark.gpu
@pytest.mark.parametrize("interleaved", [False, True])
def test_positions_outside_the_table_are_not_rotated(pkg, cuda, interleaved):
    g = torch.Generator().manual_seed(4)
    q = torch.randn(64, 2, 128, generator=g).bfloat16().to(cuda)
    table = table_for(10, 64, cuda, g)
    positions = torch.randint(0, 10, (64,), generator=g, dtype=torch.int32)
    positions[::3], positions[1], positions[2] = -1, 10, 2 ** 31 - 1
    positions = positions.to(cuda)
    y, _ = pkg.ops.qk_norm_rope(q, rotation=table, positions=positions, interleaved=interleaved)
    check(y, q, None, table, positions, interleaved)
    assert torch.equal(y[::3], pkg.ops.qk_norm_rope(q)[0][::3])


@pytest.mark.gpu
@pytest.mark.parametrize("interleaved", [False, True])
def test_infinity_stays_in_its_pair(pkg, cuda, interleaved):
    """Without the norm an infinite element reaches its own pair, and where nothing is rotated itself alone."""
    q = torch.ones(4, 1, 64, device=cuda)
    q[0, 0, 3], q[1, 0, 40], q[2, 0, 63] = math.inf, math.inf, math.inf
    table = torch.cat([torch.full((4, 16), 0.6), torch.full((4, 16), 0.8)], 1).to(cuda)
    y, _ = pkg.ops.qk_norm_rope(q, rotation=table, interleaved=interleaved, normed=False, out_dtype=torch.float32)
    pair = {0: {3, 2} if interleaved else {3, 19}, 1: {40}, 2: {63}, 3: set()}
    for t, where in pair.items():
        assert {int(j) for j in torch.nonzero(~torch.isfinite(y[t, 0]))[:, 0]} == where


@pytest.mark.gpu
def test_rows_of_zeros_and_extreme_sizes(pkg, cuda):
    q = torch.zeros(4, 2, 32, device=cuda, dtype=torch.bfloat16)
    q[1] = 1e-20
    q[2] = 1e18
    y, _ = pkg.ops.qk_norm_rope(q, eps=1e-6)
    check(y, q, None)
    assert bool((y[0] == 0).all())


@pytest.mark.gpu
def test_strides_beyond_32_bits_of_elements(pkg, cuda):
    """Tokens far apart: the last one lies past 2^32 bytes."""
    T, stride = 40, (1 << 26) + 64
    buf = torch.empty((T - 1) * stride + 256, dtype=torch.bfloat16, device=cuda)
    q = buf.as_strided((T, 2, 128), (stride, 128, 1))
    q.copy_(torch.randn(T, 2, 128, generator=torch.Generator().manual_seed(1)).bfloat16())
    y, _ = pkg.ops.qk_norm_rope(q, q_out=torch.empty(T, 2, 128, dtype=torch.bfloat16, device=cuda))
    check(y, q, None)


@pytest.mark.gpu
def test_captured_and_replayed_and_on_another_stream(pkg, cuda):
    g = torch.Generator().manual_seed(5)
    q, k = (torch.randn(2000, 4, 64, generator=g).bfloat16().to(cuda) for _ in range(2))
    table = table_for(64, 64, cuda, g)
    want = [t.clone() for t in pkg.ops.qk_norm_rope(q, k, rotation=table)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = pkg.ops.qk_norm_rope(q, k, rotation=table)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = pkg.ops.qk_norm_rope(q, k, rotation=table)
    for _ in range(3):
        for t in out:
            t.fill_(9.0)
        graph.replay()
        torch.cuda.synchronize()
        eager = pkg.ops.qk_norm_rope(q, k, rotation=table)
        assert all(torch.equal(a, b) and torch.equal(a, c) for a, b, c in zip(out, want, eager))


@pytest.mark.gpu
def test_refusals_on_the_gpu(pkg, cuda):
    ops, z = pkg.ops, lambda *s, dtype=torch.bfloat16: torch.zeros(*s, dtype=dtype, device=cuda)  # noqa: E731
    q, table = z(8, 2, 64), z(4, 64, dtype=torch.float32)
    bad = [
        dict(q=z(8, 2, 48)), dict(q=z(8, 2, 64, dtype=torch.float16)), dict(q=z(2, 64)), dict(q=z(8, 64, 2).transpose(1, 2)),
        dict(q=z(8, 2, 68)[..., 2:66]), dict(q=z(8, 2, 66)[..., :64]), dict(k=z(7, 2, 64)), dict(k=z(8, 2, 64, dtype=torch.float32)),
        dict(q_gain=z(32)), dict(q_gain=z(3, 64)), dict(k_gain=z(64)), dict(q_gain=z(64, dtype=torch.float16)),
        dict(rotation=z(4, 64)), dict(rotation=z(4, 40, dtype=torch.float32)), dict(rotation=z(4, 128, dtype=torch.float32)),
        dict(rotation=z(0, 64, dtype=torch.float32)), dict(positions=z(8, dtype=torch.int32)),
        dict(rotation=table, positions=z(8, dtype=torch.int64)), dict(rotation=table, positions=z(0, dtype=torch.int32)),
        dict(rotation=table, positions=z(16, dtype=torch.int32)[::2]), dict(q_out=z(8, 2, 32)), dict(q_out=z(1, 2, 64).expand(8, 2, 64)),
        dict(rotation=table.cpu()), dict(q=q.cpu()), dict(eps=-1.0), dict(eps=math.nan),
        dict(k=q, q_gain=z(64), k_gain=z(64, dtype=torch.float32)), dict(k=z(8, 0, 64)),
    ]
    for kw in bad:
        with pytest.raises(RuntimeError):
            ops.qk_norm_rope(**{"q": q, **kw})
    assert ops.qk_norm_rope(z(0, 2, 64))[0].shape == (0, 2, 64)


def test_refusals_without_a_gpu(pkg):
    """The entry point looks at everything on the host before anything touches a GPU."""
    L, at = pkg._lib, 1 << 20
    S = pkg.ops.QK_NORM_ROPE

    def call(part=(), n=1, tokens=4, D=64, xd=L.BF16, yd=L.BF16, gd=L.F32, eps=1e-6, rot=at, rows=4, R=64, pos=0, n_pos=0):
        f = dict(x=at, y=at, gain=0, heads=2, xt=128, xh=64, xe=1, yt=128, yh=64, ye=1, gh=0, scale=1.0)
        f.update(part)
        a = S.pack(*f.values(), *f.values(), rot, pos, tokens, D, xd, yd, gd, 1, 0, rows, R, n_pos, n, eps)
        return L.lib().aeris_qk_norm_rope_fwd(a, None)

    for kw in [dict(part={"x": 0}), dict(part={"y": 0}), dict(part={"x": at + 8}), dict(part={"gain": at + 4}), dict(part={"xt": 129}),
               dict(part={"yh": 4}), dict(part={"xe": 2}), dict(part={"ye": 0}), dict(part={"gain": at, "gh": 2}), dict(part={"heads": 0}), dict(tokens=0), dict(tokens=-1), dict(xd=2), dict(yd=-1),
               dict(gd=5), dict(eps=-1.0), dict(eps=float("nan")), dict(rot=0), dict(rot=at + 4), dict(rows=0), dict(rows=2 ** 31),
               dict(pos=at, n_pos=0), dict(pos=at + 2, n_pos=4), dict(n=0), dict(n=3)]:
        assert call(**kw) == L.EINVAL, kw
        assert "aeris_qk_norm_rope_fwd" in L.last_error()
    for kw in [dict(D=48), dict(D=256), dict(D=2 ** 32 + 64), dict(R=8), dict(R=80), dict(R=-16), dict(R=2 ** 32), dict(tokens=2 ** 31 - 1),
               dict(part={"heads": 40000}), dict(part={"heads": 32768}, n=2), dict(part={"heads": 32767}, tokens=2 ** 31 - 100)]:
        assert call(**kw) == L.EUNSUPPORTED, kw
    assert L.lib().aeris_qk_norm_rope_fwd(None, None) == L.EINVAL
    with pytest.raises(RuntimeError, match="GPU"):
        pkg.ops.qk_norm_rope(torch.zeros(4, 2, 64, dtype=torch.bfloat16))
    assert S.size == 304


def test_grids_that_cannot_be_launched(pkg):
    L, at = pkg._lib, 1 << 20

    def call(tokens, heads, D, n):
        part = (at, at, 0, heads, heads * D, D, 1, heads * D, D, 1, 0, 1.0)
        a = pkg.ops.QK_NORM_ROPE.pack(*part, *part, at, 0, tokens, D, L.BF16, L.BF16, L.BF16, 1, 0, 4, 16, 0, n, 1e-6)
        return L.lib().aeris_qk_norm_rope_fwd(a, None)

    for args in [(2 ** 31 - 100, 1, 32, 1), (2 ** 30, 1, 64, 2), (2 ** 28, 8, 128, 1), (2 ** 24, 32767, 32, 2)]:
        assert call(*args) == L.EUNSUPPORTED and "workgroups" in L.last_error(), args
