"""Training passes (``grad``) against their definitions in 64 bits, differentiated by autograd on the CPU.

Every element is held to a bound of its own.  Half a step of bf16 is U = 2^-8 of the value, of fp32 E = 2^-24; a sum of n products in
fp32, in whatever order, is off by at most (n + 2) E times the sum of their sizes.  The bounds add up, to first order, what each rounding on
the way does to a result; SLACK covers the products of two roundings.  GELU, SiLU and their derivatives are evaluated to 1e-6 of their
argument's size (at least of 1), and change by at most LIP and LIP2 times what their argument changes: |silu'| <= 1.1, |gelu'| <= 1.13,
|silu''| <= 0.5, |gelu''| <= 0.8.
"""
import math

import pytest
import torch

U, E, SLACK = 2.0 ** -8, 2.0 ** -24, 1.02
KEPT = 2.0 ** -16  # half a step of the 24-bit values (15 bits of fraction) that a forward pass keeps
LIP, LIP2, FN = 1.13, 0.8, 1e-6
BF16, F32 = torch.bfloat16, torch.float32


def close(got, want, bound, name):
    got = got.detach().double().to(want.device)
    assert got.shape == want.shape, (name, got.shape, want.shape)
    over = (got - want).abs() - SLACK * bound - 1e-30
    worst = over.max().cpu() if over.numel() else torch.tensor(-1.0)
    assert worst <= 0, f"{name}: {int((over > 0).sum())} of {over.numel()} beyond their bound, by up to {float(worst):.3g} (bound there {float(bound.flatten()[over.argmax()]):.3g})"
    assert not torch.isnan(got).any(), name


def half_step(dtype):
    return U if dtype is BF16 else E


def tokens(g, *shape):
    return torch.randn(*shape, generator=g) * (0.25 + 1.5 * torch.rand(shape[-1], generator=g)) + 0.5 * torch.randn(shape[-1], generator=g)


# ----------------------------------------------------------------------------------------------
# norm and modulation

def norm_definition(x, gamma, beta, shift, scale, kind, order, eps):
    if scale is not None or shift is not None:
        one = 1 + scale[:, None] if scale is not None else 1.0
        add = shift[:, None] if shift is not None else 0.0
    if (scale is not None or shift is not None) and order == "mod_then_norm":
        x = x * one + add
    if kind == "layernorm":
        x = x - x.mean(-1, keepdim=True)
    y = x / (x.square().mean(-1, keepdim=True) + eps).sqrt() * gamma
    if beta is not None:
        y = y + beta
    if (scale is not None or shift is not None) and order == "norm_then_mod":
        y = y * one + add
    return y


def norm_bounds(p, dy, kind, order, eps, types):
    """Bounds of the gradients, with sums over a row of at most 50 additions a lane and its shuffles, over tokens of as many as there are."""
    x, gamma, beta, shift, scale = (None if t is None else t.detach() for t in p)
    B, S, d = x.shape
    one = 1 + scale[:, None] if scale is not None else torch.ones(1, 1, 1, dtype=torch.float64)
    pre = order == "mod_then_norm" and (scale is not None or shift is not None)
    u = x * one + (shift[:, None] if shift is not None else 0) if pre else x
    size = (x * one).abs() + (shift[:, None].abs() if shift is not None else 0) if pre else x.abs()
    c = u - u.mean(-1, keepdim=True) if kind == "layernorm" else u
    r = (c.square().mean(-1, keepdim=True) + eps).rsqrt()
    n = c * r
    R = 60 * E
    en = R * (r * (size.mean(-1, keepdim=True) + size) + n.abs())
    dv = dy if pre or order == "mod_then_norm" else dy * one
    dn = (dv * gamma)
    m1, m2 = dn.abs().mean(-1, keepdim=True), (dn * n).abs().mean(-1, keepdim=True)
    c2 = (dn * n).mean(-1, keepdim=True).abs()
    e2 = (dn.abs() * en).mean(-1, keepdim=True) + R * m2
    whole = dn.abs() + m1 + n.abs() * c2
    edu = r * (R * m1 + en * c2 + n.abs() * e2 + R * whole)
    du = r * whole
    T = (B * S + 70) * E
    over = (0, 1)
    members = scale.shape[0] if scale is not None else shift.shape[0] if shift is not None else 1
    dims = (1,) if members > 1 else (0, 1)
    keep = members > 1
    factor = one.abs() if pre else 1.0  # dx = du (1 + s) for mod then norm; for norm then mod dx = du, with 1 + s inside dv already
    out = {"x": edu * factor + half_step(types["x"]) * du * factor}
    v = n * gamma + (beta if beta is not None else 0)
    ev = en * gamma.abs() + 4 * E * ((n * gamma).abs() + (beta.abs() if beta is not None else 0))
    half = half_step(types["gamma"])
    out["gamma"] = (dv.abs() * en).sum(over) + T * (dv * n).abs().sum(over) + half * (dv * n).sum(over).abs()
    if beta is not None:
        out["beta"] = T * dv.abs().sum(over) + half * dv.sum(over).abs()
    if pre:
        ds = (edu * x.abs() + T * (du * x).abs()).sum(dims) + E * (du * x).abs().sum(dims)
        dt = (edu + T * du).sum(dims)
    else:
        ds = (dy.abs() * ev + T * (dy.abs() * (n * gamma).abs() + dy.abs() * (beta.abs() if beta is not None else 0))).sum(dims) + E * (dy * v).abs().sum(dims)
        dt = T * dy.abs().sum(dims)
    if scale is not None:
        out["scale"] = ds if keep else ds[None]
    if shift is not None:
        out["shift"] = dt if keep else dt[None]
    return out


def norm_case(g, B, S, d, kind, mod, x_dtype, y_dtype, p_dtype, beta=True):
    x = tokens(g, B, S, d).to(x_dtype)
    gamma, bt = (1 + 0.2 * torch.randn(d, generator=g)).to(p_dtype), (0.2 * torch.randn(d, generator=g)).to(p_dtype) if beta else None
    shift = scale = None
    if mod != "none":
        m = 0.3 * torch.randn(B if mod == "members" else 1, 2 * d, generator=g)
        shift, scale = m[:, :d], m[:, d:]
    dy = torch.randn(B, S, d, generator=g).to(y_dtype)
    return [x, gamma, bt, shift, scale], dy


NAMES = ("x", "gamma", "beta", "shift", "scale")


def run_norm(pkg, cuda, p, dy, kind, order, eps):
    on = [None if t is None else t.to(cuda).requires_grad_() for t in p]
    if p[3] is not None:  # two columns' views of one matrix, as a modulation MLP gives them
        both = torch.cat([p[3], p[4]], dim=1).to(cuda)
        d = p[3].shape[1]
        on[3], on[4] = both[:, :d].detach().requires_grad_(), both[:, d:].detach().requires_grad_()
    y = pkg.grad.norm_modulate(*on, kind=kind, order=order, eps=eps, out_dtype=dy.dtype)
    names = [n for n, t in zip(NAMES, on) if t is not None]
    return y, dict(zip(names, torch.autograd.grad(y, [t for t in on if t is not None], dy.to(cuda)))), on


def check_norm(pkg, cuda, p, dy, kind, order, eps, types):
    y, got, on = run_norm(pkg, cuda, p, dy, kind, order, eps)
    assert torch.equal(y.detach(), pkg.ops.norm_modulate(*[None if t is None else t.detach() for t in on], kind=kind, order=order, eps=eps, out_dtype=dy.dtype))
    p64 = [None if t is None else t.double().requires_grad_() for t in p]
    want = torch.autograd.grad(norm_definition(*p64, kind, order, eps), [t for t in p64 if t is not None], dy.double())
    bounds = norm_bounds(p64, dy.double(), kind, order, eps, types)
    for n, w in zip([n for n, t in zip(NAMES, p64) if t is not None], want):
        t = dict(zip(NAMES, on))[n]
        assert got[n].dtype is t.dtype and got[n].shape == t.shape
        close(got[n], w, bounds[n], n)


@pytest.mark.gpu
@pytest.mark.parametrize("order", ["norm_then_mod", "mod_then_norm"])
@pytest.mark.parametrize("kind", ["layernorm", "rmsnorm"])
@pytest.mark.parametrize("B,S,d,mod", [(1, 1, 8, "one"), (1, 5, 64, "none"), (2, 67, 128, "members"), (3, 33, 136, "members"), (1, 130, 256, "one"),
                                       (2, 19, 264, "one"), (2, 45, 512, "members"), (1, 21, 1000, "members"), (5, 9, 1536, "members"), (2, 7, 2048, "none"),
                                       (2, 13, 2056, "members"), (1, 6, 4096, "one"), (3, 3, 6144, "members"), (1, 3000, 128, "one"), (2, 2600, 320, "members")])
def test_norm_gradients(pkg, cuda, B, S, d, mod, kind, order):
    g = torch.Generator().manual_seed(B * 1000 + S + d)
    for x_dtype, y_dtype, p_dtype in ((BF16, BF16, BF16), (F32, BF16, F32), (F32, F32, BF16), (BF16, F32, F32)):
        p, dy = norm_case(g, B, S, d, kind, mod, x_dtype, y_dtype, p_dtype, beta=kind == "layernorm")
        check_norm(pkg, cuda, p, dy, kind, order, 1e-5, {"x": x_dtype, "gamma": p_dtype})


@pytest.mark.gpu
@pytest.mark.parametrize("which", ["shift", "scale"])
@pytest.mark.parametrize("order", ["norm_then_mod", "mod_then_norm"])
def test_norm_gradients_with_half_a_modulation(pkg, cuda, which, order):
    g = torch.Generator().manual_seed(3)
    p, dy = norm_case(g, 2, 37, 192, "layernorm", "members", F32, BF16, F32, beta=False)
    keep = [t if n != {"shift": "scale", "scale": "shift"}[which] else None for n, t in zip(NAMES, p)]
    on = [None if t is None else t.to(cuda).contiguous().requires_grad_() for t in keep]
    y = pkg.grad.norm_modulate(*on, order=order)
    got = torch.autograd.grad(y, [t for t in on if t is not None], dy.to(cuda))
    p64 = [None if t is None else t.double().requires_grad_() for t in keep]
    want = torch.autograd.grad(norm_definition(*p64, "layernorm", order, 1e-5), [t for t in p64 if t is not None], dy.double())
    bounds = norm_bounds(p64, dy.double(), "layernorm", order, 1e-5, {"x": F32, "gamma": F32})
    for n, a, w in zip([n for n, t in zip(NAMES, p64) if t is not None], got, want):
        close(a, w, bounds[n], n)


@pytest.mark.gpu
def test_norm_gradients_agree_with_differences(pkg, cuda):
    """<gradient, v> against (L(p + h v) - L(p - h v)) / 2h of the definition in 64 bits: the quotient is off by some h^2 (1e-8 of the slope here)."""
    g = torch.Generator().manual_seed(5)
    for kind, order in (("layernorm", "norm_then_mod"), ("rmsnorm", "mod_then_norm")):
        p, dy = norm_case(g, 2, 40, 320, kind, "members", F32, F32, F32, beta=kind == "layernorm")
        _, got, _ = run_norm(pkg, cuda, p, dy, kind, order, 1e-5)
        p64 = [None if t is None else t.double() for t in p]
        for i, n in enumerate(NAMES):
            if p[i] is None:
                continue
            v, h = torch.randn(p[i].shape, generator=g, dtype=torch.float64), 1e-4
            up, down = [*p64], [*p64]
            up[i], down[i] = p64[i] + h * v, p64[i] - h * v
            slope = ((norm_definition(*up, kind, order, 1e-5) - norm_definition(*down, kind, order, 1e-5)) * dy.double()).sum() / (2 * h)
            mine = (got[n].double().cpu() * v).sum()
            size = (got[n].double().cpu() * v).norm()
            assert abs(mine - slope) <= 1e-5 * size * math.sqrt(v.numel()), (kind, n, float(mine), float(slope))


@pytest.mark.gpu
def test_norm_rows_of_one_value(pkg, cuda):
    """A constant row has variance 0: its normed values are 0, its gradient is eps^-1/2 of the centred dn."""
    d = 256
    x = torch.full((1, 3, d), 1.5)
    x[:, 1] = 0.0
    g = torch.Generator().manual_seed(6)
    dy, gamma = torch.randn(1, 3, d, generator=g), torch.ones(d)
    on = [x.to(cuda).requires_grad_(), gamma.to(cuda).requires_grad_()]
    y = pkg.grad.norm_modulate(*on, out_dtype=F32)
    dx, dgamma = torch.autograd.grad(y, on, dy.to(cuda))
    want = (dy.double() - dy.double().mean(-1, keepdim=True)) * 1e-5 ** -0.5
    close(dx, want, 60 * E * 1e-5 ** -0.5 * (dy.abs().double() + dy.abs().double().mean(-1, keepdim=True)) + E * want.abs(), "dx")
    assert (dgamma == 0).all() and (y == 0).all()


@pytest.mark.gpu
def test_norm_nan_and_infinity_stay_in_their_row(pkg, cuda):
    g = torch.Generator().manual_seed(7)
    p, dy = norm_case(g, 1, 40, 128, "layernorm", "none", F32, F32, F32)
    _, clean, _ = run_norm(pkg, cuda, p, dy, "layernorm", "norm_then_mod", 1e-5)
    p[0][0, 7, 3], dy[0, 21, 5] = math.nan, math.inf
    _, got, _ = run_norm(pkg, cuda, p, dy, "layernorm", "norm_then_mod", 1e-5)
    rows = [r for r in range(40) if r not in (7, 21)]
    assert torch.equal(got["x"][0, rows], clean["x"][0, rows])
    assert torch.isnan(got["x"][0, 7]).all() and not torch.isfinite(got["x"][0, 21]).all()
    assert torch.isnan(got["gamma"]).all()  # row 7 takes part in every column


# ----------------------------------------------------------------------------------------------
# projections

def kept(z):
    """Values as they are kept for the backward pass: the upper 16 bits of all of them, then bits 8 to 15."""
    bits = z.float().contiguous().flatten().view(torch.int32)
    return torch.cat([(bits >> 16).to(torch.int16).view(torch.uint8), ((bits >> 8) & 255).to(torch.uint8)])


def act_of(z, act):
    if act == "gelu":
        return z * torch.special.ndtr(z)
    return z * torch.sigmoid(z) if act == "silu" else z


def check_linear(pkg, cuda, g, M, N, K, act, bias, residual, y_dtype, lead=None, at="cpu"):
    """``at``: where the 64-bit products are made."""
    shape = lead or (M,)
    a = tokens(g, M, K).to(BF16)
    w = (torch.randn(N, K, generator=g) * K ** -0.5).to(BF16)
    b = (0.2 * torch.randn(N, generator=g)).to(BF16) if bias else None
    res = tokens(g, M, N).to(residual) if residual else None
    dy = torch.randn(M, N, generator=g).to(y_dtype)
    p = {"a": a, "w": w, "bias": b, "residual": res}
    on = {n: t.to(cuda) for n, t in p.items() if t is not None}
    for n in ("a", "residual"):
        if n in on:
            on[n] = on[n].view(*shape, -1)
    for t in on.values():
        t.requires_grad_()
    y = pkg.grad.linear(on["a"], on["w"], on.get("bias"), act=act, residual=on.get("residual"), out_dtype=y_dtype)
    assert y.shape == (*shape, N) and y.dtype is y_dtype
    got = dict(zip(on, torch.autograd.grad(y, list(on.values()), dy.to(cuda).view(y.shape))))
    # the definition
    a, w, b, dy = a.to(at), w.to(at), None if b is None else b.to(at), dy.to(at)
    p64 = {n: t.to(at).double().requires_grad_() for n, t in p.items() if t is not None}
    z = p64["a"] @ p64["w"].T + (p64["bias"] if bias else 0)
    want_y = act_of(z, act) + (p64["residual"] if residual else 0)
    want = dict(zip(p64, torch.autograd.grad(want_y, list(p64.values()), dy.double())))
    # bounds
    A, W, D = a.double().abs(), w.double().abs(), dy.double().abs()
    ez = (K + 3) * E * (A @ W.T + (b.double().abs() if bias else 0))
    z = z.detach()
    bent = act in ("gelu", "silu")
    ey = (LIP * ez + FN * z.abs().clamp_min(1)) if bent else ez
    ey = ey + (half_step(y_dtype) + 2 * E) * (want_y.detach().abs() + ey) + 2 * E * (act_of(z, act).abs())
    close(y.view(M, N), want_y.detach(), ey, "y")
    ez = ez + KEPT * z.abs()  # as kept
    zz = z.clone().requires_grad_()
    dz = torch.autograd.grad(act_of(zz, act), zz, dy.double())[0]
    edz = D * (LIP2 * ez + FN * z.abs().clamp_min(1)) if bent else torch.zeros_like(dz)
    edzr = edz + (U * (dz.abs() + edz) if bent or y_dtype is F32 else 0)  # rounded for the products
    Z = dz.abs()
    close(got["a"].view(M, K), want["a"], edzr @ W + (N + 2) * E * (Z @ W) + U * want["a"].abs(), "da")
    close(got["w"], want["w"], edzr.T @ A + (M + 70) * E * (Z.T @ A) + U * want["w"].abs(), "dw")
    if bias:
        close(got["bias"], want["bias"], edz.sum(0) + (M + 70) * E * Z.sum(0) + U * want["bias"].abs(), "dbias")
    if residual:
        close(got["residual"].view(M, N), want["residual"], (0 if residual is F32 or y_dtype is BF16 else U) * want["residual"].abs(), "dresidual")
    assert all(got[n].dtype is on[n].dtype and got[n].shape == on[n].shape for n in on)


LINEAR = [(1, 8, 64), (2, 64, 64), (9, 1536, 64), (63, 72, 128), (64, 128, 192), (65, 200, 320), (129, 136, 64), (300, 512, 384), (1000, 96, 640), (4097, 128, 128),
          (2500, 264, 128), (777, 1544, 512), (1, 6144, 64)]


@pytest.mark.gpu
@pytest.mark.parametrize("M,N,K", LINEAR)
def test_linear_gradients(pkg, cuda, M, N, K):
    g = torch.Generator().manual_seed(M + N + K)
    check_linear(pkg, cuda, g, M, N, K, None, True, None, BF16)
    check_linear(pkg, cuda, g, M, N, K, None, False, F32, F32)
    check_linear(pkg, cuda, g, M, N, K, "gelu", True, BF16, BF16)
    check_linear(pkg, cuda, g, M, N, K, "silu", True, F32, F32)


@pytest.mark.gpu
@pytest.mark.parametrize("act", [None, "gelu", "silu"])
@pytest.mark.parametrize("residual", [None, BF16, F32])
@pytest.mark.parametrize("y_dtype", [BF16, F32])
def test_linear_types(pkg, cuda, act, residual, y_dtype):
    g = torch.Generator().manual_seed(11)
    check_linear(pkg, cuda, g, 210, 144, 192, act, act != "silu", residual, y_dtype, lead=(2, 105))


@pytest.mark.gpu
@pytest.mark.parametrize("M,N,K", [(37, 64, 72), (200, 48, 8), (70, 24, 200)])
def test_linear_inner_widths_that_end_inside_a_k_tile(pkg, cuda, M, N, K):
    check_linear(pkg, cuda, torch.Generator().manual_seed(K), M, N, K, "gelu", True, None, BF16)


@pytest.mark.gpu
@pytest.mark.parametrize("M", [20000, 66001])
def test_linear_many_tokens_few_weights(pkg, cuda, M):
    """The weight's gradient is cut along the tokens."""
    check_linear(pkg, cuda, torch.Generator().manual_seed(M), M, 128, 64, None, True, None, BF16)


# Products large enough for tiles of 256: whole rounds of them, a last round cut along k, rows, columns and k that end inside a tile, in all three
# layouts and with every epilogue.
@pytest.mark.gpu
@pytest.mark.parametrize("M,N,K,act,y_dtype,residual", [(8200, 2056, 1088, None, BF16, None), (4113, 4104, 1024, "gelu", BF16, BF16), (16500, 1032, 512, "silu", F32, F32),
                                                        (33000, 520, 1536, None, F32, F32), (2304, 6152, 2048, "gelu", F32, None), (9000, 6152, 3136, None, BF16, None)])
def test_linear_large_products(pkg, cuda, M, N, K, act, y_dtype, residual):
    check_linear(pkg, cuda, torch.Generator().manual_seed(M), M, N, K, act, True, residual, y_dtype, at=cuda)


@pytest.mark.gpu
@pytest.mark.parametrize("M,d,H", [(8200, 512, 2056), (16400, 264, 1088), (4100, 1544, 3080), (20000, 1024, 2056)])
def test_feed_forward_large_products(pkg, cuda, M, d, H):
    check_feed_forward(pkg, cuda, torch.Generator().manual_seed(M), M, d, H, at=cuda)


@pytest.mark.gpu
def test_what_lies_behind_the_rows_of_a_k_tile_does_not_matter(pkg, cuda):
    """N = 72 ends inside a k-tile of da = dz w: the next row's elements, NaN here, take no part in a row's sums."""
    g = torch.Generator().manual_seed(2)
    M, N, K = 70, 72, 64
    dy, w, a = torch.randn(M, N, generator=g).to(BF16), torch.randn(N, K, generator=g).to(BF16), torch.randn(M, K, generator=g).to(BF16)
    clean = pkg.ops.linear_backward(dy.to(cuda), a.to(cuda), w.to(cuda), wanted=(True, False, False, False))[0]
    dy[33] = math.nan
    got = pkg.ops.linear_backward(dy.to(cuda), a.to(cuda), w.to(cuda), wanted=(True, False, False, False))[0]
    rows = [r for r in range(M) if r != 33]
    assert torch.equal(got[rows], clean[rows]) and torch.isnan(got[33]).all()


@pytest.mark.gpu
@pytest.mark.parametrize("act", ["gelu", "silu"])
def test_activation_gradients_of_any_value(pkg, cuda, act):
    """dz for z from the smallest to the largest bf16, through an identity weight; far out the derivatives are 0 and 1."""
    z = torch.arange(-(1 << 15), 1 << 15, dtype=torch.int32).to(torch.int16).view(BF16)
    z = z[torch.isfinite(z)]
    n = z.numel() // 8 * 8
    z = z[:n].view(-1, 8)
    dy, a, w = torch.ones_like(z), torch.zeros(z.shape[0], 8, dtype=BF16), torch.zeros(8, 8, dtype=BF16)
    dz = pkg.ops.linear_backward(dy.to(cuda), a.to(cuda), w.to(cuda), kept(z).to(cuda), act=act, wanted=(False, False, False, True))[3].double().cpu()
    x = z.double()
    if act == "gelu":
        want = torch.special.ndtr(x) + torch.where(x.abs() < 1e3, x * (-0.5 * x * x).exp(), 0.0) / math.sqrt(2 * math.pi)
    else:
        s = torch.sigmoid(x)
        want = s + torch.where(x.abs() < 1e3, x * s * (1 - s), 0.0)
    close(dz, want, U * want.abs() + FN, act)
    bad = torch.tensor([[math.nan] * 8], dtype=BF16)
    dz = pkg.ops.linear_backward(dy[:1].to(cuda), a[:1].to(cuda), w.to(cuda), kept(bad).to(cuda), act=act, wanted=(False, False, False, True))[3]
    assert torch.isnan(dz).all()


# ----------------------------------------------------------------------------------------------
# the gated MLP

def check_feed_forward(pkg, cuda, g, M, d, H, lead=None, loud=1.0, at="cpu"):
    x = (loud * tokens(g, M, d)).to(BF16)
    w1, w2 = (torch.randn(2 * H, d, generator=g) * d ** -0.5).to(BF16), (torch.randn(d, H, generator=g) * H ** -0.5).to(BF16)
    dy = torch.randn(M, d, generator=g).to(BF16)
    on = [x.to(cuda).view(*(lead or (M,)), d).requires_grad_(), w1.to(cuda).requires_grad_(), w2.to(cuda).requires_grad_()]
    y = pkg.grad.feed_forward(*on)
    assert y.shape == on[0].shape and y.dtype is BF16
    got = torch.autograd.grad(y, on, dy.to(cuda).view(y.shape))
    x, w1, w2, dy = (t.to(at) for t in (x, w1, w2, dy))
    p = [t.double().requires_grad_() for t in (x, w1, w2)]
    gate, up = (p[0] @ p[1].T).chunk(2, dim=-1)
    want_y = (gate * torch.sigmoid(gate) * up) @ p[2].T
    want = torch.autograd.grad(want_y, p, dy.double())
    gate, up, X, W1, W2, D = (t.detach() for t in (gate, up, x.double().abs(), w1.double().abs(), w2.double().abs(), dy.double().abs()))
    s = torch.sigmoid(gate)
    silu, ds = gate * s, (s * (1 + gate * (1 - s))).abs()
    e = (d + 2) * E * (X @ W1.T)
    eg, eu = e[:, :H], e[:, H:]
    fn = FN * gate.abs().clamp_min(1)
    h = (silu * up).abs()
    eh = (LIP * eg + fn) * up.abs() + silu.abs() * eu + 4 * E * h
    eh = eh + U * (h + eh)
    close(y.view(M, d), want_y.detach(), eh @ W2.T + (H + 2) * E * (h @ W2.T) + U * want_y.detach().abs(), "y")
    eg, eu = eg + KEPT * gate.abs(), eu + KEPT * up.abs()  # as kept
    dh = (dy.double() @ w2.double()).abs()
    edh = (d + 2) * E * (D @ W2)
    dup, dgate = dh * silu.abs(), dh * up.abs() * ds
    edup = edh * silu.abs() + dh * (LIP * eg + fn) + U * dup
    edgate = edh * up.abs() * ds + dh * eu * (ds + fn) + dh * up.abs() * (LIP2 * eg + fn) + U * dgate
    D1, E1 = torch.cat([dgate, dup], 1), torch.cat([edgate, edup], 1)
    close(got[0].view(M, d), want[0], E1 @ W1 + (2 * H + 2) * E * (D1 @ W1) + U * want[0].abs(), "dx")
    close(got[1], want[1], E1.T @ X + (M + 70) * E * (D1.T @ X) + U * want[1].abs(), "dw1")
    close(got[2], want[2], D.T @ eh + (M + 70) * E * (D.T @ h) + U * want[2].abs(), "dw2")


@pytest.mark.gpu
@pytest.mark.parametrize("M,d,H", [(1, 8, 8), (1, 64, 256), (9, 384, 1088), (31, 136, 72), (64, 64, 64), (65, 128, 200), (200, 256, 1024), (1030, 320, 136),
                                   (4097, 64, 128), (700, 1536, 512)])
def test_feed_forward_gradients(pkg, cuda, M, d, H):
    check_feed_forward(pkg, cuda, torch.Generator().manual_seed(M + d + H), M, d, H)


@pytest.mark.gpu
def test_feed_forward_of_loud_tokens_and_members(pkg, cuda):
    check_feed_forward(pkg, cuda, torch.Generator().manual_seed(1), 2 * 3 * 35, 128, 256, lead=(2, 3, 35), loud=8.0)


# ----------------------------------------------------------------------------------------------
# calls: what is asked for, streams, graphs, refusals

def make(pkg, cuda, seed=0, M=300, d=128, H=256):
    """A block's two branches without its attention, on leaves of its own: norm -> projection onto the stream -> norm -> gated MLP."""
    g = torch.Generator().manual_seed(seed)
    leaf = {"x": tokens(g, 1, M, d).to(cuda), "mod": (0.3 * torch.randn(1, 4 * d, generator=g)).to(cuda)}
    for n in ("g1", "g2"):
        leaf[n] = (1 + 0.2 * torch.randn(d, generator=g)).to(BF16).to(cuda)
    for n, shape in (("w", (d, d)), ("w1", (2 * H, d)), ("w2", (d, H))):
        leaf[n] = (torch.randn(*shape, generator=g) * shape[1] ** -0.5).to(BF16).to(cuda)
    leaf["b"] = (0.2 * torch.randn(d, generator=g)).to(BF16).to(cuda)
    for t in leaf.values():
        t.requires_grad_()
    return leaf, torch.randn(1, M, d, generator=g).to(BF16).to(cuda)


def branches(G, p):
    d = p["x"].shape[-1]
    m = [p["mod"][:, i * d:(i + 1) * d] for i in range(4)]
    y = G.norm_modulate(p["x"], p["g1"], None, m[0], m[1], kind="rmsnorm", order="mod_then_norm")
    x = G.linear(y, p["w"], p["b"], residual=p["x"], out_dtype=F32)
    y = G.norm_modulate(x, p["g2"], None, m[2], m[3], kind="rmsnorm", order="mod_then_norm")
    return G.feed_forward(y, p["w1"], p["w2"])


@pytest.mark.gpu
def test_branches_of_a_block_together(pkg, cuda):
    """The operators one behind the other, as a block has them, against the definition in 64 bits: gradients of every leaf to 2 percent of their
    2-norm (six roundings to bf16 of 2^-8 each, at worst, lie on the longest way)."""
    leaf, dy = make(pkg, cuda)
    y = branches(pkg.grad, leaf)
    got = dict(zip(leaf, torch.autograd.grad(y, list(leaf.values()), dy)))

    class Definition:
        norm_modulate = staticmethod(lambda x, gamma, beta, shift, scale, kind, order: norm_definition(x, gamma, beta, shift, scale, kind, order, 1e-5))
        linear = staticmethod(lambda a, w, b, residual, out_dtype: a @ w.T + b + residual)

        @staticmethod
        def feed_forward(x, w1, w2):
            gate, up = (x @ w1.T).chunk(2, dim=-1)
            return (gate * torch.sigmoid(gate) * up) @ w2.T
    p64 = {n: t.detach().double().cpu().requires_grad_() for n, t in leaf.items()}
    want_y = branches(Definition, p64)
    want = dict(zip(p64, torch.autograd.grad(want_y, list(p64.values()), dy.double().cpu())))
    for n in want:
        off = (got[n].double().cpu() - want[n]).norm() / want[n].norm()
        assert off <= 6 * U, (n, float(off))
    assert (y.detach().double().cpu() - want_y.detach()).norm() <= 6 * U * want_y.detach().norm()


@pytest.mark.gpu
def test_only_what_is_asked_for(pkg, cuda):
    leaf, dy = make(pkg, cuda, 1)
    whole = dict(zip(leaf, torch.autograd.grad(branches(pkg.grad, leaf), list(leaf.values()), dy)))
    for n in leaf:
        for t in leaf.values():
            t.requires_grad_(False)
        leaf[n].requires_grad_()
        alone, = torch.autograd.grad(branches(pkg.grad, leaf), [leaf[n]], dy)
        assert torch.equal(alone, whole[n]), n
    for t in leaf.values():
        t.requires_grad_(False)
    y = branches(pkg.grad, leaf)
    assert not y.requires_grad
    leaf["x"].requires_grad_()
    with torch.no_grad():
        assert torch.equal(branches(pkg.grad, leaf), y)


@pytest.mark.gpu
def test_equal_calls_have_equal_results(pkg, cuda):
    leaf, dy = make(pkg, cuda, 2, M=5000)
    first = torch.autograd.grad(branches(pkg.grad, leaf), list(leaf.values()), dy)
    for _ in range(3):
        again = torch.autograd.grad(branches(pkg.grad, leaf), list(leaf.values()), dy)
        assert all(torch.equal(a, b) for a, b in zip(first, again))


@pytest.mark.gpu
def test_gradients_that_arrive_expanded_or_transposed(pkg, cuda):
    leaf, dy = make(pkg, cuda, 3)
    y = branches(pkg.grad, leaf)
    a, = torch.autograd.grad(y.sum(), [leaf["w1"]], retain_graph=True)
    b, = torch.autograd.grad(y, [leaf["w1"]], torch.ones_like(y))
    assert torch.equal(a, b)
    with pytest.raises(RuntimeError):  # saved tensors are gone
        torch.autograd.grad(y, [leaf["w1"]], dy)


@pytest.mark.gpu
def test_rows_expanded_over_the_members_have_gradients_of_their_own(pkg, cuda):
    g = torch.Generator().manual_seed(4)
    p, dy = norm_case(g, 3, 20, 64, "layernorm", "one", F32, F32, F32)
    on = [t.to(cuda).requires_grad_() for t in p]
    y = pkg.grad.norm_modulate(on[0], on[1], on[2], on[3].expand(3, 64), on[4].expand(3, 64), out_dtype=F32)
    a = torch.autograd.grad(y, on, dy.to(cuda))
    y = pkg.grad.norm_modulate(*on, out_dtype=F32)
    b = torch.autograd.grad(y, on, dy.to(cuda))
    for s, t in zip(a, b):  # (the same sums in another order)
        assert s.shape == t.shape and torch.allclose(s, t, rtol=1e-4, atol=1e-4 * float(t.abs().max()))


@pytest.mark.gpu
def test_empty_batches(pkg, cuda):
    G = pkg.grad
    w, w1, w2 = (torch.ones(s, dtype=BF16, device=cuda, requires_grad=True) for s in ((16, 64), (32, 64), (64, 16)))
    gamma = torch.ones(64, dtype=BF16, device=cuda, requires_grad=True)
    for shape in ((0, 5, 64), (2, 0, 64)):
        x = torch.empty(shape, dtype=BF16, device=cuda, requires_grad=True)
        for f, ps in ((lambda: G.norm_modulate(x, gamma), (x, gamma)), (lambda: G.linear(x, w), (x, w)), (lambda: G.linear(x, w, act="gelu"), (x, w)),
                      (lambda: G.feed_forward(x, w1, w2), (x, w1, w2))):
            y = f()
            for t, p in zip(torch.autograd.grad(y, ps, torch.ones_like(y)), ps):
                assert t.shape == p.shape and (t == 0).all()


@pytest.mark.gpu
def test_two_streams_beside_each_other(pkg, cuda):
    a, da = make(pkg, cuda, 5, M=3000)
    b, db = make(pkg, cuda, 6, M=2000)
    want = [torch.autograd.grad(branches(pkg.grad, p), list(p.values()), d) for p, d in ((a, da), (b, db))]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(3):
        got = []
        for s, (p, d) in zip(streams, ((a, da), (b, db))):
            with torch.cuda.stream(s):
                got.append(torch.autograd.grad(branches(pkg.grad, p), list(p.values()), d))
        torch.cuda.synchronize()
        for g, w in zip(got, want):
            assert all(torch.equal(x, y) for x, y in zip(g, w))


@pytest.mark.gpu
def test_captured_passes_replayed_beside_eager_ones(pkg, cuda):
    a, da = make(pkg, cuda, 7, M=3000)
    b, db = make(pkg, cuda, 8, M=900)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graphs, outs = [], []
    with torch.cuda.stream(side):
        for p, d in ((a, da), (b, db)):  # warm up where the capture runs
            torch.autograd.grad(branches(pkg.grad, p), list(p.values()), d)
    torch.cuda.synchronize()
    for p, d in ((a, da), (b, db)):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            y = branches(pkg.grad, p)
            out = torch.autograd.grad(y, list(p.values()), d)
        graphs.append(graph)
        outs.append((y, *out))
    for seed in range(4):
        g = torch.Generator().manual_seed(20 + seed)
        with torch.no_grad():
            for p, d in ((a, da), (b, db)):
                p["x"].copy_(tokens(g, *p["x"].shape))
                d.copy_(torch.randn(d.shape, generator=g))
        for graph in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for (p, d), got in zip(((a, da), (b, db)), outs):
            y = branches(pkg.grad, p)
            want = (y, *torch.autograd.grad(y, list(p.values()), d))
            assert all(torch.equal(s, t) for s, t in zip(got, want))
            del y, want
        torch.cuda.synchronize()


@pytest.mark.gpu
def test_capture_beside_a_living_eager_graph_is_refused(pkg, cuda):
    leaf, dy = make(pkg, cuda, 9)
    alive = pkg.grad.linear(leaf["x"].detach().to(BF16), leaf["w"])
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="still alive"):
        with torch.cuda.graph(graph, stream=torch.cuda.Stream()):
            pkg.grad.linear(leaf["x"].detach().to(BF16), leaf["w"])
    torch.cuda.synchronize()
    del alive
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=torch.cuda.Stream()):
        y = pkg.grad.linear(leaf["x"].detach().to(BF16), leaf["w"])
        torch.autograd.grad(y, [leaf["w"]], torch.ones_like(y))
    graph.replay()
    torch.cuda.synchronize()


@pytest.mark.gpu
@pytest.mark.parametrize("through", ["view", "cast"])
def test_capture_beside_a_living_eager_graph_of_what_an_input_was_made_of(pkg, cuda, through):
    """The leaf is not an input of the call itself: a modulation matrix that is cut into vectors, an f32 weight that is cast."""
    G = pkg.grad
    x = torch.randn(1, 20, 64, device=cuda).to(BF16)
    gamma = torch.ones(64, dtype=BF16, device=cuda)
    leaf = torch.zeros(1, 128, device=cuda, requires_grad=True) if through == "view" else torch.zeros(64, 64, device=cuda, requires_grad=True)

    def call():
        return G.norm_modulate(x, gamma, None, leaf[:, :64], leaf[:, 64:]) if through == "view" else G.linear(x, leaf.to(BF16))
    alive = call()
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="still alive"):
        with torch.cuda.graph(graph, stream=torch.cuda.Stream()):
            call()
    torch.cuda.synchronize()
    del alive
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=torch.cuda.Stream()):
        y = call()
        got, = torch.autograd.grad(y, [leaf], torch.ones_like(y))
    for _ in range(2):
        graph.replay()
        torch.cuda.synchronize()
        y = call()
        want, = torch.autograd.grad(y, [leaf], torch.ones_like(y))
        assert torch.equal(got, want)
        del y


@pytest.mark.gpu
def test_captured_call_without_gradients_beside_an_eager_graph(pkg, cuda):
    leaf, _ = make(pkg, cuda, 10)
    y = branches(pkg.grad, leaf)
    graph = torch.cuda.CUDAGraph()
    with torch.no_grad(), torch.cuda.graph(graph, stream=torch.cuda.Stream()):
        out = branches(pkg.grad, leaf)
    for _ in range(3):
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, y)


@pytest.mark.gpu
def test_many_members_with_modulation_rows_of_their_own(pkg, cuda):
    g = torch.Generator().manual_seed(12)
    for B, S, d, order in ((9, 5, 64, "norm_then_mod"), (40, 3, 136, "mod_then_norm"), (300, 1, 8, "norm_then_mod"), (1500, 2, 128, "mod_then_norm")):
        p, dy = norm_case(g, B, S, d, "layernorm", "members", F32, BF16, F32)
        check_norm(pkg, cuda, p, dy, "layernorm", order, 1e-5, {"x": F32, "gamma": F32})


@pytest.mark.gpu
def test_bf16_rows_that_belong_to_several_waves(pkg, cuda):
    """bf16 tokens, the modulation ahead of the norm, enough of them for two and four waves to a row; 64-bit reference on the GPU."""
    g = torch.Generator().manual_seed(13)
    for B, S, d in ((1, 40001, 776), (2, 10007, 1536), (1, 15001, 2048)):
        for y_dtype in (BF16, F32):
            p, dy = norm_case(g, B, S, d, "rmsnorm", "members", BF16, y_dtype, BF16, beta=False)
            y, got, on = run_norm(pkg, cuda, p, dy, "rmsnorm", "mod_then_norm", 1e-6)
            p64 = [None if t is None else t.to(cuda).double().requires_grad_() for t in p]
            names = [n for n, t in zip(NAMES, p64) if t is not None]
            want = torch.autograd.grad(norm_definition(*p64, "rmsnorm", "mod_then_norm", 1e-6), [t for t in p64 if t is not None], dy.to(cuda).double())
            bounds = norm_bounds(p64, dy.to(cuda).double(), "rmsnorm", "mod_then_norm", 1e-6, {"x": BF16, "gamma": BF16})
            for n, w in zip(names, want):
                close(got[n], w, bounds[n], n)


@pytest.mark.gpu
def test_gradients_that_arrive_at_odd_addresses(pkg, cuda):
    leaf, dy = make(pkg, cuda, 14)
    y = branches(pkg.grad, leaf)
    want = torch.autograd.grad(y, list(leaf.values()), dy, retain_graph=True)
    odd = torch.empty(dy.numel() + 3, dtype=BF16, device=cuda)[3:].view(dy.shape).copy_(dy)
    assert odd.data_ptr() % 16 and odd.is_contiguous()
    got = torch.autograd.grad(y, list(leaf.values()), odd)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.gpu
def test_a_residual_of_another_shape(pkg, cuda):
    g = torch.Generator().manual_seed(15)
    x, w = torch.randn(2, 30, 64, generator=g).to(BF16).to(cuda), torch.randn(16, 64, generator=g).to(BF16).to(cuda)
    for dtype, y_dtype in ((BF16, F32), (F32, F32), (F32, BF16)):
        res = torch.randn(60, 16, generator=g).to(dtype).to(cuda).requires_grad_()
        dy = torch.randn(2, 30, 16, generator=g).to(y_dtype).to(cuda)
        got, = torch.autograd.grad(pkg.grad.linear(x, w, residual=res, out_dtype=y_dtype), [res], dy)
        assert got.dtype is dtype and torch.equal(got, dy.to(dtype).view(60, 16))


@pytest.mark.gpu
def test_gradients_of_gradients_are_refused(pkg, cuda):
    leaf, dy = make(pkg, cuda, 16)
    y = branches(pkg.grad, leaf)
    got, = torch.autograd.grad(y, [leaf["x"]], dy, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(got.sum(), [leaf["x"]])


@pytest.mark.gpu
def test_forward_mode_is_refused(pkg, cuda):
    from torch.autograd import forward_ad
    G, x, w, gamma = pkg.grad, torch.ones(1, 3, 64, dtype=BF16, device=cuda), torch.ones(64, 64, dtype=BF16, device=cuda), torch.ones(64, device=cuda)
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(x, torch.ones_like(x))
        for call in (lambda: G.norm_modulate(dual, gamma), lambda: G.linear(dual, w), lambda: G.linear(x, w, residual=dual), lambda: G.feed_forward(dual, torch.cat([w, w]), w)):
            with pytest.raises(RuntimeError, match="reverse mode"):
                call()
            with torch.no_grad(), pytest.raises(RuntimeError, match="reverse mode"):
                call()


@pytest.mark.gpu
def test_a_parameter_changed_in_place_is_noticed(pkg, cuda):
    leaf, dy = make(pkg, cuda, 17)
    y = branches(pkg.grad, leaf)
    with torch.no_grad():
        leaf["w1"].mul_(2)
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        torch.autograd.grad(y, [leaf["w1"]], dy)


@pytest.mark.gpu
def test_a_step_of_training(pkg, cuda):
    """Two eager steps with an optimizer on the leaves, through ``backward``: the gradients that accumulate are those of each step."""
    leaf, dy = make(pkg, cuda, 18)
    opt = torch.optim.SGD(list(leaf.values()), lr=1e-3)
    for _ in range(2):
        opt.zero_grad()
        want = torch.autograd.grad(branches(pkg.grad, leaf), list(leaf.values()), dy)
        branches(pkg.grad, leaf).backward(dy)
        assert all(torch.equal(t.grad, w) for t, w in zip(leaf.values(), want))
        branches(pkg.grad, leaf).backward(dy)
        assert all(torch.equal(t.grad, w + w) for t, w in zip(leaf.values(), want))
        opt.step()


@pytest.mark.gpu
@pytest.mark.parametrize("M", [5, 700])
def test_explicit_passes_have_the_same_bits(pkg, cuda, M):
    """``ops``' forward and backward calls, for callers without autograd, against the nodes of ``grad``."""
    ops, G, g = pkg.ops, pkg.grad, torch.Generator().manual_seed(M)
    x, dy = (torch.randn(1, M, 128, generator=g).to(BF16).to(cuda) for _ in range(2))
    gamma, beta = (torch.randn(128, generator=g).to(cuda) for _ in range(2))
    mod = torch.randn(1, 256, generator=g).to(cuda)
    w, b = torch.randn(128, 128, generator=g).to(BF16).to(cuda), torch.randn(128, generator=g).to(BF16).to(cuda)
    w1, w2 = torch.randn(512, 128, generator=g).to(BF16).to(cuda), torch.randn(128, 256, generator=g).to(BF16).to(cuda)
    res = torch.randn(1, M, 128, generator=g).to(cuda)

    def through(f, inputs, dy):
        leaves = [t.detach().clone().requires_grad_() for t in inputs]
        y = f(*leaves)
        return [y.detach(), *torch.autograd.grad(y, leaves, dy)]

    def same(got, want):
        assert len(got) == len(want) and all(torch.equal(s, t) for s, t in zip(got, want))
    norm = (x, gamma, beta, mod[:, :128].contiguous(), mod[:, 128:].contiguous())
    for kw in (dict(), dict(kind="rmsnorm", order="mod_then_norm", eps=1e-6)):
        same([ops.norm_modulate(*norm, **kw), *ops.norm_modulate_backward(dy, *norm, **kw)], through(lambda *a: G.norm_modulate(*a, **kw), norm, dy))
    y, z = ops.linear_train(x, w, b, act="silu")
    same([y, *ops.linear_backward(dy, x, w, z, act="silu", wanted=(True, True, True, False))[:3]], through(lambda *a: G.linear(*a, act="silu"), (x, w, b), dy))
    y, z = ops.linear_train(x, w, b, residual=res, out_dtype=F32)
    assert z is None
    same([y, *ops.linear_backward(dy.float(), x, w, wanted=(True, True, True, False))[:3], dy.float()],
         through(lambda x, w, b, r: G.linear(x, w, b, residual=r, out_dtype=F32), (x, w, b, res), dy.float()))
    assert torch.equal(ops.linear_backward(dy.float(), x, w)[3], dy) and ops.linear_backward(dy, x, w)[3] is dy
    assert ops.linear_train(x, w, act="gelu", keep=False)[1] is None and ops.feed_forward_train(x, w1, w2, keep=False)[1] is None
    y, gate_up, h = ops.feed_forward_train(x, w1, w2)
    same([y, *ops.feed_forward_backward(dy, x, w1, w2, gate_up, h)], through(G.feed_forward, (x, w1, w2), dy))


@pytest.mark.gpu
def test_one_tensor_as_several_inputs(pkg, cuda):
    """Its gradient is the sum of theirs, and the result's gradient stays what it was."""
    G, g = pkg.grad, torch.Generator().manual_seed(3)
    x, dy = (torch.randn(1, 90, 64, generator=g).to(BF16).to(cuda) for _ in range(2))
    w, gamma, m = torch.randn(64, 64, generator=g).to(BF16).to(cuda), torch.randn(64, generator=g).to(cuda), torch.randn(1, 64, generator=g).to(cuda)

    def both(f, *inputs):
        """f of the tensor for both inputs, against f of two copies of it."""
        t, *rest = inputs
        one, kept = t.clone().requires_grad_(), dy.clone()
        got = torch.autograd.grad(f(one, one, *rest), one, kept)[0]
        two = [t.clone().requires_grad_() for _ in range(2)]
        a, b = torch.autograd.grad(f(*two, *rest), two, kept)
        assert torch.equal(got, a + b) and torch.equal(kept, dy)
    both(lambda a, r: G.linear(a, w, residual=r), x)
    both(lambda a, r: G.linear(a, w, act="gelu", residual=r), x)
    both(lambda p, q: G.norm_modulate(x, p, q), gamma)
    both(lambda p, q: G.norm_modulate(x, gamma, None, p, q, order="mod_then_norm"), m)


@pytest.mark.gpu
def test_refusals(pkg, cuda):
    G = pkg.grad
    x = torch.zeros(1, 4, 64, dtype=BF16, device=cuda)
    w, gamma = torch.zeros(16, 64, dtype=BF16, device=cuda), torch.ones(64, dtype=BF16, device=cuda)
    for bad in (lambda: G.norm_modulate(x, gamma[:32]), lambda: G.norm_modulate(x[0], gamma), lambda: G.norm_modulate(x, gamma, kind="batchnorm"),
                lambda: G.norm_modulate(x, gamma, order="both"), lambda: G.norm_modulate(x.half(), gamma), lambda: G.norm_modulate(x, gamma, gamma[:8]),
                lambda: G.norm_modulate(x, gamma, None, torch.zeros(2, 64, device=cuda), torch.zeros(1, 64, device=cuda)),
                lambda: G.linear(x, w.float()), lambda: G.linear(x, w[:, :32]), lambda: G.linear(x, w, act="swiglu"), lambda: G.linear(x, w[:12].contiguous()),
                lambda: G.linear(x, w, torch.zeros(8, dtype=BF16, device=cuda)), lambda: G.linear(x, w, residual=x), lambda: G.linear(x, w, out_dtype=torch.float16),
                lambda: G.linear(x.transpose(1, 2), torch.zeros(16, 4, dtype=BF16, device=cuda)), lambda: G.linear(x, w, act="gelu", residual=torch.zeros(1, 4, 16, dtype=torch.float16, device=cuda)),
                lambda: G.feed_forward(x, w, w), lambda: G.feed_forward(x, torch.zeros(24, 64, dtype=BF16, device=cuda), torch.zeros(64, 12, dtype=BF16, device=cuda)),
                lambda: G.feed_forward(x.float(), torch.zeros(32, 64, dtype=BF16, device=cuda), torch.zeros(64, 16, dtype=BF16, device=cuda)),
                lambda: pkg.ops.linear_train(x, w, act="swiglu"), lambda: pkg.ops.linear_train(x, w.float()), lambda: pkg.ops.linear_train(x, w, residual=x),
                lambda: pkg.ops.feed_forward_train(x, w, w), lambda: pkg.ops.norm_modulate_backward(x[:, :2], x, gamma), lambda: pkg.ops.norm_modulate_backward(x, x, gamma[:32]),
                lambda: pkg.ops.norm_modulate_backward(x.expand(2, 4, 64).contiguous(), x.expand(2, 4, 64).contiguous(), gamma, None, torch.zeros(1, 64, device=cuda).expand(2, 64)),
                lambda: pkg.ops.norm_modulate_backward(x, x, gamma, None, torch.zeros(1, 64, device=cuda).expand(4, 64)[:1].expand(1, 64), torch.zeros(2, 64, device=cuda)),
                lambda: pkg.ops.linear_backward(torch.zeros(1, 4, 16, dtype=BF16, device=cuda), x, w, act="gelu")):
        with pytest.raises(RuntimeError):
            bad()


@pytest.mark.gpu
def test_calls_whose_gradients_would_be_refused_are_refused_themselves(pkg, cuda):
    G, ops = pkg.grad, pkg.ops
    a, w = torch.zeros(1, 32768, dtype=BF16, device=cuda), torch.zeros(32768, 32768, dtype=BF16, device=cuda)
    assert G.linear(a, w).shape == (1, 32768)
    with pytest.raises(RuntimeError, match="no gradients"):
        G.linear(a.requires_grad_(), w)
    x, gamma, m = torch.zeros(65536, 1, 8, dtype=BF16, device=cuda), torch.ones(8, device=cuda), torch.zeros(65536, 16, device=cuda)
    assert G.norm_modulate(x, gamma, None, m[:, :8], m[:, 8:]).shape == x.shape
    with pytest.raises(RuntimeError, match="no gradients"):
        G.norm_modulate(x, gamma, None, m[:, :8].requires_grad_(), m[:, 8:])
    y = G.norm_modulate(x.requires_grad_(), gamma, None, m[:1, :8], m[:1, 8:])  # one row for all of them
    assert torch.autograd.grad(y, x, torch.ones_like(y))[0].shape == x.shape


# More than 2^32 bytes of every operand in turn, a few rows of gradients at the start, in the middle and at the end: the weights' gradients are those
# rows' alone, and the rest of the tokens' gradients is 0.
FAR = 1_060_003


def far_rows(M):
    return torch.cat([torch.arange(0, 70), torch.arange(M // 2 - 9, M // 2 + 60), torch.arange(M - 300, M)])


def noise(cuda, seed, M, N, dtype=BF16):
    g = torch.Generator(device=cuda).manual_seed(seed)
    t = torch.empty(M, N, dtype=dtype, device=cuda)
    for r in range(0, M, 1 << 17):
        part = t[r:r + (1 << 17)]
        part.copy_(torch.randn(part.shape, generator=g, device=cuda))
    return t


def only(rows, values, M):
    dy = torch.zeros(M, values.shape[1], dtype=values.dtype, device=values.device)
    dy[rows] = values
    return dy


@pytest.mark.gpu
@pytest.mark.parametrize("N,K,act,y_dtype", [(2048, 64, "gelu", BF16), (64, 2048, None, BF16), (2048, 64, None, F32), (64, 2048, "silu", F32)])
def test_linear_offsets_past_32_bits(pkg, cuda, N, K, act, y_dtype):
    M = FAR
    rows = far_rows(M).to(cuda)
    a, w = noise(cuda, 1, M, K), (noise(cuda, 2, N, K) * K ** -0.5).to(BF16)
    res = noise(cuda, 3, M, N, y_dtype)
    dy = only(rows, noise(cuda, 4, len(rows), N, y_dtype), M)
    on = [a.requires_grad_(), w.requires_grad_(), res.requires_grad_()]
    y = pkg.grad.linear(a, w, act=act, residual=res, out_dtype=y_dtype)
    da, dw, dres = torch.autograd.grad(y, on, dy)
    near = [t.detach()[rows].requires_grad_() if t is not w else t for t in on]
    y_near = pkg.grad.linear(near[0], w, act=act, residual=near[2], out_dtype=y_dtype)
    da_near, dw_near, dres_near = torch.autograd.grad(y_near, near, dy[rows])
    # (the same numbers summed in another order, then rounded: steps of fp32 sums of K or N numbers of size 1, and one of the result's type)
    a_, w_, d_ = a.detach()[rows].double().abs(), w.detach().double().abs(), dy[rows].double().abs()
    ez = 2 * (K + 3) * E * (a_ @ w_.T)
    z = a_ @ w_.T if act is None else (a.detach()[rows].double() @ w.detach().double().T).abs()
    edz = d_ * (LIP2 * (ez + 2 * KEPT * z) + 2 * FN * z.clamp_min(1)) if act else 0 * d_
    Z = d_ * 1.2  # |act'| <= 1.13
    edz = edz + (2 * U * (Z + edz) if act or y_dtype is F32 else 0)
    top = y_near.detach().double().abs()
    close(y.detach()[rows], y_near.detach().double(), (LIP if act else 1) * ez + 2 * FN * z.clamp_min(1) * (act is not None) + 2 * half_step(y_dtype) * (top + ez) + 4 * E * (z + top), "y")
    close(da[rows], da_near.double(), edz @ w_ + 2 * (N + 2) * E * (Z @ w_) + 2 * U * da_near.double().abs(), "da")
    close(dw, dw_near.double(), edz.T @ a_ + 2 * (len(rows) + 70) * E * (Z.T @ a_) + 2 * U * dw_near.double().abs(), "dw")
    assert torch.equal(dres, dy)
    da[rows] = 0
    assert not da.any()


@pytest.mark.gpu
@pytest.mark.parametrize("d,H", [(2048, 64), (64, 2048)])
def test_feed_forward_offsets_past_32_bits(pkg, cuda, d, H):
    M = FAR
    rows = far_rows(M).to(cuda)
    x, w1, w2 = noise(cuda, 1, M, d), (noise(cuda, 2, 2 * H, d) * d ** -0.5).to(BF16), (noise(cuda, 3, d, H) * H ** -0.5).to(BF16)
    dy = only(rows, noise(cuda, 4, len(rows), d), M)
    y = pkg.grad.feed_forward(x.requires_grad_(), w1.requires_grad_(), w2.requires_grad_())
    dx, dw1, dw2 = torch.autograd.grad(y, [x, w1, w2], dy)
    near = x.detach()[rows].requires_grad_()
    y_near = pkg.grad.feed_forward(near, w1, w2)
    want = torch.autograd.grad(y_near, [near, w1, w2], dy[rows])
    # (two roundings of h and of dgate and dup that may differ by a step each: 2^-8 of the sums of the sizes)
    x_, a1, a2, d_ = near.detach().double().abs(), w1.detach().double().abs(), w2.detach().double().abs(), dy[rows].double().abs()
    gate, up = (near.detach().double() @ w1.detach().double().T).chunk(2, dim=-1)
    s = torch.sigmoid(gate)
    h, silu, ds = (gate * s * up).abs(), (gate * s).abs(), (s * (1 + gate * (1 - s))).abs()
    dh = (dy[rows].double() @ w2.detach().double()).abs()
    D1 = torch.cat([dh * up.abs() * ds, dh * silu], 1)
    small = 2 * (d + 2) * E * (x_ @ a1.T)
    eg, eu = small[:, :H] + 2 * KEPT * gate.abs(), small[:, H:] + 2 * KEPT * up.abs()
    fn = 2 * FN * gate.abs().clamp_min(1)
    eh = (LIP * eg + fn) * up.abs() + silu * eu + 2 * U * h * (1 + U)
    edh = 2 * (d + 2) * E * (d_ @ a2)
    E1 = torch.cat([edh * up.abs() * ds + dh * eu * (ds + fn) + dh * up.abs() * (LIP2 * eg + fn), edh * silu + dh * (LIP * eg + fn)], 1) + 2 * U * D1 * (1 + U)
    close(y.detach()[rows], y_near.detach().double(), eh @ a2.T + 2 * (H + 2) * E * (h @ a2.T) + 2 * U * y_near.detach().double().abs(), "y")
    close(dx[rows], want[0].double(), E1 @ a1 + 2 * (2 * H + 2) * E * (D1 @ a1) + 2 * U * want[0].double().abs(), "dx")
    close(dw1, want[1].double(), E1.T @ x_ + 2 * (len(rows) + 70) * E * (D1.T @ x_) + 2 * U * want[1].double().abs(), "dw1")
    close(dw2, want[2].double(), d_.T @ eh + 2 * (len(rows) + 70) * E * (d_.T @ h) + 2 * U * want[2].double().abs(), "dw2")
    dx[rows] = 0
    assert not dx.any()


@pytest.mark.gpu
@pytest.mark.parametrize("order", ["norm_then_mod", "mod_then_norm"])
@pytest.mark.parametrize("x_dtype", [BF16, F32])
def test_norm_offsets_past_32_bits(pkg, cuda, x_dtype, order):
    M, d = FAR, 2048
    rows = far_rows(M).to(cuda)
    x, gamma, m = noise(cuda, 1, M, d, x_dtype)[None], (1 + 0.2 * torch.randn(d)).to(cuda), (0.3 * torch.randn(1, 2 * d)).to(cuda)
    dy = only(rows, noise(cuda, 4, len(rows), d), M)[None]
    on = [x.requires_grad_(), gamma.requires_grad_(), m[:, :d].detach().requires_grad_(), m[:, d:].detach().requires_grad_()]
    y = pkg.grad.norm_modulate(on[0], gamma, None, on[2], on[3], order=order)
    got = torch.autograd.grad(y, on, dy)
    near = [x.detach()[:, rows].requires_grad_(), *on[1:]]
    p64 = [t.detach().double().cpu().requires_grad_() for t in near]
    want = torch.autograd.grad(norm_definition(p64[0], p64[1], None, p64[2], p64[3], "layernorm", order, 1e-5), p64, dy[:, rows].double().cpu())
    bounds = norm_bounds([p64[0], p64[1], None, p64[2], p64[3]], dy[:, rows].double().cpu(), "layernorm", order, 1e-5, dict(x=x_dtype, gamma=F32))
    for name, g, v in zip(("x", "gamma", "shift", "scale"), (got[0][:, rows], *got[1:]), want):
        close(g, v.to(cuda), bounds[name].to(cuda), name)
    got[0][:, rows] = 0
    assert not got[0].any()


def test_cpu_tensors_are_refused(pkg):
    G = pkg.grad
    x, w = torch.zeros(1, 4, 64, dtype=BF16), torch.zeros(16, 64, dtype=BF16)
    for bad in (lambda: G.norm_modulate(x, torch.ones(64, dtype=BF16)), lambda: G.linear(x, w), lambda: G.feed_forward(x, w, w)):
        with pytest.raises(RuntimeError, match="GPU"):
            bad()


def test_a_missing_extension_is_an_error(pkg, monkeypatch, tmp_path):
    monkeypatch.setattr(pkg.grad, "_loaded", None)
    monkeypatch.setattr(pkg.grad, "EXTENSION_PATH", str(tmp_path / "aeris_grad.so"))
    with pytest.raises(RuntimeError, match="missing"):
        pkg.grad.feed_forward(*[torch.zeros(8, 8, dtype=BF16)] * 3)


def test_packed_records_match_the_header(pkg):
    import os
    import re
    header = open(os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include", "aeris_hip.h")).read()
    header = re.sub(r"/\*.*?\*/", "", header, flags=re.S)

    def fields(name):
        body = re.search(r"typedef struct %s \{(.*?)\} %s;" % (name, name), header, flags=re.S).group(1)
        return sum(len(line.split(",")) for line in body.split(";") if line.strip())
    ops = pkg.ops
    for record, name in ((ops.NORM_GRAD, "aeris_norm_modulate_grad"), (ops.LINEAR_TRAIN, "aeris_linear_train"), (ops.LINEAR_GRAD, "aeris_linear_grad"),
                         (ops.FEED_FORWARD, "aeris_feed_forward"), (ops.FEED_FORWARD_GRAD, "aeris_feed_forward_grad")):
        assert record.size == 8 * fields(name), name


def test_native_argument_checks_need_no_gpu(pkg):
    L, ops = pkg._lib, pkg.ops
    lib, p = L.lib(), 0x1000
    norm = dict(x=p, dy=p, gamma=p, beta=0, shift=0, scale=0, dx=p, dgamma=p, dbeta=0, dshift=0, dscale=0, B=1, rows=4, d=64, stride=0, xt=0, yt=0, pt=0, kind=0, order=0, eps=1e-5)

    def norm_call(ws=None, size=0, **change):
        return lib.aeris_norm_modulate_bwd(ops.NORM_GRAD.pack(*{**norm, **change}.values()), ws, size, None)
    assert lib.aeris_norm_modulate_grad_workspace_bytes(ops.NORM_GRAD.pack(*norm.values())) == 2 * 64 * 4
    assert lib.aeris_norm_modulate_grad_workspace_bytes(ops.NORM_GRAD.pack(*{**norm, "dgamma": 0}.values())) == 0
    for change in (dict(x=0), dict(dy=0), dict(gamma=0), dict(B=0), dict(rows=-1), dict(xt=2), dict(yt=9), dict(pt=-1), dict(kind=2), dict(order=5), dict(eps=-1.0),
                   dict(eps=float("nan")), dict(stride=-4), dict(x=p + 4), dict(dgamma=p + 2), dict(dbeta=p), dict(dshift=p), dict(dscale=p)):
        assert norm_call(**change) == L.EINVAL, change
    for change in (dict(d=60), dict(d=6152), dict(d=0), dict(rows=1 << 60), dict(B=1 << 40, rows=1 << 40), dict(B=70000, rows=1, shift=p, stride=64),
                   dict(B=60000, rows=1, d=1024, shift=p, stride=1024)):
        assert norm_call(**change) == L.EUNSUPPORTED, change
    assert norm_call() == L.EINVAL and "workspace" in L.last_error()  # too small
    assert norm_call(ws=p + 8, size=1 << 20) == L.EINVAL

    train = dict(x=p, w=p, bias=0, res=0, y=p, z=p, M=4, N=16, K=64, act=1, rt=0, yt=0)
    for change, rc in ((dict(x=0), -1), (dict(y=0), -1), (dict(M=0), -1), (dict(act=0), -1), (dict(act=2), -1), (dict(yt=3), -1), (dict(res=p, rt=7), -1), (dict(bias=p + 2), -1),
                       (dict(N=12), -2), (dict(K=63), -2), (dict(N=1 << 21), -2), (dict(N=1 << 20, K=1 << 16), -2), (dict(M=1 << 31), -2), (dict(M=1 << 30, N=1 << 16), -2)):
        assert lib.aeris_linear_train_fwd(ops.LINEAR_TRAIN.pack(*{**train, **change}.values()), None) == rc, change
    lin = dict(dy=p, x=p, w=p, z=0, dx=p, dw=p, db=p, dz=0, M=4, N=16, K=64, act=0, yt=0)

    def linear_call(ws=None, size=0, **change):
        return lib.aeris_linear_bwd(ops.LINEAR_GRAD.pack(*{**lin, **change}.values()), ws, size, None)
    for change, rc in ((dict(dy=0), -1), (dict(w=0), -1), (dict(x=0), -1), (dict(act=1), -1), (dict(act=2, z=p), -1), (dict(yt=4), -1), (dict(dz=p), -1), (dict(dw=p + 8), -1),
                       (dict(N=20), -2), (dict(K=0), -1), (dict(M=-3), -1)):
        assert linear_call(**change) == rc, change
    assert linear_call() == L.EINVAL and "workspace" in L.last_error()
    ff = dict(x=p, w1=p, w2=p, gu=p, h=p, y=p, M=4, d=64, H=128)
    for change, rc in ((dict(x=0), -1), (dict(h=0), -1), (dict(M=0), -1), (dict(H=0), -1), (dict(H=12), -2), (dict(d=4), -2), (dict(H=1 << 62), -2), (dict(d=1 << 19, H=1 << 19), -2), (dict(y=p + 1), -1)):
        assert lib.aeris_feed_forward_train_fwd(ops.FEED_FORWARD.pack(*{**ff, **change}.values()), p, 1 << 40, None) == rc, change
    ffg = dict(dy=p, x=p, w1=p, w2=p, gu=p, h=p, dx=p, dw1=p, dw2=p, M=4, d=64, H=128)
    for change, rc in ((dict(dy=0), -1), (dict(x=0), -1), (dict(w1=0), -1), (dict(h=0), -1), (dict(H=-8), -1), (dict(H=4), -2), (dict(dx=p + 2), -1)):
        assert lib.aeris_feed_forward_bwd(ops.FEED_FORWARD_GRAD.pack(*{**ffg, **change}.values()), p, 1 << 40, None) == rc, change
    assert lib.aeris_feed_forward_bwd(ops.FEED_FORWARD_GRAD.pack(*ffg.values()), None, 0, None) == L.EINVAL
    for f in (lib.aeris_norm_modulate_grad_workspace_bytes, lib.aeris_linear_grad_workspace_bytes, lib.aeris_feed_forward_workspace_bytes, lib.aeris_feed_forward_grad_workspace_bytes):
        assert f(None) == 0
