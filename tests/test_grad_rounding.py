"""What training passes keep in more than one bf16: 24-bit values for the backward pass, two bf16 a value of up to 64 tokens; and that a bound
on the results notices where either is lost.

As in ``test_grad``: U = 2^-8 is half a step of bf16, E = 2^-24 of fp32, a sum of n products in fp32 is off by at most (n + 2) E times the sum of
their sizes.  A number kept as two bf16 is off by half a step of the remainder, which is itself at most half a step of the number: U * U.
"""
import pytest
import torch

from test_grad import BF16, E, F32, FN, KEPT, LIP, LIP2, U, act_of, check_linear, close, kept, norm_bounds, norm_case, norm_definition, run_norm, tokens

LOW = U * U


# ----------------------------------------------------------------------------------------------
# two bf16 a value: the formula with that precision, and its bounds

def mlp_inputs(M, d, H, at="cpu"):
    g = torch.Generator().manual_seed(M + d + H)
    x, dy = tokens(g, M, d).to(BF16).to(at), torch.randn(M, d, generator=g).to(BF16).to(at)
    w1, w2 = (torch.randn(2 * H, d, generator=g) * d ** -0.5).to(BF16).to(at), (torch.randn(d, H, generator=g) * H ** -0.5).to(BF16).to(at)
    return x, w1, w2, dy


def mlp_parts(x, w1, w2, dy):
    """h, [dgate | dup] in 64 bits."""
    x, w1, w2, dy = (t.double() for t in (x, w1, w2, dy))
    gate, up = (x @ w1.T).chunk(2, dim=-1)
    s, dh = torch.sigmoid(gate), dy @ w2
    return gate * s * up, torch.cat([dh * up * s * (1 + gate * (1 - s)), dh * gate * s], 1)


def mlp_results(h, both, x, w1, w2, dy):
    x, w1, w2, dy = (t.double() for t in (x, w1, w2, dy))
    return h @ w2.T, both @ w1, both.T @ x, dy.T @ h


def mlp_bounds(x, w1, w2, dy, rounding):
    """``rounding``: of h, dgate and dup."""
    M, d = x.shape
    H = w2.shape[1]
    X, W1, W2, D = (t.double().abs() for t in (x, w1, w2, dy))
    gate, up = (x.double() @ w1.double().T).chunk(2, dim=-1)
    s = torch.sigmoid(gate)
    silu, ds, fn = (gate * s).abs(), (s * (1 + gate * (1 - s))).abs(), FN * gate.abs().clamp_min(1)
    eg, eu = ((d + 2) * E * (X @ W1.T)).chunk(2, dim=-1)
    h, both = mlp_parts(x, w1, w2, dy)
    want, h = mlp_results(h, both, x, w1, w2, dy), h.abs()
    eh = (LIP * eg + fn) * up.abs() + silu * eu + 4 * E * h
    eh = eh + rounding * (h + eh)
    ey = eh @ W2.T + (H + 2) * E * (h @ W2.T) + U * want[0].abs()
    eg, eu = eg + KEPT * gate.abs(), eu + KEPT * up.abs()
    dh, edh = (dy.double() @ w2.double()).abs(), (d + 2) * E * (D @ W2)
    dup, dgate = dh * silu, dh * up.abs() * ds
    edup = edh * silu + dh * (LIP * eg + fn) + rounding * dup
    edgate = edh * up.abs() * ds + dh * eu * (ds + fn) + dh * up.abs() * (LIP2 * eg + fn) + rounding * dgate
    D1, E1 = torch.cat([dgate, dup], 1), torch.cat([edgate, edup], 1)
    return want, (ey, E1 @ W1 + (2 * H + 2) * E * (D1 @ W1) + U * want[1].abs(), E1.T @ X + (M + 70) * E * (D1.T @ X) + U * want[2].abs(),
                  D.T @ eh + (M + 70) * E * (D.T @ h) + U * want[3].abs())


# (the first ones have sums short enough for the bounds to notice, in each result, what is below half a step of bf16)
FEW_MLP = [(1, 64, 256), (31, 136, 72), (64, 64, 64), (1, 1536, 512), (9, 384, 1088), (64, 256, 1024), (40, 1536, 4096), (64, 2048, 8192)]


@pytest.mark.gpu
@pytest.mark.parametrize("M,d,H", FEW_MLP)
def test_gated_mlp_of_few_tokens(pkg, cuda, M, d, H):
    p = mlp_inputs(M, d, H, cuda)
    on, dy = [t.clone().requires_grad_() for t in p[:3]], p[3]
    y = pkg.grad.feed_forward(*on)
    got = (y, *torch.autograd.grad(y, on, dy))
    want, bounds = mlp_bounds(*p, LOW)
    for name, a, b, e in zip(("y", "dx", "dw1", "dw2"), got, want, bounds):
        close(a, b, e, name)


def lost(t, sign):
    """t in 64 bits as a bf16 and ``sign`` times its remainder."""
    hi = t.to(BF16)
    return hi.double() + sign * (t - hi.double()).to(BF16).double()


@pytest.mark.parametrize("M,d,H", FEW_MLP[:3])
def test_the_bounds_notice_a_gated_mlp_without_its_remainders(M, d, H):
    """The results as the kernels would have them, with the remainders, without, and with their signs turned: only the first keep to the bounds."""
    p = mlp_inputs(M, d, H)
    h, both = mlp_parts(*p)
    want, bounds = mlp_bounds(*p, LOW)
    for sign in (1, 0, -1):
        got = [t.to(BF16).double() for t in mlp_results(lost(h, sign), lost(both, sign), *p)]
        for n, (a, b, e) in enumerate(zip(got, want, bounds)):
            beyond = ((a - b).abs() > 1.02 * e + 1e-30).any()
            assert bool(beyond) == (sign != 1), (n, sign)


def linear_inputs(M, N, K, act, at="cpu"):
    g = torch.Generator().manual_seed(M + N + K)
    a, w = tokens(g, M, K).to(BF16).to(at), (torch.randn(N, K, generator=g) * K ** -0.5).to(BF16).to(at)
    return a, w, torch.randn(M, N, generator=g).to(at).to(F32 if act is None else BF16)


def linear_dz(a, w, dy, act):
    z = (a.double() @ w.double().T).requires_grad_()
    return torch.autograd.grad(act_of(z, act), z, dy.double())[0], z.detach()


def linear_bounds(a, w, dy, act, rounding):
    M, K = a.shape
    N = w.shape[0]
    dz, z = linear_dz(a, w, dy, act)
    A, W, Z = a.double().abs(), w.double().abs(), dz.abs()
    edz = dy.double().abs() * (LIP2 * ((K + 3) * E * (A @ W.T) + KEPT * z.abs()) + FN * z.abs().clamp_min(1)) if act else 0 * dz
    edz = edz + rounding * (Z + edz)
    want = dz @ w.double(), dz.T @ a.double()
    return want, (edz @ W + (N + 2) * E * (Z @ W) + U * want[0].abs(), edz.T @ A + (M + 70) * E * (Z.T @ A) + U * want[1].abs())


FEW_LINEAR = [(1, 256, 64), (9, 1536, 64), (63, 72, 128), (64, 128, 192), (17, 520, 1032), (64, 6144, 4096)]  # (the first four: as above)


@pytest.mark.gpu
@pytest.mark.parametrize("act", [None, "gelu", "silu"])
@pytest.mark.parametrize("M,N,K", FEW_LINEAR)
def test_projection_of_few_tokens(pkg, cuda, M, N, K, act):
    a, w, dy = linear_inputs(M, N, K, act, cuda)
    _, z = pkg.ops.linear_train(a, w, act=act) if act else (None, None)
    da, dw = pkg.ops.linear_backward(dy, a, w, z, act=act, wanted=(True, True, False, False))[:2]
    want, bounds = linear_bounds(a, w, dy, act, LOW)
    close(da, want[0], bounds[0], "da")
    close(dw, want[1], bounds[1], "dw")


@pytest.mark.parametrize("act", [None, "gelu", "silu"])
@pytest.mark.parametrize("M,N,K", FEW_LINEAR[:4])
def test_the_bounds_notice_a_projection_without_its_remainders(M, N, K, act):
    a, w, dy = linear_inputs(M, N, K, act)
    dz, _ = linear_dz(a, w, dy, act)
    want, bounds = linear_bounds(a, w, dy, act, LOW)
    for sign in (1, 0, -1):
        for n, (got, b, e) in enumerate(zip((lost(dz, sign) @ w.double(), lost(dz, sign).T @ a.double()), want, bounds)):
            beyond = ((got.to(BF16).double() - b).abs() > 1.02 * e + 1e-30).any()
            assert bool(beyond) == (sign != 1), (n, sign)


# ---- long sums: whole numbers of 11 bits, which two bf16 hold and one does not, times -1, 0 and 1 (most of them 0): every sum is exact in fp32 (below
# 2^24), and the only rounding is that of the result

def ones(g, *shape, density=0.125):
    return (torch.randint(0, 2, shape, generator=g) * 2 - 1.0) * (torch.rand(*shape, generator=g) < density)


def exactly(got, exact, without, notices=True):
    """``exact`` rounded once, and not what comes out ``without`` the remainders."""
    assert exact.abs().max() < 2 ** 24
    assert torch.equal(got, exact.to(BF16)) and notices != torch.equal(without.to(BF16), exact.to(BF16))


LONG = [(9, 6144, 1536), (64, 1536, 1536), (1, 520, 1032), (64, 6144, 4096), (33, 4104, 2056)]


@pytest.mark.gpu
@pytest.mark.parametrize("M,N,K", LONG)
def test_projection_of_few_tokens_to_the_last_bit(pkg, cuda, M, N, K):
    """In tiles of 64 and 128, whole and cut into parts, alone and two products in a launch."""
    g = torch.Generator().manual_seed(N)
    dy, a, w = torch.randint(-1023, 1024, (M, N), generator=g).float().to(cuda), ones(g, M, K).to(cuda), ones(g, N, K).to(cuda)
    hi = dy.to(BF16).double()
    for wanted in ((True, True), (True, False), (False, True)):
        da, dw = pkg.ops.linear_backward(dy, a.to(BF16), w.to(BF16), wanted=(*wanted, False, False))[:2]
        if wanted[0]:
            exactly(da, dy.double() @ w.double(), hi @ w.double())
        if wanted[1]:
            exactly(dw, dy.double().T @ a.double(), hi.T @ a.double(), M > 1)  # (one token: a single number, rounded)


@pytest.mark.gpu
@pytest.mark.parametrize("M,d,H", [(9, 1536, 6144), (64, 1536, 6144), (1, 64, 1032), (64, 2048, 8192), (40, 136, 2056)])
def test_gated_mlp_of_few_tokens_to_the_last_bit(pkg, cuda, M, d, H):
    """Gates of 64, whose sigmoid is 1 and whose derivative is 1 in fp32: h = 64 up, dgate = dh up, dup = 64 dh."""
    g = torch.Generator().manual_seed(H)
    ops = pkg.ops
    # forward: the first channel of x makes the gates and most of up, the others what up has besides
    x, w1 = ones(g, M, d, density=0.5), ones(g, 2 * H, d, density=0.25)
    x[:, 0], w1[:H], w1[:H, 0], w1[H:, 0] = 8.0, 0.0, 8.0, torch.randint(-100, 101, (H,), generator=g).float()
    w2 = ones(g, d, H, density=0.03)
    x, w1, w2 = x.to(cuda), w1.to(cuda), w2.to(cuda)
    up = (x.double() @ w1.double().T)[:, H:]
    on = [t.to(BF16) for t in (x, w1, w2)]
    y, gate_up, h = ops.feed_forward_train(*on)
    assert torch.equal(gate_up, kept(torch.cat([torch.full_like(up, 64.0), up], 1)))
    h64 = 64 * up
    exactly(y, h64 @ w2.double().T, h64.to(BF16).double() @ w2.double().T)
    # backward: dh is 1, 0 or -1, up of 11 bits
    dy = ones(g, M, d, density=0.5).to(cuda)
    up = torch.randint(-1023, 1024, (M, H), generator=g).float().to(cuda)
    gate_up = kept(torch.cat([torch.full_like(up, 64.0), up], 1))
    pick = torch.zeros(d, H, device=cuda)
    pick[torch.arange(H) % d, torch.arange(H)] = 1.0
    dh = dy.double() @ pick.double()
    both = torch.cat([dh * up.double(), 64 * dh], 1)
    w1, x = ones(g, 2 * H, d).to(cuda), ones(g, M, d, density=0.5).to(cuda)
    hi = both.to(BF16).double()
    for dw2 in (False, True):
        got = ops.feed_forward_backward(dy.to(BF16), x.to(BF16), w1.to(BF16), pick.to(BF16), gate_up, h, wanted=(True, True, dw2))
        exactly(got[0], both @ w1.double(), hi @ w1.double())
        exactly(got[1], both.T @ x.double(), hi.T @ x.double(), M > 1)
        if dw2:
            exactly(got[2], dy.double().T @ h64, dy.double().T @ h64.to(BF16).double(), M > 1)


# ----------------------------------------------------------------------------------------------
# 24-bit values: written by the forward passes

def whole_numbers(g, *shape):
    """Numbers that a bf16 holds and whose sums of up to 4000 products are exact in fp32 (below 2^24), most of them wider than the 16 bits that are kept."""
    return torch.randint(-63, 64, shape, generator=g).float()


def rounded(z):
    """fp32 to the nearest number of 24 bits, halves away from zero."""
    return ((z.contiguous().view(torch.int32) + 0x80) & ~0xff).view(F32)


# (tiles of 64, of 64 with few rows, of 128, whole rounds of tiles of 256, such and a rest; columns and rows that end inside a tile)
@pytest.mark.gpu
@pytest.mark.parametrize("M,d,H", [(9, 384, 1088), (700, 1536, 512), (4000, 512, 1024), (9001, 256, 1032), (8200, 512, 2056), (12480, 384, 1088), (4100, 1544, 3080)])
def test_gate_and_up_are_kept_to_the_last_bit(pkg, cuda, M, d, H):
    g = torch.Generator().manual_seed(M)
    x, w1 = whole_numbers(g, M, d).to(cuda), whole_numbers(g, 2 * H, d).to(cuda)
    want = x.double() @ w1.double().T
    assert want.abs().max() < 2 ** 24 and (want.abs() > 2 ** 16).any()
    _, gate_up, _ = pkg.ops.feed_forward_train(x.to(BF16), w1.to(BF16), torch.zeros(d, H, dtype=BF16, device=cuda))
    assert torch.equal(gate_up, kept(rounded(want.float())))


@pytest.mark.gpu
@pytest.mark.parametrize("act", ["gelu", "silu"])
@pytest.mark.parametrize("M,N,K", [(9, 1536, 64), (300, 512, 384), (3000, 520, 512), (4113, 4104, 1024), (2304, 6152, 2048), (8192, 6144, 1536)])
def test_what_an_activation_is_applied_to_is_kept_to_the_last_bit(pkg, cuda, M, N, K, act):
    g = torch.Generator().manual_seed(M)
    a, w, b = whole_numbers(g, M, K).to(cuda), whole_numbers(g, N, K).to(cuda), whole_numbers(g, N).to(cuda)
    want = a.double() @ w.double().T + b.double()
    assert want.abs().max() < 2 ** 24
    _, z = pkg.ops.linear_train(a.to(BF16), w.to(BF16), b.to(BF16), act=act)
    assert torch.equal(z, kept(rounded(want.float())))


# ---- read by the backward passes

def any_24_bits(g, *shape):
    return (torch.randn(*shape, generator=g).view(torch.int32) & ~0xff).view(F32)


# dh's product in tiles of 64 (few tokens and more), 128 and 256; with dw2 beside it in one launch where that is how they are made
@pytest.mark.gpu
@pytest.mark.parametrize("with_dw2", [False, True])
@pytest.mark.parametrize("M,d,H", [(40, 64, 136), (200, 64, 64), (3000, 256, 512), (8200, 512, 2056), (4100, 1544, 3080), (12480, 384, 1088)])
def test_gate_and_up_are_read_to_the_last_bit(pkg, cuda, M, d, H, with_dw2):
    """w2 hands each hidden channel one of dy's, x hands each row of dw1 one token: dw1 is dgate and dup, rounded once, of as many tokens as there are
    channels.  (Two bf16 a value, up to 64 tokens: their sum rounded once, whose first part is the bf16 nearest to the value.)"""
    g = torch.Generator().manual_seed(M)
    gate, up = any_24_bits(g, M, H), any_24_bits(g, M, H)
    R = min(M, d)
    at = torch.randperm(M, generator=g)[:R]
    dy, x, w2 = torch.zeros(M, d), torch.zeros(M, d), torch.zeros(d, H)
    dy[at] = torch.randn(R, d, generator=g)
    x[at, torch.arange(R)] = 1.0
    w2[torch.arange(H) % d, torch.arange(H)] = 1.0
    dy = dy.to(BF16)
    gate_up = kept(torch.cat([gate, up], 1)).to(cuda)
    h = torch.randn((M if M > 64 else 2 * M) * H, generator=g).to(BF16).to(cuda)
    w1 = torch.zeros(2 * H, d, dtype=BF16, device=cuda)
    dw1 = pkg.ops.feed_forward_backward(dy.to(cuda), x.to(BF16).to(cuda), w1, w2.to(BF16).to(cuda), gate_up, h, wanted=(False, True, with_dw2))[1]
    gt, u, dh = gate[at].double(), up[at].double(), dy[at].double()[:, torch.arange(H) % d]
    s = torch.sigmoid(gt)
    want = torch.cat([dh * u * s * (1 + gt * (1 - s)), dh * gt * s], 1)
    fn = FN * gt.abs().clamp_min(1)
    bound = U * want.abs() + torch.cat([(dh * u).abs() * fn, dh.abs() * fn], 1) * (1 + U)
    close(dw1[:, :R], want.T, bound.T, "dw1")
    assert not dw1[:, R:].any()

    def noticed(mask):  # of values whose lower plane is lost
        gt, u = ((t[at].view(torch.int32) & mask).view(F32).double() for t in (gate, up))
        s = torch.sigmoid(gt)
        got = torch.cat([dh * u * s * (1 + gt * (1 - s)), dh * gt * s], 1).to(BF16).double()
        return ((got - want).abs() > 1.02 * bound + 1e-30).any()
    assert noticed(~0xffff) and not noticed(~0xff)


@pytest.mark.gpu
@pytest.mark.parametrize("y_dtype", [BF16, F32])
@pytest.mark.parametrize("act", ["gelu", "silu"])
@pytest.mark.parametrize("M,N", [(1, 8), (9, 1536), (64, 520), (300, 1032), (5000, 2048)])
def test_what_an_activation_was_applied_to_is_read_to_the_last_bit(pkg, cuda, M, N, act, y_dtype):
    g = torch.Generator().manual_seed(M + N)
    z, dy = any_24_bits(g, M, N), torch.randn(M, N, generator=g).to(y_dtype)
    a, w = torch.zeros(M, 64, dtype=BF16, device=cuda), torch.zeros(N, 64, dtype=BF16, device=cuda)
    dz = pkg.ops.linear_backward(dy.to(cuda), a, w, kept(z).to(cuda), act=act, wanted=(False, False, False, True))[3]

    def formula(z):
        z = z.double().requires_grad_()
        return torch.autograd.grad(act_of(z, act), z, dy.double())[0]
    want, fn = formula(z), dy.double().abs() * FN * z.double().abs().clamp_min(1)
    bound = U * want.abs() + fn * (1 + U)
    close(dz, want, bound, "dz")
    without = formula((z.view(torch.int32) & ~0xffff).view(F32)).to(BF16).double()
    assert M * N < 1000 or ((without - want).abs() > 1.02 * bound + 1e-30).any()  # (a lost lower plane is noticed)


# ----------------------------------------------------------------------------------------------
# forms of the kernels that need many rows, and what else a call's documentation says

@pytest.mark.gpu
@pytest.mark.parametrize("y_dtype", [BF16, F32])
@pytest.mark.parametrize("B,S,d", [(1, 40001, 776), (2, 10007, 1536), (1, 15001, 2048)])
def test_layer_norm_of_bf16_rows_that_belong_to_several_waves(pkg, cuda, B, S, d, y_dtype):
    """Two sums over a row more than an RMS norm has, which pass between the waves; 64-bit reference on the GPU."""
    g = torch.Generator().manual_seed(d)
    p, dy = norm_case(g, B, S, d, "layernorm", "members", BF16, y_dtype, BF16)
    _, got, _ = run_norm(pkg, cuda, p, dy, "layernorm", "mod_then_norm", 1e-5)
    p64 = [t.to(cuda).double().requires_grad_() for t in p]
    names = ("x", "gamma", "beta", "shift", "scale")
    want = torch.autograd.grad(norm_definition(*p64, "layernorm", "mod_then_norm", 1e-5), p64, dy.to(cuda).double())
    bounds = norm_bounds(p64, dy.to(cuda).double(), "layernorm", "mod_then_norm", 1e-5, {"x": BF16, "gamma": BF16})
    for n, w in zip(names, want):
        close(got[n], w, bounds[n], n)


@pytest.mark.gpu
@pytest.mark.parametrize("act,y_dtype", [("silu", F32), ("gelu", BF16), (None, F32)])
def test_gradients_of_more_dz_than_the_caches_hold(pkg, cuda, act, y_dtype):
    check_linear(pkg, cuda, torch.Generator().manual_seed(1), 70001, 2048, 64, act, True, None, y_dtype, at=cuda)


@pytest.mark.gpu
def test_gradients_that_arrive_in_another_order_of_strides(pkg, cuda):
    g, G = torch.Generator().manual_seed(5), pkg.grad
    x, gamma = torch.randn(6, 50, 64, generator=g).to(BF16).to(cuda), torch.randn(64, generator=g).to(cuda)
    w, w1, w2 = (torch.randn(*s, generator=g).to(BF16).to(cuda) for s in ((72, 64), (144, 64), (64, 72)))
    for f, *inputs in ((G.norm_modulate, x, gamma), (G.linear, x, w), (lambda *a: G.linear(*a, act="silu"), x, w), (lambda *a: G.linear(*a, out_dtype=F32), x, w), (G.feed_forward, x, w1, w2)):
        inputs = [t.clone().requires_grad_() for t in inputs]
        y = f(*inputs)
        dy = torch.randn(*y.shape, generator=g).to(y.dtype).to(cuda)
        want = torch.autograd.grad(y, inputs, dy, retain_graph=True)
        for order in ((1, 0, 2), (2, 1, 0), (0, 2, 1)):
            back = [order.index(i) for i in range(3)]
            other = dy.permute(order).contiguous().permute(back)
            assert not other.is_contiguous() and torch.equal(other, dy)
            assert all(torch.equal(s, t) for s, t in zip(torch.autograd.grad(y, inputs, other, retain_graph=True), want))


@pytest.mark.gpu
@pytest.mark.parametrize("M", [5, 64, 65, 700])
def test_results_have_the_same_bits_with_and_without_gradients(pkg, cuda, M):
    g, G = torch.Generator().manual_seed(M), pkg.grad
    x, res = (torch.randn(M, 128, generator=g).to(BF16).to(cuda) for _ in range(2))
    w, w1, w2 = (torch.randn(*s, generator=g).to(BF16).to(cuda) for s in ((128, 128), (400, 128), (128, 200)))
    for f in (lambda x: G.linear(x, w), lambda x: G.linear(x, w, act="gelu", residual=res), lambda x: G.linear(x, w, act="silu", out_dtype=F32), lambda x: G.feed_forward(x, w1, w2)):
        with torch.no_grad():
            plain = f(x)
        y = f(x.clone().requires_grad_())
        assert y.requires_grad and torch.equal(plain, y.detach())


@pytest.mark.gpu
@pytest.mark.parametrize("M", [5, 64, 65, 700])
def test_results_agree_with_the_inference_calls(pkg, cuda, M):
    """Not bit for bit: other kernels, whose fp32 sums (of K products, and of the 2 H that one bf16 rounding of h stands before) and approximations of
    GELU (FN here) differ, before one rounding of the result."""
    g, G, ops = torch.Generator().manual_seed(M), pkg.grad, pkg.ops
    K, N, H = 128, 192, 256
    x, w, b = torch.randn(M, K, generator=g).to(BF16).to(cuda), (torch.randn(N, K, generator=g) * K ** -0.5).to(BF16).to(cuda), torch.randn(N, generator=g).to(BF16).to(cuda)
    size = x.double().abs() @ w.double().abs().T + b.double().abs()
    for act in ("gelu", "silu"):
        z = (x.double() @ w.double().T + b.double()).abs()
        want = ops.gemm(x, w, b, act=act).double()
        close(G.linear(x, w, b, act=act), want, 2 * (LIP * (K + 3) * E * size + FN * z.clamp_min(1)) + 2 * U * want.abs() * (1 + U), act)
    assert torch.equal(G.linear(x, w, b), ops.gemm(x, w, b))
    w1, w2 = (torch.randn(2 * H, K, generator=g) * K ** -0.5).to(BF16).to(cuda), (torch.randn(K, H, generator=g) * H ** -0.5).to(BF16).to(cuda)
    mlp = pkg.FeedForward(K, H).to(cuda).to(BF16)
    with torch.no_grad():
        ws = list(mlp.parameters())
        assert [tuple(t.shape) for t in ws] == [(2 * H, K), (K, H)]
        ws[0].copy_(w1)
        ws[1].copy_(w2)
        theirs = mlp(x[None])[0].double()
    (want, *_), (bound, *_) = mlp_bounds(x, w1, w2, torch.zeros_like(x), U)  # (either is within this of the formula)
    close(G.feed_forward(x, w1, w2), theirs, 2 * bound, "mlp")
