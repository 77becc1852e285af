"""Calls of ``grad`` beyond a single pass: gradients of gradients, gradients that accumulate, operands that hold infinities."""
import math

import pytest
import torch

BF16, F32 = torch.bfloat16, torch.float32


def normal(g, *shape, dtype=F32, std=1.0):
    return (std * torch.randn(*shape, generator=g)).to(dtype)


def operators(pkg, cuda, seed=0):
    """name -> (the call, its inputs by name), each on leaves of its own."""
    G, g = pkg.grad, torch.Generator().manual_seed(seed)

    def leaves(**tensors):
        return {n: t.to(cuda).requires_grad_() for n, t in tensors.items()}
    M, d, H = 70, 64, 96
    norm = leaves(x=normal(g, 2, 35, d), gamma=normal(g, d), beta=normal(g, d), shift=normal(g, 2, d, std=0.3), scale=normal(g, 2, d, std=0.3))
    linear = leaves(a=normal(g, M, d, dtype=BF16), w=normal(g, H, d, dtype=BF16, std=d ** -0.5), bias=normal(g, H, dtype=BF16))
    mlp = leaves(x=normal(g, M, d, dtype=BF16), w1=normal(g, 2 * H, d, dtype=BF16, std=d ** -0.5), w2=normal(g, d, H, dtype=BF16, std=H ** -0.5))
    return {
        "norm": (lambda: G.norm_modulate(*norm.values()), norm),
        "mod_norm": (lambda: G.norm_modulate(*norm.values(), order="mod_then_norm", out_dtype=F32), norm),
        "linear": (lambda: G.linear(*linear.values()), linear),
        "gelu": (lambda: G.linear(*linear.values(), act="gelu", out_dtype=F32), linear),
        "mlp": (lambda: G.feed_forward(*mlp.values()), mlp),
    }


@pytest.mark.gpu
@pytest.mark.parametrize("name", ["norm", "mod_norm", "linear", "gelu", "mlp"])
def test_a_penalty_on_a_gradient_is_refused_beside_other_terms(pkg, cuda, name):
    """A loss of the result and of a gradient: what the gradient's term adds cannot be left out without a word, whichever inputs are asked for."""
    call, inputs = operators(pkg, cuda)[name]
    once = {n: torch.autograd.grad(call().float().sum(), t)[0] for n, t in inputs.items()}
    for n, t in inputs.items():
        y = call()
        g, = torch.autograd.grad(y.float().sum(), t, create_graph=True)
        assert g.requires_grad and torch.equal(g.detach(), once[n])
        loss = y.float().square().sum() + g.float().square().sum()
        for other in inputs.values():
            with pytest.raises(RuntimeError, match="differentiable once"):
                torch.autograd.grad(loss, other, retain_graph=True)
        with pytest.raises(RuntimeError, match="differentiable once"):
            loss.backward()
    # through the result's gradient alone
    y = call()
    dy = torch.ones_like(y).requires_grad_()
    for g in torch.autograd.grad(y, list(inputs.values()), dy, create_graph=True):
        with pytest.raises(RuntimeError, match="differentiable once"):
            torch.autograd.grad(g.float().square().sum() + dy.float().sum(), dy, retain_graph=True)
    for t in inputs.values():
        t.grad = None
    call().float().sum().backward(create_graph=True)
    assert all(torch.equal(t.grad.detach(), once[n]) for n, t in inputs.items())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,y_dtype", [(BF16, BF16), (F32, F32), (BF16, F32), (F32, BF16)])
def test_a_residual_is_differentiable_more_than_once(pkg, cuda, dtype, y_dtype):
    """Its gradient is the result's, in its type: torch's own operations, whose derivative is 1."""
    g = torch.Generator().manual_seed(1)
    a, w = normal(g, 70, 64, dtype=BF16).to(cuda), normal(g, 32, 64, dtype=BF16).to(cuda)
    for shape in ((70, 32), (7, 10, 32)):
        res = normal(g, *shape, dtype=dtype).to(cuda).requires_grad_()
        dy = normal(g, 70, 32, dtype=y_dtype).to(cuda).requires_grad_()
        got, = torch.autograd.grad(pkg.grad.linear(a, w, residual=res, out_dtype=y_dtype), res, dy, create_graph=True)
        assert got.shape == shape and torch.equal(got.detach().view(70, 32), dy.detach().to(dtype))
        again, = torch.autograd.grad(got.sum(), dy)
        assert (again == 1).all()


@pytest.mark.gpu
@pytest.mark.parametrize("act", [None, "gelu"])
@pytest.mark.parametrize("dtype,y_dtype", [(BF16, BF16), (F32, F32), (BF16, F32), (F32, BF16)])
@pytest.mark.parametrize("shape", [(2, 30, 16), (60, 16)])
def test_residual_gradients_that_accumulate(pkg, cuda, shape, dtype, y_dtype, act):
    """Several passes into ``.grad`` with one gradient of the result (whole numbers, whose sums are exact in bf16): three times that gradient, which
    itself stays what it was; so does the gradient of what else the result is added to."""
    g = torch.Generator().manual_seed(2)
    a, w = normal(g, 2, 30, 64, dtype=BF16).to(cuda), normal(g, 16, 64, dtype=BF16).to(cuda).requires_grad_()
    dy = torch.randint(-8, 9, (2, 30, 16), generator=g).to(y_dtype).to(cuda)
    kept = dy.clone()
    res = torch.zeros(shape, dtype=dtype, device=cuda, requires_grad=True)
    for n in range(1, 4):
        pkg.grad.linear(a, w, act=act, residual=res, out_dtype=y_dtype).backward(dy)
        assert torch.equal(dy, kept) and torch.equal(res.grad, (n * kept).to(dtype).view(shape)), n
    # two leaves whose gradients are the same numbers, and whose gradients arrive from a graph that nobody holds
    res = torch.zeros(shape, dtype=dtype, device=cuda, requires_grad=True)
    other = torch.zeros(2, 30, 16, dtype=y_dtype, device=cuda, requires_grad=True)
    for n in range(1, 4):
        y = pkg.grad.linear(a, w, act=act, residual=res, out_dtype=y_dtype) + other
        (y * kept).sum().backward()
        assert torch.equal(res.grad, (n * kept).to(dtype).view(shape)) and torch.equal(other.grad, n * kept), n


@pytest.mark.gpu
@pytest.mark.parametrize("name", ["norm", "mod_norm", "linear", "gelu", "mlp"])
def test_a_tangent_of_the_result_s_gradient_is_refused(pkg, cuda, name):
    """Forward mode over reverse mode: nothing of the call's inputs has a tangent, but what its result is multiplied with has."""
    from torch.autograd import forward_ad
    call, inputs = operators(pkg, cuda)[name]
    with forward_ad.dual_level():
        y = call()
        factor = forward_ad.make_dual(torch.ones_like(y), torch.ones_like(y))
        for t in inputs.values():
            with pytest.raises(RuntimeError, match="reverse mode"):
                torch.autograd.grad((y * factor).sum(), t, retain_graph=True)
        assert all(torch.isfinite(t).all() for t in torch.autograd.grad(y.sum(), list(inputs.values())))


@pytest.mark.gpu
def test_a_tangent_of_the_result_s_gradient_reaches_the_residual_s(pkg, cuda):
    from torch.autograd import forward_ad
    a, w, res = torch.zeros(70, 64, dtype=BF16, device=cuda), torch.zeros(32, 64, dtype=BF16, device=cuda), torch.zeros(70, 32, device=cuda, requires_grad=True)
    with forward_ad.dual_level():
        y = pkg.grad.linear(a, w, residual=res, out_dtype=F32)
        g, = torch.autograd.grad((y * forward_ad.make_dual(torch.ones_like(y), torch.full_like(y, 3.0))).sum(), res)
        primal, tangent = forward_ad.unpack_dual(g)
        assert (primal == 1).all() and (tangent == 3).all()


@pytest.mark.gpu
@pytest.mark.parametrize("name", ["norm", "mod_norm", "linear", "gelu", "mlp"])
def test_batches_of_gradients_are_refused(pkg, cuda, name):
    """Vectorised Jacobians (vmap over the backward pass)."""
    call, inputs = operators(pkg, cuda)[name]
    y = call()
    with pytest.raises(RuntimeError):
        torch.autograd.grad(y, list(inputs.values()), torch.ones_like(y).expand(3, *y.shape), is_grads_batched=True)


def same_kind(got, want):
    """Infinities where the formula has them, with their signs, NaN where it has NaN; -> where the formula is finite."""
    got, want = got.detach().double().cpu(), want.double()
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    far = torch.isinf(want)
    assert torch.equal(torch.isinf(got), far) and torch.equal(got[far], want[far])
    return torch.isfinite(want)


@pytest.mark.gpu
@pytest.mark.parametrize("M", [1, 9, 64, 65, 300])
@pytest.mark.parametrize("act", [None, "gelu"])
def test_infinite_operands_of_a_projection_s_gradients(pkg, cuda, M, act):
    """An infinity in w or a makes infinities of the sign of the numbers that it is multiplied with, in its column of the gradient alone."""
    g = torch.Generator().manual_seed(M)
    N, K = 136, 192
    dy, a, w = normal(g, M, N), normal(g, M, K, dtype=BF16), normal(g, N, K, dtype=BF16, std=K ** -0.5)
    _, z = pkg.ops.linear_train(a.to(cuda), w.to(cuda), act=act)

    def grads(a, w):
        return pkg.ops.linear_backward(dy.to(cuda), a.to(cuda), w.to(cuda), z, act=act, wanted=(True, True, False, True))[:4]
    clean_a, clean_w, _, dz = grads(a, w)
    w_far, a_far = w.clone(), a.clone()
    w_far[3, 5], w_far[100, 7], a_far[M // 2, 11], a_far[0, 150] = math.inf, -math.inf, -math.inf, math.inf
    da, dw = grads(a_far, w_far)[:2]
    dz = dz.double().cpu()
    finite = same_kind(da, dz @ w_far.double())
    assert torch.equal(da.cpu()[finite], clean_a.cpu()[finite]) and not finite[:, [5, 7]].any() and finite.sum() == M * (K - 2)
    finite = same_kind(dw, dz.T @ a_far.double())
    assert torch.equal(dw.cpu()[finite], clean_w.cpu()[finite]) and finite.sum() == N * (K - 2)


@pytest.mark.gpu
@pytest.mark.parametrize("M", [1, 9, 64, 65, 300])
def test_infinite_operands_of_the_gated_mlp(pkg, cuda, M):
    """In w2 for the result, in the result's gradient for that of w2, in w1 and x for those of x and w1 (whose gates are kept finite here)."""
    g = torch.Generator().manual_seed(M)
    ops, d, H = pkg.ops, 64, 136
    x, dy = normal(g, M, d, dtype=BF16), normal(g, M, d, dtype=BF16)
    w1, w2 = normal(g, 2 * H, d, dtype=BF16, std=d ** -0.5), normal(g, d, H, dtype=BF16, std=H ** -0.5)
    on = [t.to(cuda) for t in (x, w1, w2)]
    clean_y, gate_up, h = ops.feed_forward_train(*on)
    clean = ops.feed_forward_backward(dy.to(cuda), *on, gate_up, h)
    gate, up = (x.double() @ w1.double().T).chunk(2, dim=-1)
    s = torch.sigmoid(gate)
    h64, dh = gate * s * up, dy.double() @ w2.double()
    both = torch.cat([dh * up * s * (1 + gate * (1 - s)), dh * gate * s], 1)

    far = w2.clone()
    far[3, 5], far[40, 100] = math.inf, -math.inf
    y = ops.feed_forward_train(on[0], on[1], far.to(cuda))[0]
    finite = same_kind(y, h64 @ far.double().T)
    assert torch.equal(y.cpu()[finite], clean_y.cpu()[finite]) and finite.sum() == M * (d - 2)

    far = dy.clone()
    far[M // 2, 9], far[0, 50] = math.inf, -math.inf
    dw2 = ops.feed_forward_backward(far.to(cuda), *on, gate_up, h, wanted=(False, False, True))[2]
    finite = same_kind(dw2, far.double().T @ h64)
    assert torch.equal(dw2.cpu()[finite], clean[2].cpu()[finite]) and finite.sum() == (d - 2) * H

    far_w1, far_x = w1.clone(), x.clone()
    far_w1[3, 5], far_w1[2 * H - 1, 60], far_x[M // 2, 1], far_x[0, 33] = math.inf, -math.inf, math.inf, -math.inf
    dx, dw1, _ = ops.feed_forward_backward(dy.to(cuda), far_x.to(cuda), far_w1.to(cuda), on[2], gate_up, h, wanted=(True, True, False))
    finite = same_kind(dx, both @ far_w1.double())
    assert torch.equal(dx.cpu()[finite], clean[0].cpu()[finite]) and finite.sum() == M * (d - 2)
    finite = same_kind(dw1, both.T @ far_x.double())
    assert torch.equal(dw1.cpu()[finite], clean[1].cpu()[finite]) and finite.sum() == 2 * H * (d - 2)


def test_an_extension_built_against_another_torch_is_an_error(pkg, monkeypatch, tmp_path):
    """It is neither loaded nor taken for up to date by the build."""
    build = pkg.grad.build
    assert build.grad_built_for_this_torch() and pkg.grad._functions().marker == build.grad_marker()
    other = tmp_path / "aeris_grad.so"
    with open(build.GRAD_LIB, "rb") as f:
        other.write_bytes(f.read().replace(build.grad_marker().encode(), build.grad_marker().encode()[::-1]))
    assert not build.grad_built_for_this_torch(str(other))
    monkeypatch.setattr(pkg.grad, "_loaded", None)
    monkeypatch.setattr(pkg.grad, "EXTENSION_PATH", str(other))
    with pytest.raises(RuntimeError, match="another torch"):
        pkg.grad.feed_forward(*[torch.zeros(8, 8, dtype=BF16)] * 3)
    # a build with everything else up to date compiles the extension, and nothing else, again
    monkeypatch.setattr(build, "_stale", lambda target, deps: False)
    made = []
    monkeypatch.setattr(build.subprocess, "run", lambda cmd, **kw: made.append(cmd) or build.subprocess.CompletedProcess(cmd, 0, "", ""))
    build.build(verbose=False)
    assert not made
    monkeypatch.setattr(build, "grad_marker", lambda: "aeris_grad for torch 0.0")
    build.build(verbose=False)
    assert len(made) == 1 and made[0][0] == "g++" and build.GRAD_SOURCE in made[0]


def test_refusals_of_sizes_name_the_limit(pkg):
    """As many tokens as the documented limit of tiles allows are taken (up to the workspace, which is missing here), one tile more is refused with
    a message that speaks of rows; the gated MLP's names H as it was given."""
    L, ops = pkg._lib, pkg.ops
    lib, p = L.lib(), 0x1000
    most = ((1 << 24) - 1) // 256 * 64  # rows of a projection to 8192 columns

    def linear(M, N=8192, K=64):
        return lib.aeris_linear_bwd(ops.LINEAR_GRAD.pack(p, p, p, 0, p, p, p, 0, M, N, K, 0, L.F32), None, 0, None)
    assert linear(most) == L.EINVAL and "workspace" in L.last_error()
    assert linear(most + 1) == L.EUNSUPPORTED and "rows: fewer than 2^31" in L.last_error() and "2^24 tiles" in L.last_error()

    def mlp(M, d=64, H=4096):
        return lib.aeris_feed_forward_bwd(ops.FEED_FORWARD_GRAD.pack(p, p, p, p, p, p, p, p, p, M, d, H), None, 0, None)
    assert mlp(most) == L.EINVAL and "workspace" in L.last_error()
    assert mlp(most + 1) == L.EUNSUPPORTED and "H=4096" in L.last_error() and "2^24 tiles" in L.last_error()
    assert mlp(1, H=1 << 20) == L.EUNSUPPORTED and f"H={1 << 20} " in L.last_error()
    assert mlp(1, H=12) == L.EUNSUPPORTED and "H=12 (H a multiple of 8" in L.last_error()
    assert mlp(1, d=0) == L.EINVAL and mlp(0) == L.EINVAL and mlp(1, H=-8) == L.EINVAL


@pytest.mark.gpu
def test_infinite_operands_of_a_wide_projection_s_gradients(pkg, cuda):
    """64 tokens, dw in tiles of 128, da cut along k: an infinity in one part, in two of the same sign, and in two of different signs."""
    g = torch.Generator().manual_seed(64)
    M, N, K = 64, 6144, 4096
    dy, a, w = normal(g, M, N).to(cuda), normal(g, M, K, dtype=BF16).to(cuda), normal(g, N, K, dtype=BF16, std=K ** -0.5).to(cuda)
    clean_a, clean_w, _, dz = pkg.ops.linear_backward(dy, a, w)
    a[40, 4000], w[5, 7], w[6000, 7], w[3, 9], w[4, 2048] = math.inf, math.inf, math.inf, -math.inf, math.inf
    da, dw = pkg.ops.linear_backward(dy, a, w, wanted=(True, True, False, False))[:2]
    dz = dz.double()
    finite = same_kind(da, (dz @ w.double()).cpu())
    assert torch.equal(da.cpu()[finite], clean_a.cpu()[finite]) and finite.sum() == M * (K - 3)
    finite = same_kind(dw, (dz.T @ a.double()).cpu())
    assert torch.equal(dw.cpu()[finite], clean_w.cpu()[finite]) and finite.sum() == N * (K - 1)


@pytest.mark.gpu
@pytest.mark.parametrize("name", ["norm", "mod_norm", "linear", "gelu", "mlp"])
def test_what_is_kept_may_pass_through_hooks(pkg, cuda, name):
    """Kept on the host, or made again by a checkpoint, as torch's own operations allow it."""
    call, inputs = operators(pkg, cuda)[name]
    y = call()
    dy = torch.randn(y.shape, generator=torch.Generator().manual_seed(3)).to(y.dtype).to(cuda)
    want = (y, *torch.autograd.grad(y, list(inputs.values()), dy))
    with torch.autograd.graph.save_on_cpu():
        y = call()
    got = (y, *torch.autograd.grad(y, list(inputs.values()), dy))
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    y = torch.utils.checkpoint.checkpoint(lambda *_: call(), *inputs.values(), use_reentrant=False)
    got = (y, *torch.autograd.grad(y, list(inputs.values()), dy))
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.gpu
@pytest.mark.parametrize("name", ["norm", "mod_norm"])
@pytest.mark.parametrize("which", [0, 1])
def test_modulation_rows_of_which_a_hook_moves_one(pkg, cuda, name, which):
    """Two columns' views of one matrix when they went in, rows of two strides when they come back."""
    call, inputs = operators(pkg, cuda)[name]
    g = torch.Generator().manual_seed(4)
    mod = normal(g, 2, 128, std=0.3).to(cuda).requires_grad_()
    x, gamma, beta, *_ = inputs.values()
    order = "mod_then_norm" if name == "mod_norm" else "norm_then_mod"

    def once(pack):
        with torch.autograd.graph.saved_tensors_hooks(pack, lambda t: t):
            y = pkg.grad.norm_modulate(x, gamma, beta, mod[:, :64], mod[:, 64:], order=order)
        return torch.autograd.grad(y.float().square().sum(), [x, gamma, beta, mod])
    rows = []

    def move_one(t):
        if t.shape == (2, 64):
            rows.append(t)
            return t.clone() if len(rows) == which + 1 else t
        return t
    want = once(lambda t: t)
    got = once(move_one)
    assert len(rows) == 2 and rows[0].stride(0) == 128
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.gpu
@pytest.mark.parametrize("name", ["norm", "mod_norm", "linear", "gelu", "mlp"])
@pytest.mark.parametrize("change", ["host", "half", "strides", "fewer", "flat"])
def test_what_hooks_bring_back_changed_is_refused(pkg, cuda, name, change):
    """A tensor that is not what was kept, one after the other: each is an error, none is read."""
    how = {"host": lambda t: t.cpu(), "half": lambda t: t.to(torch.float64), "strides": lambda t: t.as_strided(t.shape, [0] * t.dim()),
           "fewer": lambda t: t[:-1] if t.dim() == 1 else t[..., :-8].contiguous(), "flat": lambda t: t.reshape(1, -1) if t.dim() == 1 else t.flatten()}[change]
    call, inputs = operators(pkg, cuda)[name]
    kept = []
    with torch.autograd.graph.saved_tensors_hooks(lambda t: kept.append(t) or t, lambda t: t):
        call()
    assert kept
    for i in range(len(kept)):
        if change == "strides" and kept[i].shape == (2, 64):
            continue  # (rows of modulation may have any distance)
        n = []

        def unpack(t):
            n.append(t)
            return how(t) if len(n) == i + 1 else t
        with torch.autograd.graph.saved_tensors_hooks(lambda t: t, unpack):
            y = call()
        with pytest.raises(RuntimeError, match="came back as"):
            torch.autograd.grad(y.float().sum(), list(inputs.values()))


def test_an_unknown_norm_is_the_operators_own_error(pkg):
    x = torch.zeros(1, 4, 64)
    for kw in (dict(kind="batchnorm"), dict(order="both"), dict(kind=None)):
        with pytest.raises(RuntimeError, match="kind must be one of"):
            pkg.ops.norm_modulate_backward(x, x, x[0, 0], **kw)
    with pytest.raises(RuntimeError, match="GPU"):
        pkg.ops.norm_modulate_backward(x, x, x[0, 0])


@pytest.mark.gpu
def test_a_single_token_without_a_row(pkg, cuda):
    """Inputs of one dimension: the bits of a matrix of one row."""
    g, G = torch.Generator().manual_seed(6), pkg.grad
    x, res = normal(g, 64, dtype=BF16).to(cuda), normal(g, 72, dtype=BF16).to(cuda)
    w, w1, w2 = normal(g, 72, 64, dtype=BF16).to(cuda), normal(g, 96, 64, dtype=BF16).to(cuda), normal(g, 64, 48, dtype=BF16).to(cuda)
    for f, *inputs in ((lambda x, r, w: G.linear(x, w, residual=r), x, res, w), (lambda x, r, w: G.linear(x, w, act="silu", residual=r), x, res, w), (G.feed_forward, x, w1, w2)):
        flat = [t.clone().requires_grad_() for t in inputs]
        rows = [(t[None] if t.dim() == 1 else t).clone().requires_grad_() for t in inputs]
        y, want = f(*flat), f(*rows)
        assert y.dim() == 1 and torch.equal(y, want[0])
        dy = normal(g, *y.shape, dtype=BF16).to(cuda)
        for a, b, t in zip(torch.autograd.grad(y, flat, dy), torch.autograd.grad(want, rows, dy[None]), flat):
            assert a.shape == t.shape and torch.equal(a, b.view(a.shape))


@pytest.mark.gpu
def test_two_threads_at_once(pkg, cuda):
    """Each on a stream and on leaves of its own, with the bits of calls alone."""
    from concurrent.futures import ThreadPoolExecutor
    both = [operators(pkg, cuda, seed) for seed in (7, 8)]
    want = [{n: torch.autograd.grad(call().float().sum(), list(t.values())) for n, (call, t) in ops.items()} for ops in both]
    torch.cuda.synchronize()

    def work(ops):
        got = []
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(20):
                got.append({n: torch.autograd.grad(call().float().sum(), list(t.values())) for n, (call, t) in ops.items()})
            torch.cuda.current_stream().synchronize()
        return got
    with ThreadPoolExecutor(2) as pool:
        runs = list(pool.map(work, both))
    for got, w in zip(runs, want):
        for one in got:
            assert all(torch.equal(a, b) for n in w for a, b in zip(one[n], w[n]))


@pytest.mark.gpu
def test_accumulated_gradients_in_a_captured_step(pkg, cuda):
    """Forward and backward pass into ``.grad``, captured and replayed several times beside eager work: as many times the gradients of one pass, and
    the residual's apart from the result's."""
    g, G = torch.Generator().manual_seed(9), pkg.grad
    a, w = torch.randint(-3, 4, (40, 64), generator=g).to(BF16).to(cuda), torch.randint(-3, 4, (16, 64), generator=g).to(BF16).to(cuda)
    dy = torch.randint(-3, 4, (40, 16), generator=g).float().to(cuda)
    kept = dy.clone()
    leaf = {"w": w, "res": torch.zeros(40, 16, device=cuda)}
    for t in leaf.values():
        t.requires_grad_().grad = torch.zeros_like(t)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=torch.cuda.Stream()):
        G.linear(a, leaf["w"], residual=leaf["res"], out_dtype=F32).backward(dy)
    for n in range(1, 4):
        graph.replay()
        torch.cuda.synchronize()
        eager = [t.detach().clone().requires_grad_() for t in leaf.values()]
        once = torch.autograd.grad(G.linear(a, eager[0], residual=eager[1], out_dtype=F32), eager, dy)
        assert torch.equal(dy, kept) and torch.equal(leaf["res"].grad, n * kept)
        assert (leaf["w"].grad.float() - n * once[0].float()).abs().max() <= n * 2 ** -8 * leaf["w"].grad.float().abs().max()  # (a sum of n in bf16: a rounding each)
