"""GPU: the router's balance loss, its counts and the logits' gradient against
64-bit forms; and the layer's operators together around the routed experts.

Tolerances: a score is good to 2^-20 of itself (exponential, reciprocal and the
sum over the experts, each a few units of 2^-24), a block's fp32 sum over at
most 64 tokens adds 64 * 2^-24; everything after that is summed in 64 bits."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def ref64(x, idx, cu, alpha, scoring, grad_loss=None, dw=None, scale=2.5):
    """Loss, counts, tokens, mean scores and the gradient (by autograd in 64 bits, counts constant)."""
    t, e = x.shape
    k = idx.shape[1]
    bounds = cu.tolist() if cu is not None else [0, t]
    xr = x.double().requires_grad_()
    ok = (idx >= 0) & (idx < e)
    real = ok.any(1)
    s = torch.sigmoid(xr)
    p = s / (s.sum(1, keepdim=True) + 1e-20) if scoring == "sigmoid" else torch.softmax(xr, 1)
    hits = torch.zeros(t, e + 1, dtype=torch.float64, device=x.device).scatter_add_(
        1, torch.where(ok, idx, e).long(), ok.double())[:, :e]
    counts, tokens, means, losses = [], [], [], []
    for a, b in zip(bounds, bounds[1:]):
        r = real[a:b]
        n = int(r.sum())
        c = hits[a:b].sum(0)
        mean = p[a:b][r].sum(0) / max(n, 1)
        counts.append(c)
        tokens.append(n)
        means.append(mean)
        if n:
            losses.append((c * e / (k * n) * mean).sum())
    loss = alpha * torch.stack(losses).mean() if losses else torch.zeros((), dtype=torch.float64, device=x.device)
    total = torch.zeros((), dtype=torch.float64, device=x.device) + (s * 0).sum()
    if grad_loss is not None:
        total = total + loss * grad_loss
    if dw is not None:
        top = torch.where(ok, s.gather(1, idx.clamp(0, e - 1).long()), torch.zeros((), dtype=torch.float64, device=x.device))
        total = total + (dw.double() * torch.where(ok, top / (top.sum(1, keepdim=True) + 1e-20) * scale, 0.0 * top)).sum()
    grad, = torch.autograd.grad(total, xr)
    return loss.detach(), torch.stack(counts), torch.tensor(tokens), torch.stack(means).detach(), grad


def inputs(t, e, k, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(t, e, generator=g, device="cuda") * 1.5 + 0.5 * torch.randn(e, generator=g, device="cuda")
    idx = (x + 0.3 * torch.randn(t, e, generator=g, device="cuda")).topk(min(k, e), dim=1).indices.to(torch.int32)
    if t:
        idx = idx.contiguous()
    return x, idx, 0.01 * torch.randn(t, min(k, e), generator=g, device="cuda")


def verify(pkg, x, idx, cu, dw, scoring, alpha=0.02, grad_loss=0.7):
    b = pkg.balance_loss(x, idx, cu_seqlens=cu, alpha=alpha, scoring=scoring)
    g = pkg.balance_loss_backward(x, idx, b, cu_seqlens=cu, grad_loss=grad_loss, alpha=alpha, scoring=scoring, grad_topk_weights=dw)
    loss, counts, tokens, means, grad = ref64(x, idx, cu, alpha, scoring, grad_loss, dw)
    assert torch.equal(b.counts.double(), counts)
    assert b.tokens.tolist() == tokens.tolist() and int(b.sequences) == int((tokens > 0).sum())
    tol = 2.0 ** -18
    assert ((b.mean_scores.double() - means).abs() <= tol * means.abs() + 1e-30).all()
    assert abs(float(b.loss.double() - loss)) <= tol * abs(float(loss)) + 1e-30
    # the gradient is (c_e - sum_j c_j p_j) times a factor of at most max(s (1 - s)) / sum s (softmax: max p): the
    # difference is off by a few 2^-24 of the largest coefficient (it cancels to zero with one expert)
    t, e = x.shape
    bounds = cu.tolist() if cu is not None else [0, t]
    top = torch.zeros(t, 1, dtype=torch.float64, device=x.device)
    for q, (lo, hi) in enumerate(zip(bounds, bounds[1:])):
        n = max(int(tokens[q]), 1)
        top[lo:hi] = alpha * grad_loss * e / (idx.shape[1] * max(int((tokens > 0).sum()), 1) * n * n) * counts[q].max()
    sg = torch.sigmoid(x.double())
    factor = (sg * (1 - sg)).amax(1, keepdim=True) / (sg.sum(1, keepdim=True) + 1e-20) if scoring == "sigmoid" else 1.0
    parts = top * factor
    if dw is not None:
        parts = parts + 2.5 * dw.double().abs().sum(1, keepdim=True)
    assert ((g.double() - grad).abs() <= 2.0 ** -16 * parts + 1e-30).all()
    b2 = pkg.balance_loss(x, idx, cu_seqlens=cu, alpha=alpha, scoring=scoring)
    assert all(torch.equal(u, v) for u, v in zip(b, b2))
    return b, g


@pytest.mark.parametrize("t, e, k", [(1, 256, 8), (2, 8, 2), (7, 1, 1), (63, 33, 3), (64, 256, 8), (65, 64, 4), (300, 257, 6),
                                     (1000, 130, 8), (2049, 512, 8), (100, 1024, 32), (4096, 256, 8)])
@pytest.mark.parametrize("scoring", ["sigmoid", "softmax"])
def test_balance_one_sequence(pkg, t, e, k, scoring):
    x, idx, dw = inputs(t, e, k, seed=t)
    verify(pkg, x, idx, None, dw, scoring)
    verify(pkg, x, idx, None, None, scoring)


@pytest.mark.parametrize("cuts", [[0, 300], [0, 1, 2, 3, 300], [0, 0, 0, 8, 8, 9, 150, 300, 300], [5, 100, 290], [0, 56, 112, 168],
                                  [300, 300], list(range(0, 301))])
@pytest.mark.parametrize("scoring", ["sigmoid", "softmax"])
def test_balance_ragged(pkg, cuts, scoring):
    x, idx, dw = inputs(300, 96, 4, seed=len(cuts))
    cu = torch.tensor(cuts, dtype=torch.int32, device="cuda")
    verify(pkg, x, idx, cu, dw, scoring)


def test_balance_long_packed(pkg):
    t = 5000
    x, idx, dw = inputs(t, 256, 8, seed=2)
    g = torch.Generator().manual_seed(1)
    cuts = torch.cat([torch.tensor([0]), torch.randint(0, t, (37,), generator=g).sort().values, torch.tensor([t])])
    verify(pkg, x, idx, cuts.to(torch.int32).cuda(), dw, "sigmoid")


def test_balance_padding_and_repeats(pkg):
    """Picks of -1 or past E select nothing, tokens without picks count nowhere whatever their logits hold, a
    repeated pick counts twice."""
    x, idx, dw = inputs(200, 64, 4, seed=9)
    idx[3] = -1
    idx[50:90] = torch.tensor([-1, 64, 1 << 30, -(1 << 31)], dtype=torch.int32, device="cuda")
    idx[100, 1] = idx[100, 0]
    idx[101] = idx[101, 2].item()
    idx[102, 3] = -1
    cu = torch.tensor([0, 3, 4, 55, 80, 200], dtype=torch.int32, device="cuda")
    b, g = verify(pkg, x, idx, cu, dw, "sigmoid")
    assert int(b.tokens[1]) == 0 and not g[50:90].any()
    x2 = x.clone()
    x2[50:90] = float("nan")
    b2 = pkg.balance_loss(x2, idx, cu_seqlens=cu, alpha=0.02)
    assert all(torch.equal(u, v) for u, v in zip(b2, b))
    g2 = pkg.balance_loss_backward(x2, idx, b2, cu_seqlens=cu, grad_loss=0.7, alpha=0.02, grad_topk_weights=dw)
    assert torch.equal(g2, g)


@pytest.mark.parametrize("scoring", ["sigmoid", "softmax"])
def test_balance_masked_experts(pkg, scoring):
    """Experts masked by -inf or the lowest float have no score and no gradient; large logits stay finite."""
    x, idx, _ = inputs(50, 64, 4, seed=4)
    x[10] = 200.0
    x[11] = -200.0 if scoring == "softmax" else -60.0
    x[:, 5] = -float("inf")
    x[:, 6] = torch.finfo(torch.float32).min
    idx = (x + 1e-3).topk(4, dim=1).indices.to(torch.int32)
    b = pkg.balance_loss(x, idx, alpha=0.1, scoring=scoring)
    g = pkg.balance_loss_backward(x, idx, b, alpha=0.1, scoring=scoring)
    assert torch.isfinite(b.loss) and torch.isfinite(g).all()
    assert not b.mean_scores[:, 5:7].any() and not g[:, 5:7].any()
    if scoring == "softmax":
        x[12] = -float("inf")                     # a row with nothing to choose from has no scores
        b = pkg.balance_loss(x, idx, alpha=0.1, scoring=scoring)
        assert torch.isfinite(b.loss) and not pkg.balance_loss_backward(x, idx, b, alpha=0.1, scoring=scoring)[12].any()
    x[0, 0] = float("nan")
    assert torch.isnan(pkg.balance_loss(x, idx, alpha=0.1, scoring=scoring).loss)


def test_balance_empty_and_bad_boundaries(pkg):
    x, idx, dw = inputs(40, 32, 2)
    b = pkg.balance_loss(x[:0], idx[:0], cu_seqlens=torch.zeros(4, dtype=torch.int32, device="cuda"))
    assert float(b.loss) == 0 and not b.counts.any() and not b.mean_scores.any() and int(b.sequences) == 0 and b.counts.shape == (3, 32)
    assert pkg.balance_loss_backward(x[:0], idx[:0], b, cu_seqlens=torch.zeros(4, dtype=torch.int32, device="cuda")).shape == (0, 32)
    for cuts in ([0, 30, 20, 40], [-5, 10, 40], [0, 10, 41], [10, 5]):
        cu = torch.tensor(cuts, dtype=torch.int32, device="cuda")
        b = pkg.balance_loss(x, idx, cu_seqlens=cu)
        assert torch.isnan(b.loss)
        pkg.balance_loss_backward(x, idx, b, cu_seqlens=cu)          # in bounds whatever the boundaries are
    torch.cuda.synchronize()


@pytest.mark.parametrize("scoring", ["sigmoid", "softmax"])
def test_balance_bad_boundaries_leave_no_gradient(pkg, scoring):
    x, idx, dw = inputs(40, 32, 2)
    for cuts in ([0, 30, 20, 40], [-5, 10, 40], [0, 10, 41], [10, 5]):
        cu = torch.tensor(cuts, dtype=torch.int32, device="cuda")
        b = pkg.balance_loss(x, idx, cu_seqlens=cu, scoring=scoring)
        assert torch.isnan(b.loss) and int(b.sequences) == -1
        assert torch.isnan(pkg.balance_loss_backward(x, idx, b, cu_seqlens=cu, scoring=scoring)).all()


def test_balance_weights_only_and_refusals(pkg):
    x, idx, dw = inputs(40, 32, 2)
    g = pkg.balance_loss_backward(x, idx, None, grad_topk_weights=dw, routed_scaling_factor=1.5)
    want = ref64(x, idx, None, 0.1, "sigmoid", None, dw, 1.5)[4]
    assert ((g.double() - want).abs() <= 2.0 ** -16 * 1.5 * dw.double().abs().sum(1, keepdim=True)).all()
    assert not pkg.balance_loss_backward(x, idx, None).any()
    b = pkg.balance_loss(x, idx)
    one = pkg.balance_loss_backward(x, idx, b)
    assert torch.equal(one, pkg.balance_loss_backward(x, idx, b, grad_loss=torch.ones((), device="cuda")))
    for bad in (lambda: pkg.balance_loss(x.half(), idx), lambda: pkg.balance_loss(x, idx.long()), lambda: pkg.balance_loss(x, idx[:3]),
                lambda: pkg.balance_loss(x, idx, scoring="top"), lambda: pkg.balance_loss(x, idx, cu_seqlens=idx[0][:1]),
                lambda: pkg.balance_loss(x, idx, cu_seqlens=torch.zeros(2, device="cuda")), lambda: pkg.balance_loss(x.cpu(), idx),
                lambda: pkg.balance_loss_backward(x, idx, None, grad_loss=1.0),
                lambda: pkg.balance_loss_backward(x, idx, b, grad_loss=torch.ones(2, device="cuda")),
                lambda: pkg.balance_loss_backward(x, idx, b, cu_seqlens=torch.tensor([0, 10, 40], dtype=torch.int32, device="cuda")),
                lambda: pkg.balance_loss_backward(x, idx, b, grad_topk_weights=dw[:, :1])):
        with pytest.raises(ValueError):
            bad()


def test_layer_around_the_routed_experts(pkg, oracle):
    """A layer's step: gate -> routed experts -> shared expert added to them, then the router's gradients from the
    balance loss and the combine weights down to the gate's weights, and the shared expert's from 8-bit checkpoints."""
    T, H, I = 48, 7168, 2048
    x = pkg.inputs.make_inputs(T, seed=5, device="cuda", weight_experts=2)
    g = torch.Generator(device="cuda").manual_seed(6)
    rn = lambda *s, f=1.0: (torch.randn(*s, generator=g, device="cuda") * f).to(torch.bfloat16)  # noqa: E731
    h, wg, wu, wd = rn(T, H), rn(256, H, f=H ** -0.5), rn(2 * I, H, f=H ** -0.5), rn(H, I, f=I ** -0.5)
    logits, ck_gate = pkg.linear_checkpointed(h, wg, out_dtype=torch.float32)
    hq, hs = pkg.quantize_activations(h)
    args = list(x.args())
    args[0], args[2], args[3] = logits, hq, hs
    routed = pkg.run(*args)
    idx, weights, counts = pkg.route(logits, x.routing_bias, 0, 256, 2.5)
    mid, ck_up = pkg.linear_checkpointed(h, wu, activation="swiglu")
    out, ck_down = pkg.linear_checkpointed(mid, wd, residual=routed)
    z = h.double() @ wu.double().t()
    m64 = z[:, :I] * z[:, I:] * torch.sigmoid(z[:, I:])
    ref = mid.double() @ wd.double().t() + routed.double()
    assert ((mid.double() - m64).abs() <= 2.0 ** -8 * m64.abs() + 1e-2).all()
    assert ((out.double() - ref).abs() <= 2.0 ** -8 * ref.abs() + 1e-3).all()
    b = pkg.balance_loss(logits, idx, alpha=1e-2)
    assert torch.equal(b.counts[0], counts) and int(b.counts.sum()) == 8 * T
    dweights = 0.1 * torch.randn(T, 8, generator=g, device="cuda")
    dlogits = pkg.balance_loss_backward(logits, idx, b, alpha=1e-2, grad_topk_weights=dweights)
    gate = pkg.linear_backward(dlogits, ck_gate, wg, grad_dtype=torch.float32)
    href = pkg.restore_activations(ck_gate.x, ck_gate.x_scale).double()
    want = dlogits.double().t() @ href
    assert float((gate.weight.double() - want).norm() / want.norm()) < 1e-5
    dout = rn(T, H, f=0.02)
    down = pkg.linear_backward(dout, ck_down, wd)
    up = pkg.linear_backward(down.x, ck_up, wu)
    zr = pkg.restore_activations(ck_up.z, ck_up.z_scale, torch.float32).double()
    s = torch.sigmoid(zr[1])
    dmid = dout.double() @ wd.double()
    dz = torch.cat([dmid * zr[1] * s, dmid * zr[0] * (s + zr[1] * s * (1 - s))], 1)
    want = dz.t() @ href
    # bf16 roundings of dmid, dz and the result: three of 2^-8 at most, far less in the norm
    assert float((up.weight.double() - want).norm() / want.norm()) < 3 * 2.0 ** -8
    # the weights' part of the routing gradient agrees with the weights that route returned
    s = torch.sigmoid(logits.double()).gather(1, idx.long())
    w64 = s / (s.sum(1, keepdim=True) + 1e-20) * 2.5
    assert ((weights.double() - w64).abs() <= 2.0 ** -18 * w64).all()


@pytest.mark.parametrize("e, k, stride", [(8, 8, 1), (16, 8, 3), (256, 8, 5), (64, 32, 7)])
def test_same_experts_in_other_pick_positions(pkg, e, k, stride):
    """Tokens one after the other pick the same experts, each in another position than the token before."""
    t = 20000
    x, _, _ = inputs(t, e, 1, seed=12)
    turn = (torch.arange(t, device="cuda") * stride)[:, None] + torch.arange(k, device="cuda")
    idx = ((turn % k) * (e // k)).to(torch.int32)
    dw = 0.01 * torch.randn(t, k, generator=torch.Generator(device="cuda").manual_seed(3), device="cuda")
    g = pkg.balance_loss_backward(x, idx, None, grad_topk_weights=dw)
    want = ref64(x, idx, None, 0.1, "sigmoid", None, dw)[4]
    assert ((g.double() - want).abs() <= 2.0 ** -16 * 2.5 * dw.double().abs().sum(1, keepdim=True)).all()
    for _ in range(10):
        assert torch.equal(pkg.balance_loss_backward(x, idx, None, grad_topk_weights=dw), g)


@pytest.mark.parametrize("cuts", [[0, 30, 20, 40], [-5, 10, 40], [0, 10, 41], [10, 5], [0, 5, 10, 39, 7, 12, 40], [0, 8, 16, 24, 50]])
def test_bad_boundaries_leave_no_counts_behind(pkg, cuts):
    """Wrong boundaries give the same outputs for every sequence, whatever the workspace and the outputs held before."""
    import ctypes
    import sys
    layer = sys.modules[pkg.__name__ + ".layer"]
    lib = layer._library()
    t, e, k, s = 40, 96, 2, len(cuts) - 1
    x, idx, _ = inputs(t, e, k)
    cu = torch.tensor(cuts, dtype=torch.int32, device="cuda")
    need = lib.moe_balance_workspace_bytes(t, e, s)
    for fill in (0, 1, 127):
        ws = torch.full((need,), fill, dtype=torch.uint8, device="cuda")
        out = torch.full((2 + s + 2 * s * e,), fill, dtype=torch.int32, device="cuda")
        loss, live, tokens, counts, mean = out[:1].view(torch.float32), out[1:2], out[2:2 + s], out[2 + s:2 + s + s * e], out[2 + s + s * e:].view(torch.float32)
        a = layer.MoeBalanceArgs(x.data_ptr(), idx.data_ptr(), cu.data_ptr(), loss.data_ptr(), counts.data_ptr(), tokens.data_ptr(),
                                 mean.data_ptr(), live.data_ptr(), ws.data_ptr(), need, t, e, k, s, 0, 0.1)
        assert lib.moe_balance_loss(ctypes.byref(a), torch.cuda.current_stream().cuda_stream) == 0
        torch.cuda.synchronize()
        assert torch.isnan(loss).all() and torch.isnan(mean).all() and not counts.any()
        assert (tokens == -1).all() and int(live) == -1


def test_boundaries_of_no_tokens(pkg):
    """Without tokens the only right boundaries are zeros."""
    x, idx, _ = inputs(4, 32, 2)
    for cuts, ok in (([0, 0, 0], True), ([0, 3], False), ([0, 0, -1], False), ([2, 2], False)):
        b = pkg.balance_loss(x[:0], idx[:0], cu_seqlens=torch.tensor(cuts, dtype=torch.int32, device="cuda"))
        assert not b.counts.any()
        if ok:
            assert float(b.loss) == 0 and int(b.sequences) == 0 and not b.tokens.any() and not b.mean_scores.any()
        else:
            assert torch.isnan(b.loss) and int(b.sequences) == -1 and (b.tokens == -1).all() and torch.isnan(b.mean_scores).all()


@pytest.mark.parametrize("k", [1, 2, 8])
@pytest.mark.parametrize("masked", [False, True])
def test_what_the_weights_have_in_common_has_no_gradient(pkg, k, masked):
    """A token's combine weights add up to the scale whatever its logits are, so the part of their gradients that is the same for all
    picks of a token cancels: for one pick that is everything, and it is not a remainder of rounding that is left."""
    t, e = 3000, 64
    x, idx, _ = inputs(t, e, k, seed=7)
    if masked and k > 1:
        idx[:, 0] = -1
    common = torch.randn(t, 1, generator=torch.Generator(device="cuda").manual_seed(1), device="cuda").expand(t, k).contiguous()
    g = pkg.balance_loss_backward(x, idx, None, grad_topk_weights=common)
    # what is left is dw scale 1e-20 / S^2 s (1 - s); S is above 1e-4 here
    assert (g.abs() <= 2.5 * common.abs().amax(1, keepdim=True) * 1e-20 * 1e8).all()
    own = common + 0.01 * torch.randn(t, k, generator=torch.Generator(device="cuda").manual_seed(2), device="cuda")
    g = pkg.balance_loss_backward(x, idx, None, grad_topk_weights=own)
    ok = (idx >= 0)
    spread = torch.where(ok, own - own[:, -1:], 0.0).double().abs().sum(1, keepdim=True)
    want = ref64(x, idx, None, 0.1, "sigmoid", None, own, 2.5)[4]
    assert ((g.double() - want).abs() <= 2.0 ** -16 * 2.5 * spread + 1e-12).all()


@pytest.mark.parametrize("e, k", [(1, 1), (8, 2), (64, 4), (256, 8)])
@pytest.mark.parametrize("scoring", ["sigmoid", "softmax"])
def test_balanced_counts_have_no_gradient(pkg, e, k, scoring):
    """Where every expert is picked equally often the loss does not depend on the logits; one pick more leaves that pick's part,
    not a remainder of rounding of the rest."""
    t = 8 * e // k * 32
    x, _, _ = inputs(t, e, 1, seed=3)
    idx = (torch.arange(t * k, device="cuda") % e).view(t, k).to(torch.int32)
    b = pkg.balance_loss(x, idx, alpha=1.0, scoring=scoring)
    assert (b.counts == t * k // e).all()
    g = pkg.balance_loss_backward(x, idx, b, alpha=1.0, scoring=scoring)
    # what is left of c (1 - sum p): c 1e-20 / S, twice over S, with S above 1e-4 and c = e / (k t^2) t k / e = 1 / t
    assert (g.abs() <= 1e-20 * 1e8 / t).all()
    if e > 1:
        idx[5, 0] = idx[5, k - 1] if k > 1 else (idx[5, 0] + 1) % e
        b = pkg.balance_loss(x, idx, alpha=1.0, scoring=scoring)
        g = pkg.balance_loss_backward(x, idx, b, alpha=1.0, scoring=scoring)
        want = ref64(x, idx, None, 1.0, scoring, 1.0)[4]
        # two coefficients are off the common one by e / (k t^2); the factors are good to 2^-20
        s = torch.sigmoid(x.double())
        factor = (s * (1 - s)).amax(1, keepdim=True) / (s.sum(1, keepdim=True) + 1e-20) if scoring == "sigmoid" else 1.0
        assert ((g.double() - want).abs() <= 2.0 ** -16 * e / (k * t * t) * factor + 1e-12 / t).all()


@pytest.mark.parametrize("t, cuts", [(65534, list(range(65535))), (100, [0] * 30000 + [50] * 30000 + [100])])
def test_balance_most_sequences(pkg, t, cuts):
    """A sequence per token, and tens of thousands of empty ones in one place."""
    e, k, s = 8, 2, len(cuts) - 1
    x, idx, _ = inputs(t, e, k, seed=5)
    cu = torch.tensor(cuts, dtype=torch.int32, device="cuda")
    b = pkg.balance_loss(x, idx, cu_seqlens=cu, alpha=0.1)
    g = pkg.balance_loss_backward(x, idx, b, cu_seqlens=cu, alpha=0.1)
    tokens = cu.diff().double()[:, None]
    seq = torch.repeat_interleave(torch.arange(s, device="cuda"), cu.diff().long())
    counts = torch.zeros(s, e, dtype=torch.float64, device="cuda").index_put_(
        (seq[:, None].expand(t, k), idx.long()), torch.ones((), dtype=torch.float64, device="cuda"), accumulate=True)
    sg = torch.sigmoid(x.double())
    p = sg / (sg.sum(1, keepdim=True) + 1e-20)
    freq = counts * e / (k * tokens.clamp(min=1))
    live = int((tokens > 0).sum())
    mean = torch.zeros_like(counts).index_add_(0, seq, p) / tokens.clamp(min=1)
    loss = 0.1 * (freq * mean).sum() / live
    assert torch.equal(b.counts.double(), counts) and torch.equal(b.tokens.double(), tokens[:, 0]) and int(b.sequences) == live
    assert abs(float(b.loss.double() - loss)) <= 2.0 ** -18 * float(loss)
    c = (0.1 * freq / (tokens.clamp(min=1) * live))[seq]
    want = (c - (c * p).sum(1, keepdim=True)) / (sg.sum(1, keepdim=True) + 1e-20) * sg * (1 - sg)
    top = c.amax(1, keepdim=True) * (sg * (1 - sg)).amax(1, keepdim=True) / sg.sum(1, keepdim=True)
    assert ((g.double() - want).abs() <= 2.0 ** -16 * top).all()
