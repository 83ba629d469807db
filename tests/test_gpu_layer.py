"""GPU: dense products, 8-bit checkpoints and gradients against 64-bit forms.

Tolerances. A product summed in fp32 is off by at most K * 2^-23 * sum |x||w|
(an addition that truncates loses up to 2^-23 of the running sum); rounding to
bf16 loses at most 2^-8 of the value, to e4m3 2^-4 of it (2^-10 of the block's
scale below the normal numbers). The activations' slopes are at most 1.13 and
their own fp32 evaluation is good to 2^-20 of 1 + |z|."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

ACTS = ("none", "relu", "gelu", "silu", "swiglu")
BF, F32 = torch.bfloat16, torch.float32


def randn(*shape, seed=0, scale=1.0, dtype=BF):
    g = torch.Generator(device="cuda").manual_seed(seed + 1000 * sum(shape))
    return (torch.randn(*shape, generator=g, device="cuda") * scale).to(dtype)


def act64(z, act):
    if act == "none":
        return z
    if act == "relu":
        return z.clamp(min=0)
    if act == "gelu":
        return z * 0.5 * torch.erfc(-z / math.sqrt(2))
    if act == "silu":
        return z * torch.sigmoid(z)
    a, b = z.chunk(2, dim=-1)
    return a * b * torch.sigmoid(b)


def dense64(x, w, b=None):
    z = x.double() @ w.double().t()
    mag = x.double().abs() @ w.double().abs().t()
    if b is not None:
        z, mag = z + b.double(), mag + b.double().abs()
    return z, mag * ((x.shape[1] + 2) * 2.0 ** -23) + 1e-30


def tol_act(z, tz, act):
    """Error of act(z) in fp32 from an error tz of z."""
    if act == "swiglu":
        a, b = z.chunk(2, dim=-1)
        ta, tb = tz.chunk(2, dim=-1)
        return ta * (b.abs() + 1) + (a.abs() + ta) * 1.13 * tb + 2.0 ** -20 * (1 + b.abs()) * a.abs()
    return 1.13 * tz + (2.0 ** -20 * (1 + z.abs()) if act != "none" else 0)


def check(got, ref, tol, what):
    got = got.double()
    assert got.shape == ref.shape, what
    bad = ~((got - ref).abs() <= tol)
    assert not bad.any(), (f"{what}: {int(bad.sum())} of {bad.numel()} outside, worst "
                           f"{float(((got - ref).abs() - tol).max()):.3e} over, first at {bad.nonzero()[0].tolist()}")


def rounded(ref, tol, dtype):
    return tol + (ref.abs() + tol) * (2.0 ** -8 if dtype == BF else 2.0 ** -23) + 1e-38


def linear_case(pkg, m, k, n, act="none", bias=False, res=False, dtype=BF, x=None, w=None):
    x = randn(m, k, seed=1) if x is None else x
    w = randn(n, k, seed=2, scale=k ** -0.5) if w is None else w
    b = randn(n, seed=3, scale=0.3) if bias else None
    o = n // 2 if act == "swiglu" else n
    r = randn(m, o, seed=4) if res else None
    y = pkg.linear(x, w, bias=b, residual=r, activation=act, out_dtype=dtype)
    z, tz = dense64(x, w, b)
    ref, tol = act64(z, act), tol_act(z, tz, act)
    if res:
        ref = ref + r.double()
        tol = tol + ref.abs() * 2.0 ** -23
    assert y.dtype == dtype
    check(y, ref, rounded(ref, tol, dtype), f"linear {m}x{k}x{n} {act}")
    return y


SIZES = [(1, 7168, 256), (1, 8, 1), (2, 64, 16), (3, 72, 130), (7, 7168, 64), (8, 2048, 512), (9, 128, 264), (16, 256, 48),
         (17, 320, 96), (32, 512, 128), (33, 512, 128), (64, 7168, 512), (127, 64, 256), (128, 192, 256), (129, 200, 264),
         (255, 640, 96), (256, 64, 512), (257, 72, 520), (300, 7168, 256), (600, 2048, 1032), (1000, 136, 2050)]


@pytest.mark.parametrize("m, k, n", SIZES)
@pytest.mark.parametrize("act", ["none", "swiglu"])
def test_linear_sizes(pkg, m, k, n, act):
    if act == "swiglu" and n % 2:
        n += 1
    linear_case(pkg, m, k, n, act)


@pytest.mark.parametrize("m", [33, 64, 65, 97, 128])
@pytest.mark.parametrize("k, n, act, dtype", [(7168, 1030, "swiglu", BF), (2048, 7168, "none", BF), (7168, 300, "none", F32),
                                              (520, 515, "gelu", BF), (20000, 130, "silu", F32)])
def test_linear_few_tokens(pkg, m, k, n, act, dtype):
    linear_case(pkg, m, k, n, act, True, True, dtype)


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("m, k, n", [(5, 96, 80), (40, 96, 80), (300, 520, 390), (520, 1024, 768)])
def test_linear_epilogues(pkg, m, k, n, act):
    for bias, res, dtype in ((True, False, BF), (False, True, BF), (True, True, F32), (False, False, F32)):
        linear_case(pkg, m, k, n, act, bias, res, dtype)


@pytest.mark.parametrize("m", [1, 6, 31, 70, 400])
@pytest.mark.parametrize("k, n", [(1, 1), (7, 3), (65, 33), (129, 257), (1001, 130)])
def test_linear_odd_sizes(pkg, m, k, n):
    linear_case(pkg, m, k, n, "gelu", True, True)
    linear_case(pkg, m, k, 2 * n, "swiglu", True, True, F32)


@pytest.mark.parametrize("m", [4, 50, 300])
def test_linear_strides_and_offsets(pkg, m):
    """Row strides, misaligned bases, transposed and expanded inputs."""
    big = randn(m + 1, 300, seed=5)
    wbig = randn(200, 300, seed=6, scale=0.1)
    for c0, k in ((0, 128), (8, 128), (1, 128), (3, 77)):
        linear_case(pkg, m, k, 96, "silu", x=big[1:, c0:c0 + k], w=wbig[7:103, c0:c0 + k])
    linear_case(pkg, m, 64, 96, x=randn(64, m, seed=7).t(), w=randn(64, 96, seed=8).t())
    linear_case(pkg, m, 64, 96, x=randn(1, 64, seed=9).expand(m, 64))
    x, w = randn(m, 64, seed=10), randn(96, 64, seed=11)
    r = randn(1, 96, seed=12).expand(m, 96)
    wide = randn(m, 200, seed=13)
    for out in (None, torch.empty(m, 96, dtype=BF, device="cuda"), wide[:, 3:99], torch.empty(96, m, dtype=BF, device="cuda").t()):
        before = wide.clone()
        y = pkg.linear(x, w, residual=r, output=out)
        z, tz = dense64(x, w)
        check(y, z + r.double(), rounded(z + r.double(), tz * 2, BF), "strided")
        if out is not None:
            assert y is out
        assert torch.equal(wide[:, :3], before[:, :3]) and torch.equal(wide[:, 99:], before[:, 99:])


@pytest.mark.parametrize("m", [5, 200])
def test_linear_in_place_residual(pkg, m):
    x, w, r = randn(m, 256, seed=1), randn(128, 256, seed=2, scale=0.06), randn(m, 128, seed=3)
    want = pkg.linear(x, w, residual=r)
    got = pkg.linear(x, w, residual=r, output=r)
    assert got is r and torch.equal(got, want)


@pytest.mark.parametrize("m", [1, 12, 90, 700])
def test_linear_non_finite(pkg, m):
    """A NaN or infinity stays in its row (x) or column (weight); rows past the matrix do not leak in."""
    x, w = randn(m, 192, seed=1), randn(80, 192, seed=2)
    clean = pkg.linear(x, w)
    x2 = x.clone()
    x2[m // 2, 100] = float("nan")
    y = pkg.linear(x2, w)
    assert torch.isnan(y[m // 2]).all()
    keep = torch.arange(m, device="cuda") != m // 2
    assert torch.equal(y[keep], clean[keep])
    w2 = w.clone()
    w2[11, 3] = float("inf")
    y = pkg.linear(x, w2)
    cols = torch.arange(80, device="cuda") != 11
    assert torch.equal(y[:, cols], clean[:, cols]) and not torch.isfinite(y[:, 11]).any()
    big = torch.full((m, 192), float("nan"), dtype=BF, device="cuda")
    xs = torch.cat([x, big])[:m]                   # NaN rows lie right behind the last one
    assert torch.equal(pkg.linear(xs, w), clean)


def test_linear_empty_and_refusals(pkg):
    x, w = randn(4, 64), randn(32, 64)
    assert pkg.linear(x[:0], w).shape == (0, 32)
    bad = [dict(x=x[0]), dict(x=x.float()), dict(weight=w[:, :32]), dict(weight=w.float()), dict(weight=w.cpu()),
           dict(bias=randn(31)), dict(bias=randn(32).float()), dict(residual=randn(4, 31)), dict(residual=randn(4, 32).float()),
           dict(activation="tanh"), dict(weight=randn(31, 64), activation="swiglu"), dict(out_dtype=torch.float16),
           dict(output=torch.empty(4, 31, dtype=BF, device="cuda")), dict(output=torch.empty(4, 32, device="cuda")),
           dict(output=torch.empty(4, 32, dtype=BF)), dict(weight=w[:0]), dict(x=x[:, :0], weight=w[:, :0])]
    for kw in bad:
        with pytest.raises(ValueError):
            pkg.linear(**{"x": x, "weight": w, **kw})
    sq = randn(64, 64)
    with pytest.raises(ValueError, match="overlaps x"):
        pkg.linear(sq, sq.clone(), output=sq)
    r = randn(9, 64)
    with pytest.raises(ValueError, match="residual"):
        pkg.linear(sq[:8], sq, residual=r[:8], output=r[1:])


@pytest.mark.parametrize("m, k, n", [(5, 64, 40), (90, 72, 37), (700, 128, 96)])
def test_linear_columns_of_one_buffer(pkg, m, k, n):
    """x, y and the residual as columns side by side: the neighbours stay as they are."""
    buf = randn(m, k + 2 * n + 3, seed=5)
    before, w = buf.clone(), randn(n, k, seed=6, scale=0.1)
    x, y, r = buf[:, :k], buf[:, k:k + n], buf[:, k + n:k + 2 * n]
    want = pkg.linear(x, w, residual=r)
    pkg.linear(x, w, residual=r, output=y)
    assert torch.equal(y, want)
    buf[:, k:k + n] = before[:, k:k + n]
    assert torch.equal(buf, before)
    with pytest.raises(ValueError, match="overlaps x"):
        pkg.linear(x, w, output=buf[:, k - 1:k - 1 + n])


def test_linear_residual_of_another_type_in_the_same_place(pkg):
    x, w, out = randn(8, 64), randn(64, 64), torch.zeros(8, 64, device="cuda")
    r = out.view(BF).as_strided((8, 64), (64, 1))
    with pytest.raises(ValueError, match="residual"):
        pkg.linear(x, w, residual=r, output=out, out_dtype=F32)


# --------------------------------------------------------------------------------- checkpoints
def quantize64(x):
    """(values, codes) of the format, element by element in 64 bits."""
    t, k = x.shape
    v = torch.nn.functional.pad(x.double(), (0, -k % 128)).view(t, -1, 128)
    amax = v.abs().amax(-1, keepdim=True)
    e = torch.full_like(amax, -117.0)
    for p in range(-116, 121):                      # the least e with amax <= 448 * 2^e
        e = torch.where(amax > 448.0 * 2.0 ** (p - 1), torch.full_like(e, p), e)
    s = v / torch.exp2(e)
    s = torch.where(e == 120, s.clamp(-240, 240), s)          # 256 * 2^120 would be infinite
    ex = torch.floor(torch.log2(s.abs().clamp(min=2.0 ** -30))).clamp(min=-6)
    step = torch.exp2(ex - 3)
    out = torch.round(s / step) * step * torch.exp2(e)
    return out.flatten(1)[:, :k], (e.squeeze(-1).t() + 127).to(torch.uint8)


@pytest.mark.parametrize("t, k", [(1, 1), (1, 128), (2, 7168), (3, 129), (31, 1000), (33, 136), (64, 7168), (65, 2047),
                                  (513, 1024), (4099, 264)])
@pytest.mark.parametrize("dtype", [BF, F32])
def test_checkpoint_round_trip(pkg, t, k, dtype):
    x = randn(t, k, dtype=F32)
    x = (x * torch.exp(2 * randn(1, k, seed=5, dtype=F32)) * torch.exp2(randn(t, 1, seed=6, dtype=F32) * 20)).to(dtype)
    x[0, : k // 2] = 0
    q, s = pkg.checkpoint_activations(x)
    assert q.dtype == torch.float8_e4m3fn and s.dtype == torch.float8_e8m0fnu and s.shape == (-(-k // 128), t)
    want, codes = quantize64(x)
    assert torch.equal(s.view(torch.uint8), codes)
    for out in (BF, F32):
        r = pkg.restore_activations(q, s, out)
        assert r.dtype == out and torch.equal(r.double(), want)
    assert ((want - x.double()).abs() <= 2.0 ** -4 * x.double().abs() + torch.exp2(
        codes.double() - 127 - 10).t().repeat_interleave(128, 1)[:, :k]).all()


def test_checkpoint_edges(pkg):
    """Borders of the scale (448 * 2^e and its neighbours), the smallest and largest values, zero blocks, NaN and infinity."""
    tops = []
    for e in (-140, -126, -125, -117, -100, -3, 0, 5, 90, 118, 119):
        v = 448.0 * 2.0 ** e
        tops += [v, v * (1 + 2.0 ** -7), v * (1 - 2.0 ** -8), v / 1.75, v / 1.75 * (2 - 2.0 ** -7)]
    tops += [0.0, 1e-45, 1.1754944e-38, 3.38e38]
    x = torch.zeros(len(tops), 128, device="cuda", dtype=F32)
    x[:, 17] = torch.tensor(tops, dtype=torch.float64).to(F32)
    x[:, 18] = -x[:, 17] / 3
    x[:, 19] = x[:, 17] * 2.0 ** -17
    q, s = pkg.checkpoint_activations(x)
    want, codes = quantize64(x)
    assert torch.equal(s.view(torch.uint8), codes)
    assert torch.equal(pkg.restore_activations(q, s).double(), want)
    y = randn(4, 300)
    clean = pkg.restore_activations(*pkg.checkpoint_activations(y))
    for bad in (float("nan"), float("inf"), -float("inf")):
        z = y.clone()
        z[2, 140] = bad
        got = pkg.restore_activations(*pkg.checkpoint_activations(z))
        assert torch.isnan(got[2, 128:256]).all()
        got[2, 128:256] = clean[2, 128:256]
        assert torch.equal(got, clean)


def test_checkpoint_strides_batch_and_refusals(pkg):
    x = randn(40, 700)
    for v in (x[3:30, 5:400], x[::2, 8:264], x.t(), x[:1, 1:129]):
        q, s = pkg.checkpoint_activations(v)
        q2, s2 = pkg.checkpoint_activations(v.contiguous())
        assert torch.equal(q.view(torch.uint8), q2.view(torch.uint8)) and torch.equal(s.view(torch.uint8), s2.view(torch.uint8))
    a, b = pkg.checkpoint_activations(x), pkg.checkpoint_activations(-x)
    q, s = torch.stack([a[0].view(torch.uint8), b[0].view(torch.uint8)]), torch.stack([a[1].view(torch.uint8), b[1].view(torch.uint8)])
    r = pkg.restore_activations(q.view(torch.float8_e4m3fn), s.view(torch.float8_e8m0fnu))
    assert torch.equal(r[0], pkg.restore_activations(*a)) and torch.equal(r[1], -r[0])
    q, s = pkg.checkpoint_activations(x[:0])
    assert q.shape == (0, 700) and pkg.restore_activations(q, s).shape == (0, 700)
    for bad in (lambda: pkg.checkpoint_activations(x.half()), lambda: pkg.checkpoint_activations(x.cpu()),
                lambda: pkg.restore_activations(a[0], a[1][1:]), lambda: pkg.restore_activations(x, a[1]),
                lambda: pkg.restore_activations(a[0], a[1], torch.float16), lambda: pkg.restore_activations(a[0], a[1].cpu())):
        with pytest.raises(ValueError):
            bad()


# --------------------------------------------------------------------------------- training pass
def act_slope64(z, act):
    if act == "relu":
        return (z > 0).double()
    s = torch.sigmoid(z)
    if act == "silu":
        return s * (1 + z * (1 - s))
    return 0.5 * torch.erfc(-z / math.sqrt(2)) + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)


def grads64(pkg, dy, ck, w):
    """64-bit gradients from the checkpoint's values, with the magnitudes the tolerances need."""
    x = pkg.restore_activations(ck.x, ck.x_scale, F32).double()
    dz = dy.double()
    if ck.activation == "swiglu":
        a, b = pkg.restore_activations(ck.z, ck.z_scale, F32).double()
        s = torch.sigmoid(b)
        dz = torch.cat([dz * b * s, dz * a * (s + b * s * (1 - s))], 1)
    elif ck.activation != "none":
        dz = dz * act_slope64(pkg.restore_activations(ck.z, ck.z_scale, F32).double(), ck.activation)
    return x, dz


TRAIN = [(1, 64, 32), (3, 8, 2), (30, 200, 130), (64, 128, 256), (130, 96, 264), (300, 1000, 390), (513, 512, 512),
         (600, 7168, 256), (1100, 264, 1040)]


@pytest.mark.parametrize("m, k, n", TRAIN)
@pytest.mark.parametrize("act", ACTS)
def test_linear_checkpointed(pkg, m, k, n, act):
    x, w, b = randn(m, k, seed=1), randn(n, k, seed=2, scale=k ** -0.5), randn(n, seed=3)
    y, ck = pkg.linear_checkpointed(x, w, bias=b, activation=act)
    z, tz = dense64(x, w, b)
    ref = act64(z, act)
    check(y, ref, rounded(ref, tol_act(z, tz, act), BF), "y")
    q, s = pkg.checkpoint_activations(x)
    assert torch.equal(ck.x.view(torch.uint8), q.view(torch.uint8)) and torch.equal(ck.x_scale.view(torch.uint8), s.view(torch.uint8))
    assert ck.activation == act
    if act == "none":
        assert ck.z is None and ck.z_scale is None
        return
    zs = z.chunk(2, 1) if act == "swiglu" else (z,)
    ts = tz.chunk(2, 1) if act == "swiglu" else (tz,)
    got = pkg.restore_activations(ck.z, ck.z_scale, F32)
    got = got if act == "swiglu" else got[None]
    codes = ck.z_scale.view(torch.uint8)
    codes = codes if act == "swiglu" else codes[None]
    for h, (zz, tt) in enumerate(zip(zs, ts)):
        scale = torch.exp2(codes[h].double() - 127).t().repeat_interleave(128, 1)[:, : zz.shape[1]]
        check(got[h], zz, 2.0 ** -4 * (zz.abs() + tt) + 2.0 ** -10 * scale + tt, "z")
        # the scale is the least that holds the block, up to the error of its largest value
        amax = torch.nn.functional.pad(zz.abs(), (0, -zz.shape[1] % 128)).unflatten(1, (-1, 128)).amax(-1).t()
        slack = torch.nn.functional.pad(tt, (0, -tt.shape[1] % 128)).unflatten(1, (-1, 128)).amax(-1).t()
        sc = torch.exp2(codes[h].double() - 127)
        assert (amax - slack <= 448 * sc).all() and ((amax + slack > 224 * sc) | (codes[h] == 10)).all()


@pytest.mark.parametrize("m, k, n", [(20, 64, 64), (300, 192, 512), (700, 264, 1040), (2600, 128, 2048)])
@pytest.mark.parametrize("act", ["none", "gelu", "swiglu"])
@pytest.mark.parametrize("dtype", [BF, F32])
def test_linear_checkpointed_with_residual(pkg, m, k, n, act, dtype):
    """The kept blocks do not change with a residual or the output's type, and y is linear()'s up to its rounding."""
    x, w, b = randn(m, k, seed=1), randn(n, k, seed=2, scale=k ** -0.5), randn(n, seed=3)
    r = randn(m, n // 2 if act == "swiglu" else n, seed=4)
    y, ck = pkg.linear_checkpointed(x, w, bias=b, residual=r, activation=act, out_dtype=dtype)
    z, tz = dense64(x, w, b)
    ref = act64(z, act) + r.double()
    check(y, ref, rounded(ref, tol_act(z, tz, act) + ref.abs() * 2.0 ** -23, dtype), "y")
    plain = pkg.linear_checkpointed(x, w, bias=b, activation=act)[1]
    if act != "none":
        assert torch.equal(ck.z.view(torch.uint8), plain.z.view(torch.uint8))
        assert torch.equal(ck.z_scale.view(torch.uint8), plain.z_scale.view(torch.uint8))
    own = r.clone() if dtype == BF else None
    if own is not None:
        got = pkg.linear_checkpointed(x, w, bias=b, residual=own, activation=act, output=own)[0]
        assert got is own and torch.equal(own, y)


@pytest.mark.parametrize("m, k, n", TRAIN)
@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("gin, gout", [(BF, BF), (F32, F32), (F32, BF), (BF, F32)])
def test_linear_backward(pkg, m, k, n, act, gin, gout):
    x, w = randn(m, k, seed=1), randn(n, k, seed=2, scale=k ** -0.5)
    y, ck = pkg.linear_checkpointed(x, w, activation=act)
    dy = randn(m, y.shape[1], seed=5, dtype=gin)
    g = pkg.linear_backward(dy, ck, w, need_bias=True, grad_dtype=gout)
    xr, dz = grads64(pkg, dy, ck, w)
    # dz: fp32 evaluation (2^-20 of its factors), then bf16 (2^-8), or three bf16 terms (its 24 bits)
    exact = act == "none" and gin == BF
    rel = (0 if act == "none" else 2.0 ** -19) + (0 if exact else 2.0 ** -8 if gout == BF else 2.0 ** -23)
    mag = dz.abs() + 2.0 ** -6 * dy.double().abs().repeat(1, 2 if act == "swiglu" else 1) * (act != "none")
    zmag = 1.0
    if act == "swiglu":
        zr = pkg.restore_activations(ck.z, ck.z_scale, F32).double().abs()
        zmag = 1 + torch.cat([zr[1], zr[0]], 1)
    ez = mag * rel + (2.0 ** -19 * dy.double().abs().repeat(1, 2 if act == "swiglu" else 1) * zmag if act != "none" else 0)
    ww = w.double()
    ref = dz @ ww
    check(g.x, ref, rounded(ref, ez @ ww.abs() + 3 * (n + 2) * 2.0 ** -23 * (dz.abs() @ ww.abs()) + 1e-30, gout), "grad_x")
    ref = dz.t() @ xr
    check(g.weight, ref, rounded(ref, ez.t() @ xr.abs() + 3 * (m + 2) * 2.0 ** -23 * (dz.abs().t() @ xr.abs()) + 1e-30, gout), "grad_weight")
    ref = dz.sum(0)
    eb = (mag * (0 if act == "none" else 2.0 ** -19)).sum(0) + (ez.sum(0) if act == "swiglu" else 0) + (m + 2) * 2.0 ** -23 * dz.abs().sum(0)
    eb = eb + (2.0 ** -19 * dy.double().abs().sum(0) if act not in ("none", "swiglu") else 0)
    check(g.bias, ref, rounded(ref, eb + 1e-30, gout), "grad_bias")
    assert g.x.dtype == g.weight.dtype == g.bias.dtype == gout
    again = pkg.linear_backward(dy, ck, w, need_bias=True, grad_dtype=gout)
    assert all(torch.equal(a, b) for a, b in zip(g, again))
    only = pkg.linear_backward(dy, ck, w, need_x=False, need_weight=False, need_bias=True, grad_dtype=gout)
    assert only.x is None and only.weight is None and torch.equal(only.bias, g.bias)
    assert torch.equal(pkg.linear_backward(dy, ck, w, need_weight=False, grad_dtype=gout).x, g.x)
    assert torch.equal(pkg.linear_backward(dy, ck, w, need_x=False, grad_dtype=gout).weight, g.weight)


@pytest.mark.parametrize("m, n", [(4, 1), (40, 1), (300, 96), (300, 97)])
@pytest.mark.parametrize("keep", [False, True])
def test_gelu_far_below_zero(pkg, m, n, keep):
    """gelu(z) = z Phi(z) keeps its value down to where Phi leaves the normal numbers. In fp32 a value is
    off by the rounding of z^2 / 2, whose exponential multiplies it (z^2 / 4 units of 2^-23), and by a few units of the
    exponential, a reciprocal and a product of polynomials: z^2 + 8 together."""
    z = torch.linspace(-13, 1, m * n, device="cuda").view(m, n)
    x = torch.zeros(m, 128, device="cuda", dtype=BF)
    w = torch.zeros(n, 128, device="cuda", dtype=BF)
    x[:, 0] = 1                                                # z = bias + x_1: both in bf16
    x[:, 1] = z[:, 0].to(BF)
    w[:, 1] = 1
    b = (z[0] - z[0, 0]).to(BF)
    z = x[:, 1:2].double() + b.double()
    z32 = z.float().double()                                   # what fp32 holds of it
    f = pkg.linear_checkpointed if keep else pkg.linear
    y = f(x, w, bias=b, activation="gelu", out_dtype=F32)
    y = y[0] if keep else y
    ref = act64(z32, "gelu")
    assert ((y.double() - ref).abs() <= ref.abs() * (z32 * z32 + 8) * 2.0 ** -23 + 1e-37).all()
    yb = f(x, w, bias=b, activation="gelu")
    yb = yb[0] if keep else yb
    assert ((yb.double() - ref).abs() <= ref.abs() * (2.0 ** -8 + (z32 * z32 + 8) * 2.0 ** -22) + 1e-37).all()


@pytest.mark.parametrize("gout", [BF, F32])
@pytest.mark.parametrize("n", [8, 9])
def test_gelu_slope_far_below_zero(pkg, gout, n):
    """Phi(z) + z phi(z) at values that the checkpoint holds exactly; for bf16 gradients the exponential is the hardware's,
    2^-21 of the larger of 1 and its exponent z^2 / 2."""
    z = torch.tensor([-12.0, -11, -10, -9, -8, -7.5, -7, -6.5, -6, -5.5, -5, -4, -3.5, -3, -2, -1, -0.5, 0, 0.5, 1, 3, 8], device="cuda")
    z8, zs = pkg.checkpoint_activations(z[:, None].expand(-1, n).contiguous())
    assert torch.equal(pkg.restore_activations(z8, zs, F32)[:, 0], z)
    x8, xs = pkg.checkpoint_activations(torch.ones(z.numel(), n, device="cuda"))
    g = pkg.linear_backward(torch.ones(z.numel(), n, device="cuda"), pkg.LinearCheckpoint(x8, xs, z8, zs, "gelu"),
                            torch.eye(n, device="cuda").to(BF), grad_dtype=gout)
    zz = z.double()
    phi, cdf = zz * torch.exp(-zz * zz / 2) / math.sqrt(2 * math.pi), 0.5 * torch.erfc(-zz / math.sqrt(2))
    tol = (cdf + phi.abs()) * (zz * zz + 8) * (2.0 ** -20 if gout == BF else 2.0 ** -22)
    tol = tol + ((cdf + phi).abs() + tol) * (2.0 ** -8 if gout == BF else 2.0 ** -23) + 1e-36
    assert ((g.x.double() - (cdf + phi)[:, None]).abs() <= tol[:, None]).all()


@pytest.mark.parametrize("act", ACTS)
def test_backward_against_differences(pkg, act):
    """The gradients are those of the forward: with inputs whose checkpoints are exact (few-bit values, one
    scale), a central difference of sum(y * dy) in 64 bits agrees to the difference's own error."""
    g = torch.Generator(device="cuda").manual_seed(3)
    m, k, n = 5, 16, 8
    x = torch.randint(-4, 5, (m, k), generator=g, device="cuda").double() / 4
    w = torch.randint(-4, 5, (n, k), generator=g, device="cuda").double() / 8
    x8, xs = pkg.checkpoint_activations(x.to(BF))
    assert torch.equal(pkg.restore_activations(x8, xs).double(), x)
    z = x @ w.t()
    if act == "relu":
        z = torch.where(z == 0, z + 0.5, z)
    zq = torch.stack(z.chunk(2, 1)) if act == "swiglu" else z
    pairs = [pkg.checkpoint_activations(h.float().contiguous()) for h in (zq if act == "swiglu" else zq[None])]
    st = lambda i, d: torch.stack([p[i].view(torch.uint8) for p in pairs]).view(d)  # noqa: E731
    z8, zs = st(0, torch.float8_e4m3fn), st(1, torch.float8_e8m0fnu)
    zr = pkg.restore_activations(z8, zs, F32).double()
    zr = torch.cat(list(zr), 1) if act == "swiglu" else zr[0]
    ck = pkg.LinearCheckpoint(x8, xs, None if act == "none" else z8 if act == "swiglu" else z8[0],
                              None if act == "none" else zs if act == "swiglu" else zs[0], act)
    if act == "none":
        zr = z
    o = n // 2 if act == "swiglu" else n
    dy = torch.randint(-8, 9, (m, o), generator=g, device="cuda").double() / 8
    got = pkg.linear_backward(dy.float(), ck, w.to(BF), need_bias=True, grad_dtype=F32)
    h = 1e-4

    def f(dz):      # the loss along a change of the pre-activation, from the checkpoint's own point
        return (act64(zr + dz, act) * dy).sum()

    for name, grad, shape, change in (("x", got.x, (m, k), lambda d: d @ w.t()), ("weight", got.weight, (n, k), lambda d: x @ d.t()),
                                      ("bias", got.bias, (n,), lambda d: d.expand(m, n))):
        for t in range(6):
            d = torch.randn(shape, generator=g, device="cuda", dtype=torch.float64)
            dz = change(d)
            diff = (f(h * dz) - f(-h * dz)) / (2 * h)
            # third derivatives of the activations are below 2 (times the other factor for swiglu)
            tol = h * h * (dz.abs() ** 3).sum() * 4 + 1e-4 * (grad.double() * d).abs().sum() + 1e-9
            assert abs(float((grad.double() * d).sum() - diff)) <= float(tol), (act, name)


def test_backward_refusals_and_empty(pkg):
    x, w = randn(4, 64), randn(32, 64)
    y, ck = pkg.linear_checkpointed(x, w, activation="silu")
    dy = torch.ones_like(y)
    for dt in (BF, F32):
        e = pkg.LinearCheckpoint(ck.x[:0], ck.x_scale[:, :0], ck.z[:0], ck.z_scale[:, :0], "silu")
        g = pkg.linear_backward(dy[:0], e, w, need_bias=True, grad_dtype=dt)
        assert g.x.shape == (0, 64) and not g.weight.any() and not g.bias.any() and g.weight.shape == (32, 64)
    for args in ((dy[:3], ck, w), (dy.half(), ck, w), (dy, ck, w[:, :32]), (dy, ck, w.float()), (dy.cpu(), ck, w),
                 (dy, ck._replace(z=None), w), (dy, ck._replace(z_scale=ck.x_scale[:, :2]), w), (dy, ck._replace(x=ck.z), w),
                 (dy, ck._replace(activation="swiglu"), w), (dy, ck._replace(activation="x"), w)):
        with pytest.raises(ValueError):
            pkg.linear_backward(*args)
    with pytest.raises(ValueError):
        pkg.linear_backward(dy, ck, w, grad_dtype=torch.float16)


# --------------------------------------------------------------------------------- streams, graphs, devices
@pytest.mark.parametrize("m", [3, 300])
def test_streams_and_graphs(pkg, m):
    """Calls on two side streams at once, and two captured graphs replayed together, give the eager results."""
    xs = [randn(m, 1024, seed=s) for s in (1, 2)]
    w = randn(512, 1024, seed=3, scale=0.03)
    dys = [randn(m, 256, seed=s) for s in (4, 5)]

    def step(i):
        y, ck = pkg.linear_checkpointed(xs[i], w, activation="swiglu")
        return (y, *pkg.linear_backward(dys[i], ck, w, need_bias=True))

    want = [step(i) for i in range(2)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [None, None]
    for _ in range(3):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i] = step(i)
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(a, b) for a, b in zip(got[i], want[i]))
    graphs, outs = [], []
    for i, st in enumerate(streams):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=st):
            outs.append(step(i))
        graphs.append(g)
    for _ in range(3):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                graphs[i].replay()
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(a, b) for a, b in zip(outs[i], want[i]))
    xs[0].copy_(xs[1])
    dys[0].copy_(dys[1])
    graphs[0].replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(outs[0], want[1]))


def test_graph_between_copies(pkg):
    """Captured calls whose inputs come from copies and other kernels right before them, and whose outputs are
    copied right after, replay to the eager results (the kernels start while their predecessors end)."""
    x, w = randn(200, 512, seed=1), randn(256, 512, seed=2, scale=0.05)
    xs = torch.empty_like(x)
    outs = [torch.empty(200, 256, dtype=BF, device="cuda") for _ in range(2)]

    def step():
        xs.copy_(x)
        a = pkg.linear(xs, w)
        outs[0].copy_(a)
        xs.mul_(2)
        q, s = pkg.checkpoint_activations(xs)
        b = pkg.linear(pkg.restore_activations(q, s), w)
        outs[1].copy_(b)

    step()
    torch.cuda.synchronize()
    want = [o.clone() for o in outs]
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        step()
    for _ in range(20):
        for o in outs:
            o.zero_()
        g.replay()
        assert all(torch.equal(o, v) for o, v in zip(outs, want))
    for _ in range(50):
        step()
    assert all(torch.equal(o, v) for o, v in zip(outs, want))


@pytest.mark.parametrize("m, n, act", [(300, 512, "none"), (100, 4096, "swiglu"), (300, 130, "gelu")])
def test_wait_that_runs_out_gives_nan(pkg, m, n, act):
    """A product whose accumulators never come (a host-set test hook) returns NaN after the shortened limit, and the
    next call is right again."""
    x, w = randn(m, 256, seed=1), randn(n, 256, seed=2, scale=0.06)
    want = pkg.linear(x, w, activation=act)
    lib = pkg.load_library()
    torch.cuda.synchronize()
    assert lib.moe_fp8_debug_set_waits(20_000_000, 1) == 0
    try:
        bad = pkg.linear(x, w, activation=act)
        bad32 = pkg.linear(x, w, activation=act, out_dtype=F32)
        torch.cuda.synchronize()
    finally:
        assert lib.moe_fp8_debug_set_waits(2_000_000_000, 0) == 0
    assert torch.isnan(bad).all() and torch.isnan(bad32).all()
    assert torch.equal(pkg.linear(x, w, activation=act), want)


@pytest.mark.parametrize("m, k, n, act", [(4096, 256, 7168, "none"), (2048, 2048, 4096, "swiglu")])
def test_wait_that_runs_out_with_residual_and_checkpoint(pkg, m, k, n, act):
    """The same over many tiles per SM, where the residual's boxes are fetched ahead of the products."""
    o = n // 2 if act == "swiglu" else n
    x, w, r = randn(m, k, seed=1), randn(n, k, seed=2, scale=0.06), randn(m, o, seed=3)
    want = pkg.linear(x, w, residual=r, activation=act)
    lib = pkg.load_library()
    torch.cuda.synchronize()
    assert lib.moe_fp8_debug_set_waits(20_000_000, 1) == 0
    try:
        bad = pkg.linear(x, w, residual=r, activation=act)
        bad32 = pkg.linear(x, w, residual=r, activation=act, out_dtype=F32)
        kept, ck = pkg.linear_checkpointed(x, w, residual=r, activation=act)
        torch.cuda.synchronize()
    finally:
        assert lib.moe_fp8_debug_set_waits(2_000_000_000, 0) == 0
    assert torch.isnan(bad).all() and torch.isnan(bad32).all() and torch.isnan(kept).all()
    if act != "none":
        assert torch.isnan(pkg.restore_activations(ck.z, ck.z_scale)).all()
    assert torch.equal(pkg.linear(x, w, residual=r, activation=act), want)


def bits(t):
    return t.view(torch.uint8) if t.element_size() == 1 else t


@pytest.mark.parametrize("t, k", [(9, 8), (9, 127), (30, 129), (7, 1001), (40, 3), (5, 1)])
def test_restore_at_any_offset(pkg, t, k):
    """Rows cut out of a checkpoint start anywhere in memory."""
    x = randn(t, k, seed=8, scale=3.0)
    q, s = pkg.checkpoint_activations(x)
    for dtype in (BF, F32):
        whole = pkg.restore_activations(q, s, dtype)
        for a, b in ((0, t), (1, t), (2, t - 1), (3, 4)):
            assert torch.equal(pkg.restore_activations(q[a:b], s[:, a:b], dtype), whole[a:b])
        both = pkg.restore_activations(torch.stack([q, q.flip(0)]), torch.stack([s, s.flip(1)]), dtype)
        assert torch.equal(both[0], whole) and torch.equal(both[1], whole.flip(0))
    w, dy = randn(16, k, seed=9), randn(t, 16, seed=10)
    ck = pkg.LinearCheckpoint(q, s, None, None, "none")
    cut = pkg.LinearCheckpoint(q[1:], s[:, 1:], None, None, "none")
    again = pkg.LinearCheckpoint(q[1:].clone(), s[:, 1:].clone(), None, None, "none")
    assert torch.equal(pkg.linear_backward(dy[1:], cut, w).weight, pkg.linear_backward(dy[1:], again, w).weight)
    assert torch.equal(pkg.linear_backward(dy, ck, w).x[1:], pkg.linear_backward(dy[1:], cut, w).x)


@pytest.mark.parametrize("dtype, t", [(BF, 33), (F32, 8)])
@pytest.mark.parametrize("k", [128, 136, 131, 258])
def test_checkpoint_rows_at_any_offset(pkg, dtype, t, k):
    """Rows of a wider buffer, starting at any element: the same bytes as from a copy."""
    wide = randn(t, 700, seed=11, dtype=dtype)
    for c in (0, 1, 2, 3, 4, 7):
        q, s = pkg.checkpoint_activations(wide[:, c:c + k])
        q2, s2 = pkg.checkpoint_activations(wide[:, c:c + k].clone())
        assert torch.equal(bits(q), bits(q2)) and torch.equal(bits(s), bits(s2))


@pytest.mark.parametrize("m, k, n, act, grad", [(40, 64, 48, "gelu", BF), (300, 333, 130, "swiglu", F32), (600, 512, 1024, "none", BF),
                                                (5, 2000, 777, "relu", F32)])
def test_backward_reads_inputs_written_just_before(pkg, m, k, n, act, grad):
    """The kernels of a gradient call overlap, but none runs ahead of what was launched before the call."""
    o = n // 2 if act == "swiglu" else n
    cases, want = [], []
    for i in range(3):
        x, w, dy = randn(m, k, seed=20 + i), randn(n, k, seed=30 + i, scale=0.1), randn(m, o, seed=40 + i)
        _, ck = pkg.linear_checkpointed(x, w, activation=act)
        cases.append((dy, w, ck))
        g = pkg.linear_backward(dy, ck, w, need_bias=True, grad_dtype=grad)
        torch.cuda.synchronize()
        want.append(g)
    dy, w, ck = (cases[0][0].clone(), cases[0][1].clone(), pkg.LinearCheckpoint(*[v.clone() if torch.is_tensor(v) else v for v in cases[0][2]]))
    got = []
    for r in range(60):
        for live, src in zip((dy, w, *ck[:4]), (cases[r % 3][0], cases[r % 3][1], *cases[r % 3][2][:4])):
            if live is not None:
                bits(live).copy_(bits(src))
        got.append(pkg.linear_backward(dy, ck, w, need_bias=True, grad_dtype=grad))
    for r, g in enumerate(got):
        assert all(torch.equal(a, b) for a, b in zip(g, want[r % 3]))


def test_restore_past_32_bits(pkg):
    """More than 2^32 values in rows of odd width."""
    t, k = 1_050_000, 4099
    if torch.cuda.mem_get_info()[0] < 24 << 30:
        pytest.skip("needs 24 GB")
    q = torch.zeros(t, k, dtype=torch.uint8, device="cuda")
    q[-20:] = torch.randint(0, 120, (20, k), device="cuda", generator=torch.Generator(device="cuda").manual_seed(1)).to(torch.uint8)
    s = torch.randint(100, 150, ((k + 127) // 128, t), device="cuda", generator=torch.Generator(device="cuda").manual_seed(2)).to(torch.uint8)
    q, s = q.view(torch.float8_e4m3fn), s.view(torch.float8_e8m0fnu)
    r = pkg.restore_activations(q, s)
    assert torch.equal(r[-20:], pkg.restore_activations(q[-20:].clone(), s[:, -20:]))
    assert not r[:1000].any() and not r[-1000:-20].any()


def test_offsets_past_32_bits(pkg):
    """More than 2^31 elements: the last rows of a product and of a checkpoint are those of the rows alone."""
    m, k, n = 300_100, 64, 7168
    if torch.cuda.mem_get_info()[0] < 24 << 30:
        pytest.skip("needs 24 GB")
    x, w = randn(m, k, seed=1), randn(n, k, seed=2, scale=0.1)
    y = pkg.linear(x, w)
    z, tz = dense64(x[-40:], w)
    check(y[-40:], z, rounded(z, tz, BF), "last rows")
    q, s = pkg.checkpoint_activations(y)
    q2, s2 = pkg.checkpoint_activations(y[-40:])
    assert torch.equal(q[-40:].view(torch.uint8), q2.view(torch.uint8))
    assert torch.equal(s[:, -40:].contiguous().view(torch.uint8), s2.view(torch.uint8))
    r = pkg.restore_activations(q, s)
    assert torch.equal(r[-40:], pkg.restore_activations(q2, s2))
    del r, z, tz
    dy = y[:, :1].expand(m, 8)                        # a broadcast gradient of a product with 8 outputs
    ck = pkg.LinearCheckpoint(q, s, None, None, "none")
    g = pkg.linear_backward(dy, ck, randn(8, n, seed=3), need_x=True, need_bias=True, grad_dtype=F32)
    ref = dy[-40:].double() @ randn(8, n, seed=3).double()
    check(g.x[-40:], ref, ref.abs() * 2.0 ** -20 + 1e-4, "grad_x of the last rows")
    want = dy[:, 0].double().sum()
    assert abs(float(g.bias[0].double() - want)) <= 2.0 ** -16 * float(dy[:, 0].double().abs().sum())


# --------------------------------------------------------------------------------- far and non-finite values
@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("gin, gout", [(BF, BF), (F32, F32)])
@pytest.mark.parametrize("m, k, n", [(40, 64, 512), (300, 130, 390)])
def test_backward_non_finite(pkg, act, gin, gout, m, k, n):
    """A NaN or infinity in grad_output or in a kept block reaches the gradients it is part of, and no others."""
    x, w = randn(m, k, seed=1), randn(n, k, seed=2, scale=k ** -0.5)
    y, ck = pkg.linear_checkpointed(x, w, activation=act)
    o = y.shape[1]
    dy = randn(m, o, seed=5, dtype=gin)
    clean = pkg.linear_backward(dy, ck, w, need_bias=True, grad_dtype=gout)
    rows = torch.arange(m, device="cuda")

    def compare(g, row, cols):
        out = torch.zeros(n, dtype=torch.bool, device="cuda")
        for c in cols:
            out[c] = True
        assert not torch.isfinite(g.x[row]).any() and torch.equal(g.x[rows != row], clean.x[rows != row])
        assert not torch.isfinite(g.weight[out]).any() and torch.equal(g.weight[~out], clean.weight[~out])
        assert not torch.isfinite(g.bias[out]).any() and torch.equal(g.bias[~out], clean.bias[~out])

    halves = (0, o) if act == "swiglu" else (0,)
    for bad in (float("nan"), float("inf"), -float("inf")):
        d = dy.clone()
        row, col = m // 2, 3
        if act == "relu":                                      # an infinity times a slope of 0 is a NaN too
            col = int(torch.nonzero(y[row] > 0)[0])
        d[row, col] = bad
        compare(pkg.linear_backward(d, ck, w, need_bias=True, grad_dtype=gout), row, [h + col for h in halves])
    if act == "none":
        return
    z = ck.z.clone().view(torch.uint8)
    s = ck.z_scale.clone().view(torch.uint8)
    row = m - 1
    for h in range(len(halves)):                               # the NaN scale of one block, as an overflow leaves it
        zs = s.clone()
        (zs[h] if act == "swiglu" else zs)[1, row] = 255
        c = ck._replace(z_scale=zs.view(torch.float8_e8m0fnu))
        cols = slice(128, min(256, o))
        # d/da = dy silu(b) does not see a; d/db = dy a silu'(b) sees both
        hit = [cols] if act != "swiglu" else [slice(o + cols.start, o + cols.stop)] + ([cols] if h == 1 else [])
        compare(pkg.linear_backward(dy, c, w, need_bias=True, grad_dtype=gout), row, hit)
    zq = z.clone()                                             # a NaN byte
    (zq[0] if act == "swiglu" else zq)[row, 5] = 0x7f
    c = ck._replace(z=zq.view(torch.float8_e4m3fn))
    compare(pkg.linear_backward(dy, c, w, need_bias=True, grad_dtype=gout), row, [5] if act != "swiglu" else [o + 5])


# --------------------------------------------------------------------------------- aligned slices of wider buffers
@pytest.mark.parametrize("m, k, n", [(9, 128, 72), (60, 192, 104), (300, 520, 264), (1500, 192, 1096), (9000, 64, 328), (64, 7168, 520)])
@pytest.mark.parametrize("act", ["none", "silu", "swiglu"])
@pytest.mark.parametrize("dtype", [BF, F32])
def test_linear_aligned_slices(pkg, m, k, n, act, dtype):
    """x, weight, residual and output as slices of wider buffers whose rows bulk copies reach (strides of multiples of 16 bytes
    beyond the width), the last box cut off beside live neighbours: the same bits as from tensors of their own, and nothing
    else is written."""
    o = n // 2 if act == "swiglu" else n
    xb, wb = randn(m + 2, k + 72, seed=1), randn(n + 3, k + 40, seed=2, scale=k ** -0.5)
    x, w, b = xb[1:m + 1, 8:8 + k], wb[2:2 + n, 32:32 + k], randn(n, seed=3)
    rb, ob = randn(m, o + 56, seed=4), randn(m + 2, o + 80, seed=6, dtype=dtype)
    for r in (None, rb[:, 24:24 + o]):
        want = pkg.linear(x.contiguous(), w.contiguous(), bias=b, residual=None if r is None else r.contiguous(), activation=act, out_dtype=dtype)
        z, tz = dense64(x, w, b)
        ref, tol = act64(z, act), tol_act(z, tz, act)
        if r is not None:
            ref = ref + r.double()
            tol = tol + ref.abs() * 2.0 ** -23
        check(want, ref, rounded(ref, tol, dtype), "own tensors")
        for c0 in (16, 4 if dtype == F32 else 8):
            out = ob.clone()
            y = out[1:m + 1, c0:c0 + o]
            got = pkg.linear(x, w, bias=b, residual=r, activation=act, out_dtype=dtype, output=y)
            assert got is y
            if o % 8 == 0:                                     # else the contiguous rows go another way
                assert torch.equal(y, want)
            check(y, ref, rounded(ref, tol, dtype), "slices")
            out[1:m + 1, c0:c0 + o] = ob[1:m + 1, c0:c0 + o]
            assert torch.equal(out, ob)
    if dtype == BF:                                            # in place, in the residual's wider rows
        out = rb.clone()
        r = out[:, 24:24 + o]
        want = pkg.linear(x, w, bias=b, residual=r.clone(), activation=act)
        pkg.linear(x, w, bias=b, residual=r, activation=act, output=r)
        if o % 8 == 0:
            assert torch.equal(r, want)
        out[:, 24:24 + o] = rb[:, 24:24 + o]
        assert torch.equal(out, rb)


@pytest.mark.parametrize("m, k, n", [(40, 128, 96), (300, 520, 288), (1500, 192, 1120), (300, 136, 264)])
@pytest.mark.parametrize("act", ["none", "gelu", "swiglu"])
@pytest.mark.parametrize("dtype", [BF, F32])
def test_training_step_on_aligned_slices(pkg, m, k, n, act, dtype):
    """The same for a checkpointed product and its gradients."""
    o = n // 2 if act == "swiglu" else n
    x = randn(m + 2, k + 72, seed=1)[1:m + 1, 8:8 + k]
    w = randn(n + 3, k + 40, seed=2, scale=k ** -0.5)[2:2 + n, 32:32 + k]
    ob = randn(m, o + 80, seed=6, dtype=dtype)
    out = ob.clone()
    y, ck = pkg.linear_checkpointed(x, w, activation=act, out_dtype=dtype, output=out[:, 16:16 + o])
    yc, cc = pkg.linear_checkpointed(x.contiguous(), w.contiguous(), activation=act, out_dtype=dtype)
    if o % 8 == 0:
        assert torch.equal(y, yc)
    for a, c in zip(ck[:4], cc[:4]):
        assert (a is None and c is None) or torch.equal(bits(a), bits(c))
    out[:, 16:16 + o] = ob[:, 16:16 + o]
    assert torch.equal(out, ob)
    dy = randn(m + 1, o + 64, seed=7, dtype=dtype)[1:, 16:16 + o]
    for need in (dict(), dict(need_weight=False), dict(need_x=False, need_bias=True)):
        g = pkg.linear_backward(dy, ck, w, grad_dtype=dtype, **need)
        gc = pkg.linear_backward(dy.contiguous(), cc, w.contiguous(), grad_dtype=dtype, **need)
        assert all((a is None and c is None) or torch.equal(a, c) for a, c in zip(g, gc))


def test_graph_that_forks_and_joins(pkg):
    """A capture whose calls run on two streams and wait for one another replays to the eager results."""
    x, w1, w2 = randn(300, 512, seed=1), randn(512, 512, seed=2, scale=0.05), randn(512, 512, seed=3, scale=0.05)
    dy, side = randn(300, 512, seed=4), torch.cuda.Stream()

    def step():
        a = pkg.linear(x, w1)
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            b, ck = pkg.linear_checkpointed(a, w2, activation="silu")
            g = pkg.linear_backward(dy, ck, w2, need_bias=True)
        c = pkg.linear(a, w1)
        torch.cuda.current_stream().wait_stream(side)
        d = pkg.linear(b, w1, residual=c)
        e, ck = pkg.linear_checkpointed(d, w1, activation="swiglu")
        return (a, b, c, d, e, *g, *pkg.linear_backward(dy[:, :256], ck, w1, need_bias=True))

    want = step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for _ in range(10):
        for o in out:
            o.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want))
