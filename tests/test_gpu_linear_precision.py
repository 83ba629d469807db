"""GPU: how far the dense products, their kept pre-activations and their gradients are from 64-bit forms as a whole.

What the bounds rest on. The tensor core adds to its fp32 sum by truncation, which loses half a unit of the running sum on
average, 2^-23 * 0.36 of its value (a unit is 2^-23 to 2^-24 of the value, 0.72 * 2^-23 on average over significands). A
chain of n such additions (4 per 64 of K) of independent terms has running sums that grow as sqrt(i / n), so it loses at
most the sum of 0.36 * 2^-23 * sqrt(i / n), 0.24 n * 2^-23 of the chain's norm. Chains are joined in fp32 with rounding to
nearest, which is smaller by a factor of ten. The chains are 12 K-blocks (n = 48) for fp32 results, 6 for gated ones, 8
(n = 32) at most for kept pre-activations."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

BF, F32 = torch.bfloat16, torch.float32
CHAIN12 = 0.24 * 48 * 2.0 ** -23          # 1.4e-6


def randn(*shape, seed=0, scale=1.0, dtype=BF):
    g = torch.Generator(device="cuda").manual_seed(seed + 1000 * sum(shape))
    return (torch.randn(*shape, generator=g, device="cuda") * scale).to(dtype)


def off(got, want):
    return float((got.double() - want).norm() / want.norm())


@pytest.mark.parametrize("m", [1, 16, 64, 128, 300, 1500, 4096])
@pytest.mark.parametrize("k, n", [(512, 1024), (7168, 256), (7168, 2050), (20000, 640)])
def test_fp32_products(pkg, m, k, n):
    x, w = randn(m, k, seed=1), randn(n, k, seed=2, scale=k ** -0.5)
    assert off(pkg.linear(x, w, out_dtype=F32), x.double() @ w.double().t()) <= CHAIN12 + 2.0 ** -23


@pytest.mark.parametrize("m", [1, 100, 300, 2048])
@pytest.mark.parametrize("k, n", [(768, 1024), (7168, 512), (20000, 260)])
def test_fp32_gated_products(pkg, m, k, n):
    """Both factors drift by a chain of 6; the exact sigmoid's fp32 is a few 2^-24 of 1 + |z|."""
    x, w = randn(m, k, seed=1), randn(n, k, seed=2, scale=k ** -0.5)
    a, b = (x.double() @ w.double().t()).chunk(2, 1)
    want = a * b * torch.sigmoid(b)
    assert off(pkg.linear(x, w, activation="swiglu", out_dtype=F32), want) <= CHAIN12 + 4 * 2.0 ** -23


@pytest.mark.parametrize("m, k, n", [(600, 512, 1024), (4096, 7168, 256), (1500, 768, 4096)])
@pytest.mark.parametrize("act", ["none", "silu", "swiglu"])
def test_fp32_gradients(pkg, m, k, n, act):
    """dz enters with all its 24 bits; its own evaluation is good to 2^-20 (activations)."""
    x, w = randn(m, k, seed=1), randn(n, k, seed=2, scale=k ** -0.5)
    y, ck = pkg.linear_checkpointed(x, w, activation=act)
    dz = dy = randn(*y.shape, seed=3, dtype=F32)
    g = pkg.linear_backward(dy, ck, w, grad_dtype=F32)
    dz = dy.double()
    if act != "none":
        z = pkg.restore_activations(ck.z, ck.z_scale, F32).double()
        b = z[1] if act == "swiglu" else z
        s = torch.sigmoid(b)
        slope = s * (1 + b * (1 - s))
        dz = torch.cat([dz * b * s, dz * z[0] * slope], 1) if act == "swiglu" else dz * slope
    xr = pkg.restore_activations(ck.x, ck.x_scale, F32).double()
    bound = CHAIN12 + 2.0 ** -23 + (0 if act == "none" else 2.0 ** -20)
    assert off(g.x, dz @ w.double()) <= bound
    assert off(g.weight, dz.t() @ xr) <= bound


def kept64(z):
    """The values of the 8-bit format, from 64-bit ones."""
    k = z.shape[1]
    v = torch.nn.functional.pad(z, (0, -k % 128)).unflatten(1, (-1, 128))
    amax = v.abs().amax(-1, keepdim=True)
    e = torch.floor(torch.log2(amax.clamp(min=1e-300))) - 8
    e = torch.where(amax > 448 * torch.exp2(e), e + 1, e)
    s = v / torch.exp2(e)
    step = torch.exp2(torch.floor(torch.log2(s.abs().clamp(min=2.0 ** -30))).clamp(min=-6) - 3)
    return (torch.round(s / step) * step * torch.exp2(e)).flatten(1)[:, :k]


@pytest.mark.parametrize("m, k, n", [(2048, 7168, 1024), (8192, 512, 1024), (2048, 20000, 520)])
@pytest.mark.parametrize("act", ["silu", "swiglu"])
@pytest.mark.parametrize("dtype", [BF, F32])
def test_kept_values(pkg, m, k, n, act, dtype):
    """A value off by an error e of its sum falls on the other side of a border of the format, a step away, with the
    probability e / step: the squares add up to E[e step], and the steps are an eighth of a power of two, 0.07 of the norm
    on average for normal values. A chain of 8 K-blocks (0.24 * 32 * 2^-23) and the fp32 joins (a tenth) give 2.7e-4 of the norm,
    and a few dozen such values in a case make that good to a tenth."""
    x, w = randn(m, k, seed=1), randn(n, k, seed=2, scale=k ** -0.5)
    _, ck = pkg.linear_checkpointed(x, w, activation=act, out_dtype=dtype)
    got = pkg.restore_activations(ck.z, ck.z_scale, F32).double()
    z = x.double() @ w.double().t()
    want = torch.stack([kept64(h) for h in z.chunk(2, 1)]) if act == "swiglu" else kept64(z)
    assert off(got, want) <= 1.1 * math.sqrt(0.07 * 1.1 * 0.24 * 32 * 2.0 ** -23)


@pytest.mark.parametrize("k", [64, 128, 256, 400, 512, 832, 1024, 1536, 2048, 3283, 4096])
@pytest.mark.parametrize("act", ["silu", "swiglu"])
def test_kept_values_like_those_of_an_fp32_product(pkg, k, act):
    """Chains of sqrt(K / 64) K-blocks drift like the roundings of an fp32 product, so about as many values fall on another
    step: some 30 of the 2^24 here, which makes the ratio of the two norms good to 18 % (30^-1/2)."""
    m, n = 8192, 2048
    x, w = randn(m, k, seed=1), randn(n, k, seed=2, scale=k ** -0.5)
    z, z32 = x.double() @ w.double().t(), x.float() @ w.float().t()
    if act == "swiglu":
        cut = lambda v: torch.stack([kept64(h.double()) for h in v.chunk(2, 1)])  # noqa: E731
    else:
        cut = lambda v: kept64(v.double())  # noqa: E731
    _, ck = pkg.linear_checkpointed(x, w, activation=act)
    got = pkg.restore_activations(ck.z, ck.z_scale, F32).double()
    assert off(got, cut(z)) <= 1.5 * off(cut(z32), cut(z))


@pytest.mark.parametrize("m, k, n", [(300, 768, 512), (700, 2048, 512), (2048, 7168, 1024), (513, 1100, 1040)])
@pytest.mark.parametrize("act", ["gelu", "swiglu"])
def test_kept_bytes_do_not_depend_on_the_output_type(pkg, m, k, n, act):
    x, w = randn(m, k, seed=1), randn(n, k, seed=2, scale=k ** -0.5)
    a = pkg.linear_checkpointed(x, w, activation=act)[1]
    b = pkg.linear_checkpointed(x, w, activation=act, out_dtype=F32)[1]
    assert torch.equal(a.z.view(torch.uint8), b.z.view(torch.uint8))
    assert torch.equal(a.z_scale.view(torch.uint8), b.z_scale.view(torch.uint8))


def positive(rows, cols, seed):
    """Values of one sign, rows at different scales so that sums of the same size round everywhere between two steps."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.rand(rows, cols, generator=g, device="cuda") + 0.5
    return (x * (1 + torch.rand(rows, 1, generator=g, device="cuda"))).to(BF)


def product64(x, w):
    """x w^T in 64 bits, a piece of K at a time."""
    z = torch.zeros(x.shape[0], w.shape[0], dtype=torch.float64, device="cuda")
    for i in range(0, x.shape[1], 32768):
        z.addmm_(x[:, i:i + 32768].double(), w[:, i:i + 32768].double().t())
    return z


def drift(got, want):
    """Mean relative error, with its sign: roundings to nearest cancel in it, truncation does not."""
    return float(((got.double() - want) / want).mean())


@pytest.fixture
def room():
    torch.cuda.empty_cache()
    if torch.cuda.mem_get_info()[0] < 40 << 30:
        pytest.skip("needs 40 GB")
    yield
    torch.cuda.empty_cache()


# A bf16 rounding is off by 2^-9 of the value at the most typical, either way: over 16384 values and more the mean is below
# 2^-9 / sqrt(16384) = 1.5e-5. The tensor core cuts the 16 products of an addition and the running sum at one place before
# it adds them, so terms of one sign lose more than the sum's own half unit: 3.7e-7 per K-block of 64 (measured), 9.5e-5 in a
# chain of 256. Together 1.1e-4, under the bound of 1.18e-4; uncut chains of 4096 K-blocks lose 1.5e-3.
LONG = 0.18 * 4096 * 2.0 ** -23 + 3e-5


@pytest.mark.parametrize("m, k, n", [(2560, 262144, 2048), (64, 4194304, 256)])
def test_bf16_products_of_a_long_contraction(pkg, room, m, k, n):
    x, w = positive(m, k, 1), positive(n, k, 2)
    assert abs(drift(pkg.linear(x, w), product64(x, w))) <= LONG


def test_bf16_weight_gradient_of_many_tokens(pkg, room):
    m, k, n = 262144, 4096, 4096
    x = positive(k, m, 1).t().contiguous()
    dy = positive(n, m, 2).t().contiguous()
    x8, xs = pkg.checkpoint_activations(x)
    del x
    g = pkg.linear_backward(dy, pkg.LinearCheckpoint(x8, xs, None, None, "none"), randn(n, k), need_x=False)
    xr = pkg.restore_activations(x8, xs)
    assert abs(drift(g.weight, product64(dy.t(), xr.t()))) <= LONG


def test_fp32_product_of_few_tokens_and_a_long_contraction(pkg, room):
    """A warp's chain is joined after 16 additions of terms of one sign or fewer, each of which loses up to 9e-8 of the running
    sum (see LONG); half of that on average, and the fp32 joins round to nearest."""
    x, w = positive(8, 262144, 1), positive(7168, 262144, 2)
    assert abs(drift(pkg.linear(x, w, out_dtype=F32), product64(x, w))) <= 0.18 * 64 * 2.0 ** -23 + 2.0 ** -23
