"""GPU: dense products whose tiles follow one another closely on every pair of SMs, and whose waits run out.

The inputs are small integers, so every product sum is a whole number below 2^24 and exact in fp32 in any order: y is
the 64-bit form rounded once, bit for bit."""
import pytest
import torch

pytestmark = pytest.mark.gpu

BF, F32 = torch.bfloat16, torch.float32


def whole(*shape, seed=0, top=3):
    g = torch.Generator(device="cuda").manual_seed(seed + 1000 * sum(shape))
    return torch.randint(-top, top + 1, shape, generator=g, device="cuda").to(BF)


def bits(t):
    return t.view(torch.uint8) if t.element_size() == 1 else t


# Tiles of 192 columns leave three boxes of 32 per warp, 64 (and 128 of a gated product) one, and a last column tile that
# is cut off any number: the next tile's first box must not be the one that is still being read. Few K-blocks, so that
# the next accumulator is always there already.
@pytest.mark.parametrize("m, k, n, act, keep", [
    (4096, 1024, 5120, "none", False), (8192, 512, 1048, "none", False), (4096, 64, 1280, "relu", False),
    (20000, 64, 272, "relu", False), (20000, 64, 64, "relu", False), (40000, 128, 64, "none", False),
    (60000, 64, 80, "relu", False), (4096, 64, 1536, "swiglu", False), (4096, 256, 1536, "swiglu", False),
    (40000, 64, 80, "relu", True), (20000, 64, 272, "relu", True), (8192, 64, 1304, "relu", True),
    (20000, 64, 160, "swiglu", True)])
def test_many_short_tiles(pkg, m, k, n, act, keep):
    x, w, b = whole(m, k, seed=1), whole(n, k, seed=2), whole(n, seed=3)
    z = x.double() @ w.double().t() + b.double()
    if act == "swiglu":
        f, s = z.chunk(2, 1)
        want = f * s * torch.sigmoid(s)
        # the product of the whole numbers and the sigmoid (2^-20 of 1 + |z|), rounded to bf16
        tol = 2.0 ** -8 * want.abs() + 2.0 ** -19 * f.abs() * (1 + s.abs()) * 1.01 + 1e-30
    else:
        want, tol = z.clamp(min=0) if act == "relu" else z, None
    first = None
    for _ in range(12):
        if keep:
            y, ck = pkg.linear_checkpointed(x, w, bias=b, activation=act)
            out = (y, bits(ck.z), bits(ck.z_scale))
        else:
            out = (pkg.linear(x, w, bias=b, activation=act),)
        if first is None:
            first = out
            if tol is None:
                assert torch.equal(out[0], want.to(BF))
            else:
                assert ((out[0].double() - want).abs() <= tol).all()
            if keep:
                halves = z.chunk(2, 1) if act == "swiglu" else (z,)
                q = [pkg.checkpoint_activations(h.float().contiguous()) for h in halves]
                stack = torch.stack if act == "swiglu" else lambda v: v[0]
                assert torch.equal(out[1], stack([bits(v[0]) for v in q]))
                assert torch.equal(out[2], stack([bits(v[1]) for v in q]))
        else:
            assert all(torch.equal(a, c) for a, c in zip(out, first))


@pytest.mark.parametrize("m, k, n, act, grad", [(300, 512, 512, "none", BF), (600, 2048, 1024, "silu", F32), (4096, 256, 2048, "none", BF)])
def test_wait_that_runs_out_in_the_gradients(pkg, m, k, n, act, grad):
    """Gradients whose accumulators never come (a host-set test hook) are NaN after the shortened limit, the bias gradient, which
    needs none, is not, and the next call is right again. The two products overlap."""
    x, w, dy = whole(m, k, seed=1), whole(n, k, seed=2), whole(m, n, seed=3)
    ck = pkg.linear_checkpointed(x, w, activation=act)[1]
    want = pkg.linear_backward(dy, ck, w, need_bias=True, grad_dtype=grad)
    lib = pkg.load_library()
    torch.cuda.synchronize()
    assert lib.moe_fp8_debug_set_waits(20_000_000, 1) == 0
    try:
        bad = pkg.linear_backward(dy, ck, w, need_bias=True, grad_dtype=grad)
        torch.cuda.synchronize()
    finally:
        assert lib.moe_fp8_debug_set_waits(2_000_000_000, 0) == 0
    assert torch.isnan(bad.x).all() and torch.isnan(bad.weight).all() and torch.equal(bad.bias, want.bias)
    again = pkg.linear_backward(dy, ck, w, need_bias=True, grad_dtype=grad)
    assert all(torch.equal(a, b) for a, b in zip(again, want))


@pytest.mark.parametrize("m, n, act, dtype", [(64, 512, "none", BF), (128, 4096, "swiglu", BF), (40, 256, "none", F32)])
def test_wait_that_runs_out_with_few_tokens(pkg, m, n, act, dtype):
    """The same where the weights' rows are the tile's."""
    x, w = whole(m, 7168, seed=1, top=1), whole(n, 7168, seed=2, top=1)
    want = pkg.linear(x, w, activation=act, out_dtype=dtype)
    lib = pkg.load_library()
    torch.cuda.synchronize()
    assert lib.moe_fp8_debug_set_waits(20_000_000, 1) == 0
    try:
        bad = pkg.linear(x, w, activation=act, out_dtype=dtype)
        torch.cuda.synchronize()
    finally:
        assert lib.moe_fp8_debug_set_waits(2_000_000_000, 0) == 0
    assert torch.isnan(bad).all()
    assert torch.equal(pkg.linear(x, w, activation=act, out_dtype=dtype), want)
