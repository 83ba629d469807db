"""CPU: argument checks of the layer operators (dense products, 8-bit
checkpoints, gradients, balance loss), made before anything is launched."""
import ctypes

import pytest
import torch


@pytest.fixture(scope="module")
def layer(pkg):
    import sys
    return sys.modules[pkg.__name__ + ".layer"]


@pytest.fixture(scope="module")
def lib(layer):
    return layer._library()


FAKE = 4096          # never dereferenced: the checks fail first


def linear_args(layer, **kw):
    a = layer.MoeLinearArgs()
    a.x = a.weight = a.y = FAKE
    a.m, a.k, a.n = 4, 64, 32
    a.ldx = a.ldw = 64
    a.ldy = 32
    for k, v in kw.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("kw, text", [
    ({"m": -1}, b"m must be"), ({"k": 0}, b"m must be"), ({"n": 0}, b"m must be"), ({"m": (1 << 30) + 1}, b"m must be"),
    ({"activation": 5}, b"activation"), ({"activation": -1}, b"activation"), ({"activation": 4, "n": 31}, b"even"),
    ({"x": None}, b"NULL"), ({"weight": None}, b"NULL"), ({"y": None}, b"NULL"),
    ({"z8": FAKE}, b"go together"), ({"z_scale": FAKE}, b"go together"),
    ({"x": FAKE + 1}, b"aligned"), ({"weight": FAKE + 1}, b"aligned"), ({"bias": FAKE + 1}, b"aligned"),
    ({"residual": FAKE + 1}, b"aligned"), ({"y": FAKE + 2, "y_f32": 1}, b"aligned"),
    ({"ldx": 63}, b"stride"), ({"ldw": 63}, b"stride"), ({"ldy": 31}, b"stride"),
    ({"residual": FAKE, "ldr": -1}, b"stride"),
])
def test_linear_refusals(layer, lib, pkg, kw, text):
    a = linear_args(layer, **kw)
    assert lib.moe_linear_run(ctypes.byref(a), None) == 1
    assert text in lib.moe_fp8_last_error()


@pytest.mark.parametrize("kw", [{"y_f32": 1, "ldr": 32}, {"ldr": 40}])
def test_linear_residual_that_is_not_y_itself(layer, lib, kw):
    a = linear_args(layer, residual=FAKE, **kw)
    assert lib.moe_linear_run(ctypes.byref(a), None) == 1
    assert b"residual itself" in lib.moe_fp8_last_error()


def test_linear_workspace_refusal_and_empty(layer, lib):
    a = linear_args(layer, m=600, k=7168, n=4096, ldx=7168, ldw=7168, ldy=4096)
    need = lib.moe_linear_workspace_bytes(ctypes.byref(a))
    if need:
        for ws, size in ((None, need), (FAKE + 8, need), (FAKE, need - 1)):
            a.workspace, a.workspace_bytes = ws, size
            assert lib.moe_linear_run(ctypes.byref(a), None) == 2
            assert b"workspace" in lib.moe_fp8_last_error()
    assert lib.moe_linear_run(None, None) == 1
    assert lib.moe_linear_run(ctypes.byref(linear_args(layer, m=0)), None) == 0


def grad_args(layer, **kw):
    a = layer.MoeLinearGradArgs()
    a.grad_y = a.x8 = a.x_scale = a.z8 = a.z_scale = a.weight = a.grad_x = a.grad_weight = a.grad_bias = FAKE
    a.m, a.k, a.n, a.activation = 4, 64, 32, 3
    a.ldg, a.ldw = 32, 64
    a.workspace, a.workspace_bytes = FAKE, 1 << 40
    for k, v in kw.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("kw, rc, text", [
    ({"m": -1}, 1, b"m must be"), ({"k": 0}, 1, b"m must be"), ({"activation": 9}, 1, b"activation"),
    ({"activation": 4, "n": 31}, 1, b"even"),
    ({"grad_y": None}, 1, b"NULL"), ({"z8": None}, 1, b"NULL"), ({"z_scale": None}, 1, b"NULL"),
    ({"weight": None}, 1, b"NULL"), ({"x8": None}, 1, b"NULL"), ({"x_scale": None}, 1, b"NULL"),
    ({"grad_y": FAKE + 1}, 1, b"aligned"), ({"grad_y": FAKE + 2, "grad_y_f32": 1}, 1, b"aligned"),
    ({"grad_x": FAKE + 1}, 1, b"aligned"), ({"grad_weight": FAKE + 2, "grad_f32": 1}, 1, b"aligned"),
    ({"grad_bias": FAKE + 1}, 1, b"aligned"), ({"ldw": 63}, 1, b"stride"), ({"ldg": -1}, 1, b"stride"),
    ({"workspace": None}, 2, b"workspace"), ({"workspace": FAKE + 16}, 2, b"workspace"),
    ({"workspace_bytes": 16}, 2, b"workspace"),
])
def test_linear_grad_refusals(layer, lib, kw, rc, text):
    a = grad_args(layer, **kw)
    assert lib.moe_linear_grad(ctypes.byref(a), None) == rc
    assert text in lib.moe_fp8_last_error()
    assert lib.moe_linear_grad(None, None) == 1


def test_nothing_asked_is_a_no_op(layer, lib):
    a = grad_args(layer, grad_x=None, grad_weight=None, grad_bias=None)
    assert lib.moe_linear_grad(ctypes.byref(a), None) == 0


def test_checkpoint_refusals(lib):
    c, r = lib.moe_checkpoint_activations, lib.moe_restore_activations
    assert c(FAKE, 1, -1, 8, 8, FAKE, FAKE, None) == 1
    assert c(FAKE, 1, 1, 65535 * 1024 + 1, 8, FAKE, FAKE, None) == 1
    assert c(None, 1, 1, 8, 8, FAKE, FAKE, None) == 1
    assert c(FAKE + 2, 0, 1, 8, 8, FAKE, FAKE, None) == 1
    assert c(FAKE, 1, 1, 8, -8, FAKE, FAKE, None) == 1
    assert c(None, 1, 0, 8, 8, None, None, None) == 0
    assert r(FAKE, FAKE, 65536, 1, 8, FAKE, 0, None) == 1
    assert r(FAKE, None, 1, 1, 8, FAKE, 0, None) == 1
    assert r(FAKE, FAKE, 1, 1, 8, FAKE + 2, 1, None) == 1
    assert r(None, None, 1, 0, 8, None, 0, None) == 0


def balance_args(layer, cls="MoeBalanceArgs", **kw):
    a = getattr(layer, cls)()
    for name, kind in a._fields_:
        if kind is ctypes.c_void_p:
            setattr(a, name, FAKE)
    a.num_tokens, a.num_experts, a.top_k, a.num_sequences = 4, 256, 8, 2
    if cls == "MoeBalanceArgs":
        a.workspace_bytes = 1 << 40
    for k, v in kw.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("kw", [{"num_tokens": -1}, {"num_experts": 0}, {"num_experts": 1025}, {"top_k": 0}, {"top_k": 33},
                                {"num_sequences": 0}, {"num_sequences": 65536}, {"scoring": 2}, {"routing_logits": None},
                                {"topk_idx": None}, {"routing_logits": FAKE + 2}, {"cu_seqlens": None}])
def test_balance_refusals(layer, lib, kw):
    assert lib.moe_balance_loss(ctypes.byref(balance_args(layer, **kw)), None) == 1
    assert lib.moe_balance_loss_grad(ctypes.byref(balance_args(layer, "MoeBalanceGradArgs", **kw)), None) == 1


@pytest.mark.parametrize("name", ["cu_seqlens", "counts", "tokens", "sequences"])
def test_balance_misaligned_pointers(layer, lib, name):
    for entry, cls in ((lib.moe_balance_loss, "MoeBalanceArgs"), (lib.moe_balance_loss_grad, "MoeBalanceGradArgs")):
        assert entry(ctypes.byref(balance_args(layer, cls, **{name: FAKE + 2})), None) == 1
        assert b"aligned" in lib.moe_fp8_last_error()


def test_balance_refusals_of_one_entry(layer, lib):
    for kw in ({"loss": None}, {"counts": None}, {"tokens": None}, {"mean_scores": None}, {"sequences": None}):
        assert lib.moe_balance_loss(ctypes.byref(balance_args(layer, **kw)), None) == 1
    for kw in ({"workspace": None}, {"workspace": FAKE + 8}, {"workspace_bytes": 8}):
        assert lib.moe_balance_loss(ctypes.byref(balance_args(layer, **kw)), None) == 2
    g = "MoeBalanceGradArgs"
    for kw in ({"grad_logits": None}, {"counts": None}, {"tokens": None}, {"sequences": None},
               {"grad_topk_weights": FAKE + 2}):
        assert lib.moe_balance_loss_grad(ctypes.byref(balance_args(layer, g, **kw)), None) == 1
    assert lib.moe_balance_loss_grad(ctypes.byref(balance_args(layer, g, num_tokens=0)), None) == 0


def test_python_refusals_without_a_gpu(pkg):
    x, w = torch.zeros(2, 8, dtype=torch.bfloat16), torch.zeros(4, 8, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="CUDA"):
        pkg.linear(x, w)
    with pytest.raises(ValueError, match="activation"):
        pkg.linear(x, w, activation="tanh")
    with pytest.raises(ValueError, match="bfloat16"):
        pkg.linear(x.float(), w)
    with pytest.raises(ValueError, match="CUDA"):
        pkg.checkpoint_activations(x)
    with pytest.raises(ValueError, match="2-d"):
        pkg.checkpoint_activations(x[0])
    with pytest.raises(ValueError, match="q must be"):
        pkg.restore_activations(x[0], x)
    with pytest.raises(ValueError, match="CUDA"):
        pkg.balance_loss(torch.zeros(2, 8), torch.zeros(2, 2, dtype=torch.int32))
    with pytest.raises(ValueError, match="float32"):
        pkg.balance_loss(x, torch.zeros(2, 2, dtype=torch.int32))


def test_build_without_torch_headers(monkeypatch, tmp_path, capsys):
    """Where torch has no C++ headers the binding is left out and the build goes on."""
    import importlib.util
    import pathlib
    path = pathlib.Path(__file__).resolve().parents[1] / "starter-kit-fused-moe_b200" / "build.py"
    spec = importlib.util.spec_from_file_location("_moe_build_layer", path)
    b = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(b)
    assert b.torch_root() is not None
    monkeypatch.setattr(torch, "__file__", str(tmp_path / "torch" / "__init__.py"))
    assert b.torch_root() is None
    monkeypatch.setattr(b, "build", lambda *a, **k: None)
    assert b.build_layer_binding(force=True) is None
    assert "headers" in capsys.readouterr().err
