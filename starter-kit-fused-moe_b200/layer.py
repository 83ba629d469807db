"""Operators around the routed experts, for layers that are trained: dense
products (the router's gate, the shared expert) with their 8-bit activation
checkpoints and gradients, and the router's balance loss with its gradient.

Everything is computed by the library's own kernels through its C ABI
(`moe_linear_*`, `moe_checkpoint_*`, `moe_restore_*`, `moe_balance_*` in
include/moe_fp8.h) on the current stream of the tensors' device, without host
synchronisation. The calls go through a native binding (binding/layer_binding.cc:
argument checks, outputs, workspaces); the ctypes declarations below serve
callers who bring their own buffers. If either library is missing, every call
raises. No autograd graph is recorded: gradients are computed by the
`*_backward` functions. Outputs and workspaces come from torch's allocator per
call, so calls on several streams and in several captured graphs do not share
memory. Wrong shapes, types, devices or overlapping buffers raise ValueError.
The reference holds the routed operator alone and has no counterpart.
"""
from __future__ import annotations

import ctypes
import importlib.util
import pathlib
from typing import NamedTuple, Optional

import torch

BINDING_PATH = pathlib.Path(__file__).resolve().parent / "moe_b200_layer.so"

_vp, _i32, _i64, _sz, _f32 = ctypes.c_void_p, ctypes.c_int32, ctypes.c_int64, ctypes.c_size_t, ctypes.c_float


class MoeLinearArgs(ctypes.Structure):
    _fields_ = [("x", _vp), ("weight", _vp), ("bias", _vp), ("residual", _vp), ("y", _vp), ("z8", _vp),
                ("z_scale", _vp), ("workspace", _vp), ("workspace_bytes", _sz), ("ldx", _i64), ("ldw", _i64),
                ("ldr", _i64), ("ldy", _i64), ("m", _i32), ("k", _i32), ("n", _i32), ("activation", _i32),
                ("y_f32", _i32)]


class MoeLinearGradArgs(ctypes.Structure):
    _fields_ = [("grad_y", _vp), ("x8", _vp), ("x_scale", _vp), ("z8", _vp), ("z_scale", _vp), ("weight", _vp),
                ("grad_x", _vp), ("grad_weight", _vp), ("grad_bias", _vp), ("workspace", _vp),
                ("workspace_bytes", _sz), ("ldg", _i64), ("ldw", _i64), ("m", _i32), ("k", _i32), ("n", _i32),
                ("activation", _i32), ("grad_y_f32", _i32), ("grad_f32", _i32)]


class MoeBalanceArgs(ctypes.Structure):
    _fields_ = [("routing_logits", _vp), ("topk_idx", _vp), ("cu_seqlens", _vp), ("loss", _vp), ("counts", _vp),
                ("tokens", _vp), ("mean_scores", _vp), ("sequences", _vp), ("workspace", _vp),
                ("workspace_bytes", _sz), ("num_tokens", _i32), ("num_experts", _i32), ("top_k", _i32),
                ("num_sequences", _i32), ("scoring", _i32), ("alpha", _f32)]


class MoeBalanceGradArgs(ctypes.Structure):
    _fields_ = [("routing_logits", _vp), ("topk_idx", _vp), ("cu_seqlens", _vp), ("counts", _vp), ("tokens", _vp),
                ("sequences", _vp), ("grad_loss", _vp), ("grad_topk_weights", _vp), ("grad_logits", _vp),
                ("num_tokens", _i32), ("num_experts", _i32), ("top_k", _i32), ("num_sequences", _i32),
                ("scoring", _i32), ("alpha", _f32), ("routed_scaling_factor", _f32)]


class LinearCheckpoint(NamedTuple):
    """What `linear_backward` needs of a forward pass: the input and, with an
    activation, the pre-activation, both as 8-bit checkpoints."""
    x: torch.Tensor                     # e4m3 [M, K]
    x_scale: torch.Tensor               # e8m0 [ceil(K / 128), M]
    z: Optional[torch.Tensor]           # e4m3 [M, N]; [2, M, N / 2] for swiglu; None for "none"
    z_scale: Optional[torch.Tensor]     # e8m0 [ceil(N / 128), M]; [2, ceil(N / 2 / 128), M]
    activation: str


class LinearGrads(NamedTuple):
    x: Optional[torch.Tensor]
    weight: Optional[torch.Tensor]
    bias: Optional[torch.Tensor]


class BalanceLoss(NamedTuple):
    loss: torch.Tensor                  # f32 []
    counts: torch.Tensor                # int32 [S, E] picks per sequence and expert
    tokens: torch.Tensor                # int32 [S] tokens per sequence, padding left out
    mean_scores: torch.Tensor           # f32 [S, E]
    sequences: torch.Tensor             # int32 [] sequences with tokens


_declared = None
_binding = None


def _native():
    """The native binding, loaded after the library it calls."""
    global _binding
    if _binding is None:
        _library()
        if not BINDING_PATH.exists():
            raise RuntimeError(f"{BINDING_PATH.name} is not built; run `python starter-kit-fused-moe_b200/build.py`")
        spec = importlib.util.spec_from_file_location("moe_b200_layer", BINDING_PATH)
        mod = importlib.util.module_from_spec(spec)
        spec.loader.exec_module(mod)
        _binding = mod
    return _binding


def _library():
    global _declared
    if _declared is None:
        from . import load_library
        lib = load_library()
        for name, args, res in (
                ("moe_linear_workspace_bytes", [_vp], _sz), ("moe_linear_run", [_vp, _vp], ctypes.c_int),
                ("moe_linear_grad_workspace_bytes", [_vp], _sz), ("moe_linear_grad", [_vp, _vp], ctypes.c_int),
                ("moe_checkpoint_activations", [_vp, _i32, _i64, _i64, _i64, _vp, _vp, _vp], ctypes.c_int),
                ("moe_restore_activations", [_vp, _vp, _i64, _i64, _i64, _vp, _i32, _vp], ctypes.c_int),
                ("moe_balance_workspace_bytes", [_i32, _i32, _i32], _sz),
                ("moe_balance_loss", [_vp, _vp], ctypes.c_int), ("moe_balance_loss_grad", [_vp, _vp], ctypes.c_int)):
            f = getattr(lib, name)
            f.argtypes, f.restype = args, res
        _declared = lib
    return _declared


def linear(x, weight, bias=None, residual=None, activation="none", out_dtype=torch.bfloat16, output=None):
    """y = act(x W^T + bias) + residual.

    x bf16 [M, K], weight bf16 [N, K], bias bf16 [N], residual bf16 [M, O];
    activation "none", "relu", "gelu" (erf form), "silu" or "swiglu" (first half
    of the N columns times silu of the second half, as in the routed experts;
    O = N / 2, otherwise O = N). Products are summed in fp32; the result is
    rounded once to `out_dtype` (bf16 or f32). `output` [M, O] is written in
    place when given and returned; it may be the residual itself (bf16) or columns
    beside x or the residual in the same rows, but not overlap an input. Any sizes with
    K, N >= 1 and any strides (rows that are not contiguous are copied first).
    f32 logits for `route` and `run` come from `out_dtype=torch.float32`.
    """
    return _native().linear(x, weight, bias, residual, activation, out_dtype, output, False)[0]


def linear_checkpointed(x, weight, bias=None, residual=None, activation="none", out_dtype=torch.bfloat16, output=None):
    """`linear` for a training step: returns (y, LinearCheckpoint). The checkpoint keeps
    x and, with an activation, the pre-activation z = x W^T + bias in 8 bits each."""
    y, *kept = _native().linear_checkpointed(x, weight, bias, residual, activation, out_dtype, output)
    return y, LinearCheckpoint(*kept, activation)


def linear_backward(grad_output, checkpoint, weight, need_x=True, need_weight=True, need_bias=False,
                    grad_dtype=torch.bfloat16):
    """Gradients of `linear_checkpointed`: LinearGrads(x [M, K], weight [N, K], bias [N]).

    dz = grad_output * act'(z^); x: dz W, weight: dz^T x^, bias: the sum of dz
    over the tokens, with x^ and z^ the checkpoint's values; a gradient that is
    not asked for is None. (The residual's gradient is grad_output.)
    grad_output is bf16 or f32 [M, O]. With grad_dtype bf16, dz is rounded to
    bf16 for the products; with f32 it enters them as the sum of three bf16 terms.
    Repeated calls give the same bits.
    """
    c = checkpoint
    return LinearGrads(*_native().linear_backward(grad_output, c.x, c.x_scale, c.z, c.z_scale, c.activation, weight,
                                                  need_x, need_weight, need_bias, grad_dtype))


def checkpoint_activations(x):
    """x bf16 or f32 [T, K] -> (e4m3 [T, K], e8m0 scales [ceil(K / 128), T]).

    Per 1x128 block the scale is the least power of two 2^e with
    amax <= 448 * 2^e (e >= -117) and the bytes are e4m3(x / 2^e), round to
    nearest even; a block with an infinity or NaN comes back as NaN. Restored
    values are exact in bf16.
    """
    return _native().checkpoint(x)


def restore_activations(q, scale, dtype=torch.bfloat16):
    """The values of an 8-bit checkpoint (e4m3 [.., T, K], e8m0 [.., ceil(K / 128), T]), as bf16 or f32."""
    return _native().restore(q, scale, dtype)


def balance_loss(routing_logits, topk_idx, cu_seqlens=None, alpha=1e-4, scoring="sigmoid"):
    """The router's balance loss and the picks per expert.

    routing_logits f32 [T, E], topk_idx int32 [T, k] (as `route` returns it),
    cu_seqlens int32 [S + 1] on the device, or None for one sequence. With
    p = sigmoid scores over their sum (or softmax), T_q the tokens of sequence q:

        loss = alpha * mean over sequences with tokens of sum_e f_qe P_qe,
        f_qe = E / (k T_q) * counts_qe,  P_qe = mean over the sequence of p_te.

    A pick outside [0, E) selects nothing and a token without picks is padding:
    it counts nowhere. Boundaries that decrease or leave [0, T], one or several, give
    a NaN loss, -1 for `sequences` and all `tokens`, counts of 0, NaN mean scores and
    NaN gradients. The outputs share one allocation: keep `loss.clone()` where losses
    are kept over many steps.
    """
    return BalanceLoss(*_native().balance_loss(routing_logits, topk_idx, cu_seqlens, alpha, scoring))


def balance_loss_backward(routing_logits, topk_idx, balance, cu_seqlens=None, grad_loss=None, alpha=1e-4,
                          scoring="sigmoid", grad_topk_weights=None, routed_scaling_factor=2.5):
    """Gradient of the routing logits, f32 [T, E].

    The balance loss's part is grad_loss (a number or an f32 device scalar; None: 1)
    times the gradient of `balance_loss` with the same arguments, the counts held
    constant; `balance` is what it returned, or None to leave this part out. With
    grad_topk_weights f32 [T, k] the gradient of the combine weights of `route`
    (w = s / (sum of the picked s + 1e-20) * routed_scaling_factor, s the sigmoid)
    is added for every token, so one pass trains the router on both.
    """
    counts = tokens = sequences = None
    if balance is not None:
        counts, tokens, sequences = balance.counts, balance.tokens, balance.sequences
        if grad_loss is not None and not isinstance(grad_loss, torch.Tensor):
            alpha, grad_loss = alpha * float(grad_loss), None
    elif grad_loss is not None:
        raise ValueError("grad_loss needs what balance_loss returned")
    return _native().balance_loss_backward(routing_logits, topk_idx, counts, tokens, sequences, cu_seqlens, grad_loss,
                                           alpha, scoring, grad_topk_weights, routed_scaling_factor)
