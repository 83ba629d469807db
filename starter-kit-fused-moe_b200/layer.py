"""Operators around the routed experts, for layers that are trained: dense
products (the router's gate, the shared expert) with their 8-bit activation
checkpoints and gradients, and the router's balance loss with its gradient.

Everything is computed by the library's own kernels through its C ABI
(`moe_linear_*`, `moe_checkpoint_*`, `moe_restore_*`, `moe_balance_*` in
include/moe_fp8.h) on the current stream of the tensors' device, without host
synchronisation. No autograd graph is recorded: gradients are computed by the
`*_backward` functions. Outputs and workspaces come from torch's allocator per
call, so calls on several streams and in several captured graphs do not share
memory. The reference holds the routed operator alone and has no counterpart.
"""
from __future__ import annotations

import ctypes
from typing import NamedTuple, Optional

import torch

ACTIVATIONS = {"none": 0, "relu": 1, "gelu": 2, "silu": 3, "swiglu": 4}
SCORINGS = {"sigmoid": 0, "softmax": 1}
_BF16, _F32, _E4M3, _E8M0 = torch.bfloat16, torch.float32, torch.float8_e4m3fn, torch.float8_e8m0fnu

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


def _check(rc, what):
    if rc:
        from . import _check as check
        check(rc, what)


def _tensor(t, name, dims, dtypes, device=None):
    if not isinstance(t, torch.Tensor):
        raise ValueError(f"{name} must be a tensor, got {type(t).__name__}")
    if t.dim() != dims or t.dtype not in dtypes:
        raise ValueError(f"{name} must be a {dims}-d tensor of {' or '.join(str(d) for d in dtypes)}, "
                         f"got {t.dtype} {tuple(t.shape)}")
    if not t.is_cuda:
        raise ValueError(f"{name} must be a CUDA tensor")
    if device is not None and t.device != device:
        raise ValueError(f"{name} must be on {device}, got {t.device}")


def _shape(t, name, shape):
    if tuple(t.shape) != tuple(shape):
        raise ValueError(f"{name} must have shape {tuple(shape)}, got {tuple(t.shape)}")


def _rows(t):
    """(tensor, row stride) of a matrix whose rows the kernels can read in place, copied if they cannot."""
    m, n = t.shape
    s0, s1 = t.stride()
    if (s1 == 1 or n == 1) and (s0 >= n or m == 1):
        return t, (s0 if m > 1 else n)
    return t.contiguous(), n


def _span(t):
    """Byte range that a tensor's values lie in."""
    a = t.data_ptr()
    return a, a + (sum((n - 1) * s for n, s in zip(t.shape, t.stride())) + 1) * t.element_size() if t.numel() else a


def _overlap(a, b):
    (a0, a1), (b0, b1) = _span(a), _span(b)
    return a0 < b1 and b0 < a1


def _stream(device):
    return torch.cuda.current_stream(device).cuda_stream


def _activation(name):
    if name not in ACTIVATIONS:
        raise ValueError(f"activation must be one of {', '.join(ACTIVATIONS)}, got {name!r}")
    return ACTIVATIONS[name]


def _call(function, what, args, device):
    with torch.cuda.device(device):
        _check(function(ctypes.byref(args), _stream(device)), what)


def _linear(x, weight, bias, residual, activation, out_dtype, output, keep):
    act = _activation(activation)
    _tensor(x, "x", 2, (_BF16,))
    dev = x.device
    _tensor(weight, "weight", 2, (_BF16,), dev)
    M, K = x.shape
    N = weight.shape[0]
    if K < 1 or N < 1 or weight.shape[1] != K:
        raise ValueError(f"weight must be [N, {K}] with N and K at least 1, got {tuple(weight.shape)}")
    if act == 4 and N % 2:
        raise ValueError(f"swiglu needs an even number of weight rows, got {N}")
    O = N // 2 if act == 4 else N
    if out_dtype not in (_BF16, _F32):
        raise ValueError(f"out_dtype must be bfloat16 or float32, got {out_dtype}")
    a = MoeLinearArgs()
    if bias is not None:
        _tensor(bias, "bias", 1, (_BF16,), dev)
        _shape(bias, "bias", (N,))
        bias = bias.contiguous()
        a.bias = bias.data_ptr()
    xr, a.ldx = _rows(x)
    wr, a.ldw = _rows(weight)
    if residual is not None:
        _tensor(residual, "residual", 2, (_BF16,), dev)
        _shape(residual, "residual", (M, O))
    y = output
    if output is not None:
        _tensor(output, "output", 2, (out_dtype,), dev)
        _shape(output, "output", (M, O))
        for name, t in (("x", x), ("weight", weight), ("bias", bias)):
            if t is not None and _overlap(output, t):
                raise ValueError(f"output overlaps {name}")
        if residual is not None and _overlap(output, residual) and not (
                output.data_ptr() == residual.data_ptr() and output.stride() == residual.stride()):
            raise ValueError("output may be the residual itself but not overlap it otherwise")
        s0, s1 = output.stride()
        if not ((s1 == 1 or O == 1) and (s0 >= O or M == 1)):
            y = None
    if y is None:
        y = torch.empty(M, O, dtype=out_dtype, device=dev)
    a.y, a.ldy, a.y_f32 = y.data_ptr(), (y.stride(0) if M > 1 else O), int(out_dtype == _F32)
    if residual is not None:
        rr, a.ldr = _rows(residual)
        a.residual = rr.data_ptr()
    a.x, a.weight, a.m, a.k, a.n, a.activation = xr.data_ptr(), wr.data_ptr(), M, K, N, act
    z = z_scale = None
    if keep and act:
        halves = (2,) if act == 4 else ()
        z = torch.empty(*halves, M, O, dtype=_E4M3, device=dev)
        z_scale = torch.empty(*halves, -(-O // 128), M, dtype=_E8M0, device=dev)
        a.z8, a.z_scale = z.data_ptr(), z_scale.data_ptr()
    if M > 0:
        lib = _library()
        need = lib.moe_linear_workspace_bytes(ctypes.byref(a))
        if need:
            ws = torch.empty(need, dtype=torch.uint8, device=dev)
            a.workspace, a.workspace_bytes = ws.data_ptr(), need
        _call(lib.moe_linear_run, "moe_linear_run", a, dev)
    if output is not None and y is not output:
        output.copy_(y)
        y = output
    return y, z, z_scale


@torch.no_grad()
def linear(x, weight, bias=None, residual=None, activation="none", out_dtype=torch.bfloat16, output=None):
    """y = act(x W^T + bias) + residual.

    x bf16 [M, K], weight bf16 [N, K], bias bf16 [N], residual bf16 [M, O];
    activation "none", "relu", "gelu" (erf form), "silu" or "swiglu" (first half
    of the N columns times silu of the second half, as in the routed experts;
    O = N / 2, otherwise O = N). Products are summed in fp32; the result is
    rounded once to `out_dtype` (bf16 or f32). `output` [M, O] is written in
    place when given and returned; it may be the residual itself. Any sizes with
    K, N >= 1 and any strides (rows that are not contiguous are copied first).
    f32 logits for `route` and `run` come from `out_dtype=torch.float32`.
    """
    return _linear(x, weight, bias, residual, activation, out_dtype, output, False)[0]


@torch.no_grad()
def linear_checkpointed(x, weight, bias=None, residual=None, activation="none", out_dtype=torch.bfloat16, output=None):
    """`linear` for a training step: returns (y, LinearCheckpoint). The checkpoint keeps
    x and, with an activation, the pre-activation z = x W^T + bias in 8 bits each."""
    y, z, z_scale = _linear(x, weight, bias, residual, activation, out_dtype, output, True)
    q, s = checkpoint_activations(x)
    return y, LinearCheckpoint(q, s, z, z_scale, activation)


@torch.no_grad()
def linear_backward(grad_output, checkpoint, weight, need_x=True, need_weight=True, need_bias=False,
                    grad_dtype=torch.bfloat16):
    """Gradients of `linear_checkpointed`: LinearGrads(x [M, K], weight [N, K], bias [N]).

    dz = grad_output * act'(z^); x: dz W, weight: dz^T x^, bias: the sum of dz
    over the tokens, with x^ and z^ the checkpoint's values; a gradient that is
    not asked for is None. (The residual's gradient is grad_output.)
    grad_output is bf16 or f32 [M, O]. With grad_dtype bf16, dz is rounded to
    bf16 for the products; with f32 it enters them as the sum of two bf16 terms.
    Repeated calls give the same bits.
    """
    act = _activation(checkpoint.activation)
    _tensor(weight, "weight", 2, (_BF16,))
    dev = weight.device
    N, K = weight.shape
    if K < 1 or N < 1 or (act == 4 and N % 2):
        raise ValueError(f"weight must be [N, K] with K and N at least 1 (N even for swiglu), got {tuple(weight.shape)}")
    O = N // 2 if act == 4 else N
    _tensor(grad_output, "grad_output", 2, (_BF16, _F32), dev)
    M = grad_output.shape[0]
    _shape(grad_output, "grad_output", (M, O))
    if grad_dtype not in (_BF16, _F32):
        raise ValueError(f"grad_dtype must be bfloat16 or float32, got {grad_dtype}")
    a = MoeLinearGradArgs()
    keep = []

    def pair(q, s, name, shape, scale_shape, lead):
        _tensor(q, f"checkpoint.{name}", 2 + lead, (_E4M3,), dev)
        _tensor(s, f"checkpoint.{name}_scale", 2 + lead, (_E8M0,), dev)
        _shape(q, f"checkpoint.{name}", shape)
        _shape(s, f"checkpoint.{name}_scale", scale_shape)
        q, s = q.contiguous(), s.contiguous()
        keep.extend((q, s))
        return q.data_ptr(), s.data_ptr()

    a.x8, a.x_scale = pair(checkpoint.x, checkpoint.x_scale, "x", (M, K), (-(-K // 128), M), 0)
    if act:
        lead = (2,) if act == 4 else ()
        a.z8, a.z_scale = pair(checkpoint.z, checkpoint.z_scale, "z", (*lead, M, O), (*lead, -(-O // 128), M), len(lead))
    wr, a.ldw = _rows(weight)
    gr, a.ldg = _rows(grad_output)
    a.weight, a.grad_y = wr.data_ptr(), gr.data_ptr()
    a.m, a.k, a.n, a.activation = M, K, N, act
    a.grad_y_f32, a.grad_f32 = int(grad_output.dtype == _F32), int(grad_dtype == _F32)
    gx = torch.empty(M, K, dtype=grad_dtype, device=dev) if need_x else None
    gw = torch.empty(N, K, dtype=grad_dtype, device=dev) if need_weight else None
    gb = torch.empty(N, dtype=grad_dtype, device=dev) if need_bias else None
    a.grad_x, a.grad_weight, a.grad_bias = (t.data_ptr() if t is not None and t.numel() else None for t in (gx, gw, gb))
    lib = _library()
    need = lib.moe_linear_grad_workspace_bytes(ctypes.byref(a))
    if need:
        ws = torch.empty(need, dtype=torch.uint8, device=dev)
        a.workspace, a.workspace_bytes = ws.data_ptr(), need
    _call(lib.moe_linear_grad, "moe_linear_grad", a, dev)
    return LinearGrads(gx, gw, gb)


@torch.no_grad()
def checkpoint_activations(x):
    """x bf16 or f32 [T, K] -> (e4m3 [T, K], e8m0 scales [ceil(K / 128), T]).

    Per 1x128 block the scale is the least power of two 2^e with
    amax <= 448 * 2^e (e >= -117) and the bytes are e4m3(x / 2^e), round to
    nearest even; a block with an infinity or NaN comes back as NaN. Restored
    values are exact in bf16.
    """
    _tensor(x, "x", 2, (_BF16, _F32))
    T, K = x.shape
    dev = x.device
    q = torch.empty(T, K, dtype=_E4M3, device=dev)
    s = torch.empty(-(-K // 128), T, dtype=_E8M0, device=dev)
    if x.numel():
        xr, ld = _rows(x)
        with torch.cuda.device(dev):
            _check(_library().moe_checkpoint_activations(xr.data_ptr(), int(x.dtype == _BF16), T, K, ld, q.data_ptr(),
                                                         s.data_ptr(), _stream(dev)), "moe_checkpoint_activations")
    return q, s


@torch.no_grad()
def restore_activations(q, scale, dtype=torch.bfloat16):
    """The values of an 8-bit checkpoint (e4m3 [.., T, K], e8m0 [.., ceil(K / 128), T]), as bf16 or f32."""
    if not isinstance(q, torch.Tensor) or q.dim() not in (2, 3):
        raise ValueError("q must be a tensor of 2 or 3 dimensions")
    _tensor(q, "q", q.dim(), (_E4M3,))
    _tensor(scale, "scale", q.dim(), (_E8M0,), q.device)
    T, K = q.shape[-2:]
    _shape(scale, "scale", (*q.shape[:-2], -(-K // 128), T))
    if dtype not in (_BF16, _F32):
        raise ValueError(f"dtype must be bfloat16 or float32, got {dtype}")
    dev = q.device
    out = torch.empty(q.shape, dtype=dtype, device=dev)
    if q.numel():
        qc, sc = q.contiguous(), scale.contiguous()
        with torch.cuda.device(dev):
            _check(_library().moe_restore_activations(qc.data_ptr(), sc.data_ptr(), q.shape[0] if q.dim() == 3 else 1,
                                                      T, K, out.data_ptr(), int(dtype == _F32), _stream(dev)),
                   "moe_restore_activations")
    return out


def _router_inputs(routing_logits, topk_idx, cu_seqlens, scoring):
    _tensor(routing_logits, "routing_logits", 2, (_F32,))
    dev = routing_logits.device
    _tensor(topk_idx, "topk_idx", 2, (torch.int32,), dev)
    T, E = routing_logits.shape
    if topk_idx.shape[0] != T or not 1 <= E <= 1024 or not 1 <= topk_idx.shape[1] <= 32:
        raise ValueError(f"routing_logits must be [T, E] with E in [1, 1024] and topk_idx [T, k] with k in [1, 32], "
                         f"got {tuple(routing_logits.shape)} and {tuple(topk_idx.shape)}")
    if scoring not in SCORINGS:
        raise ValueError(f"scoring must be one of {', '.join(SCORINGS)}, got {scoring!r}")
    S = 1
    if cu_seqlens is not None:
        _tensor(cu_seqlens, "cu_seqlens", 1, (torch.int32,), dev)
        S = cu_seqlens.shape[0] - 1
        if not 1 <= S <= 65535:
            raise ValueError(f"cu_seqlens must hold 2 to 65536 boundaries, got {S + 1}")
        cu_seqlens = cu_seqlens.contiguous()
    return routing_logits.contiguous(), topk_idx.contiguous(), cu_seqlens, S


@torch.no_grad()
def balance_loss(routing_logits, topk_idx, cu_seqlens=None, alpha=1e-4, scoring="sigmoid"):
    """The router's balance loss and the picks per expert.

    routing_logits f32 [T, E], topk_idx int32 [T, k] (as `route` returns it),
    cu_seqlens int32 [S + 1] on the device, or None for one sequence. With
    p = sigmoid scores over their sum (or softmax), T_q the tokens of sequence q:

        loss = alpha * mean over sequences with tokens of sum_e f_qe P_qe,
        f_qe = E / (k T_q) * counts_qe,  P_qe = mean over the sequence of p_te.

    A pick outside [0, E) selects nothing and a token without picks is padding:
    it counts nowhere. Boundaries that decrease or leave [0, T] give a NaN loss.
    """
    logits, idx, cu, S = _router_inputs(routing_logits, topk_idx, cu_seqlens, scoring)
    T, E = logits.shape
    dev = logits.device
    out = BalanceLoss(torch.empty((), dtype=_F32, device=dev), torch.empty(S, E, dtype=torch.int32, device=dev),
                      torch.empty(S, dtype=torch.int32, device=dev), torch.empty(S, E, dtype=_F32, device=dev),
                      torch.empty((), dtype=torch.int32, device=dev))
    lib = _library()
    need = lib.moe_balance_workspace_bytes(T, E, S)
    ws = torch.empty(need, dtype=torch.uint8, device=dev)
    a = MoeBalanceArgs(logits.data_ptr(), idx.data_ptr(), cu.data_ptr() if cu is not None else None,
                       out.loss.data_ptr(), out.counts.data_ptr(), out.tokens.data_ptr(), out.mean_scores.data_ptr(),
                       out.sequences.data_ptr(), ws.data_ptr(), need, T, E, idx.shape[1], S, SCORINGS[scoring],
                       float(alpha))
    _call(lib.moe_balance_loss, "moe_balance_loss", a, dev)
    return out


@torch.no_grad()
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
    logits, idx, cu, S = _router_inputs(routing_logits, topk_idx, cu_seqlens, scoring)
    T, E = logits.shape
    k = idx.shape[1]
    dev = logits.device
    a = MoeBalanceGradArgs()
    keep = []
    if balance is not None:
        if grad_loss is None or not isinstance(grad_loss, torch.Tensor):
            grad_loss = torch.full((), 1.0 if grad_loss is None else float(grad_loss), dtype=_F32, device=dev)
        if grad_loss.numel() != 1 or grad_loss.dtype != _F32 or grad_loss.device != dev:
            raise ValueError("grad_loss must be a number or one f32 value on the logits' device")
        for name, t, shape in (("counts", balance.counts, (S, E)), ("tokens", balance.tokens, (S,)),
                               ("sequences", balance.sequences, ())):
            _tensor(t, f"balance.{name}", len(shape), (torch.int32,), dev)
            _shape(t, f"balance.{name}", shape)
            t = t.contiguous()
            keep.append(t)
            setattr(a, name, t.data_ptr())
        a.grad_loss = grad_loss.data_ptr()
    elif grad_loss is not None:
        raise ValueError("grad_loss needs what balance_loss returned")
    if grad_topk_weights is not None:
        _tensor(grad_topk_weights, "grad_topk_weights", 2, (_F32,), dev)
        _shape(grad_topk_weights, "grad_topk_weights", (T, k))
        grad_topk_weights = grad_topk_weights.contiguous()
        a.grad_topk_weights = grad_topk_weights.data_ptr()
    grad = torch.empty(T, E, dtype=_F32, device=dev)
    a.routing_logits, a.topk_idx, a.grad_logits = logits.data_ptr(), idx.data_ptr(), grad.data_ptr()
    a.cu_seqlens = cu.data_ptr() if cu is not None else None
    a.num_tokens, a.num_experts, a.top_k, a.num_sequences = T, E, k, S
    a.scoring, a.alpha, a.routed_scaling_factor = SCORINGS[scoring], float(alpha), float(routed_scaling_factor)
    if T > 0:
        _call(_library().moe_balance_loss_grad, "moe_balance_loss_grad", a, dev)
    return grad
