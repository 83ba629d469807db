"""Measured cases of the operators that stand around the routed experts of a layer in training.

* ``linear``: y = act(x W^T + b) + r, the dense products of the layer: the router's gate (f32 logits),
  the shared expert's gate/up product (SwiGLU) and its down product with the routed experts' output as the residual.
* ``linear_checkpointed`` / ``linear_backward``: the same product keeping its input and pre-activation in 8 bits
  (e4m3 with one power-of-two scale per 1x128 block), and the gradients computed from those checkpoints.
* ``checkpoint_activations`` / ``restore_activations``: the 8-bit checkpoints on their own.
* ``balance_loss`` / ``balance_loss_backward``: the per-sequence balance loss of the router with the counts per
  expert, and the gradient of the loss and of the combine weights with respect to the routing logits.

Hidden size 7168, intermediate size 2048 (gate and up rows: 4096) and 256 experts with 8 picks are the
framework's own geometry; 1, 64, 600, 4096 and 16384 tokens are those of its benchmark and tests.
"""
import math

import torch

own = False

HIDDEN, INTER, EXPERTS, PICKS = 7168, 2048, 256, 8
ACTIVATIONS = ("none", "relu", "gelu", "silu", "swiglu")
BLOCK = 128
MOST_MACS = 16384 * HIDDEN * 2 * INTER     # of one product of the largest listed case


def _linear(name, m, k, n, act="none", bias=False, residual=False, out="bf16"):
    c = {"op": "linear", "m": m, "k": k, "n": n, "act": act, "bias": bias, "residual": residual, "out": out}
    return {"name": name, **c} if name else c


def _backward(name, m, k, n, act="none", bias=False, grad_in="bf16", grad="bf16"):
    c = {"op": "backward", "m": m, "k": k, "n": n, "act": act, "bias": bias, "grad_in": grad_in, "grad": grad}
    return {"name": name, **c} if name else c


def _balance(name, t, e, k, seqs, scoring="sigmoid", weights=True):
    c = {"op": "balance", "t": t, "e": e, "k": k, "seqs": seqs, "scoring": scoring, "weights": weights}
    return {"name": name, **c} if name else c


def listed():
    return [
        # the router's gate for one token of a serving step: a weight stream of 3.7 MB, latency counts
        _linear("gate 1 token", 1, HIDDEN, EXPERTS, out="f32"),
        # the shared expert's gate/up product in a decode step of 64 tokens: a weight stream of 59 MB
        _linear("up 64 tokens", 64, HIDDEN, 2 * INTER, act="swiglu"),
        # the shared expert's down product of a prompt, added to the routed experts' output
        _linear("down 4096 tokens", 4096, INTER, HIDDEN, residual=True),
        # a small projection with nothing aligned: rows that no bulk copy can read, edges in every tile
        _linear("odd projection", 1037, 1111, 515, act="gelu", bias=True, residual=True),
        # a training step's forward: SwiGLU product keeping its 8-bit checkpoints
        {"name": "train up 4096 tokens", "op": "train", "m": 4096, "k": HIDDEN, "n": 2 * INTER, "act": "swiglu", "bias": False},
        # gradients of the down product of a short batch
        _backward("backward down 600 tokens", 600, INTER, HIDDEN),
        # gradients of the gate, from f32 gradients of the logits to f32 gradients
        _backward("backward gate 4096 tokens", 4096, HIDDEN, EXPERTS, grad_in="f32", grad="f32"),
        # gradients of the SwiGLU product over the largest token count
        _backward("backward up 16384 tokens", 16384, HIDDEN, 2 * INTER, act="swiglu"),
        # the layer's input kept in 8 bits and brought back, at the largest token count and at an odd size
        {"name": "checkpoint 16384 tokens", "op": "checkpoint", "t": 16384, "k": HIDDEN, "dtype": "bf16"},
        {"name": "checkpoint odd", "op": "checkpoint", "t": 333, "k": 1001, "dtype": "f32"},
        # the balance loss of one short sequence, and of a packed batch of ragged sequences
        _balance("balance 64 tokens", 64, EXPERTS, PICKS, 1),
        _balance("balance 16384 tokens", 16384, EXPERTS, PICKS, 13),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("linear", "linear", "train", "backward", "backward", "checkpoint", "balance"))
    if op == "checkpoint":
        return {"op": op, "t": _log(rng, 1, 16384), "k": _log(rng, 16, HIDDEN), "dtype": rng.choice(("bf16", "f32"))}
    if op == "balance":
        t = _log(rng, 1, 16384)
        e = rng.choice((EXPERTS, _log(rng, 8, 512)))
        return _balance(None, t, e, rng.randint(1, 8), _log(rng, 1, min(t, 128)), rng.choice(("sigmoid", "softmax")),
                        rng.choice((False, True)))
    while True:
        m, k, n = _log(rng, 1, 16384), _log(rng, 32, HIDDEN), _log(rng, 16, HIDDEN)
        if rng.random() < 0.5:          # half of the cases as models have them, half as they come
            k, n = max(64, k // 64 * 64), max(64, n // 64 * 64)
        if m * k * n <= MOST_MACS // 2:
            break
    act = rng.choice(ACTIVATIONS)
    n += n % 2 if act == "swiglu" else 0
    bias = rng.choice((False, True))
    if op == "linear":
        return _linear(None, m, k, n, act, bias, rng.choice((False, True)), rng.choice(("bf16", "bf16", "f32")))
    if op == "train":
        return {"op": op, "m": m, "k": k, "n": n, "act": act, "bias": bias}
    return _backward(None, m, k, n, act, bias, rng.choice(("bf16", "bf16", "f32")), rng.choice(("bf16", "bf16", "f32")))


def _out_width(c):
    return c["n"] // 2 if c["act"] == "swiglu" else c["n"]


# ------------------------------------------------------------------------------------------------ inputs
_DT = {"bf16": torch.bfloat16, "f32": torch.float32}


def _activations(t, k, g):
    """Normal values with some channels much larger than the rest, as the inputs of a layer have."""
    x = torch.randn(t, k, generator=g, device="cuda")
    return x * torch.exp(0.7 * torch.randn(k, generator=g, device="cuda"))


def _block_exponents(x):
    """Per 1x128 block of x [..., T, K]: the least e with amax <= 448 * 2^e, at least -117; [..., blocks, T]."""
    k = x.shape[-1]
    xb = torch.nn.functional.pad(x.abs(), (0, -k % BLOCK)).unflatten(-1, (-1, BLOCK))
    amax = xb.amax(-1)
    m, e = torch.frexp(amax)
    e = torch.where(m <= 0.875, e - 9, e - 8)
    e = torch.where(amax == 0, torch.full_like(e, -117), e).clamp(min=-117)
    return e.to(torch.int32).transpose(-1, -2).contiguous()


def _spread(e, k):
    """Block exponents [..., blocks, T] for every value [..., T, K]."""
    return e.transpose(-1, -2).repeat_interleave(BLOCK, -1)[..., :k]


def _quantize(x):
    """x f32 [..., T, K] -> (e4m3 values, e8m0 scales [..., blocks, T])."""
    e = _block_exponents(x)
    q = torch.ldexp(x, -_spread(e, x.shape[-1])).to(torch.float8_e4m3fn)
    return q, (e + 127).to(torch.uint8).view(torch.float8_e8m0fnu)


def _dequantize(q, s):
    e = s.view(torch.uint8).to(torch.int32) - 127
    return torch.ldexp(q.float(), _spread(e, q.shape[-1]))


def _cu_seqlens(t, seqs, g):
    """Ragged packed sequences covering the t tokens, one of them empty where there are several."""
    cuts = torch.randint(0, t + 1, (seqs - 1,), generator=g, device="cuda").sort().values
    if seqs > 2:
        cuts[1] = cuts[0]
    ends = torch.tensor([0, t], device="cuda")
    return torch.cat([ends[:1], cuts, ends[1:]]).to(torch.int32)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    c = dict(case)
    s = {"case": c}
    if c["op"] == "checkpoint":
        s["x"] = _activations(c["t"], c["k"], g).to(_DT[c["dtype"]])
        return s
    if c["op"] == "balance":
        t, e, k = c["t"], c["e"], c["k"]
        bias = 0.5 * torch.randn(e, generator=g, device="cuda")       # some experts are much more popular
        s["logits"] = torch.randn(t, e, generator=g, device="cuda") + bias
        noise = 0.3 * torch.randn(t, e, generator=g, device="cuda")   # the selection bias keeps changing
        s["idx"] = (s["logits"] + noise).topk(min(k, e), dim=1).indices.to(torch.int32)
        s["cu"] = _cu_seqlens(t, c["seqs"], g) if c["seqs"] > 1 else None
        s["grad_weights"] = 0.01 * torch.randn(t, min(k, e), generator=g, device="cuda") if c["weights"] else None
        s["grad_loss"] = 0.5 + torch.rand((), generator=g, device="cuda")
        return s
    m, k, n, o = c["m"], c["k"], c["n"], _out_width(c)
    x = _activations(m, k, g).to(torch.bfloat16)
    s["w"] = (torch.randn(n, k, generator=g, device="cuda") / math.sqrt(k)).to(torch.bfloat16)
    s["b"] = (0.1 * torch.randn(n, generator=g, device="cuda")).to(torch.bfloat16) if c["bias"] else None
    if c["op"] == "backward":
        s["x8"], s["xs"] = _quantize(x.float())
        s["z8"] = s["zs"] = None
        if c["act"] != "none":
            shape = (2, m, o) if c["act"] == "swiglu" else (m, n)
            s["z8"], s["zs"] = _quantize(1.3 * torch.randn(shape, generator=g, device="cuda"))
        s["dy"] = (0.02 * torch.randn(m, o, generator=g, device="cuda")).to(_DT[c["grad_in"]])
        return s
    s["x"] = x
    s["r"] = torch.randn(m, o, generator=g, device="cuda").to(torch.bfloat16) if c.get("residual") else None
    return s


# ------------------------------------------------------------------------------------------------ plain forms, 32 bits
def _phi(z):
    return 0.5 * (1 + torch.erf(z * math.sqrt(0.5)))


def _act(z, act):
    """z [..., N], or [2, ..., N] for swiglu (first half times silu of the second half)."""
    if act == "none":
        return z
    if act == "relu":
        return z.clamp(min=0)
    if act == "gelu":
        return z * _phi(z)
    if act == "silu":
        return z * torch.sigmoid(z)
    return z[0] * (z[1] * torch.sigmoid(z[1]))


def _act_backward(dy, z, act):
    """Gradient of the pre-activation; [M, 2 I] (first half, then second half) for swiglu."""
    if act == "none":
        return dy
    if act == "relu":
        return dy * (z > 0)
    if act == "gelu":
        return dy * (_phi(z) + z * torch.exp(-0.5 * z * z) / math.sqrt(2 * math.pi))
    if act == "silu":
        sg = torch.sigmoid(z)
        return dy * (sg * (1 + z * (1 - sg)))
    a, b = z[0], z[1]
    sg = torch.sigmoid(b)
    return torch.cat([dy * (b * sg), dy * a * (sg * (1 + b * (1 - sg)))], 1)


def _halves(z, act):
    return torch.stack(z.chunk(2, dim=1)) if act == "swiglu" else z


def _plain_linear(s):
    c = s["case"]
    z = s["x"].float() @ s["w"].float().t()
    if s["b"] is not None:
        z = z + s["b"].float()
    z = _halves(z, c["act"])
    y = _act(z, c["act"])
    if s["r"] is not None:
        y = y + s["r"].float()
    return y, z


def _plain_balance(s):
    c = s["case"]
    x, idx, t = s["logits"], s["idx"].long(), c["t"]
    e, k = c["e"], idx.shape[1]
    cu = s["cu"] if s["cu"] is not None else torch.tensor([0, t], device=x.device, dtype=torch.int32)
    n_seq = cu.numel() - 1
    seq = torch.searchsorted(cu[1:].contiguous(), torch.arange(t, device=x.device, dtype=torch.int32), right=True)
    sg = torch.sigmoid(x)
    if c["scoring"] == "sigmoid":
        den = sg.sum(1, keepdim=True) + 1e-20
        p = sg / den
    else:
        p = torch.softmax(x, 1)
    tokens = torch.bincount(seq, minlength=n_seq)
    counts = torch.bincount((seq[:, None] * e + idx).reshape(-1), minlength=n_seq * e).view(n_seq, e)
    sums = torch.zeros(n_seq, e, device=x.device, dtype=torch.float64).index_add_(0, seq, p.double())
    length = tokens.clamp(min=1)[:, None].double()
    mean = sums / length
    freq = counts.double() * (e / k) / length
    live = (tokens > 0).sum()
    alpha = 1e-3
    loss = alpha * (freq * mean).sum() / live
    # d loss / d p of every token of a sequence is the same row
    coef = (alpha * s["grad_loss"].double() * freq / (length * live)).float()[seq]
    inner = (coef * p).sum(1, keepdim=True)
    if c["scoring"] == "sigmoid":
        dx = (coef - inner) / den * (sg * (1 - sg))
    else:
        dx = p * (coef - inner)
    if s["grad_weights"] is not None:
        top = sg.gather(1, idx)
        total = top.sum(1, keepdim=True) + 1e-20
        dw = s["grad_weights"] * 2.5
        ds = (dw - (dw * top).sum(1, keepdim=True) / total) / total
        dx = dx + torch.zeros_like(dx).scatter_add_(1, idx, ds * top * (1 - top))
    return {"loss": loss.float(), "counts": counts.int(), "tokens": tokens.int(), "mean_scores": mean.float(),
            "grad_logits": dx}


def _plain(s):
    c = s["case"]
    if c["op"] == "linear":
        return {"y": _plain_linear(s)[0].to(_DT[c["out"]])}
    if c["op"] == "train":
        y, z = _plain_linear({**s, "r": None})
        x8, xs = _quantize(s["x"].float())
        out = {"y": y.to(torch.bfloat16), "x": _dequantize(x8, xs).to(torch.bfloat16)}
        if c["act"] != "none":
            out["z"] = _dequantize(*_quantize(z)).to(torch.bfloat16)
        return out
    if c["op"] == "backward":
        x = _dequantize(s["x8"], s["xs"])
        z = _dequantize(s["z8"], s["zs"]) if s["z8"] is not None else None
        dz = _act_backward(s["dy"].float(), z, c["act"])
        dt = _DT[c["grad"]]
        out = {"grad_x": (dz @ s["w"].float()).to(dt), "grad_weight": (dz.t() @ x).to(dt)}
        if c["bias"]:
            out["grad_bias"] = dz.sum(0, dtype=torch.float64).to(dt)
        return out
    if c["op"] == "checkpoint":
        q, sc = _quantize(s["x"].float())
        return {"x": _dequantize(q, sc).to(torch.bfloat16), "scale": sc.view(torch.uint8)}
    return _plain_balance(s)


# ------------------------------------------------------------------------------------------------ the framework's calls
_pkg = None


def _package():
    global _pkg
    if _pkg is None:
        import __graft_entry__
        _pkg = __graft_entry__.load_package()
    return _pkg


def _calls(s):
    P, c = _package(), s["case"]
    if c["op"] == "linear":
        return {"y": P.linear(s["x"], s["w"], bias=s["b"], residual=s["r"], activation=c["act"], out_dtype=_DT[c["out"]])}
    if c["op"] == "train":
        y, ck = P.linear_checkpointed(s["x"], s["w"], bias=s["b"], activation=c["act"])
        out = {"y": y, "x": P.restore_activations(ck.x, ck.x_scale)}
        if ck.z is not None:
            out["z"] = P.restore_activations(ck.z, ck.z_scale)
        return out
    if c["op"] == "backward":
        ck = P.LinearCheckpoint(s["x8"], s["xs"], s["z8"], s["zs"], c["act"])
        g = P.linear_backward(s["dy"], ck, s["w"], need_bias=c["bias"], grad_dtype=_DT[c["grad"]])
        out = {"grad_x": g.x, "grad_weight": g.weight}
        if c["bias"]:
            out["grad_bias"] = g.bias
        return out
    if c["op"] == "checkpoint":
        q, sc = P.checkpoint_activations(s["x"])
        return {"x": P.restore_activations(q, sc), "scale": sc.view(torch.uint8)}
    b = P.balance_loss(s["logits"], s["idx"], cu_seqlens=s["cu"], alpha=1e-3, scoring=c["scoring"])
    dx = P.balance_loss_backward(s["logits"], s["idx"], b, cu_seqlens=s["cu"], grad_loss=s["grad_loss"], alpha=1e-3,
                                 scoring=c["scoring"], grad_topk_weights=s["grad_weights"], routed_scaling_factor=2.5)
    return {"loss": b.loss, "counts": b.counts, "tokens": b.tokens, "mean_scores": b.mean_scores, "grad_logits": dx}


def run(state):
    return _calls(state) if own else _plain(state)


def work(case):
    c = case
    if c["op"] == "checkpoint":
        size = 4 if c["dtype"] == "f32" else 2
        n, blocks = c["t"] * c["k"], c["t"] * -(-c["k"] // BLOCK)
        # written in 8 bits, read again and brought back to 16 bits
        return {"bytes": n * (size + 1) + blocks + n * (1 + 2) + blocks, "flops": 0}
    if c["op"] == "balance":
        t, e, k, s = c["t"], c["e"], min(c["k"], c["e"]), c["seqs"]
        # logits and picks once, counts and mean scores written, the logits' gradient written
        return {"bytes": t * e * 4 + t * k * 4 * (2 if c["weights"] else 1) + s * e * 8 + t * e * 4, "flops": 0}
    m, k, n, o = c["m"], c["k"], c["n"], _out_width(c)
    small = 2 * n if c["bias"] else 0
    if c["op"] == "linear":
        out = m * o * (4 if c["out"] == "f32" else 2)
        return {"bytes": 2 * (m * k + n * k) + small + out + (2 * m * o if c["residual"] else 0), "flops": 2 * m * n * k}
    blocks = m * -(-k // BLOCK)
    zb = 0 if c["act"] == "none" else m * n + m * -(-n // BLOCK)
    if c["op"] == "train":
        # the 8-bit copies are written, read and returned as 16-bit values
        kept = m * k + blocks + zb
        return {"bytes": 2 * (m * k + n * k) + small + 2 * m * o + 2 * kept + 2 * m * k + (2 * m * n if zb else 0),
                "flops": 2 * m * n * k}
    gin, gout = (4 if c[x] == "f32" else 2 for x in ("grad_in", "grad"))
    return {"bytes": m * o * gin + m * k + blocks + zb + 2 * n * k + gout * (m * k + n * k + (n if c["bias"] else 0)),
            "flops": 4 * m * n * k}


# ------------------------------------------------------------------------------------------------ 64 bits
def _exact_checkpoint(x):
    """The values that the 8-bit checkpoint of x (float64 [..., T, K]) stands for: per block of 128 the power of
    two that brings the largest value to at most 448, then the nearest e4m3 number (3 fraction bits, least
    exponent -6), ties to even."""
    k = x.shape[-1]
    blocks = torch.nn.functional.pad(x, (0, -k % BLOCK)).unflatten(-1, (-1, BLOCK))
    amax = blocks.abs().amax(-1, keepdim=True)
    e = torch.ceil(torch.log2(amax.clamp(min=1e-300) / 448.0))
    e = torch.where(amax > 448.0 * torch.exp2(e), e + 1, e)       # the logarithm may be a hair off at a border
    e = torch.where(amax <= 448.0 * torch.exp2(e - 1), e - 1, e).clamp(min=-117.0)
    v = blocks / torch.exp2(e)
    top = torch.floor(torch.log2(v.abs().clamp(min=1e-300)))
    top = torch.where(torch.exp2(top + 1) <= v.abs(), top + 1, top)
    top = torch.where(torch.exp2(top) > v.abs(), top - 1, top).clamp(min=-6.0)
    step = torch.exp2(top - 3)
    q = torch.round(v / step) * step * torch.exp2(e)
    return q.flatten(-2)[..., :k], (e.squeeze(-1).transpose(-1, -2) + 127).to(torch.uint8)


def _exact_values(q8, s8):
    """Values of an 8-bit checkpoint, from the bytes."""
    b = q8.view(torch.uint8).long()
    sign, ex, fr = 1.0 - 2.0 * (b >> 7).double(), (b >> 3) & 15, (b & 7).double()
    mag = torch.where(ex > 0, (1 + fr / 8) * torch.exp2((ex - 7).double()), fr / 8 * 2.0 ** -6)
    scale = torch.exp2(s8.view(torch.uint8).double() - 127)
    return sign * mag * scale.transpose(-1, -2).repeat_interleave(BLOCK, -1)[..., : q8.shape[-1]]


def _normal_cdf(z):
    return 0.5 * torch.erfc(-z / math.sqrt(2.0))


def _logistic(z):
    return 1.0 / (1.0 + torch.exp(-z))


def _exact_dense(s, c):
    z = torch.einsum("mk,nk->mn", s["x"].double(), s["w"].double())
    if s["b"] is not None:
        z += s["b"].double()
    half = z.shape[1] // 2
    forms = {
        "none": lambda: z,
        "relu": lambda: torch.where(z > 0, z, 0.0),
        "gelu": lambda: z * _normal_cdf(z),
        "silu": lambda: z * _logistic(z),
        "swiglu": lambda: z[:, :half] * z[:, half:] * _logistic(z[:, half:]),
    }
    return forms[c["act"]](), z


def exact(case, seed):
    s = prepare(case, seed)
    c = s["case"]
    if c["op"] == "linear":
        y = _exact_dense(s, c)[0]
        return {"y": y + s["r"].double() if s["r"] is not None else y}
    if c["op"] == "train":
        y, z = _exact_dense(s, c)
        out = {"y": y, "x": _exact_checkpoint(s["x"].double())[0]}
        if c["act"] != "none":
            if c["act"] == "swiglu":
                z = torch.stack([z[:, : z.shape[1] // 2], z[:, z.shape[1] // 2:]])
            out["z"] = _exact_checkpoint(z)[0]
        return out
    if c["op"] == "checkpoint":
        v, code = _exact_checkpoint(s["x"].double())
        return {"x": v, "scale": code}
    if c["op"] == "backward":
        x = _exact_values(s["x8"], s["xs"])
        dz = s["dy"].double()
        if c["act"] != "none":
            z = _exact_values(s["z8"], s["zs"])
            gate = z[1] if c["act"] == "swiglu" else z
            sig = _logistic(gate)
            if c["act"] == "relu":
                dz = torch.where(z > 0, dz, 0.0)
            elif c["act"] == "gelu":
                dz = dz * (_normal_cdf(z) + z * torch.exp(-z.square() / 2) / math.sqrt(2 * math.pi))
            elif c["act"] == "silu":
                dz = dz * (sig + z * sig * (1 - sig))
            else:
                dz = torch.cat([dz * gate * sig, dz * z[0] * (sig + gate * sig * (1 - sig))], dim=1)
        out = {"grad_x": torch.einsum("mn,nk->mk", dz, s["w"].double()), "grad_weight": torch.einsum("mn,mk->nk", dz, x)}
        if c["bias"]:
            out["grad_bias"] = dz.sum(0)
        return out
    # balance: the definition's sums, sequence by sequence; gradients by hand for one row per token
    x, idx, t, e = s["logits"].double(), s["idx"].long(), c["t"], c["e"]
    k = idx.shape[1]
    bounds = s["cu"].tolist() if s["cu"] is not None else [0, t]
    sig = _logistic(x)
    score = sig if c["scoring"] == "sigmoid" else torch.exp(x - x.amax(1, keepdim=True))
    den = score.sum(1, keepdim=True) + (1e-20 if c["scoring"] == "sigmoid" else 0.0)
    p = score / den
    live = sum(b > a for a, b in zip(bounds, bounds[1:]))
    n_seq = len(bounds) - 1
    counts = torch.zeros(n_seq, e, device=x.device, dtype=torch.float64)
    mean = torch.zeros_like(counts)
    loss = torch.zeros((), device=x.device, dtype=torch.float64)
    dp = torch.zeros_like(p)
    picked = torch.zeros_like(p).scatter_add_(1, idx, torch.ones_like(idx, dtype=torch.float64))
    for q, (a, b) in enumerate(zip(bounds, bounds[1:])):
        if b > a:
            counts[q], mean[q] = picked[a:b].sum(0), p[a:b].mean(0)
            freq = counts[q] * e / (k * (b - a))
            loss += 1e-3 / live * (freq * mean[q]).sum()
            dp[a:b] = s["grad_loss"].double() * 1e-3 / live / (b - a) * freq
    dscore = (dp - (dp * p).sum(1, keepdim=True)) / den
    dx = dscore * (sig * (1 - sig) if c["scoring"] == "sigmoid" else score)
    if s["grad_weights"] is not None:
        top = sig.gather(1, idx)
        total = top.sum(1, keepdim=True) + 1e-20
        dw = 2.5 * s["grad_weights"].double()
        dtop = dw / total - (dw * top).sum(1, keepdim=True) / total.square()
        dx = dx.scatter_add(1, idx, dtop * top * (1 - top))
    return {"loss": loss, "counts": counts.int(), "tokens": torch.tensor([b - a for a, b in zip(bounds, bounds[1:])],
                                                                        dtype=torch.int32),
            "mean_scores": mean, "grad_logits": dx}
