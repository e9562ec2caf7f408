"""The operators of a transformer block and its scoring head, as programs call them.

A pre-norm block runs layer norm, then products in 16 bits whose epilogue adds the bias,
applies the activation and adds the residual stream; behind the last norm and product the
logits become log probabilities.  `listed()` names twelve cases; `draw(rng)` gives more of
the same ranges.

Operators and their ranges (odd sizes among the drawn ones):

  ln_fwd   y = (x - mean) * rstd * weight + bias over rows, with the rows' mean and rstd
  ln_bwd   its gradients: dx, dweight and dbias
  gemm     y = act(a b + bias) + residual, bf16 or fp16 operands, 1 token to a long prompt
  lp_fwd   log probabilities of given tokens, entropy and the top alternatives, one pass over
           logits whose rows may be padded
  lp_bwd   the gradient of log probabilities and entropies in the logits
"""
from __future__ import annotations

import math

import torch

own = False

ACTS = ("none", "relu", "gelu_erf", "gelu_tanh")
MAX_FLOPS = 2 * 4096 * 4096 * 16384
MAX_ELEMENTS = 1 << 27
EPS = 1e-5

_TORCH = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
_SIZE = {"f32": 4, "f16": 2, "bf16": 2}


def listed():
    return [
        # Decoding: the norm of eight sequences' single tokens, one short launch.
        {"name": "ln_fwd_decode", "op": "ln_fwd", "rows": 8, "cols": 4096, "dtype": "bf16",
         "param": "bf16"},
        # A training or prefill batch.
        {"name": "ln_fwd_batch", "op": "ln_fwd", "rows": 16384, "cols": 4096, "dtype": "bf16",
         "param": "bf16"},
        # The same batch's backward pass.
        {"name": "ln_bwd_batch", "op": "ln_bwd", "rows": 16384, "cols": 4096, "dtype": "bf16",
         "param": "bf16"},
        # A small model in fp32 over a ragged batch, rows of odd width.
        {"name": "ln_bwd_odd", "op": "ln_bwd", "rows": 5003, "cols": 1021, "dtype": "f32",
         "param": "f32"},
        # Decoding: the up projection of one token, bound by reading the weights.
        {"name": "gemm_decode", "op": "gemm", "m": 1, "n": 16384, "k": 4096, "ab": "bf16",
         "y": "bf16", "act": "gelu_tanh", "bias": "bf16", "residual": False},
        # The down projection of a long prompt, added to the residual stream.
        {"name": "gemm_down_4096", "op": "gemm", "m": 4096, "n": 4096, "k": 16384, "ab": "bf16",
         "y": "bf16", "act": "none", "bias": "bf16", "residual": True},
        # Odd in every extent, fp16 operands and an fp32 residual stream.
        {"name": "gemm_odd", "op": "gemm", "m": 1531, "n": 2053, "k": 1021, "ab": "f16",
         "y": "f32", "act": "gelu_erf", "bias": "f32", "residual": True},
        # Decoding: the log probabilities of four sampled tokens with the top twenty.
        {"name": "lp_fwd_decode", "op": "lp_fwd", "rows": 4, "vocab": 131072, "pad": 0,
         "dtype": "bf16", "scale": 1.0, "top": 20},
        # Scoring a prompt with its top twenty alternatives at each place.
        {"name": "lp_fwd_score", "op": "lp_fwd", "rows": 1024, "vocab": 131072, "pad": 0,
         "dtype": "bf16", "scale": 1.0, "top": 20},
        # A policy's log probabilities and entropies in training, at a temperature; fp32
        # logits, an odd vocabulary padded to whole rows of 64.
        {"name": "lp_fwd_policy", "op": "lp_fwd", "rows": 2047, "vocab": 32001, "pad": 63,
         "dtype": "f32", "scale": 1.25, "top": 0},
        # The gradient of a cross entropy loss with an entropy bonus.
        {"name": "lp_bwd_train", "op": "lp_bwd", "rows": 1024, "vocab": 131072, "pad": 0,
         "dtype": "bf16", "scale": 1.0},
        # The policy's gradient.
        {"name": "lp_bwd_policy", "op": "lp_bwd", "rows": 2047, "vocab": 32001, "pad": 63,
         "dtype": "f32", "scale": 1.25},
    ]


def _log_int(rng, lo, hi):
    return int(min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _extent(rng, lo, hi):
    """An extent in [lo, hi], log-uniform: a multiple of 64, a multiple of 8, or any."""
    v = _log_int(rng, lo, hi)
    step = rng.choice((64, 8, 1, 1))
    return min(hi, max(lo, v // step * step)) if v >= step else v


def draw(rng):
    op = rng.choice(("ln_fwd", "ln_bwd", "gemm", "gemm", "lp_fwd", "lp_fwd", "lp_bwd"))
    if op == "gemm":
        while True:
            # One product in two has few tokens.
            m = _log_int(rng, 1, 64) if rng.random() < 0.5 else _extent(rng, 64, 8192)
            n, k = _extent(rng, 64, 16384), _extent(rng, 64, 16384)
            if 2 * m * n * k <= MAX_FLOPS and max(m * n, n * k, m * k) <= MAX_ELEMENTS:
                break
        ab = rng.choice(("bf16", "f16"))
        return {"op": op, "m": m, "n": n, "k": k, "ab": ab, "y": rng.choice((ab, ab, "f32")),
                "act": rng.choice(ACTS), "bias": rng.choice((ab, "f32")),
                "residual": rng.random() < 0.5}
    dtype = rng.choice(("bf16", "f16", "f32"))
    if op in ("ln_fwd", "ln_bwd"):
        cols = _extent(rng, 64, 32768)
        return {"op": op, "rows": _log_int(rng, 1, min(65536, MAX_ELEMENTS // cols)), "cols": cols,
                "dtype": dtype, "param": rng.choice((dtype, "f32"))}
    vocab = _extent(rng, 1000, 262144)
    rows = _log_int(rng, 1, min(4096, MAX_ELEMENTS // vocab))
    case = {"op": op, "rows": rows, "vocab": vocab, "pad": rng.choice((0, -vocab % 64)),
            "dtype": dtype, "scale": rng.choice((1.0, 1.25, 0.5))}
    if op == "lp_fwd":
        case["top"] = rng.choice((0, 1, 5, 20, 32))
    return case


# ---------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------
def _normal(g, shape, sigma, mean=0.0):
    return torch.empty(shape, device="cuda", dtype=torch.float32).normal_(mean, sigma, generator=g)


def _inputs(case, seed):
    """The case's input tensors, from the seed alone."""
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    op = case["op"]
    if op in ("ln_fwd", "ln_bwd"):
        rows, cols, t, p = case["rows"], case["cols"], _TORCH[case["dtype"]], _TORCH[case["param"]]
        # Activations of a residual stream: rows of different size, a mean that is not zero.
        x = (_normal(g, (rows, cols), 1.0, 0.2) * (0.5 + _normal(g, (rows, 1), 1.0).abs())).to(t)
        s = {"x": x, "weight": _normal(g, (cols,), 0.1, 1.0).to(p),
             "bias": _normal(g, (cols,), 0.1).to(p)}
        if op == "ln_bwd":
            d = x.double()
            mean = d.mean(dim=1)
            rstd = torch.rsqrt(((d - mean[:, None]) ** 2).mean(dim=1) + EPS)
            s["mean"], s["rstd"] = mean.float(), rstd.float()
            s["dy"] = _normal(g, (rows, cols), 0.05).to(t)
        return s
    if op == "gemm":
        m, n, k, t = case["m"], case["n"], case["k"], _TORCH[case["ab"]]
        s = {"a": _normal(g, (m, k), 1.0).to(t), "b": _normal(g, (k, n), 1.0 / math.sqrt(k)).to(t),
             "bias": _normal(g, (n,), 0.1).to(_TORCH[case["bias"]]), "residual": None}
        if case["residual"]:
            s["residual"] = _normal(g, (m, n), 1.0).to(_TORCH[case["y"]])
        return s
    rows, vocab = case["rows"], case["vocab"]
    # Logits N(0, 2.5^2) with a few likely tokens in each row, and one column in a hundred
    # ruled out; the given tokens are a likely one or any that is not ruled out.
    x = _normal(g, (rows, vocab + case["pad"]), 2.5)
    allowed = torch.randperm(vocab, device="cuda", generator=g)[vocab // 100:]
    likely = allowed[torch.randint(len(allowed), (rows, 8), device="cuda", generator=g)]
    x.scatter_add_(1, likely, 4.0 + _normal(g, (rows, 8), 2.0).abs())
    ruled_out = torch.ones(vocab + case["pad"], device="cuda", dtype=torch.bool)
    ruled_out[allowed] = False
    x.masked_fill_(ruled_out, -math.inf)
    other = allowed[torch.randint(len(allowed), (rows,), device="cuda", generator=g)]
    tokens = torch.where(torch.rand(rows, device="cuda", generator=g) < 0.8, likely[:, 0], other)
    # One row in sixteen is padding behind a sequence: it has no token.
    tokens[torch.rand(rows, device="cuda", generator=g) < 1 / 16] = -100
    s = {"logits": x.to(_TORCH[case["dtype"]]), "tokens": tokens}
    if op == "lp_bwd":
        lse, entropy = _statistics64(s["logits"][:, :vocab], case["scale"], tokens)
        s["lse"], s["entropy"] = lse.float(), entropy.float()
        s["dlogprobs"] = _normal(g, (rows,), 1.0)
        s["dentropy"] = _normal(g, (rows,), 0.1)
    return s


def _statistics64(logits, scale, tokens):
    """Each row's log of the sum of exponentials and entropy, in 64 bits; 0 without a token."""
    z = logits.double() * scale
    m = z.amax(dim=1, keepdim=True)
    e = torch.exp(z - m)
    d = e.sum(dim=1)
    lse = m[:, 0] + torch.log(d)
    entropy = torch.log(d) - (e * torch.where(e > 0, z - m, 0.0)).sum(dim=1) / d
    return torch.where(tokens < 0, 0.0, lse), torch.where(tokens < 0, 0.0, entropy)


def prepare(case, seed):
    s = {"case": case}
    s.update(_inputs(case, seed))
    op = case["op"]

    def buffer(shape, dtype):
        return torch.empty(shape, device="cuda", dtype=dtype)

    if op == "ln_fwd":
        s["out"] = (torch.empty_like(s["x"]), buffer(case["rows"], torch.float32),
                    buffer(case["rows"], torch.float32))
    elif op == "ln_bwd":
        s["out"] = (torch.empty_like(s["x"]), torch.empty_like(s["weight"]),
                    torch.empty_like(s["bias"]))
    elif op == "gemm":
        s["out"] = buffer((case["m"], case["n"]), _TORCH[case["y"]])
    elif op == "lp_fwd":
        s["out"] = tuple(buffer(case["rows"], torch.float32) for _ in range(3))
        if case["top"]:
            s["out"] += (buffer((case["rows"], case["top"]), torch.float32),
                         buffer((case["rows"], case["top"]), torch.int64))
    else:
        s["out"] = torch.empty_like(s["logits"])
    if own:
        _plan(s)
    return s


def _plan(s):
    """What a program keeps beside its tensors: the types' names, the tile, the workspace."""
    from __graft_entry__ import load_package
    mcke = load_package()
    mcke.lib()
    case, op = s["case"], s["case"]["op"]
    kinds = {"f32": mcke.DType.kF32, "f16": mcke.DType.kF16, "bf16": mcke.DType.kBF16}
    s["mcke"] = mcke
    s["types"] = [kinds[case[t]] for t in ("dtype", "param", "ab", "y", "bias") if t in case]
    s["ws"], s["ws_bytes"] = None, 0
    if op == "gemm":
        s["tile"] = mcke.gemm_lp_default_tile(case["m"], case["n"], case["k"])
        s["act"] = mcke.Activation(ACTS.index(case["act"]))
    elif op == "ln_bwd":
        s["ws_bytes"] = mcke.layer_norm_backward_workspace_bytes(case["rows"], case["cols"])
    elif op == "lp_fwd":
        s["ws_bytes"] = mcke.token_logprobs_workspace_bytes(case["rows"], case["vocab"],
                                                            case["top"])
    if s["ws_bytes"]:
        s["ws"] = torch.empty(s["ws_bytes"], device="cuda", dtype=torch.uint8)


# ---------------------------------------------------------------------------
# One pass
# ---------------------------------------------------------------------------
def run(s):
    if own:
        return _run_own(s)
    return _PLAIN[s["case"]["op"]](s)


def _run_own(s):
    case, mcke, out = s["case"], s["mcke"], s["out"]
    op = case["op"]
    if op == "ln_fwd":
        st = mcke.launch_layer_norm(s["x"], s["weight"], s["bias"], *out, *s["types"],
                                    case["rows"], case["cols"], EPS)
    elif op == "ln_bwd":
        st = mcke.launch_layer_norm_backward(s["dy"], s["x"], s["weight"], s["mean"], s["rstd"],
                                             *out, *s["types"], case["rows"], case["cols"],
                                             s["ws"], s["ws_bytes"])
    elif op == "gemm":
        st = mcke.launch_gemm_lp_bias_act(s["a"], s["b"], s["bias"], s["residual"], out,
                                          *s["types"], case["m"], case["n"], case["k"], 1.0,
                                          s["act"], s["tile"])
    elif op == "lp_fwd":
        top = out[3:] if case["top"] else (None, None)
        st = mcke.launch_token_logprobs(s["logits"], s["tokens"], *out[:3], *top, *s["types"],
                                        case["rows"], case["vocab"], case["vocab"] + case["pad"],
                                        case["scale"], case["top"], s["ws"], s["ws_bytes"])
    else:
        st = mcke.launch_token_logprobs_backward(
            s["logits"], s["tokens"], s["lse"], s["entropy"], s["dlogprobs"], s["dentropy"], out,
            *s["types"], case["rows"], case["vocab"], case["vocab"] + case["pad"], case["scale"])
        out = out[:, :case["vocab"]]
    st.throw_if_error()
    return out


def _plain_ln_fwd(s):
    x = s["x"].float()
    mean = x.mean(dim=1, keepdim=True)
    c = x - mean
    rstd = torch.rsqrt((c * c).mean(dim=1, keepdim=True) + EPS)
    y = c * rstd * s["weight"].float() + s["bias"].float()
    return y.to(s["x"].dtype), mean[:, 0], rstd[:, 0]


def _plain_ln_bwd(s):
    dy, rstd = s["dy"].float(), s["rstd"][:, None]
    xhat = (s["x"].float() - s["mean"][:, None]) * rstd
    g = dy * s["weight"].float()
    dx = (g - g.mean(dim=1, keepdim=True) - xhat * (g * xhat).mean(dim=1, keepdim=True)) * rstd
    p = s["weight"].dtype
    return dx.to(s["x"].dtype), (dy * xhat).sum(dim=0).to(p), dy.sum(dim=0).to(p)


def _act(v, act):
    if act == "relu":
        return torch.clamp(v, min=0.0)
    if act == "gelu_erf":
        return 0.5 * v * (1.0 + torch.erf(v * math.sqrt(0.5)))
    if act == "gelu_tanh":
        return 0.5 * v * (1.0 + torch.tanh(math.sqrt(2.0 / math.pi) * (v + 0.044715 * v * v * v)))
    return v


def _plain_gemm(s):
    y = _act(s["a"].float() @ s["b"].float() + s["bias"].float(), s["case"]["act"])
    if s["residual"] is not None:
        y = y + s["residual"].float()
    return y.to(s["out"].dtype)


def _plain_lp_fwd(s):
    case, tokens = s["case"], s["tokens"]
    none = tokens < 0
    x = s["logits"][:, :case["vocab"]].float()
    z = x * case["scale"]
    m = z.amax(dim=1, keepdim=True)
    e = torch.exp(z - m)
    d = e.sum(dim=1, keepdim=True)
    lse = m + torch.log(d)
    lp = z - lse
    entropy = -(e / d * torch.where(e > 0, lp, 0.0)).sum(dim=1)
    given = lp.gather(1, tokens.clamp(min=0)[:, None])[:, 0]
    out = tuple(torch.where(none, 0.0, v) for v in (given, entropy, lse[:, 0]))
    if not case["top"]:
        return out
    # The largest by (value, then lowest index), as one whole number each: the value's bits,
    # in an order that whole numbers have too, above the index counted down.
    bits = (x + 0.0).view(torch.int32)
    order = torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits).long()
    down = 0xFFFFFFFF - torch.arange(case["vocab"], device=x.device)
    key = (order << 32) + down
    ids = 0xFFFFFFFF - (key.topk(case["top"], dim=1).values & 0xFFFFFFFF)
    top = torch.where(none[:, None], 0.0, lp.gather(1, ids))
    return out + (top, torch.where(none[:, None], -1, ids))


def _plain_lp_bwd(s):
    case, tokens = s["case"], s["tokens"]
    lp = s["logits"][:, :case["vocab"]].float() * case["scale"] - s["lse"][:, None]
    p = torch.exp(lp)
    h = torch.where(p > 0, lp + s["entropy"][:, None], 0.0)
    d = -p * (s["dlogprobs"][:, None] + s["dentropy"][:, None] * h)
    d.scatter_add_(1, tokens.clamp(min=0)[:, None], s["dlogprobs"][:, None])
    return torch.where(tokens[:, None] < 0, 0.0, d * case["scale"]).to(s["logits"].dtype)


_PLAIN = {"ln_fwd": _plain_ln_fwd, "ln_bwd": _plain_ln_bwd, "gemm": _plain_gemm,
          "lp_fwd": _plain_lp_fwd, "lp_bwd": _plain_lp_bwd}


# ---------------------------------------------------------------------------
# What a pass cannot do without, and its results in 64 bits
# ---------------------------------------------------------------------------
def work(case):
    op = case["op"]
    if op == "gemm":
        m, n, k = case["m"], case["n"], case["k"]
        y = m * n * _SIZE[case["y"]] * (2 if case["residual"] else 1)
        return {"bytes": _SIZE[case["ab"]] * (m * k + k * n) + y + n * _SIZE[case["bias"]],
                "flops": 2 * m * n * k}
    t = _SIZE[case["dtype"]]
    if op in ("ln_fwd", "ln_bwd"):
        rows, cols, p = case["rows"], case["cols"], _SIZE[case["param"]]
        passes, vectors = (2, 2) if op == "ln_fwd" else (3, 3)
        return {"bytes": passes * t * rows * cols + vectors * p * cols + 8 * rows,
                "flops": (8 if op == "ln_fwd" else 14) * rows * cols}
    rows, vocab = case["rows"], case["vocab"]
    if op == "lp_fwd":
        return {"bytes": t * rows * vocab + rows * (20 + 12 * case["top"]),
                "flops": 5 * rows * vocab}
    return {"bytes": 2 * t * rows * vocab + 24 * rows, "flops": 7 * rows * vocab}


def exact(case, seed):
    s = _inputs(case, seed)
    op = case["op"]
    if op == "ln_fwd":
        x = s["x"].double()
        var, mean = torch.var_mean(x, dim=1, correction=0)
        rstd = 1.0 / torch.sqrt(var + EPS)
        y = (x - mean[:, None]) * (rstd[:, None] * s["weight"].double()) + s["bias"].double()
        return y, mean, rstd
    if op == "ln_bwd":
        # The gradients as the transposed Jacobian gives them: with xhat the normalised row,
        # dx = rstd (g - proj(g)), proj the part of g along the ones vector and along xhat.
        x, dy, rstd = s["x"].double(), s["dy"].double(), s["rstd"].double()
        xhat = rstd[:, None] * x - (rstd * s["mean"].double())[:, None]
        g = dy * s["weight"].double()[None, :]
        along = (torch.sum(g * xhat, 1, True) * xhat + torch.sum(g, 1, True)) / case["cols"]
        ones = torch.ones(case["rows"], device="cuda", dtype=torch.float64)
        return rstd[:, None] * (g - along), ones @ (dy * xhat), ones @ dy
    if op == "gemm":
        v = torch.addmm(s["bias"].double(), s["a"].double(), s["b"].double())
        if case["act"] == "relu":
            v = torch.where(v > 0, v, 0.0)
        elif case["act"] == "gelu_erf":
            v = 0.5 * v * torch.special.erfc(-v / math.sqrt(2.0))
        elif case["act"] == "gelu_tanh":
            v = v / (1.0 + torch.exp(-math.sqrt(8.0 / math.pi) * (v + 0.044715 * v ** 3)))
        return v if s["residual"] is None else v + s["residual"].double()
    x, tokens = s["logits"][:, :case["vocab"]], s["tokens"]
    none, at = tokens < 0, tokens.clamp(min=0)[:, None]
    if op == "lp_fwd":
        lse, entropy = _statistics64(x, case["scale"], tokens)
        given = x.gather(1, at)[:, 0].double() * case["scale"] - lse
        out = (torch.where(none, 0.0, given), entropy, lse)
        if not case["top"]:
            return out
        top = x.double().topk(case["top"], dim=1).values * case["scale"] - lse[:, None]
        return out + (torch.where(none[:, None], 0.0, top), None)
    # d logprob / d z = onehot - p, and d entropy / d z_j = -p_j (log p_j + entropy).
    lp = x.double() * case["scale"] - s["lse"].double()[:, None]
    p = lp.exp()
    onehot = torch.zeros_like(p).scatter_(1, at, 1.0)
    slope = torch.where(p > 0, p * (lp + s["entropy"].double()[:, None]), 0.0)
    d = s["dlogprobs"].double()[:, None] * (onehot - p) - s["dentropy"].double()[:, None] * slope
    return torch.where(none[:, None], 0.0, d * case["scale"])
