"""The ends of a language model in training, and what is kept between its passes.

Tokens become rows of the embedding table; bias and activation of the blocks keep what
their gradient needs in 8 bits; the last hidden states become a cross entropy over the
vocabulary without the logits being kept; and the gradients come back the same way, those
of the loss and of the embedding into one table where the weights are tied.  `listed()`
names twelve cases; `draw(rng)` gives more of the same ranges.

Operators and their ranges (odd sizes among the drawn ones):

  embed_fwd  rows of a table by token, scaled
  embed_bwd  the table's gradient: each token's rows of the output's gradient, added up
  act_fwd    y = act(x + bias), and x + bias as it is restored from 8 bits
  act_bwd    from those 8 bits: dx = dy act'(u), dbias, and y = act(u) once more
  lce_fwd    cross entropy of hidden states and a vocabulary's weights, one token to a batch
  lce_bwd    its gradients in the hidden states and in the weights
"""
from __future__ import annotations

import math

import torch

own = False

ACTS = ("none", "relu", "gelu_erf", "gelu_tanh")
BLOCK = 32                       # columns that share a power of two
MAX_ROWS_COLS = 1 << 26          # of an activation
MAX_TABLE = 1 << 29              # values of a table
MAX_PRODUCTS = 1 << 42           # rows * vocab * dim of a forward pass

_TORCH = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
_SIZE = {"f32": 4, "f16": 2, "bf16": 2}


def listed():
    return [
        # Decoding: the rows of eight sequences' single tokens, one short launch.
        {"name": "embed_fwd_decode", "op": "embed_fwd", "rows": 8, "vocab": 131072, "cols": 4096,
         "table": "bf16", "out": "bf16"},
        # A training batch.
        {"name": "embed_fwd_batch", "op": "embed_fwd", "rows": 16384, "vocab": 131072,
         "cols": 4096, "table": "bf16", "out": "bf16"},
        # The same batch's backward pass: a dense gradient of the whole table.
        {"name": "embed_bwd_batch", "op": "embed_bwd", "rows": 16384, "vocab": 131072,
         "cols": 4096, "table": "bf16", "out": "bf16"},
        # A small model in fp32 over a ragged batch, rows of odd width.
        {"name": "embed_bwd_odd", "op": "embed_bwd", "rows": 5003, "vocab": 32001, "cols": 1021,
         "table": "f32", "out": "f32"},
        # The wide layer of an MLP block 4096 -> 16384 -> 4096 over a batch.
        {"name": "act_fwd_batch", "op": "act_fwd", "rows": 4096, "cols": 16384, "dtype": "bf16",
         "bias": "bf16", "act": "gelu_tanh"},
        # A small model in fp32, odd rows whose last block is cut.
        {"name": "act_fwd_odd", "op": "act_fwd", "rows": 1531, "cols": 2053, "dtype": "f32",
         "bias": "f32", "act": "gelu_erf"},
        # The same MLP block's backward pass.
        {"name": "act_bwd_batch", "op": "act_bwd", "rows": 4096, "cols": 16384, "dtype": "bf16",
         "bias": "bf16", "act": "gelu_tanh"},
        # fp16 activations over a ragged batch.
        {"name": "act_bwd_odd", "op": "act_bwd", "rows": 5003, "cols": 1021, "dtype": "f16",
         "bias": "f32", "act": "gelu_erf"},
        # Scoring one token each of four sequences, bound by reading the weights.
        {"name": "lce_fwd_few", "op": "lce_fwd", "rows": 4, "vocab": 131072, "dim": 4096,
         "dtype": "bf16", "scale": 1.0},
        # The loss of a training batch.
        {"name": "lce_fwd_train", "op": "lce_fwd", "rows": 8192, "vocab": 131072, "dim": 4096,
         "dtype": "bf16", "scale": 1.0},
        # The gradients of half that batch.
        {"name": "lce_bwd_train", "op": "lce_bwd", "rows": 4096, "vocab": 131072, "dim": 4096,
         "dtype": "bf16", "scale": 1.0},
        # A small model in fp16 under loss scaling, odd vocabulary and rows, a temperature.
        {"name": "lce_bwd_odd", "op": "lce_bwd", "rows": 2047, "vocab": 32001, "dim": 1024,
         "dtype": "f16", "scale": 1.25},
    ]


def _log_int(rng, lo, hi):
    return int(min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _extent(rng, lo, hi):
    """An extent in [lo, hi], log-uniform: a multiple of 64, a multiple of 8, or any."""
    v = _log_int(rng, lo, hi)
    step = rng.choice((64, 8, 1, 1))
    return min(hi, max(lo, v // step * step)) if v >= step else v


def draw(rng):
    op = rng.choice(("embed_fwd", "embed_bwd", "act_fwd", "act_bwd", "lce_fwd", "lce_bwd"))
    if op in ("embed_fwd", "embed_bwd"):
        cols = _extent(rng, 64, 8192)
        vocab = _extent(rng, 1000, min(262144, MAX_TABLE // cols))
        table = rng.choice(("bf16", "f16", "f32"))
        return {"op": op, "rows": _log_int(rng, 1, min(65536, MAX_ROWS_COLS // cols)),
                "vocab": vocab, "cols": cols, "table": table, "out": rng.choice((table, "f32"))}
    if op in ("act_fwd", "act_bwd"):
        cols = _extent(rng, 64, 32768)
        dtype = rng.choice(("bf16", "f16", "f32"))
        return {"op": op, "rows": _log_int(rng, 1, min(65536, MAX_ROWS_COLS // cols)),
                "cols": cols, "dtype": dtype, "bias": rng.choice((dtype, "f32")),
                "act": rng.choice(ACTS)}
    dim = _extent(rng, 64, 8192)
    vocab = _extent(rng, 1000, min(262144, MAX_TABLE // dim))
    most = MAX_PRODUCTS // (vocab * dim) // (1 if op == "lce_fwd" else 2)
    # One in three has few tokens.
    rows = _log_int(rng, 1, 64) if rng.random() < 1 / 3 else _extent(rng, 64, min(8192, most))
    return {"op": op, "rows": rows, "vocab": vocab, "dim": dim,
            "dtype": rng.choice(("bf16", "f16")), "scale": rng.choice((1.0, 1.25, 0.5))}


# ---------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------
def _normal(g, shape, sigma, mean=0.0):
    return torch.empty(shape, device="cuda", dtype=torch.float32).normal_(mean, sigma, generator=g)


def _tokens(g, rows, vocab):
    """Tokens as text has them, a few of them often and most of them rarely (log-uniform
    ranks, spread over the vocabulary); one in sixteen is padding."""
    u = torch.rand(rows, device="cuda", generator=g, dtype=torch.float64)
    rank = (torch.exp(u * math.log(vocab)) - 1.0).long().clamp(0, vocab - 1)
    names = torch.randperm(vocab, device="cuda", generator=g)
    tokens = names[rank]
    tokens[torch.rand(rows, device="cuda", generator=g) < 1 / 16] = -100
    return tokens


def _exponent(amax):
    """The power of two of a block: the smallest 2^E, E >= -126, with amax <= 448 * 2^E."""
    m, e = torch.frexp(amax)
    return (e - 9 + (m > 0.875).int()).clamp(min=-126)


def _blocks(u):
    """Rows of u as blocks of 32 columns, zeros behind the last."""
    rows, cols = u.shape
    n = (cols + BLOCK - 1) // BLOCK
    if n * BLOCK != cols:
        u = torch.cat((u, u.new_zeros(rows, n * BLOCK - cols)), dim=1)
    return u.view(rows, n, BLOCK)


def _save8(u):
    """fp32 values in 8 bits: e4m3 codes and a biased exponent for each block."""
    rows, cols = u.shape
    b = _blocks(u)
    e = _exponent(b.abs().amax(dim=2))
    codes = torch.ldexp(b, -e[:, :, None]).to(torch.float8_e4m3fn)
    codes = codes.view(torch.uint8).reshape(rows, -1)[:, :cols].contiguous()
    return codes, (e + 127).to(torch.uint8)


def _restore8(codes, exponents):
    """The values that codes and exponents stand for, in fp32."""
    cols = codes.shape[1]
    v = codes.view(torch.float8_e4m3fn).float()
    e = exponents.int() - 127
    return torch.ldexp(v, e.repeat_interleave(BLOCK, dim=1)[:, :cols])


def _inputs(case, seed):
    """The case's input tensors, from the seed alone."""
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    op, rows = case["op"], case["rows"]
    if op in ("embed_fwd", "embed_bwd"):
        vocab, cols = case["vocab"], case["cols"]
        s = {"tokens": _tokens(g, rows, vocab), "scale": math.sqrt(cols)}
        if op == "embed_fwd":
            s["table"] = _normal(g, (vocab, cols), 1.0 / math.sqrt(cols)).to(_TORCH[case["table"]])
        else:
            s["dout"] = _normal(g, (rows, cols), 0.05).to(_TORCH[case["out"]])
        return s
    if op in ("act_fwd", "act_bwd"):
        cols, t = case["cols"], _TORCH[case["dtype"]]
        # Pre-activations: columns of different size, a few of them large.
        size = 0.5 + _normal(g, (1, cols), 0.7).abs()
        x = (_normal(g, (rows, cols), 1.0) * size).to(t)
        bias = _normal(g, (cols,), 0.1).to(_TORCH[case["bias"]])
        if op == "act_fwd":
            return {"x": x, "bias": bias}
        codes, exponents = _save8(x.float() + bias.float())
        return {"codes": codes, "exponents": exponents,
                "dy": _normal(g, (rows, cols), 0.05).to(t)}
    vocab, dim, t = case["vocab"], case["dim"], _TORCH[case["dtype"]]
    # Logits of size 2, the target's about 4 larger, as in a model that has learnt something;
    # one row in sixteen is padding behind a sequence.
    weight = _normal(g, (vocab, dim), 2.0 / math.sqrt(dim)).to(t)
    targets = _tokens(g, rows, vocab)
    hidden = (_normal(g, (rows, dim), 1.0) + weight[targets.clamp(min=0)].float()).to(t)
    s = {"hidden": hidden, "weight": weight, "targets": targets}
    if op == "lce_bwd":
        # The mean over the rows; fp16 gradients are scaled up as training in fp16 does.
        s["lse"] = _lse64(hidden, weight, case["scale"], targets).float()
        s["dloss"] = torch.full((rows,), (1.0 if case["dtype"] == "bf16" else 16384.0) / rows,
                                device="cuda")
    return s


def _lse64(hidden, weight, scale, targets):
    """Each row's log of the sum of exponentials, in 64 bits; 0 without a target."""
    w = weight.double().t()
    out = []
    for h in hidden.split(2048):
        z = (h.double() @ w).mul_(scale)
        m = z.amax(dim=1, keepdim=True)
        out.append(m[:, 0] + torch.log(z.sub_(m).exp_().sum(dim=1)))
    return torch.where(targets < 0, 0.0, torch.cat(out))


def prepare(case, seed):
    s = {"case": case}
    s.update(_inputs(case, seed))
    op, rows = case["op"], case["rows"]

    def buffer(shape, dtype):
        return torch.empty(shape, device="cuda", dtype=dtype)

    if op == "embed_fwd":
        s["out"] = buffer((rows, case["cols"]), _TORCH[case["out"]])
    elif op == "embed_bwd":
        s["out"] = buffer((case["vocab"], case["cols"]), _TORCH[case["table"]])
    elif op == "act_fwd":
        cols = case["cols"]
        s["codes"] = buffer((rows, cols), torch.uint8)
        s["exponents"] = buffer((rows, (cols + BLOCK - 1) // BLOCK), torch.uint8)
        s["out"] = (torch.empty_like(s["x"]), torch.empty_like(s["x"]))
    elif op == "act_bwd":
        s["out"] = (torch.empty_like(s["dy"]), torch.empty_like(s["dy"]),
                    buffer(case["cols"], _TORCH[case["bias"]]))
    elif op == "lce_fwd":
        s["out"] = (buffer(rows, torch.float32), buffer(rows, torch.float32))
    else:
        s["out"] = (torch.empty_like(s["hidden"]), torch.empty_like(s["weight"]))
    if own:
        _plan(s)
    return s


def _plan(s):
    """What a program keeps beside its tensors: the types' names and the workspace."""
    from __graft_entry__ import load_package
    mcke = load_package()
    mcke.lib()
    case, op, rows = s["case"], s["case"]["op"], s["case"]["rows"]
    kinds = {"f32": mcke.DType.kF32, "f16": mcke.DType.kF16, "bf16": mcke.DType.kBF16}
    s["mcke"] = mcke
    s["ws"], s["ws_bytes"] = None, 0
    if op in ("embed_fwd", "embed_bwd"):
        s["table_type"], s["out_type"] = kinds[case["table"]], kinds[case["out"]]
        if op == "embed_bwd":
            s["ws_bytes"] = mcke.embedding_backward_workspace_bytes(rows, case["vocab"],
                                                                    case["cols"])
    elif op in ("act_fwd", "act_bwd"):
        s["type"], s["bias_type"] = kinds[case["dtype"]], kinds[case["bias"]]
        s["act"] = mcke.Activation(ACTS.index(case["act"]))
        if op == "act_bwd":
            s["ws_bytes"] = mcke.bias_act_checkpoint8_backward_workspace_bytes(rows, case["cols"])
    else:
        s["type"] = kinds[case["dtype"]]
        f = (mcke.linear_cross_entropy_workspace_bytes if op == "lce_fwd"
             else mcke.linear_cross_entropy_backward_workspace_bytes)
        s["ws_bytes"] = f(rows, case["vocab"], case["dim"])
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
    op, rows = case["op"], case["rows"]
    if op == "embed_fwd":
        st = mcke.launch_embedding(s["tokens"], s["table"], out, s["table_type"], s["out_type"],
                                   rows, case["vocab"], case["cols"], s["scale"])
    elif op == "embed_bwd":
        st = mcke.launch_embedding_backward(s["tokens"], s["dout"], out, s["out_type"],
                                            s["table_type"], rows, case["vocab"], case["cols"],
                                            s["scale"], False, s["ws"], s["ws_bytes"])
    elif op == "act_fwd":
        # Saved, and restored as a backward pass would have it (identity, no gradient).
        y, u = out
        mcke.launch_bias_act_checkpoint8(s["x"], s["bias"], y, s["codes"], s["exponents"],
                                         s["type"], s["bias_type"], rows, case["cols"],
                                         s["act"]).throw_if_error()
        st = mcke.launch_bias_act_checkpoint8_backward(None, s["codes"], s["exponents"], None, u,
                                                       None, s["type"], s["bias_type"], rows,
                                                       case["cols"], mcke.Activation.kNone)
    elif op == "act_bwd":
        dx, y, dbias = out
        st = mcke.launch_bias_act_checkpoint8_backward(s["dy"], s["codes"], s["exponents"], dx, y,
                                                       dbias, s["type"], s["bias_type"], rows,
                                                       case["cols"], s["act"], s["ws"],
                                                       s["ws_bytes"])
    elif op == "lce_fwd":
        st = mcke.launch_linear_cross_entropy(s["hidden"], s["weight"], s["targets"], *out,
                                              s["type"], rows, case["vocab"], case["dim"],
                                              case["scale"], s["ws"], s["ws_bytes"])
    else:
        st = mcke.launch_linear_cross_entropy_backward(
            s["hidden"], s["weight"], s["targets"], s["lse"], s["dloss"], None, *out, s["type"],
            rows, case["vocab"], case["dim"], case["scale"], s["ws"], s["ws_bytes"])
    st.throw_if_error()
    return out


def _plain_embed_fwd(s):
    tokens = s["tokens"]
    rows = s["table"][tokens.clamp(min=0)].float() * s["scale"]
    return torch.where(tokens[:, None] < 0, 0.0, rows).to(s["out"].dtype)


def _plain_embed_bwd(s):
    tokens = s["tokens"]
    d = torch.where(tokens[:, None] < 0, 0.0, s["dout"].float())
    sums = torch.zeros(s["out"].shape, device=d.device)
    sums.index_add_(0, tokens.clamp(min=0), d)
    return sums.mul_(s["scale"]).to(s["out"].dtype)


def _act(v, act):
    if act == "relu":
        return torch.clamp(v, min=0.0)
    if act == "gelu_erf":
        return 0.5 * v * (1.0 + torch.erf(v * math.sqrt(0.5)))
    if act == "gelu_tanh":
        return 0.5 * v * (1.0 + torch.tanh(math.sqrt(2.0 / math.pi) * (v + 0.044715 * v * v * v)))
    return v


def _act_slope(v, act):
    if act == "relu":
        return (v > 0).to(v.dtype)
    if act == "gelu_erf":
        return (0.5 * (1.0 + torch.erf(v * math.sqrt(0.5)))
                + v * torch.exp(-0.5 * v * v) * (1.0 / math.sqrt(2.0 * math.pi)))
    if act == "gelu_tanh":
        c = math.sqrt(2.0 / math.pi)
        t = torch.tanh(c * (v + 0.044715 * v * v * v))
        return 0.5 * (1.0 + t) + 0.5 * v * (1.0 - t * t) * (c * (1.0 + 3 * 0.044715 * v * v))
    return torch.ones_like(v)


def _plain_act_fwd(s):
    u = s["x"].float() + s["bias"].float()
    t = s["x"].dtype
    return _act(u, s["case"]["act"]).to(t), _restore8(*_save8(u)).to(t)


def _plain_act_bwd(s):
    u, t = _restore8(s["codes"], s["exponents"]), s["dy"].dtype
    dx = s["dy"].float() * _act_slope(u, s["case"]["act"])
    return dx.to(t), _act(u, s["case"]["act"]).to(t), dx.sum(dim=0).to(s["out"][2].dtype)


def _plain_lce_fwd(s):
    targets = s["targets"]
    z = (s["hidden"].float() @ s["weight"].float().t()) * s["case"]["scale"]
    m = z.amax(dim=1, keepdim=True)
    lse = (m + torch.log(torch.exp(z - m).sum(dim=1, keepdim=True)))[:, 0]
    loss = lse - z.gather(1, targets.clamp(min=0)[:, None])[:, 0]
    return torch.where(targets < 0, 0.0, loss), torch.where(targets < 0, 0.0, lse)


def _plain_lce_bwd(s):
    targets, scale, t = s["targets"], s["case"]["scale"], s["hidden"].dtype
    h, w = s["hidden"].float(), s["weight"].float()
    p = torch.exp((h @ w.t()) * scale - s["lse"][:, None])
    d = torch.where(targets < 0, 0.0, s["dloss"] * scale)
    dz = p * d[:, None]
    dz.scatter_add_(1, targets.clamp(min=0)[:, None], -d[:, None])
    # (A row without a target has a lse of 0, and what exp makes of that.)
    dz = torch.where(targets[:, None] < 0, 0.0, dz)
    return (dz @ w).to(t), (dz.t() @ h).to(t)


_PLAIN = {"embed_fwd": _plain_embed_fwd, "embed_bwd": _plain_embed_bwd, "act_fwd": _plain_act_fwd,
          "act_bwd": _plain_act_bwd, "lce_fwd": _plain_lce_fwd, "lce_bwd": _plain_lce_bwd}


# ---------------------------------------------------------------------------
# What a pass cannot do without, and its results in 64 bits
# ---------------------------------------------------------------------------
def work(case):
    op, rows = case["op"], case["rows"]
    if op in ("embed_fwd", "embed_bwd"):
        n, vocab = rows * case["cols"], case["vocab"] * case["cols"]
        table, out = _SIZE[case["table"]], _SIZE[case["out"]]
        if op == "embed_fwd":
            # No more rows of the table than it has.
            return {"bytes": table * min(n, vocab) + out * n + 8 * rows, "flops": n}
        return {"bytes": out * n + table * vocab + 8 * rows, "flops": n + vocab}
    if op in ("act_fwd", "act_bwd"):
        cols, t = case["cols"], _SIZE[case["dtype"]]
        n, blocks = rows * cols, rows * ((cols + BLOCK - 1) // BLOCK)
        # Forward: x in, y out, the 8 bits out and in again, the restored values out.  Backward:
        # dy and the 8 bits in, dx and y out.
        saved = (n + blocks) * (2 if op == "act_fwd" else 1)
        return {"bytes": 3 * t * n + saved + _SIZE[case["bias"]] * cols,
                "flops": (20 if op == "act_fwd" else 30) * n}
    vocab, dim, t = case["vocab"], case["dim"], _SIZE[case["dtype"]]
    operands = t * dim * (rows + vocab)
    if op == "lce_fwd":
        return {"bytes": operands + 16 * rows, "flops": 2 * rows * vocab * dim + 4 * rows * vocab}
    # The logits once more, and a product for each gradient.
    return {"bytes": 2 * operands + 16 * rows, "flops": 6 * rows * vocab * dim + 4 * rows * vocab}


def _round_e4m3(v):
    """To four bits of significand, exponents from -6 on, ties to even; |v| <= 448."""
    _, e = torch.frexp(v)
    step = torch.exp2((e - 1).clamp(min=-6).double() - 3.0)
    return torch.round(v / step) * step


def exact(case, seed):
    s = _inputs(case, seed)
    op = case["op"]
    if op == "embed_fwd":
        out = s["table"].double().index_select(0, s["tokens"].clamp(min=0)) * s["scale"]
        return out.masked_fill_((s["tokens"] < 0)[:, None], 0.0)
    if op == "embed_bwd":
        keep = s["tokens"] >= 0
        out = torch.zeros(case["vocab"], case["cols"], device="cuda", dtype=torch.float64)
        out.index_put_((s["tokens"][keep],), s["dout"][keep].double(), accumulate=True)
        return out * s["scale"]
    if op in ("act_fwd", "act_bwd"):
        act = case["act"]
        if op == "act_fwd":
            v = s["x"].double() + s["bias"].double()
            # What is saved is the sum in fp32.
            u, cols = _blocks(v.float().double()), case["cols"]
            big = u.abs().amax(dim=2, keepdim=True)
            e = torch.ceil(torch.log2(big.clamp(min=2.0**-160) / 448.0)).clamp(min=-126)
            # (The logarithm may be off by one step next to a power of two.)
            e = torch.where(big > 448.0 * torch.exp2(e), e + 1, e)
            e = torch.where((big <= 448.0 * torch.exp2(e - 1)) & (e > -126), e - 1, e)
            u = (_round_e4m3(u * torch.exp2(-e)) * torch.exp2(e)).flatten(1)[:, :cols]
        else:
            code = s["codes"].int()
            m, x = (code & 7).double(), (code >> 3 & 15).double()
            v = torch.where(x > 0, (8.0 + m) * torch.exp2(x - 10.0), m * 2.0**-9)
            v = torch.where(code > 127, -v, v)
            scale = torch.exp2(s["exponents"].double() - 127.0)
            v = v * scale.repeat_interleave(BLOCK, dim=1)[:, :case["cols"]]
        if act == "relu":
            y, slope = torch.where(v > 0, v, 0.0), torch.where(v > 0, 1.0, 0.0).double()
        elif act == "gelu_erf":
            cdf = 0.5 * torch.special.erfc(-v / math.sqrt(2.0))
            y, slope = v * cdf, cdf + v * torch.exp(-v * v / 2.0) / math.sqrt(2.0 * math.pi)
        elif act == "gelu_tanh":
            b = math.sqrt(8.0 / math.pi)
            q = torch.sigmoid(b * (v + 0.044715 * v ** 3))
            y, slope = v * q, q + v * q * (1.0 - q) * b * (1.0 + 0.134145 * v ** 2)
        else:
            y, slope = v, torch.ones_like(v)
        if op == "act_fwd":
            return y, u
        dx = s["dy"].double() * slope
        return dx, y, torch.ones(case["rows"], device="cuda", dtype=torch.float64) @ dx
    hidden, weight, targets, scale = s["hidden"], s["weight"], s["targets"], case["scale"]
    none = targets < 0
    if op == "lce_fwd":
        lse = _lse64(hidden, weight, scale, targets)
        at = (hidden.double() * weight[targets.clamp(min=0)].double()).sum(dim=1) * scale
        return torch.where(none, 0.0, lse - at), lse
    # Rows with a target alone: those without have no gradient and give none.
    keep = (~none).nonzero()[:, 0]
    w = weight.double()
    dh = torch.zeros(case["rows"], case["dim"], device="cuda", dtype=torch.float64)
    dw = torch.zeros(case["vocab"], case["dim"], device="cuda", dtype=torch.float64)
    for rows in keep.split(1024):
        h = hidden[rows].double()
        dz = torch.exp(torch.mm(h, w.t()) * scale - s["lse"][rows].double()[:, None])
        dz[torch.arange(len(rows), device="cuda"), targets[rows]] -= 1.0
        dz *= (s["dloss"][rows].double() * scale)[:, None]
        dh[rows] = torch.mm(dz, w)
        dw.addmm_(dz.t(), h)
    return dh, dw
