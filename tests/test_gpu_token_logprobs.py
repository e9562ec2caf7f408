"""Token log probabilities, entropy, alternatives and their gradient (mcke_launch_token_logprobs,
..._backward) on the GPU against the formulas in 64 bits.

Tolerances are counts of fp32 roundings (U each).  With z = scale x, M = max z, delta = M - z,
S = sum p delta, and D the length of a chain of additions and joins (vocab / 256 values and their
rescalings in a lane of the narrowest kernel, then the tree: vocab / 256 + 32):
  a term 2^u of the sum d is off by (3 delta + 4) U of itself (difference, product, the
  constant, a hardware exponential of one ulp), a rescaling by as much of its shift, and all
  shifts of a term add up to at most delta: d is off by R = (6 S + 6 D) U of itself
  lse          R + 3 U (|lse| + |M|)
  z - lse      2 U |z - M| + R + 3 U |ln d| + U |z - lse|
  entropy      (6 sum p delta^2 + (6 D + 6) S) U + S R + R + 3 U |ln d|
The gradient takes lse and entropy as they are; with lp = z - lse, q = g + h (lp + H):
  p            (|z| + 4 |lp| + 6) U of itself
  dlogits      scale (p ((|z| + 4 |lp| + 6) U |q| + (2 |z| + 8) U (|g| + |h| (|H| + |lp| + 1))) +
               3 U |g| at the token), and the output's rounding
"""
from __future__ import annotations

import math

import numpy as np
import pytest
import torch

from tests.operator_util import (BF16, DTYPES, F16, F32, HALF, ID, TINY, TORCH, U, Captured, Dev,
                                 check, out, same_bits, workspace)

pytestmark = pytest.mark.gpu

INF = float("inf")
# One logit, less than a 16-byte vector, around vectors, waves and workgroups, rows that
# several workgroups share and rows that do not, odd widths.
SHAPES = [(1, 1), (1, 3), (2, 7), (3, 8), (5, 9), (2, 255), (1, 2048), (1, 2049), (3, 4100),
          (4, 50021), (1, 131072), (40, 20003), (300, 1000), (1030, 77), (1100, 2500), (9, 12345)]


def _logits(rows, vocab, dt, seed, sigma=2.5):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, vocab, generator=g, dtype=torch.float64) * sigma
    x[torch.arange(rows), torch.randint(vocab, (rows,), generator=g)] += 8
    tokens = torch.randint(vocab, (rows,), generator=g)
    return x.to(TORCH[dt]), tokens


def _best(x, k):
    """Ids of the k largest by value, ties to the lowest index; x has no NaN."""
    return torch.sort(x.double() + 0.0, dim=1, descending=True, stable=True).indices[:, :k]


def _reference(x, tokens, scale, k):
    """{name: (value, tolerance)} in 64 bits, for rows with a finite maximum."""
    z = x.double() * scale
    vocab = z.shape[1]
    M = z.amax(1, keepdim=True)
    delta = torch.where(z > -INF, M - z, 0.0)
    w = torch.exp(z - M)
    d = w.sum(1, keepdim=True)
    ln_d = torch.log(d)
    p, lse = w / d, M + ln_d
    S = (p * delta).sum(1, keepdim=True)
    D = vocab / 256 + 32
    R = (6 * S + 6 * D) * U

    def lp_of(ids):
        zi = z.gather(1, ids)
        lp = zi - M - ln_d                            # lse itself may swallow ln_d, in 64 bits too
        far = torch.where(zi > -INF, M - zi, 0.0)
        return lp, torch.where(lp > -INF, 2 * U * far + R + 3 * U * ln_d + U * lp.abs(), 0.0)

    r = {"lse": (lse[:, 0], (R + 3 * U * (lse.abs() + M.abs()))[:, 0])}
    entropy = ln_d + S
    te = ((6 * (p * delta**2).sum(1, keepdim=True) + (6 * D + 6) * S) * U + S * R + R +
          3 * U * ln_d)
    r["entropy"] = (entropy[:, 0], te[:, 0])
    if tokens is not None:
        lp, t = lp_of(tokens.clamp(0, vocab - 1)[:, None])
        r["logprobs"] = (lp[:, 0], t[:, 0])
    if k:
        r["top_ids"] = (_best(x, k), None)
        r["top_logprobs"] = lp_of(r["top_ids"][0])
    return r


NAMES = ("logprobs", "entropy", "lse", "top_logprobs", "top_ids")


def run(m, x, tokens, scale=1.0, k=0, pad=0, shift=0, dt=None, skip=(), stream=None):
    """One launch; the columns behind vocab hold NaN, which nobody may read."""
    rows, vocab = x.shape
    full = torch.full((rows, vocab + pad), float("nan"), dtype=x.dtype)
    full[:, :vocab] = x
    dl = Dev(m, full, shift)
    dtk = Dev(m, tokens) if tokens is not None else None
    outs = {n: out(m, (rows,), torch.float32) for n in NAMES[:3]}
    if tokens is None:
        outs["logprobs"] = None
    outs["top_logprobs"] = out(m, (rows, k), torch.float32) if k else None
    outs["top_ids"] = out(m, (rows, k), torch.int64) if k else None
    for n in skip:
        outs[n] = None
    nbytes = m.token_logprobs_workspace_bytes(rows, vocab, k)
    ws = workspace(m, nbytes)
    dt = {v: t for t, v in TORCH.items()}[x.dtype]
    m.launch_token_logprobs(dl, dtk, *(outs[n] for n in NAMES), dt, rows, vocab, vocab + pad,
                            scale, k, ws, nbytes, stream).throw_if_error()
    m.device_synchronize()
    if ws is not None:
        ws.get()
    return {n: o.get() for n, o in outs.items() if o is not None}


def compare(got, want):
    for n, (w, t) in want.items():
        if t is None:
            assert torch.equal(got[n], w), n
        else:
            check(n, got[n], w, t)


@pytest.mark.parametrize("dt", DTYPES, ids=ID.get)
@pytest.mark.parametrize("rows,vocab", SHAPES)
def test_forward(gpu, rows, vocab, dt):
    x, tokens = _logits(rows, vocab, dt, rows * 7 + vocab)
    k = min(vocab, (0, 1, 5, 20, 64)[(rows + vocab) % 5])
    scale = (1.0, 0.7, 1.25)[vocab % 3]
    got = run(gpu, x, tokens, scale, k, pad=(0, 5)[rows % 2], shift=rows % 3)
    compare(got, _reference(x, tokens, scale, k))


# Rows of one, two and four vectors a lane, whole up to 32768 logits, and shared by workgroups from
# there on where there are few of them.
@pytest.mark.parametrize("dt", DTYPES, ids=ID.get)
@pytest.mark.parametrize("rows,vocab", [(7, 1024), (5, 1025), (6, 2051), (5, 3000), (4, 4096),
                                        (3, 4097), (3, 32768), (40, 32769), (130, 65537),
                                        (127, 33003), (128, 40001), (260, 33003)])
def test_vectors_a_lane_and_parts(gpu, rows, vocab, dt):
    test_forward(gpu, rows, vocab, dt)


@pytest.mark.parametrize("rows,vocab,k,dt", [
    (r, v, k, dt) for r, v in ((1, 40000), (1, 70001), (16, 50003), (64, 60001))
    for k in (0, 20, 40) for dt in DTYPES] + [
        (65, 130003, 20, BF16), (65, 130003, 40, BF16), (130, 131077, 0, F16), (256, 131073, 0, F32),
        (257, 131073, 0, F32), (200, 66001, 1, F32), (200, 66001, 0, F32)])
def test_whole_and_shared_rows(gpu, rows, vocab, k, dt):
    """Rows that one workgroup takes, or several, by their bytes, their number and the
    alternatives, with a workspace for any type."""
    x, tokens = _logits(rows, vocab, dt, rows + vocab)
    compare(run(gpu, x, tokens, 1.0, k, pad=3, shift=1), _reference(x, tokens, 1.0, k))


@pytest.mark.parametrize("k", [1, 20, 64])
@pytest.mark.parametrize("rows,vocab", [(2, 2049), (3, 4095), (1, 32768), (33, 50003), (260, 2500)])
def test_top_k_of_more_rows(gpu, rows, vocab, k):
    test_top_k(gpu, rows, vocab, k)


@pytest.mark.parametrize("k", [1, 2, 20, 63, 64])
@pytest.mark.parametrize("rows,vocab", [(1, 64), (1, 70000), (33, 5000), (1025, 300)])
def test_top_k(gpu, rows, vocab, k):
    x, tokens = _logits(rows, vocab, BF16, k + vocab)
    compare(run(gpu, x, tokens, 1.0, k), _reference(x, tokens, 1.0, k))


def _patterned(kind, rows, vocab, dt):
    """Rows in orders and with ties that a search for the largest meets."""
    i = torch.arange(vocab, dtype=torch.float64).expand(rows, vocab).clone()
    g = torch.Generator().manual_seed(vocab)
    if kind == "constant":
        x = torch.full((rows, vocab), 1.5, dtype=torch.float64)
    elif kind == "ascending":
        x = i / vocab * 20
    elif kind == "descending":
        x = -i / vocab * 20
    elif kind == "few_values":
        x = torch.randint(4, (rows, vocab), generator=g).double()
    elif kind == "zeros":
        x = torch.where(torch.randint(2, (rows, vocab), generator=g) > 0, 0.0, -0.0).double()
    elif kind == "mostly_masked":
        x = torch.full((rows, vocab), -INF, dtype=torch.float64)
        at = torch.randint(vocab, (rows, 3), generator=g)
        x.scatter_(1, at, torch.randn(rows, 3, generator=g, dtype=torch.float64))
    else:
        assert kind == "one_hot"
        x = torch.full((rows, vocab), -80.0, dtype=torch.float64)
        x[:, vocab // 2] = 80.0
    return x.to(TORCH[dt])


KINDS = ["constant", "ascending", "descending", "few_values", "zeros", "mostly_masked", "one_hot"]


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("rows,vocab", [(1, 9), (2, 9000), (1, 33000), (1024, 1100)])
def test_ties_orders_and_masks(gpu, rows, vocab, kind):
    dt = (BF16, F32)[vocab % 2]
    x = _patterned(kind, rows, vocab, dt)
    tokens = torch.arange(rows) * 31 % vocab
    k = min(20, vocab)
    compare(run(gpu, x, tokens, 1.0, k), _reference(x, tokens, 1.0, k))


@pytest.mark.parametrize("rows,vocab", [(8, 100), (8, 30000), (1030, 600)])
def test_special_rows(gpu, rows, vocab):
    """Rows of nothing but masks, rows without a token, tokens that do not exist, NaN and +inf:
    each does what the header says, and the rows beside them are untouched by it."""
    x, tokens = _logits(rows, vocab, F32, 5)
    clean = run(gpu, x, tokens, 1.0, 4)
    x[1] = -INF
    tokens[2] = -1
    x[2] = float("nan")                              # not read
    tokens[3] = vocab
    x[4, vocab // 3] = float("nan")
    x[5, vocab - 1] = INF
    tokens[6] = -(1 << 40)
    x[7] = float("nan")
    got = run(gpu, x, tokens, 1.0, 4)
    assert got["logprobs"][1] == -INF and got["lse"][1] == -INF and got["entropy"][1] == 0
    assert (got["top_logprobs"][1] == -INF).all()
    assert got["top_ids"][1].tolist() == [0, 1, 2, 3]
    for r in (2, 6):
        assert all((got[n][r] == 0).all() for n in NAMES[:4]) and (got["top_ids"][r] == -1).all()
    assert got["logprobs"][3].isnan()
    for n in ("entropy", "lse", "top_logprobs", "top_ids"):
        assert same_bits(got[n][3], clean[n][3])
    for r in (4, 5, 7):
        assert all(got[n][r].isnan().all() for n in NAMES[:4])
    keep = x[4].clone()
    keep[vocab // 3] = -INF
    assert torch.equal(got["top_ids"][4], _best(keep[None], 4)[0])
    assert got["top_ids"][5][0] == vocab - 1 and (got["top_ids"][7] == -1).all()
    for r in (0, *range(8, rows)):
        assert all(same_bits(got[n][r], clean[n][r]) for n in NAMES)


@pytest.mark.parametrize("rows,vocab", [(3, 50), (2, 40000), (1050, 500)])
def test_optional_outputs(gpu, rows, vocab):
    """What is not asked for is not written and changes no bit of what is."""
    x, tokens = _logits(rows, vocab, F16, 77)
    full = run(gpu, x, tokens, 1.0, 7)
    for skip in (("entropy",), ("logprobs", "lse"), ("top_ids",), ("top_logprobs",),
                 ("logprobs", "entropy", "lse"), ("lse", "entropy", "top_ids")):
        got = run(gpu, x, tokens, 1.0, 7, skip=skip)
        assert all(same_bits(got[n], full[n]) for n in got)
    got = run(gpu, x, None, 1.0, 7)
    assert all(same_bits(got[n], full[n]) for n in got) and "logprobs" not in got
    got = run(gpu, x, tokens, 1.0, 0)
    compare(got, _reference(x, tokens, 1.0, 0))


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("rows,vocab", [(2, 2600), (2, 4800), (3, 40000)])
def test_ties_orders_and_masks_of_more_rows(gpu, rows, vocab, kind):
    test_ties_orders_and_masks(gpu, rows, vocab, kind)


@pytest.mark.parametrize("rows,vocab", [(8, 40000), (9, 2500), (9, 3600)])
def test_special_rows_of_more_widths(gpu, rows, vocab):
    test_special_rows(gpu, rows, vocab)


@pytest.mark.parametrize("shift,pad", [(1, 0), (3, 1), (0, 7)])
def test_any_alignment(gpu, shift, pad):
    """Row starts off 16 bytes: the same bits."""
    for dt in DTYPES:
        x, tokens = _logits(5, 10007, dt, 6)
        a, b = run(gpu, x, tokens, 1.0, 9), run(gpu, x, tokens, 1.0, 9, pad=pad, shift=shift)
        assert all(same_bits(a[n], b[n]) for n in NAMES)


@pytest.mark.parametrize("dt", [BF16, F16], ids=ID.get)
@pytest.mark.parametrize("rows,vocab,pad", [(4, 8193, 0), (5, 16384, 1), (5, 16385, 0), (4, 16391, 2),
                                            (3, 24577, 4), (3, 60001, 0), (40, 40003, 0),
                                            (130, 66001, 0), (7, 2049, 0), (7, 4097, 0)])
def test_rows_at_odd_addresses(gpu, rows, vocab, pad, dt):
    """Every other row starts off a 4-byte address (all of them, or all but those, with the buffer
    moved by an element): the bits of rows that start at 16 bytes, for one round of vectors and
    several, whole rows and shared ones, rounds that end with the row and an element before."""
    x, tokens = _logits(rows, vocab, dt, vocab)
    x[-1, -1] = x[-1].max() + 1                      # the last logit there is
    x[1, 0] = x[1].max() + 1
    tokens[-1], tokens[1] = vocab - 1, 0
    for k in (0, 20, 40):
        want = run(gpu, x, tokens, 1.0, k, pad=-vocab % 8)
        for shift in (0, 1):
            got = run(gpu, x, tokens, 1.0, k, pad=pad, shift=shift)
            assert all(same_bits(got[n], want[n]) for n in got), (k, shift)


@pytest.mark.parametrize("dt", [BF16, F16], ids=ID.get)
@pytest.mark.parametrize("vocab", [2048, 2049, 4101, 16385, 60001])
def test_first_logits_of_rows_at_odd_addresses(gpu, vocab, dt):
    """A row's first logit, its largest and its token, at odd addresses with NaN before it: the
    bits of aligned rows, the first row's too."""
    x, tokens = _logits(4, vocab, dt, 15)
    x[:, 0] = x.amax(1) + 1
    tokens[:] = 0
    want = run(gpu, x, tokens, 1.0, 20)
    for pad, shift in ((1, 1), (-vocab % 8, 1), (-vocab % 2 + 1, 0)):
        got = run(gpu, x, tokens, 1.0, 20, pad=pad, shift=shift)
        assert all(same_bits(got[n], want[n]) for n in got), (pad, shift)


@pytest.mark.parametrize("rows,vocab,k", [(3, 60001, 40), (1, 131072, 64), (2, 50000, 64),
                                          (40, 70000, 20), (3, 20000, 64)])
def test_same_bits_on_every_run(gpu, rows, vocab, k):
    """Which lane writes an alternative depends on the order of the keys, its value does not."""
    x, tokens = _logits(rows, vocab, BF16, 8)
    first = run(gpu, x, tokens, 1.0, k)
    for _ in range(6):
        again = run(gpu, x, tokens, 1.0, k)
        assert all(same_bits(again[n], first[n]) for n in NAMES)


def test_large_logits(gpu):
    """Logits of 1e4 and more, whose exponentials' arguments must not be rounded at the logits'
    size; from 1e9 on any two that differ are far apart."""
    for mag in (1e4, 1e6, -1e6, 1e9, 1e12, -1e12, 1e30, -3e38):
        x, tokens = _logits(3, 5000, F32, 8)
        x = x + mag
        compare(run(gpu, x, tokens, 1.0, 5), _reference(x, tokens, 1.0, 5))


# ---------------------------------------------------------------------------
# The gradient
# ---------------------------------------------------------------------------
def run_backward(m, x, tokens, lse, entropy, g, h, scale=1.0, pad=0, shift=0):
    rows, vocab = x.shape
    full = torch.full((rows, vocab + pad), float("nan"), dtype=x.dtype)
    full[:, :vocab] = x
    dt = {v: t for t, v in TORCH.items()}[x.dtype]
    ins = [Dev(m, t) if t is not None else None for t in (tokens, lse, entropy, g, h)]
    dx = out(m, (rows, vocab + pad), x.dtype, shift)
    before = dx.get()
    m.launch_token_logprobs_backward(Dev(m, full, shift), *ins, dx, dt, rows, vocab, vocab + pad,
                                     scale).throw_if_error()
    m.device_synchronize()
    got = dx.get()
    assert same_bits(got[:, vocab:], before[:, vocab:]), "columns behind vocab"
    return got[:, :vocab]


def _gradient(x, tokens, lse, entropy, g, h, scale, dt):
    z = x.double() * scale
    lse = lse.double()[:, None]
    H = entropy.double()[:, None] if entropy is not None else torch.zeros_like(lse)
    g = g.double()[:, None] if g is not None else torch.zeros_like(lse)
    h = h.double()[:, None] if h is not None else torch.zeros_like(lse)
    lp = z - lse
    p = torch.exp(lp)
    lp, az = torch.where(p > 0, lp, 0.0), torch.where(p > 0, z.abs(), 0.0)
    q = torch.where(p > 0, g + h * (lp + H), 0.0)
    d = -p * q
    t = p * ((az + 4 * lp.abs() + 6) * U * q.abs() +
             (2 * az + 8) * U * (g.abs() + h.abs() * (H.abs() + lp.abs() + 1)))
    if tokens is not None:
        hot = torch.zeros_like(d).scatter_(1, tokens.clamp(min=0)[:, None], 1.0)
        d, t = d + hot * g, t + 3 * U * hot * g.abs()
    d, t = d * scale, t * scale
    return d, t + HALF[dt] * (d.abs() + t) + TINY[dt]


@pytest.mark.parametrize("dt", DTYPES, ids=ID.get)
@pytest.mark.parametrize("rows,vocab", SHAPES)
def test_backward(gpu, rows, vocab, dt):
    x, tokens = _logits(rows, vocab, dt, rows + vocab)
    if vocab > 4:
        x[:, 1] = -INF                                # a masked column
        tokens[tokens == 1] = 0
    scale = (1.0, 0.7, 1.25)[vocab % 3]
    r = _reference(x, tokens, scale, 0)
    lse, entropy = r["lse"][0].float(), r["entropy"][0].float()
    gen = torch.Generator().manual_seed(1)
    g, h = torch.randn(rows, generator=gen), torch.randn(rows, generator=gen) * 0.3
    for gg, hh in ((g, h), (g, None), (None, h)):
        got = run_backward(gpu, x, tokens, lse, entropy if hh is not None else None, gg, hh, scale,
                           pad=rows % 3, shift=vocab % 2)
        check("dlogits", got, *_gradient(x, tokens, lse, entropy, gg, hh, scale, dt))


@pytest.mark.parametrize("vocab", [40, 9001])
def test_backward_special_rows(gpu, vocab):
    x, tokens = _logits(6, vocab, F32, 12)
    r = _reference(x, tokens, 1.0, 0)
    lse, entropy = r["lse"][0].float(), r["entropy"][0].float()
    g, h = torch.ones(6), torch.ones(6)
    clean = run_backward(gpu, x, tokens, lse, entropy, g, h)
    x[1], lse[1], entropy[1] = -INF, -INF, 0.0        # every logit masked
    tokens[2], x[2], lse[2] = -100, float("nan"), 0.0
    tokens[3] = vocab
    x[4, 3], lse[4], entropy[4] = float("nan"), float("nan"), float("nan")
    got = run_backward(gpu, x, tokens, lse, entropy, g, h)
    assert (got[1] == 0).all() and (got[2] == 0).all()
    assert got[3].isnan().all() and got[4].isnan().all()
    assert same_bits(got[0], clean[0]) and same_bits(got[5], clean[5])
    # Without tokens every row has its entropy's gradient.
    x, tokens = _logits(4, vocab, F32, 13)
    r = _reference(x, None, 1.0, 0)
    lse, entropy = r["lse"][0].float(), r["entropy"][0].float()
    got = run_backward(gpu, x, None, lse, entropy, None, torch.ones(4))
    check("dlogits", got, *_gradient(x, None, lse, entropy, None, torch.ones(4), 1.0, F32))


def test_gradient_against_differences(gpu):
    """dlogits of sum(g logprob + h entropy) against central differences of the 64-bit formula:
    with steps of 1e-4 their own error is below 1e-7 of the largest gradient; lse and entropy
    as the forward pass rounded them add 64 U of it."""
    rows, vocab, scale = 3, 29, 1.25
    x, tokens = _logits(rows, vocab, F32, 4, sigma=1.0)
    g, h = torch.tensor([1.0, -0.5, 0.3]), torch.tensor([0.2, 0.7, -1.0])

    def loss(z):
        lp = torch.log_softmax(z * scale, 1)
        ent = -(lp.exp() * lp).sum(1)
        return float((g.double() * lp.gather(1, tokens[:, None])[:, 0] + h.double() * ent).sum())

    f = run(gpu, x, tokens, scale)
    got = run_backward(gpu, x, tokens, f["lse"], f["entropy"], g, h, scale)
    _, tol = _gradient(x, tokens, f["lse"], f["entropy"], g, h, scale, F32)
    want = torch.zeros(rows, vocab, dtype=torch.float64)
    for i in np.ndindex(rows, vocab):
        hi, lo = x.double(), x.double()
        hi[i] += 1e-4
        lo[i] -= 1e-4
        want[i] = (loss(hi) - loss(lo)) / 2e-4
    check("dlogits", got, want, tol + (64 * U + 1e-7) * want.abs().max())


@pytest.mark.parametrize("vocab", [20011, 50021])
def test_captured(gpu, vocab):
    """Forward (whole rows, and parts with their join) and backward, captured: every replay gives
    the eager bits, with eager work between them and outputs and workspace overwritten."""
    m = gpu
    rows, k = 3, 10
    x, tokens = _logits(rows, vocab, BF16, 31)
    eager = run(m, x, tokens, 1.0, k)
    g, h = torch.ones(rows), torch.full((rows,), 0.5)
    egrad = run_backward(m, x, tokens, eager["lse"], eager["entropy"], g, h)
    dx, dt, dg, dh = (Dev(m, t) for t in (x, tokens, g, h))
    outs = {n: out(m, eager[n].shape, eager[n].dtype) for n in NAMES}
    grad = out(m, x.shape, x.dtype)
    nbytes = m.token_logprobs_workspace_bytes(rows, vocab, k)
    assert (nbytes > 0) == (vocab == 50021)
    ws = workspace(m, nbytes)

    def launch(stream):
        m.launch_token_logprobs(dx, dt, *(outs[n] for n in NAMES), BF16, rows, vocab, vocab, 1.0,
                                k, ws, nbytes, stream).throw_if_error()
        m.launch_token_logprobs_backward(dx, dt, outs["lse"], outs["entropy"], dg, dh, grad, BF16,
                                         rows, vocab, vocab, 1.0, stream).throw_if_error()

    graph = Captured(m, launch)
    try:
        for i in range(4):
            graph.replay()
            assert all(same_bits(outs[n].get(), eager[n]) for n in NAMES), i
            assert same_bits(grad.get(), egrad), i
            for o in (*outs.values(), grad, *([ws] if ws else [])):
                o.buf.upload(np.full(o.buf.nbytes, 0xA5, np.uint8))
            again = run(m, x, tokens, 1.0, k)
            assert all(same_bits(again[n], eager[n]) for n in NAMES)
    finally:
        graph.close()


def test_two_streams_at_once(gpu):
    """Two launches with a workspace each on two streams do not meet."""
    m = gpu
    jobs = []
    for s in range(2):
        x, tokens = _logits(2, 60000 + s, BF16, 90 + s)
        want = run(m, x, tokens, 1.0, 12)
        nbytes = m.token_logprobs_workspace_bytes(2, 60000 + s, 12)
        outs = {n: out(m, want[n].shape, want[n].dtype) for n in NAMES}
        jobs.append((want, outs, Dev(m, x), Dev(m, tokens), workspace(m, nbytes), nbytes,
                     60000 + s, m.Stream()))
    for _ in range(5):
        for want, outs, dx, dt, ws, nbytes, vocab, st in jobs:
            m.launch_token_logprobs(dx, dt, *(outs[n] for n in NAMES), BF16, 2, vocab, vocab, 1.0,
                                    12, ws, nbytes, st).throw_if_error()
    m.device_synchronize()
    for want, outs, *_, st in jobs:
        assert all(same_bits(outs[n].get(), want[n]) for n in NAMES)
        st.close()


def test_offsets_past_32_bits(gpu):
    """A second row more than 2^31 logits behind the first."""
    m = gpu
    vocab, stride = 5000, (1 << 31) + 8
    x, tokens = _logits(2, vocab, BF16, 14)
    want = run(m, x, tokens, 1.0, 5)
    g, h = torch.ones(2), torch.ones(2)
    wgrad = run_backward(m, x, tokens, want["lse"], want["entropy"], g, h)
    bufs = [m.DeviceBuffer(2 * (stride + vocab)) for _ in range(2)]
    L = m.lib()
    for r in range(2):
        raw = x[r].view(torch.int16).numpy()
        m._check(L.mcke_rt_memcpy_async(bufs[0].ptr + 2 * r * stride, raw.ctypes.data, raw.nbytes,
                                        0, None))
        m.device_synchronize()
    outs = {n: out(m, want[n].shape, want[n].dtype) for n in NAMES}
    nbytes = m.token_logprobs_workspace_bytes(2, vocab, 5)
    ws, dt = workspace(m, nbytes), Dev(m, tokens)
    m.launch_token_logprobs(bufs[0], dt, *(outs[n] for n in NAMES), BF16, 2, vocab, stride, 1.0, 5,
                            ws, nbytes).throw_if_error()
    m.launch_token_logprobs_backward(bufs[0], dt, outs["lse"], outs["entropy"], Dev(m, g),
                                     Dev(m, h), bufs[1], BF16, 2, vocab, stride).throw_if_error()
    m.device_synchronize()
    assert all(same_bits(outs[n].get(), want[n]) for n in NAMES)
    for r in range(2):
        got = np.empty(vocab, np.int16)
        m._check(L.mcke_rt_memcpy_async(got.ctypes.data, bufs[1].ptr + 2 * r * stride, got.nbytes,
                                        1, None))
        m.device_synchronize()
        assert same_bits(torch.from_numpy(got).view(torch.bfloat16), wgrad[r])


def test_rows_without_a_token_cost_no_reads(gpu):
    """The gradient of rows without a token is written and nothing of them read: half the bytes
    of a row with one (measured: 0.6 of the time; read all the same, 0.99)."""
    m = gpu
    rows, vocab = 1024, 131072
    x = Dev(m, torch.ones(rows, vocab, dtype=torch.bfloat16))
    dx = m.DeviceBuffer(2 * rows * vocab)
    lse, g = Dev(m, torch.full((rows,), 12.78)), Dev(m, torch.ones(rows))
    some, none = (Dev(m, torch.full((rows,), t, dtype=torch.int64)) for t in (5, -1))
    e0, e1 = m.Event(), m.Event()
    best = {}
    for _ in range(12):
        for name, tokens in (("some", some), ("none", none)):
            e0.record()
            for _ in range(4):
                m.launch_token_logprobs_backward(x, tokens, lse, None, g, None, dx, BF16, rows,
                                                 vocab, vocab).throw_if_error()
            e1.record()
            e1.synchronize()
            best[name] = min(best.get(name, INF), e0.elapsed_ms(e1))
    assert best["none"] < 0.85 * best["some"], best
