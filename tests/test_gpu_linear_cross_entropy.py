"""Cross entropy of hidden states and a vocabulary's weights, and its gradients
(mcke_launch_linear_cross_entropy, ..._backward), on the GPU against the formulas in 64 bits.

Tolerances are counts of roundings (U is one in fp32; exp2 and log2 of the hardware are off by
at most 2 U), D dim:
  z      D products, each exact in fp32, and their sum: D U sum |h w|, times scale, and 2 U |z|
  lse    the largest of its row's z errors; exponents (z - m) c are off by 3 U of themselves, which
         the sum weighs by p: below 3 U times 40 (p |z - m| adds up to the entropy plus m - lse);
         2 U for exp2; V / 16 + 64 additions of positive terms; the logarithm 2 U and its product
  loss   lse's, z's of the target, one subtraction
  p      z's, and 4 U (|z| + |lse|) + 2 U of the exponent and exp2, relative
  dz     p's times |dloss + dlse|, 4 U of its terms, and the rounding to 16 bits, half a step of
         the value (in fp16 at least half its smallest subnormal, 2^-25, where the largest row's
         gradient is 2^14 or more)
  dH     sum over V of dz's |w|, V U sum |dz w|, the output's rounding;  dW the same over rows
"""
from __future__ import annotations

import math

import numpy as np
import pytest
import torch

from tests.operator_util import (BF16, F16, F32, HALF, ID, TINY, TORCH, U, Captured, Dev, check,
                                 out, same_bits, workspace)

pytestmark = pytest.mark.gpu

TYPES = [BF16, F16]
# rows, vocab, dim: every tile (64 x 128 up to 64 rows, 128 x 128, 256 x 256 from 192 of them), one
# token, one logit, widths that are not 64s down to one (odd: padded copies; even: rows that cross
# 16-byte loads), vocabularies that end inside a tile and inside a stage, rows that do, dH in parts and
# whole.
SHAPES = [(1, 1, 64), (1, 1000, 128), (3, 130, 1), (5, 257, 33), (2, 256, 2), (70, 513, 6), (9, 514, 2),
          (40, 128, 1000), (150, 1100, 222), (300, 25001, 190), (64, 128, 64), (17, 5003, 192),
          (65, 64, 320), (100, 1021, 100), (128, 300, 256), (200, 4100, 64), (300, 25000, 512),
          (700, 3001, 130), (1500, 8200, 64)]


def _draw(rows, vocab, dim, dt, seed, spread=2.0):
    g = torch.Generator().manual_seed(seed)
    w = (torch.randn(vocab, dim, generator=g) * spread / math.sqrt(dim)).to(TORCH[dt])
    h = torch.randn(rows, dim, generator=g).to(TORCH[dt])
    t = torch.randint(vocab, (rows,), generator=g)
    t[torch.rand(rows, generator=g) < 0.2] = -100
    return h, w, t


def _logits(h, w, scale):
    """(z, its tolerance) in 64 bits."""
    hd, wd = h.double(), w.double()
    z = scale * (hd @ wd.t())
    return z, h.shape[1] * U * scale * (hd.abs() @ wd.abs().t()) + 2 * U * z.abs()


def forward_reference(h, w, t, scale):
    """((loss, lse), tolerances); zeros for rows without a target."""
    vocab = w.shape[0]
    z, tz = _logits(h, w, scale)
    lse = torch.logsumexp(z, 1)
    tl = tz.amax(1) + U * (120 + 2 + vocab / 16 + 64 + 4) + 4 * U * (lse.abs() + z.amax(1).abs())
    at = t.clamp(0, vocab - 1)[:, None]
    loss = lse - z.gather(1, at)[:, 0]
    tloss = tl + tz.gather(1, at)[:, 0] + U * loss.abs()
    loss = torch.where(t >= vocab, torch.nan, loss)
    none = t < 0
    return ((torch.where(none, 0.0, loss), torch.where(none, 0.0, lse)),
            (torch.where(none, 0.0, tloss), torch.where(none, 0.0, tl)))


def backward_reference(h, w, t, lse, dloss, dlse, scale, dt):
    """((dhidden, dweight), tolerances), from the lse that the forward pass gave."""
    rows, vocab = len(t), w.shape[0]
    hd, wd = h.double(), w.double()
    z, tz = _logits(h, w, scale)
    a = dloss.double() if dloss is not None else torch.zeros(rows, dtype=torch.float64)
    b = dlse.double() if dlse is not None else torch.zeros(rows, dtype=torch.float64)
    none = (t < 0)[:, None]
    lse = lse.double()[:, None]
    p = torch.exp(torch.where(none, -math.inf, z - lse))
    cp, ct = (scale * (a + b))[:, None], (scale * a)[:, None]
    hot = torch.zeros(rows, vocab, dtype=torch.float64)
    hot[torch.arange(rows)[t >= 0], t[t >= 0]] = 1.0
    dz = cp * p - ct * hot
    dz = torch.where(none, 0.0, dz)
    tp = p * (tz + 4 * U * (z.abs() + lse.abs()) + 2 * U)
    tdz = cp.abs() * tp + 4 * U * (cp.abs() * p + ct.abs() * hot)
    tdz = tdz + HALF[dt] * (dz.abs() + tdz)
    if dt == F16:
        tdz = tdz + 2.0**-39 * (scale * (a.abs() + b.abs())[t >= 0]).max() if (t >= 0).any() else tdz
    tdz = torch.where(none, 0.0, tdz)
    hd = torch.where(none, 0.0, hd)
    res = []
    for x, tx, y in ((dz, tdz, wd), (dz.t(), tdz.t(), hd)):
        want = x @ y
        tol = tx @ y.abs() + x.shape[1] * U * (x.abs() @ y.abs())
        res.append((want, tol + HALF[dt] * (want.abs() + tol) + TINY[dt]))
    return (res[0][0], res[1][0]), (res[0][1], res[1][1])


def run_forward(m, h, w, t, dt, scale, shift=0, want=(True, True), stream=None):
    rows, (vocab, dim) = len(t), w.shape
    outs = [out(m, (rows,), torch.float32) if k else None for k in want]
    n = m.linear_cross_entropy_workspace_bytes(rows, vocab, dim)
    ws = workspace(m, n)
    m.launch_linear_cross_entropy(Dev(m, h, shift), Dev(m, w, shift if dim % 2 else 2 * shift),
                                  Dev(m, t), *outs, dt, rows, vocab, dim, scale, ws, n,
                                  stream).throw_if_error()
    m.device_synchronize()
    ws.get()
    return [o.get() if o is not None else None for o in outs]


def run_backward(m, h, w, t, lse, dloss, dlse, dt, scale, shift=0, want=(True, True), stream=None):
    rows, (vocab, dim) = len(t), w.shape
    outs = [out(m, x.shape, x.dtype, shift) if k else None for x, k in zip((h, w), want)]
    n = m.linear_cross_entropy_backward_workspace_bytes(rows, vocab, dim)
    ws = workspace(m, n)
    vec = [Dev(m, v) if v is not None else None for v in (lse, dloss, dlse)]
    m.launch_linear_cross_entropy_backward(
        Dev(m, h, shift), Dev(m, w, shift if dim % 2 else 2 * shift), Dev(m, t), *vec, *outs, dt, rows,
        vocab, dim, scale, ws, n, stream).throw_if_error()
    m.device_synchronize()
    ws.get()
    return [o.get() if o is not None else None for o in outs]


def _grads(rows, seed, dt):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(rows, generator=g) / rows, 0.3 * torch.randn(rows, generator=g) / rows


@pytest.mark.parametrize("dt", TYPES, ids=[ID[t] for t in TYPES])
@pytest.mark.parametrize("i,shape", enumerate(SHAPES), ids=[str(s) for s in SHAPES])
def test_loss_and_gradients(gpu, i, shape, dt):
    scale = (1.0, 1.25, 0.5)[i % 3]
    h, w, t = _draw(*shape, dt, i)
    if i % 4 == 0:
        t = t.abs() % shape[1]               # every row has a target
    loss, lse = run_forward(gpu, h, w, t, dt, scale, shift=i % 3)
    want, tol = forward_reference(h, w, t, scale)
    check("loss", loss, want[0], tol[0])
    check("lse", lse, want[1], tol[1])
    dloss, dlse = _grads(shape[0], i, dt)
    dlse = None if i % 2 else dlse
    got = run_backward(gpu, h, w, t, lse, dloss, dlse, dt, scale, shift=i % 3)
    want, tol = backward_reference(h, w, t, lse, dloss, dlse, scale, dt)
    check("dhidden", got[0], want[0], tol[0])
    check("dweight", got[1], want[1], tol[1])


@pytest.mark.parametrize("shape", [(12300, 7000, 64), (12300, 7001, 66), (12300, 300, 1024), (5, 9000, 8191),
                                   (12300, 7001, 130), (12300, 7040, 192)], ids=str)
def test_pieces(gpu, shape):
    """Vocabularies in several pieces, of the weights as they are and of padded copies; logits
    at 128 x 128 and 256 x 256 tiles, dH at 256 x 256."""
    h, w, t = _draw(*shape, BF16, 1)
    loss, lse = run_forward(gpu, h, w, t, BF16, 1.0)
    want, tol = forward_reference(h, w, t, 1.0)
    check("loss", loss, want[0], tol[0])
    dloss, dlse = _grads(shape[0], 1, BF16)
    got = run_backward(gpu, h, w, t, lse, dloss, dlse, BF16, 1.0)
    want, tol = backward_reference(h, w, t, lse, dloss, dlse, 1.0, BF16)
    check("dhidden", got[0], want[0], tol[0])
    check("dweight", got[1], want[1], tol[1])


@pytest.mark.parametrize("dt", TYPES, ids=[ID[t] for t in TYPES])
@pytest.mark.parametrize("keep", ["none", "one", "last 64", "all"])
@pytest.mark.parametrize("rows", [333, 1024, 1025])
def test_rows_without_a_target(gpu, dt, keep, rows):
    """They are not read (NaN in their place changes no bit), give zeros and add nothing; by either
    way of packing the others (up to 1024 rows, and more)."""
    vocab, dim = 700, 128
    h, w, t = _draw(rows, vocab, dim, dt, 5)
    t = t.abs() % vocab
    if keep != "all":
        t[:] = -1
    if keep == "one":
        t[200] = 13
    if keep == "last 64":
        t[-64:] = torch.arange(64)
    none = t < 0
    loss, lse = run_forward(gpu, h, w, t, dt, 1.0)
    want, tol = forward_reference(h, w, t, 1.0)
    check("loss", loss, want[0], tol[0])
    dloss, dlse = _grads(rows, 5, dt)
    got = run_backward(gpu, h, w, t, lse, dloss, dlse, dt, 1.0)
    want, tol = backward_reference(h, w, t, lse, dloss, dlse, 1.0, dt)
    check("dhidden", got[0], want[0], tol[0])
    check("dweight", got[1], want[1], tol[1])
    assert not loss[none].any() and not lse[none].any() and not got[0][none].any()
    bad = h.clone()
    bad[none] = torch.nan
    lse2, dloss[none], dlse[none] = lse.clone(), torch.nan, torch.inf
    lse2[none] = torch.nan
    assert same_bits(run_forward(gpu, bad, w, t, dt, 1.0)[0], loss)
    again = run_backward(gpu, bad, w, t, lse2, dloss, dlse, dt, 1.0)
    assert all(same_bits(a, g) for a, g in zip(again, got))


def test_targets_past_the_vocabulary(gpu):
    rows, vocab, dim = 70, 300, 64
    h, w, t = _draw(rows, vocab, dim, BF16, 6)
    t[3], t[50] = vocab, torch.iinfo(torch.int64).max
    loss, lse = run_forward(gpu, h, w, t, BF16, 1.0)
    want, tol = forward_reference(h, w, t, 1.0)
    check("loss", loss, want[0], tol[0])
    check("lse", lse, want[1], tol[1])
    dloss, _ = _grads(rows, 6, BF16)
    dh, dw = run_backward(gpu, h, w, t, lse, dloss, None, BF16, 1.0)
    past = t >= vocab
    assert dh[past].isnan().all() and not dh[~past].isnan().any()
    assert dw.isnan().all()


def test_large_and_equal_logits(gpu):
    """Logits of several hundred (one exponential is left) and all equal ones (lse = z + ln V)."""
    rows, vocab, dim = 100, 1500, 64
    h, w, t = _draw(rows, vocab, dim, BF16, 7, spread=150.0)
    (_, lse), tol = forward_reference(h, w, t, 1.0)
    loss, got = run_forward(gpu, h, w, t, BF16, 1.0)
    check("lse", got, lse, tol[1])
    h[:] = 0
    loss, got = run_forward(gpu, h, w, t, BF16, 1.0)
    have = t >= 0
    check("loss", loss[have], torch.full_like(loss[have], math.log(vocab)), 200 * U)
    dloss, _ = _grads(rows, 7, BF16)
    grads = run_backward(gpu, h, w, t, got, dloss, None, BF16, 1.0)
    want, tol = backward_reference(h, w, t, got, dloss, None, 1.0, BF16)
    check("dhidden", grads[0], want[0], tol[0])
    assert not grads[1].any()                      # hidden states of zeros


@pytest.mark.parametrize("size", [2.0**-40, 1e-12, 1.0, 3e4])
def test_small_and_large_gradients_in_fp16(gpu, size):
    """dloss far below fp16's smallest value, as the mean over a batch is: dz is scaled by a power
    of two and the sums scaled back, so gradients that fp16 can hold are right.  Hidden states and
    weights are large where dloss is small, and small where it is large; what is past fp16's largest
    value all the same (from 65520 on) is infinite."""
    rows, vocab, dim = 90, 600, 64
    h, w, t = _draw(rows, vocab, dim, F16, 8)
    k = min(max(round(math.log2(1 / size) / 2), -6), 6)
    w, h = w * 2.0**-k, h * 2.0**k
    loss, lse = run_forward(gpu, h, w, t, F16, 1.0)
    dloss = torch.full((rows,), size)
    got = run_backward(gpu, h, w, t, lse, dloss, None, F16, 1.0)
    want, tol = backward_reference(h, w, t, lse, dloss, None, 1.0, F16)
    for name, g, x, e in zip(("dhidden", "dweight"), got, want, tol):
        over, under = x.abs() - e >= 65520, x.abs() + e < 65520
        assert torch.equal(g[over].double(), torch.sign(x[over]) * math.inf)
        assert (g[~over & ~under].abs() >= 60000).all()
        check(name, g[under], x[under], e[under])


def test_outputs_apart(gpu):
    rows, vocab, dim = 150, 900, 128
    h, w, t = _draw(rows, vocab, dim, BF16, 9)
    loss, lse = run_forward(gpu, h, w, t, BF16, 1.0)
    assert same_bits(run_forward(gpu, h, w, t, BF16, 1.0, want=(True, False))[0], loss)
    assert same_bits(run_forward(gpu, h, w, t, BF16, 1.0, want=(False, True))[1], lse)
    dloss, dlse = _grads(rows, 9, BF16)
    both = run_backward(gpu, h, w, t, lse, dloss, dlse, BF16, 1.0)
    for k in range(2):
        got = run_backward(gpu, h, w, t, lse, dloss, dlse, BF16, 1.0, want=(k == 0, k == 1))
        assert same_bits(got[k], both[k])
    alone = run_backward(gpu, h, w, t, lse, None, dlse, BF16, 1.0)
    want, tol = backward_reference(h, w, t, lse, None, dlse, 1.0, BF16)
    for g, x, e in zip(alone, want, tol):
        check("of lse alone", g, x, e)


def test_gradient_against_differences(gpu):
    """sum(dloss loss) along a direction in the weights, by central differences of the formula in 64
    bits, against <dweight, v>: off by h^2 / 6 times a third derivative below that of exp's sums
    (|v . h|^3 scale^3, below 1e3 here), 2e-4 of sum |dloss| at h = 1e-3, and by dweight's
    tolerance."""
    rows, vocab, dim = 40, 300, 64
    h, w, t = _draw(rows, vocab, dim, BF16, 10)
    t = t.abs() % vocab
    _, lse = run_forward(gpu, h, w, t, BF16, 1.0)
    dloss = torch.rand(rows, generator=torch.Generator().manual_seed(3)) + 0.5
    _, dw = run_backward(gpu, h, w, t, lse, dloss, None, BF16, 1.0)
    v = torch.randn(vocab, dim, generator=torch.Generator().manual_seed(4), dtype=torch.float64)
    v = v / math.sqrt(dim)

    def f(s):
        z = h.double() @ (w.double() + s * v).t()
        return (dloss.double() * (torch.logsumexp(z, 1) - z[torch.arange(rows), t])).sum()

    eps = 1e-3
    slope = (f(eps) - f(-eps)) / (2 * eps)
    tol = backward_reference(h, w, t, lse, dloss, None, 1.0, BF16)[1][1]
    third = ((v @ h.double().t()).abs().amax(0)**3 * dloss.double()).sum()
    assert abs(slope - (dw.double() * v).sum()) <= eps**2 / 6 * 8 * third + (tol * v.abs()).sum()


def test_no_rows(gpu):
    m = gpu
    dw = out(m, (77, 65), torch.bfloat16)
    m.launch_linear_cross_entropy_backward(None, None, None, None, None, None, None, dw, BF16, 0, 77,
                                           65).throw_if_error()
    m.device_synchronize()
    assert not dw.get().any()


def test_same_bits_capture_and_streams(gpu):
    m = gpu
    rows, vocab, dim = 260, 2001, 192
    h, w, t = _draw(rows, vocab, dim, BF16, 11)
    dloss, dlse = _grads(rows, 11, BF16)
    fwd = run_forward(m, h, w, t, BF16, 1.0)
    bwd = run_backward(m, h, w, t, fwd[1], dloss, dlse, BF16, 1.0)
    ins = [Dev(m, x) for x in (h, w, t, dloss, dlse)]
    f, b = ([out(m, x.shape, x.dtype) for x in r] for r in (fwd, bwd))
    nf = m.linear_cross_entropy_workspace_bytes(rows, vocab, dim)
    nb = m.linear_cross_entropy_backward_workspace_bytes(rows, vocab, dim)
    wf, wb = workspace(m, nf), workspace(m, nb)

    def launch(stream):
        m.launch_linear_cross_entropy(*ins[:3], *f, BF16, rows, vocab, dim, 1.0, wf, nf,
                                      stream).throw_if_error()
        m.launch_linear_cross_entropy_backward(*ins[:3], f[1], *ins[3:], *b, BF16, rows, vocab, dim,
                                               1.0, wb, nb, stream).throw_if_error()

    graph = Captured(m, launch)
    try:
        for _ in range(3):
            graph.replay()
            assert all(same_bits(o.get(), x) for o, x in zip(f + b, fwd + bwd))
            for o in f + b:
                o.buf.upload(np.full(o.buf.nbytes, 0xA5, np.uint8))
            assert same_bits(run_forward(m, h, w, t, BF16, 1.0)[0], fwd[0])
    finally:
        graph.close()
    st = m.Stream()
    try:
        assert same_bits(run_forward(m, h, w, t, BF16, 1.0, stream=st)[0], fwd[0])
        again = run_backward(m, h, w, t, fwd[1], dloss, dlse, BF16, 1.0, stream=st)
        assert all(same_bits(a, x) for a, x in zip(again, bwd))
    finally:
        st.close()


def test_offsets_past_32_bits(gpu):
    """Weights of more than 2^31 values, zeros but for their last rows: V - 3 logits of 0."""
    m = gpu
    import ctypes as C
    rows, dim = 3, 4096
    vocab = (1 << 31) // dim + 130
    h, w, _ = _draw(rows, 3, dim, BF16, 12)
    L = m.lib()
    L.mcke_fill_u32_async.argtypes = [C.c_void_p, C.c_uint32, C.c_size_t, C.c_void_p]
    big, grad = m.DeviceBuffer(2 * vocab * dim), m.DeviceBuffer(2 * vocab * dim)
    for buf, v in ((big, 0), (grad, 0xA5A5A5A5)):
        m._check(L.mcke_fill_u32_async(buf.ptr, v, vocab * dim // 2, None))
    raw = w.view(torch.int16).numpy()
    at = 2 * (vocab - 3) * dim
    m._check(L.mcke_rt_memcpy_async(big.ptr + at, raw.ctypes.data, raw.nbytes, 0, None))
    m.device_synchronize()
    t = torch.tensor([vocab - 1, vocab - 3, vocab - 2])
    loss, lse = (out(m, (rows,), torch.float32) for _ in range(2))
    dh, dt_ = Dev(m, h), Dev(m, t)
    n = m.linear_cross_entropy_workspace_bytes(rows, vocab, dim)
    m.launch_linear_cross_entropy(dh, big, dt_, loss, lse, BF16, rows, vocab, dim, 1.0,
                                  workspace(m, n), n).throw_if_error()
    m.device_synchronize()
    z, tz = _logits(h, w, 1.0)
    want = torch.logaddexp(torch.logsumexp(z, 1), torch.tensor(math.log(vocab - 3)))
    tol = tz.amax(1) + U * (300 + vocab / 16) + 4 * U * want.abs()
    check("lse", lse.get(), want, tol)
    check("loss", loss.get(), want - z[torch.arange(3), t - (vocab - 3)], tol + tz.amax(1) + U * want)
    n = m.linear_cross_entropy_backward_workspace_bytes(rows, vocab, dim)
    one = Dev(m, torch.ones(rows))
    m.launch_linear_cross_entropy_backward(dh, big, dt_, lse, one, None, None, grad, BF16, rows,
                                           vocab, dim, 1.0, workspace(m, n), n).throw_if_error()
    m.device_synchronize()
    got = np.empty((3, dim), np.int16)
    m._check(L.mcke_rt_memcpy_async(got.ctypes.data, grad.ptr + at, got.nbytes, 1, None))
    m.device_synchronize()
    got = torch.from_numpy(got).view(torch.bfloat16)
    l = lse.get()
    dz = torch.exp(z - l.double()[:, None])
    dz[torch.arange(3), t - (vocab - 3)] -= 1
    tdz = HALF[BF16] * dz.abs() + 2 * tz + 1e-5
    want = dz.t() @ h.double()
    tol = tdz.t() @ h.double().abs()
    check("dweight", got, want, tol + HALF[BF16] * (want.abs() + tol) + TINY[BF16])


@pytest.mark.parametrize("dt", TYPES, ids=[ID[t] for t in TYPES])
@pytest.mark.parametrize("shape", [(40, 1000, 192), (200, 4100, 64), (150, 300, 1024), (300, 25000, 512),
                                   (700, 3001, 4096)], ids=str)
def test_aligned_weight_gradient(gpu, shape, dt):
    """dweight at whole 128-byte lines, as allocators give it, of one stage, 128 x 128 and 256 x 256
    tiles: right, and the bits of one off the lines."""
    m = gpu
    rows, vocab, dim = shape
    h, w, t = _draw(*shape, dt, 13)
    _, lse = run_forward(m, h, w, t, dt, 1.0)
    dloss, _ = _grads(rows, 13, dt)
    ins = [Dev(m, x) for x in (h, w, t, lse, dloss)]
    n = m.linear_cross_entropy_backward_workspace_bytes(rows, vocab, dim)
    ws = workspace(m, n)
    got = []
    for shift in (32, 0):                       # values behind 64 bytes past a line of 256
        dw = out(m, w.shape, w.dtype, shift)
        assert (dw.ptr % 128 == 0) == (shift == 32)
        m.launch_linear_cross_entropy_backward(*ins, None, None, dw, dt, rows, vocab, dim, 1.0, ws, n
                                               ).throw_if_error()
        m.device_synchronize()
        got.append(dw.get())
    want, tol = backward_reference(h, w, t, lse, dloss, None, 1.0, dt)
    check("dweight", got[0], want[1], tol[1])
    assert same_bits(*got)


def test_more_logits_than_small_tiles(gpu):
    """2^19 rows x 2^18 logits, one 128 x 128 tile too many for a launch: some rows of both passes."""
    m = gpu
    rows, vocab, dim = 1 << 19, 1 << 18, 128
    h, w, t = _draw(rows, vocab, dim, BF16, 14)
    t = torch.where(t < 0, t, (t * 7919 + 5) % vocab)
    some = torch.tensor([0, 1, 255, 131072, 300001, rows - 129, rows - 2, rows - 1])
    t[some] = torch.tensor([vocab - 1, 0, 128, 131071, 77777, 200000, 1, vocab - 2])
    ins = [Dev(m, x) for x in (h, w, t)]
    loss, lse = (out(m, (rows,), torch.float32) for _ in range(2))
    n = m.linear_cross_entropy_workspace_bytes(rows, vocab, dim)
    ws = m.DeviceBuffer(n)
    m.launch_linear_cross_entropy(*ins, loss, lse, BF16, rows, vocab, dim, 1.0, ws, n).throw_if_error()
    m.device_synchronize()
    got = [x.get() for x in (loss, lse)]
    want, tol = forward_reference(h[some], w, t[some], 1.0)
    check("loss", got[0][some], want[0], tol[0])
    check("lse", got[1][some], want[1], tol[1])
    dloss = torch.full((rows,), 1.0 / rows)
    dh, dw = out(m, h.shape, h.dtype), out(m, w.shape, w.dtype)
    n = m.linear_cross_entropy_backward_workspace_bytes(rows, vocab, dim)
    ws = m.DeviceBuffer(n)
    m.launch_linear_cross_entropy_backward(*ins, lse, Dev(m, dloss), None, dh, dw, BF16, rows, vocab, dim,
                                           1.0, ws, n).throw_if_error()
    m.device_synchronize()
    dh, dw = dh.get(), dw.get()
    want, tol = backward_reference(h[some], w, t[some], got[1][some], dloss[some], None, 1.0, BF16)
    check("dhidden", dh[some], want[0], tol[0])
    # Some rows of dweight, over all rows of the batch: dz in 64 bits for those columns alone.
    cols = torch.tensor([0, 255, 256, 131072, vocab - 1])
    z, tz = _logits(h, w[cols], 1.0)
    have = (t >= 0)[:, None]
    p = torch.where(have, torch.exp(z - got[1].double()[:, None]), 0.0)
    dz = (p - (t[:, None] == cols).double()) * (have.double() / rows)
    tdz = p * (tz + 4 * U * (z.abs() + got[1].double().abs()[:, None]) + 2 * U) / rows
    tdz = tdz + 4 * U * dz.abs()
    tdz = torch.where(have, tdz + HALF[BF16] * (dz.abs() + tdz), 0.0)
    hd = h.double()
    want = dz.t() @ hd
    tol = tdz.t() @ hd.abs() + rows * U * (dz.abs().t() @ hd.abs())
    check("dweight", dw[cols], want, tol + HALF[BF16] * (want.abs() + tol) + TINY[BF16])


@pytest.mark.parametrize("shape", [(5, 65, 2), (7, 66, 2), (3, 129, 4), (70, 321, 2), (9, 322, 2), (5, 449, 6),
                                   (131100, 513, 2), (131100, 514, 4)], ids=str)
def test_narrow_rows_at_the_end(gpu, shape):
    """Vocabularies that end one or two narrow rows into a stage, whose loads in the stage before it
    reach past them; with pieces of 256 rows, the copy of the last ones begins a piece earlier."""
    h, w, t = _draw(*shape, BF16, 15)
    loss, lse = run_forward(gpu, h, w, t, BF16, 1.25)
    want, tol = forward_reference(h, w, t, 1.25)
    check("loss", loss, want[0], tol[0])
    check("lse", lse, want[1], tol[1])
    dloss, dlse = _grads(shape[0], 15, BF16)
    got = run_backward(gpu, h, w, t, lse, dloss, dlse, BF16, 1.25)
    want, tol = backward_reference(h, w, t, lse, dloss, dlse, 1.25, BF16)
    check("dhidden", got[0], want[0], tol[0])
    check("dweight", got[1], want[1], tol[1])
