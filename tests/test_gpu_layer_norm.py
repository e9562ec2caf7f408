"""Layer norm forward and backward (mcke_launch_layer_norm, ..._backward) on the GPU against
the formulas in 64 bits.

Tolerances are counts of roundings.  U is one fp32 rounding, D the length of a row's chain of
additions: the widest kernel adds cols / 256 values in a lane, then the lanes; cols / 64 + 16
covers every kernel.  With A = mean |x|:
  mean    e_m = D U A
  rstd    e_r = ((D + 12) / 2) U rstd + e_m^2 rstd^3 / 2  (the variance about a mean off by e_m
          is off by e_m^2, as the differences sum to zero), 6 more roundings for the square,
          the division, the sum with eps, the root and its reciprocal
  y       |w| (rstd e_m + |xhat| (e_r / rstd + 3 U)) + 3 U (|xhat w| + |b|), and y's rounding
The backward pass takes mean and rstd as they are, so xhat is off by 3 U of itself:
  dx      rstd U (5 |g| + (D + 5) mean|g| + (D + 12) |xhat| mean|g xhat|), and dx's rounding
  dweight (R + 5) U sum |dy xhat|, dbias (R + 1) U sum |dy|, and their rounding; R = rows / 64 + 200
          covers a part's rows and the fold of the parts
"""
from __future__ import annotations

import numpy as np
import pytest
import torch

from tests.operator_util import (BF16, DTYPES, F16, F32, HALF, ID, TINY, TORCH, U, Captured, Dev,
                                 check, out, same_bits, workspace)

pytestmark = pytest.mark.gpu

EPS = 1e-5
# One element, rows shorter than a 16-byte vector, around 8, 64, 256 lanes' vectors, odd widths,
# several rounds of workgroups, and past what a workgroup's registers hold.
SHAPES = [(1, 1), (3, 2), (2, 3), (5, 7), (4, 8), (7, 9), (33, 64), (3, 127), (65, 255), (9, 512),
          (4, 1021), (517, 128), (6, 2048), (3, 2050), (700, 771), (5, 4096), (2, 8199), (3, 16384),
          (2, 16391), (2, 32771), (2, 65536), (1, 70001), (1, 140001)]


def _data(rows, cols, dt, pt, seed, offset=0.3, sigma=1.0):
    g = torch.Generator().manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, generator=g, dtype=torch.float64)

    x = (normal(rows, cols) * sigma + offset).to(TORCH[dt])
    w = (1 + 0.2 * normal(cols)).to(TORCH[pt])
    b = (0.2 * normal(cols)).to(TORCH[pt])
    dy = (0.1 * normal(rows, cols)).to(TORCH[dt])
    return x, w, b, dy


def _chain(cols):
    return cols / 64 + 16


def _stats(x, eps=EPS):
    x = x.double()
    mean = x.mean(1, keepdim=True)
    var = ((x - mean) ** 2).mean(1, keepdim=True)
    return mean, 1 / torch.sqrt(var + eps)


def _forward(x, w, b, dt, eps=EPS):
    """(y, mean, rstd) in 64 bits and their tolerances."""
    mean, rstd = _stats(x, eps)
    xhat = (x.double() - mean) * rstd
    wd = w.double() if w is not None else torch.ones(x.shape[1], dtype=torch.float64)
    bd = b.double() if b is not None else torch.zeros(x.shape[1], dtype=torch.float64)
    y = xhat * wd + bd
    D = _chain(x.shape[1])
    em = D * U * x.double().abs().mean(1, keepdim=True)
    er = (D + 12) / 2 * U * rstd + em**2 * rstd**3 / 2
    ty = (wd.abs() * (rstd * em + xhat.abs() * (er / rstd + 3 * U)) +
          3 * U * ((xhat * wd).abs() + bd.abs()))
    ty = ty + HALF[dt] * (y.abs() + ty) + TINY[dt]
    return (y, mean[:, 0], rstd[:, 0]), (ty, em[:, 0] + U * mean[:, 0].abs(), er[:, 0])


def _backward(dy, x, w, mean, rstd, dt, pt):
    x, dy, mean, rstd = x.double(), dy.double(), mean.double()[:, None], rstd.double()[:, None]
    rows, cols = x.shape
    wd = w.double() if w is not None else torch.ones(cols, dtype=torch.float64)
    xhat, g = (x - mean) * rstd, dy * wd
    dx = rstd * (g - g.mean(1, keepdim=True) - xhat * (g * xhat).mean(1, keepdim=True))
    dw, db = (dy * xhat).sum(0), dy.sum(0)
    D, R = _chain(cols), rows / 64 + 200
    tx = rstd * U * (5 * g.abs() + (D + 5) * g.abs().mean(1, keepdim=True) +
                     (D + 12) * xhat.abs() * (g * xhat).abs().mean(1, keepdim=True))
    tw, tb = (R + 5) * U * (dy * xhat).abs().sum(0), (R + 1) * U * dy.abs().sum(0)
    return ((dx, dw, db), (tx + HALF[dt] * (dx.abs() + tx) + TINY[dt],
                           tw + HALF[pt] * (dw.abs() + tw) + TINY[pt],
                           tb + HALF[pt] * (db.abs() + tb) + TINY[pt]))


def run_forward(m, x, w, b, dt, pt, eps=EPS, shift=0, stats=True, stream=None):
    rows, cols = x.shape
    dx, dw, db = (Dev(m, t, shift) if t is not None else None for t in (x, w, b))
    y = out(m, (rows, cols), TORCH[dt], shift)
    mean, rstd = ((out(m, (rows,), torch.float32, shift) for _ in range(2)) if stats
                  else (None, None))
    m.launch_layer_norm(dx, dw, db, y, mean, rstd, dt, pt, rows, cols, eps,
                        stream).throw_if_error()
    m.device_synchronize()
    return (y.get(), mean.get(), rstd.get()) if stats else y.get()


def run_backward(m, dy, x, w, mean, rstd, dt, pt, shift=0, want=(True, True, True)):
    rows, cols = x.shape
    ins = [Dev(m, t, shift) if t is not None else None for t in (dy, x, w, mean, rstd)]
    outs = [out(m, s, TORCH[t], shift) if k else None
            for s, t, k in zip(((rows, cols), (cols,), (cols,)), (dt, pt, pt), want)]
    nbytes = m.layer_norm_backward_workspace_bytes(rows, cols) if want[1] or want[2] else 0
    ws = workspace(m, nbytes)
    m.launch_layer_norm_backward(*ins, *outs, dt, pt, rows, cols, ws, nbytes).throw_if_error()
    m.device_synchronize()
    if ws is not None:
        ws.get()                                   # its guards
    return tuple(o.get() if o is not None else None for o in outs)


@pytest.mark.parametrize("dt", DTYPES, ids=ID.get)
@pytest.mark.parametrize("rows,cols", SHAPES)
def test_forward(gpu, rows, cols, dt):
    pt = F32 if (rows + cols) % 2 else dt
    x, w, b, _ = _data(rows, cols, dt, pt, 1000 + rows + cols)
    got = run_forward(gpu, x, w, b, dt, pt)
    for name, g, r, t in zip(("y", "mean", "rstd"), got, *_forward(x, w, b, dt)):
        check(name, g, r, t)


@pytest.mark.parametrize("dt", DTYPES, ids=ID.get)
@pytest.mark.parametrize("rows,cols", SHAPES)
def test_backward(gpu, rows, cols, dt):
    pt = F32 if (rows + cols) % 2 else dt
    x, w, _, dy = _data(rows, cols, dt, pt, 2000 + rows + cols)
    mean, rstd = (t[:, 0].float() for t in _stats(x))
    got = run_backward(gpu, dy, x, w, mean, rstd, dt, pt)
    for name, g, r, t in zip(("dx", "dweight", "dbias"), got,
                             *_backward(dy, x, w, mean, rstd, dt, pt)):
        check(name, g, r, t)


@pytest.mark.parametrize("rows,cols", [(20000, 40), (4099, 264), (9001, 33), (2500, 1024),
                                       (1300, 4096), (777, 5000)])
def test_backward_many_rows(gpu, rows, cols):
    """More rows than partial sums, in numbers that do not divide evenly."""
    x, w, _, dy = _data(rows, cols, BF16, BF16, rows + cols)
    mean, rstd = (t[:, 0].float() for t in _stats(x))
    got = run_backward(gpu, dy, x, w, mean, rstd, BF16, BF16)
    for name, g, r, t in zip(("dx", "dweight", "dbias"), got,
                             *_backward(dy, x, w, mean, rstd, BF16, BF16)):
        check(name, g, r, t)


# Widths of 513 to 1024 vectors, whole and not, in either element size, and rows enough for a
# workgroup to walk several of them.
@pytest.mark.parametrize("dt", DTYPES, ids=ID.get)
@pytest.mark.parametrize("rows,cols", [(5, 2500), (3, 2501), (4, 3500), (3, 3501), (5, 4999),
                                       (3, 5000), (1500, 6143), (3, 6500), (5, 6501),
                                       (1100, 8191), (2, 8192)])
def test_backward_between_powers_of_two(gpu, rows, cols, dt):
    test_backward(gpu, rows, cols, dt)


@pytest.mark.parametrize("dt", DTYPES, ids=ID.get)
@pytest.mark.parametrize("shift", [1, 3])
@pytest.mark.parametrize("rows,cols", [(5, 64), (9, 1024), (3, 4099), (2, 16384)])
def test_any_alignment(gpu, rows, cols, shift, dt):
    """Operands that start off 16 bytes give the bits of aligned ones."""
    x, w, b, dy = _data(rows, cols, dt, dt, 7)
    for a, c in zip(run_forward(gpu, x, w, b, dt, dt),
                    run_forward(gpu, x, w, b, dt, dt, shift=shift)):
        assert same_bits(a, c)
    mean, rstd = (t[:, 0].float() for t in _stats(x))
    for a, c in zip(run_backward(gpu, dy, x, w, mean, rstd, dt, dt),
                    run_backward(gpu, dy, x, w, mean, rstd, dt, dt, shift=shift)):
        assert same_bits(a, c)


@pytest.mark.parametrize("cols", [5, 100, 1024, 20000])
def test_optional_operands(gpu, cols):
    """No weight is ones, no bias zeros; statistics and gradients that are not asked for are
    not written, and the others keep their bits."""
    x, w, b, dy = _data(4, cols, BF16, F32, cols)
    for ww, bb in ((None, None), (w, None), (None, b)):
        y, mean, rstd = run_forward(gpu, x, ww, bb, BF16, F32)
        want, tol = _forward(x, ww, bb, BF16)
        check("y", y, want[0], tol[0])
        assert same_bits(run_forward(gpu, x, ww, bb, BF16, F32, stats=False), y)
    full = run_backward(gpu, dy, x, w, mean, rstd, BF16, F32)
    for want in ((True, False, False), (False, True, False), (False, False, True),
                 (False, True, True), (True, True, False)):
        for a, c, k in zip(run_backward(gpu, dy, x, w, mean, rstd, BF16, F32, want=want), full,
                           want):
            assert (a is None) if not k else same_bits(a, c)
    got = run_backward(gpu, dy, x, None, mean, rstd, BF16, F32)
    for g, r, t in zip(got, *_backward(dy, x, None, mean, rstd, BF16, F32)):
        check("no weight", g, r, t)


def test_no_rows(gpu):
    """A sum over no rows is zero; nothing else is touched."""
    m = gpu
    dw, db = out(m, (100,), torch.float16), out(m, (100,), torch.float16)
    m.launch_layer_norm_backward(None, None, None, None, None, None, dw, db, F16, F16, 0, 100, None,
                                 0).throw_if_error()
    m.device_synchronize()
    assert (dw.get() == 0).all() and (db.get() == 0).all()


@pytest.mark.parametrize("cols", [8, 1000, 4096, 70001])
def test_constant_rows_and_eps(gpu, cols):
    """A row of one value has variance 0: y is the bias and rstd is 1 / sqrt(eps).  The mean of
    equal powers of two is exact, so nothing else is left."""
    x = torch.full((2, cols), 4.0)
    x[1] = -0.5
    b = torch.arange(cols, dtype=torch.float32) / 64
    # Sums of 4 and 0.5 stay below 2^24 steps: exact; cols divides its own multiple exactly.
    y, mean, rstd = run_forward(gpu, x, None, b, F32, F32, eps=0.25)
    assert torch.equal(mean, x[:, 0]) and torch.equal(rstd, torch.full((2,), 2.0))
    assert torch.equal(y, b.expand(2, cols))


def test_large_mean(gpu):
    """Rows far from zero: a sum of squares less a squared mean would lose the variance."""
    x, w, b, _ = _data(6, 2049, F32, F32, 5, offset=1000.0, sigma=0.5)
    got = run_forward(gpu, x, w, b, F32, F32)
    for name, g, r, t in zip(("y", "mean", "rstd"), got, *_forward(x, w, b, F32)):
        check(name, g, r, t)


@pytest.mark.parametrize("cols", [6, 512, 4100, 70001])
def test_special_values(gpu, cols):
    """A NaN or an infinity spoils its own row alone."""
    x, w, b, dy = _data(5, cols, F32, F32, 11)
    clean = run_forward(gpu, x, w, b, F32, F32)
    bad = x.clone()
    bad[1, cols // 2], bad[3, cols - 1] = float("nan"), float("inf")
    y, mean, rstd = run_forward(gpu, bad, w, b, F32, F32)
    for r in (1, 3):
        assert y[r].isnan().all() and rstd[r].isnan()
    assert mean[1].isnan() and mean[3] == float("inf")
    for r in (0, 2, 4):
        assert same_bits(y[r], clean[0][r])


@pytest.mark.parametrize("cols", [100, 99, 8])
def test_large_constant_rows_backward(gpu, cols):
    """Equal values of 2^120: their sum is exact and finite and xhat is 0 everywhere, while
    mean * rstd is past fp32's range; lanes that hold none of the row add nothing to it."""
    x = torch.full((3, cols), 2.0**120)
    dy = (torch.arange(3 * cols).reshape(3, cols) % 5 - 2).float()
    _, mean, rstd = run_forward(gpu, x, None, None, F32, F32)
    assert (mean == 2.0**120).all() and 2.0**120 * float(rstd[0]) > torch.finfo(torch.float32).max
    got = run_backward(gpu, dy, x, None, mean, rstd, F32, F32)
    for name, g, r, t in zip(("dx", "dweight", "dbias"), got,
                             *_backward(dy, x, None, mean, rstd, F32, F32)):
        check(name, g, r, t)


def test_gradient_against_differences(gpu):
    """dx, dweight and dbias of sum(dy y) against central differences of the forward formula in
    64 bits: with steps of 1e-4 their own error is below 1e-7 of the largest gradient."""
    rows, cols = 3, 37
    x, w, b, dy = _data(rows, cols, F32, F32, 3)

    def loss(x, w, b):
        mean, rstd = _stats(x)
        return float(((x - mean) * rstd * w + b).mul(dy.double()).sum())

    _, mean, rstd = run_forward(gpu, x, w, b, F32, F32)
    got = run_backward(gpu, dy, x, w, mean, rstd, F32, F32)
    _, tol = _backward(dy, x, w, mean, rstd, F32, F32)
    # mean and rstd as the forward pass rounded them: 32 U of each term covers their error.
    args = [t.double() for t in (x, w, b)]
    h = 1e-4
    for k in range(3):
        want = torch.zeros_like(args[k])
        for i in np.ndindex(*args[k].shape):
            hi, lo = [a.clone() for a in args], [a.clone() for a in args]
            hi[k][i] += h
            lo[k][i] -= h
            want[i] = (loss(*hi) - loss(*lo)) / (2 * h)
        check(("dx", "dw", "db")[k], got[k], want,
              tol[k] + (32 * U * (cols if k == 0 else rows) + 1e-7) * want.abs().max())


def test_captured_and_on_a_stream(gpu):
    """A captured forward and backward pass replays to the eager bits, with eager work between
    the replays."""
    m = gpu
    rows, cols = 300, 1030
    x, w, b, dy = _data(rows, cols, BF16, BF16, 21)
    eager = run_forward(m, x, w, b, BF16, BF16)
    eager += run_backward(m, dy, x, w, eager[1], eager[2], BF16, BF16)
    ins = [Dev(m, t) for t in (x, w, b, dy)]
    outs = [out(m, t.shape, t.dtype) for t in eager]
    nbytes = m.layer_norm_backward_workspace_bytes(rows, cols)
    ws = workspace(m, nbytes)

    def launch(stream):
        dx_, dw_, db_, ddy = ins
        y, mean, rstd, dx, dw, db = outs
        m.launch_layer_norm(dx_, dw_, db_, y, mean, rstd, BF16, BF16, rows, cols, EPS,
                            stream).throw_if_error()
        m.launch_layer_norm_backward(ddy, dx_, dw_, mean, rstd, dx, dw, db, BF16, BF16, rows, cols,
                                     ws, nbytes, stream).throw_if_error()

    graph = Captured(m, launch)
    try:
        for i in range(4):
            graph.replay()
            assert all(same_bits(o.get(), e) for o, e in zip(outs, eager)), i
            for o in outs:
                o.buf.upload(np.full(o.buf.nbytes, 0xA5, np.uint8))
            assert same_bits(run_forward(m, x, w, b, BF16, BF16)[0], eager[0])
    finally:
        graph.close()
    st = m.Stream()
    try:
        assert same_bits(run_forward(m, x, w, b, BF16, BF16, stream=st)[0], eager[0])
    finally:
        st.close()


def test_offsets_past_32_bits(gpu):
    """More than 2^31 elements: the last rows are their own."""
    m = gpu
    cols = 4096
    rows = (1 << 31) // cols + 3
    x, w, b, dy = _data(3, cols, BF16, BF16, 9)
    want = run_forward(m, x, w, b, BF16, BF16)
    big_x, big_y = m.DeviceBuffer(2 * rows * cols), m.DeviceBuffer(2 * rows * cols)
    import ctypes as C
    L = m.lib()
    L.mcke_fill_u32_async.argtypes = [C.c_void_p, C.c_uint32, C.c_size_t, C.c_void_p]
    for buf in (big_x, big_y):
        m._check(L.mcke_fill_u32_async(buf.ptr, 0x3F803F80, rows * cols // 2, None))
    tail = (rows - 3) * cols * 2
    raw = x.view(torch.int16).numpy()
    m._check(L.mcke_rt_memcpy_async(big_x.ptr + tail, raw.ctypes.data, raw.nbytes, 0, None))
    m.device_synchronize()
    dw, db = Dev(m, w), Dev(m, b)
    m.launch_layer_norm(big_x, dw, db, big_y, None, None, BF16, BF16, rows, cols,
                        EPS).throw_if_error()
    m.device_synchronize()
    got = np.empty((4, cols), np.int16)
    m._check(L.mcke_rt_memcpy_async(got.ctypes.data, big_y.ptr + tail - 2 * cols, got.nbytes, 1,
                                    None))
    m.device_synchronize()
    got = torch.from_numpy(got).view(torch.bfloat16)
    assert same_bits(got[0], b)                       # a constant row: the bias
    assert same_bits(got[1:], want[0])


def test_more_columns_than_a_grid_of_their_sums(gpu):
    """Past 2^27 columns the sums' fold walks them.  Quarters, a mean of a quarter and rstd of 1
    and 2: every product and sum is exact, and so is its bf16 value (at most 7 bits)."""
    m = gpu
    rows, cols = 2, (1 << 27) + 4099
    i = torch.arange(cols, dtype=torch.int32)
    x = torch.stack([(i % 7 - 3), (i % 5 - 2)]).to(torch.bfloat16) / 4
    dy = torch.stack([(i % 3 - 1), (i // 1021 % 3 - 1)]).to(torch.bfloat16)
    mean, rstd = torch.full((rows,), 0.25), torch.tensor([1.0, 2.0])
    _, dw, db = run_backward(m, dy, x, None, mean, rstd, BF16, BF16, want=(False, True, True))
    assert torch.equal(db, dy[0] + dy[1])
    del db
    assert torch.equal(dw, dy[0] * (x[0] - 0.25) + dy[1] * (x[1] - 0.25) * 2)
