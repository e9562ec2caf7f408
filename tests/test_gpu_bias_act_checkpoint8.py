"""Bias + activation whose input is kept in 8 bits, and its backward pass
(mcke_launch_bias_act_checkpoint8, ..._backward) on the GPU against the formulas in 64 bits.

What is saved is exact: u = fl32(x + bias), a power of two and a rounding to e4m3 have one right
answer each, so codes and exponents are compared as what they stand for, with no tolerance.

Tolerances are counts of roundings (U is one in fp32), as the hardware's exp2 and reciprocal
are off by at most one unit in the last place (2 U):
  y      the activations' documented bound, 1e-6 + 1e-6 |u| (tests of the products use it too),
         u's own rounding with a slope below 1.2, the output's rounding
  slope  GELU_tanh, with A = 2 |z|, q = (1 + tanh z) / 2 and w = 2 v z': the exponent is off by 4 U
         of itself, so e = exp(-2 z) by 4 U A + 2 U, q by 3 U + (1 - q)(4 U A + 2 U), e q^2 by
         20 U + 12 U A at most, w by 4 U, and the sum by U.  Below v = -10 the argument is held
         there, where q is 2^-126, w is -229 and the slope -228 2^-126; the right one lies
         between that and 0, less than 256 2^-126 from it
         GELU_erf: Phi is half an erfc whose approximation is off by 1.5e-7 and its dozen
         operations, of terms below 1, by 12 U; v phi by (1.5 v^2 + 6) U of itself; U for the sum
  dx     |dy| times the slope's, one product, the output's rounding
  dbias  sum |dy| times the slope's; a chain of additions of at most D = rows / 8 + 100 (a part's
         rows, its row groups, the fold of the parts), each U of sum |dx|; the output's
         rounding
"""
from __future__ import annotations

import math

import numpy as np
import pytest
import torch

from tests.operator_util import (BF16, DTYPES, F16, F32, HALF, ID, TINY, TORCH, U, Captured, Dev,
                                 check, out, same_bits, workspace)

pytestmark = pytest.mark.gpu

NONE, RELU, ERF, TANH = range(4)
# One element, cut vectors and blocks, whole ones, odd widths, several rounds of lanes and of
# rows.
SHAPES = [(1, 1), (3, 7), (2, 8), (5, 31), (4, 32), (9, 33), (33, 64), (257, 40), (70, 255),
          (1031, 129), (3, 2048), (517, 1021), (6, 4104), (2, 16391), (5003, 96), (2, 140001)]


def _draw(rows, cols, dt, bt, seed, sigma=1.5):
    g = torch.Generator().manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, generator=g, dtype=torch.float64)

    x = (normal(rows, cols) * sigma * torch.exp(normal(1, cols))).to(TORCH[dt])
    return x, (0.3 * normal(cols)).to(TORCH[bt]), (0.1 * normal(rows, cols)).to(TORCH[dt])


def blocks(cols):
    return (cols + 31) // 32


def saved(u):
    """(restored values, exponent bytes) of fp32 u, by the definition in 64 bits."""
    rows, cols = u.shape
    n = blocks(cols)
    b = torch.zeros(rows, n * 32, dtype=torch.float64)
    b[:, :cols] = u.double()
    b = b.view(rows, n, 32)
    size = torch.where(b.isfinite(), b.abs(), 0.0).amax(2, keepdim=True)
    e = torch.full_like(size, -126.0)
    big = size > 448.0 * 2.0**-126
    # The smallest E with size <= 448 2^E, from a logarithm that may be one off.
    guess = torch.ceil(torch.log2(torch.where(big, size, 448.0) / 448.0))
    for k in (1.0, 0.0, -1.0):
        fits = size <= 448.0 * torch.exp2(guess + k)
        e = torch.where(big & fits, guess + k, e)
    v = b * torch.exp2(-e)
    step = torch.exp2((torch.frexp(v)[1] - 1).clamp(min=-6).double() - 3)
    v = torch.where(b.isfinite(), torch.round(v / step) * step * torch.exp2(e), torch.nan)
    return v.reshape(rows, -1)[:, :cols], (e[:, :, 0] + 127).to(torch.uint8)


def restored(codes, exponents):
    """What codes and exponents stand for."""
    v = codes.view(torch.float8_e4m3fn).double()
    e = torch.exp2(exponents.double() - 127)
    return v * e.repeat_interleave(32, dim=1)[:, :codes.shape[1]]


def act_of(v, act):
    if act == RELU:
        return torch.where(v > 0, v, 0.0)
    if act == ERF:
        return 0.5 * v * torch.special.erfc(-v / math.sqrt(2))
    if act == TANH:
        return v * torch.sigmoid(math.sqrt(8 / math.pi) * (v + 0.044715 * v**3))
    return v


def slope_of(v, act):
    """(slope, its tolerance)."""
    if act == NONE:
        return torch.where(v.isnan(), v, 1.0), torch.zeros_like(v)
    if act == RELU:
        return (v > 0).double(), torch.zeros_like(v)
    if act == ERF:
        cdf = 0.5 * torch.special.erfc(-v / math.sqrt(2))
        w = v * torch.exp(-v * v / 2) / math.sqrt(2 * math.pi)
        s = cdf + w
        return s, (1.5e-7 + 12 * U) / 2 + U + (1.5 * v * v + 6) * U * w.abs() + U * s.abs()
    b = math.sqrt(8 / math.pi)
    z2 = b * (v + 0.044715 * v**3)
    q, p = torch.sigmoid(z2), torch.sigmoid(-z2)
    w = v * b * (1 + 0.134145 * v * v)
    s = q + w * q * p
    return s, U * (q * (3 + p * (4 * z2.abs() + 2)) + w.abs() * q * p * (24 + 12 * z2.abs())
                   + s.abs()) + 256 * 2.0**-126


def y_reference(u, act, dt):
    y = act_of(u, act)
    t = 1.2 * U * u.abs() + (1e-6 + 1e-6 * u.abs() if act >= ERF else 0)
    return y, t + HALF[dt] * (y.abs() + t) + TINY[dt]


def backward_reference(u, dy, act, dt, bt):
    """((dx, y, dbias), tolerances) from the restored values u."""
    dy = dy.double()
    s, ts = slope_of(u, act)
    dx = dy * s
    tx = dy.abs() * ts + U * dx.abs()
    D = u.shape[0] / 8 + 100
    db = dx.sum(0)
    tb = tx.sum(0) + D * U * dx.abs().sum(0)
    y, ty = y_reference(u, act, dt)
    return ((dx, y, db), (tx + HALF[dt] * (dx.abs() + tx) + TINY[dt], ty,
                          tb + HALF[bt] * (db.abs() + tb) + TINY[bt]))


def run_forward(m, x, bias, dt, bt, act, shift=0, want_y=True, stream=None):
    rows, cols = x.shape
    y = out(m, (rows, cols), TORCH[dt], shift) if want_y else None
    codes, ex = (out(m, s, torch.uint8, shift) for s in ((rows, cols), (rows, blocks(cols))))
    m.launch_bias_act_checkpoint8(Dev(m, x, shift), Dev(m, bias, shift) if bias is not None else None,
                                  y, codes, ex, dt, bt, rows, cols, act, stream).throw_if_error()
    m.device_synchronize()
    return (y.get() if want_y else None), codes.get(), ex.get()


def run_backward(m, dy, codes, ex, dt, bt, act, shift=0, want=(True, True, True), stream=None):
    rows, cols = codes.shape
    outs = [out(m, s, TORCH[t], shift) if k else None
            for s, t, k in zip(((rows, cols), (rows, cols), (cols,)), (dt, dt, bt), want)]
    n = m.bias_act_checkpoint8_backward_workspace_bytes(rows, cols) if want[2] else 0
    ws = workspace(m, n)
    m.launch_bias_act_checkpoint8_backward(
        Dev(m, dy, shift) if dy is not None else None, Dev(m, codes, shift), Dev(m, ex, shift),
        *outs, dt, bt, rows, cols, act, ws, n, stream).throw_if_error()
    m.device_synchronize()
    if ws is not None:
        ws.get()
    return [o.get() if o is not None else None for o in outs]


@pytest.mark.parametrize("dt", DTYPES, ids=[ID[t] for t in DTYPES])
@pytest.mark.parametrize("i,shape", enumerate(SHAPES), ids=[f"{r}x{c}" for r, c in SHAPES])
def test_forward_and_backward(gpu, i, shape, dt):
    bt = (dt, F32)[i % 2]
    for act in range(4):
        x, bias, dy = _draw(*shape, dt, bt, 10 * i + act)
        u = x.float() + bias.float()
        y, codes, ex = run_forward(gpu, x, bias, dt, bt, act, shift=i % 4)
        v, e = saved(u)
        assert torch.equal(ex, e), act
        assert torch.equal(restored(codes, ex), v), act
        check("y", y, *y_reference(x.double() + bias.double(), act, dt))
        got = run_backward(gpu, dy, codes, ex, dt, bt, act, shift=i % 3)
        for name, g, w, t in zip(("dx", "y again", "dbias"), got,
                                 *backward_reference(v, dy, act, dt, bt)):
            check(name, g, w, t)


def test_every_code(gpu):
    """Each e4m3 value in a block whose largest is 448, at powers of two over fp32's range; the
    values half way between two of them, and next to those."""
    codes = torch.arange(127, dtype=torch.uint8).view(torch.float8_e4m3fn).float()
    mid = (codes[1:] + codes[:-1]) / 2
    near = torch.cat((mid, torch.nextafter(mid, mid + 1), torch.nextafter(mid, mid - 1)))
    values = torch.cat((codes, -codes, near, -near))
    values = torch.cat((values, values.new_zeros(-len(values) % 31))).view(-1, 31)
    block = torch.cat((values, torch.full((len(values), 1), 448.0)), dim=1)
    for e in (-126, -125, -60, 0, 1, 60, 118):
        x = torch.ldexp(block, torch.tensor(e))
        got = run_forward(gpu, x, None, F32, F32, NONE, want_y=False)
        v, ex = saved(x)
        assert torch.equal(got[2], ex) and torch.equal(restored(got[1], got[2]), v), e


def test_every_bf16_value(gpu):
    """All 2^16 patterns, each in blocks of its own and next to others: subnormal and largest
    values, zeros, infinities and NaN."""
    bits = torch.arange(1 << 16, dtype=torch.int32).to(torch.int16)
    x = bits.view(torch.bfloat16)
    alone = torch.zeros(1 << 16, 32, dtype=torch.bfloat16)
    alone[torch.arange(1 << 16), torch.arange(1 << 16) % 32] = x
    for t in (alone, x.view(-1, 64), x[torch.randperm(1 << 16, generator=torch.Generator()
                                                      .manual_seed(1))].view(-1, 64)):
        _, codes, ex = run_forward(gpu, t.contiguous(), None, BF16, BF16, NONE, want_y=False)
        v, e = saved(t.float())
        r = restored(codes, ex)
        assert torch.equal(ex, e)
        assert torch.equal(r.isnan(), v.isnan()) and torch.equal(r.nan_to_num(), v.nan_to_num())


@pytest.mark.parametrize("act", range(4))
def test_infinities_and_nan(gpu, act):
    """They are lost as NaN, in their places alone: the block's other values keep their scale."""
    x, bias, dy = _draw(6, 100, F32, F32, act)
    bad = torch.zeros(6, 100, dtype=torch.bool)
    for r, c, v in ((0, 3, math.inf), (1, 40, -math.inf), (2, 99, math.nan), (3, 31, math.inf)):
        x[r, c], bad[r, c] = v, True
    x[4, :] = math.nan
    bad[4, :] = True
    _, codes, ex = run_forward(gpu, x, bias, F32, F32, act)
    v, e = saved(x + bias)
    assert torch.equal(ex, e)
    r = restored(codes, ex)
    assert torch.equal(r.isnan(), bad) and torch.equal(r[~bad], v[~bad])
    dx, y, _ = run_backward(gpu, dy, codes, ex, F32, F32, act)
    (wx, wy, _), (tx, ty, _) = backward_reference(v, dy, act, F32, F32)
    assert torch.equal(dx.isnan(), wx.isnan()) and torch.equal(y.isnan(), wy.isnan())
    check("dx", dx[~bad], wx[~bad], tx[~bad])
    check("y", y[~bad], wy[~bad], ty[~bad])


@pytest.mark.parametrize("act", [ERF, TANH])
def test_slopes_over_the_range(gpu, act):
    """Codes whose values go from 0 to 2^127 either way: slopes of 0 and 1 at the ends, no NaN."""
    ex = torch.arange(1, 248, dtype=torch.uint8)[:, None].repeat(1, 8)
    code = torch.arange(256, dtype=torch.int32).to(torch.uint8)[None].repeat(247, 1)
    code[:, 127], code[:, 255] = 0, 0
    dy = torch.ones(247, 256)
    dx, y, _ = run_backward(gpu, dy, code, ex, F32, F32, act, want=(True, True, False))
    u = restored(code, ex)
    s, t = slope_of(u, act)
    s = torch.where(u > 20, 1.0, torch.where(u < -20, 0.0, s))
    t = torch.where(u.abs() > 20, 2 * U, t)
    check("dx", dx, s, t + 2 * U * s.abs() + TINY[F32])
    assert (y[u > 20] == u[u > 20].float()).all()


def test_outputs_apart(gpu):
    """Each output alone has the bits of all together; what is not asked for is not needed."""
    x, bias, dy = _draw(300, 217, BF16, F32, 1)
    _, codes, ex = run_forward(gpu, x, bias, BF16, F32, TANH)
    none = run_forward(gpu, x, bias, BF16, F32, TANH, want_y=False)
    assert same_bits(none[1], codes) and same_bits(none[2], ex)
    both = run_backward(gpu, dy, codes, ex, BF16, F32, TANH)
    for k in range(3):
        want = tuple(i == k for i in range(3))
        got = run_backward(gpu, None if k == 1 else dy, codes, ex, BF16, F32, TANH, want=want)
        assert same_bits(got[k], both[k]), k
    plain = run_backward(gpu, None, codes, ex, BF16, F32, NONE, want=(False, True, False))[1]
    assert torch.equal(plain.double(), restored(codes, ex).to(torch.bfloat16).double())


def test_gradient_against_differences(gpu):
    """The slope that dx has is the difference quotient of y = act(u) around the restored u.

    Central differences in 64 bits of the formula are off by h^2 / 6 times its third derivative
    (below 2 for both GELUs): with h = 1e-3, 4e-7 of dy."""
    x, bias, dy = _draw(40, 130, F32, F32, 3)
    for act in (ERF, TANH):
        _, codes, ex = run_forward(gpu, x, bias, F32, F32, act)
        u = restored(codes, ex)
        h = 1e-3
        slope = (act_of(u + h, act) - act_of(u - h, act)) / (2 * h)
        dx = run_backward(gpu, dy, codes, ex, F32, F32, act, want=(True, False, False))[0]
        tol = dy.double().abs() * (4e-7 + slope_of(u, act)[1] + 3 * U)
        check("dx", dx, dy.double() * slope, tol)


def test_no_rows_and_no_bias(gpu):
    m = gpu
    db = out(m, (9,), torch.float32)
    m.launch_bias_act_checkpoint8_backward(None, None, None, None, None, db, BF16, F32, 0, 9,
                                           TANH).throw_if_error()
    m.device_synchronize()
    assert not db.get().any()
    x, _, _ = _draw(5, 77, F16, F16, 2)
    y, codes, ex = run_forward(m, x, None, F16, F16, ERF)
    check("y", y, *y_reference(x.double(), ERF, F16))
    assert torch.equal(restored(codes, ex), saved(x.float())[0])


def test_same_bits_capture_and_streams(gpu):
    m = gpu
    rows, cols = 3001, 290
    x, bias, dy = _draw(rows, cols, BF16, BF16, 4)
    fwd = run_forward(m, x, bias, BF16, BF16, TANH)
    bwd = run_backward(m, dy, fwd[1], fwd[2], BF16, BF16, TANH)
    ins = [Dev(m, t) for t in (x, bias, dy)]
    f = [out(m, t.shape, t.dtype) for t in fwd]
    b = [out(m, t.shape, t.dtype) for t in bwd]
    n = m.bias_act_checkpoint8_backward_workspace_bytes(rows, cols)
    ws = workspace(m, n)

    def launch(stream):
        m.launch_bias_act_checkpoint8(ins[0], ins[1], *f, BF16, BF16, rows, cols, TANH,
                                      stream).throw_if_error()
        m.launch_bias_act_checkpoint8_backward(ins[2], f[1], f[2], *b, BF16, BF16, rows, cols, TANH,
                                               ws, n, stream).throw_if_error()

    graph = Captured(m, launch)
    try:
        for _ in range(3):
            graph.replay()
            assert all(same_bits(o.get(), w) for o, w in zip(f + b, list(fwd) + bwd))
            for o in f + b:
                o.buf.upload(np.full(o.buf.nbytes, 0xA5, np.uint8))
            assert same_bits(run_backward(m, dy, fwd[1], fwd[2], BF16, BF16, TANH)[2], bwd[2])
    finally:
        graph.close()
    st = m.Stream()
    try:
        assert all(same_bits(a, w) for a, w in
                   zip(run_forward(m, x, bias, BF16, BF16, TANH, stream=st), fwd))
        assert all(same_bits(a, w) for a, w in
                   zip(run_backward(m, dy, fwd[1], fwd[2], BF16, BF16, TANH, stream=st), bwd))
    finally:
        st.close()


def test_offsets_past_32_bits(gpu):
    """More than 2^31 values: the last row is its own."""
    m = gpu
    cols = 16384
    rows = (1 << 31) // cols + 2
    import ctypes as C
    L = m.lib()
    L.mcke_fill_u32_async.argtypes = [C.c_void_p, C.c_uint32, C.c_size_t, C.c_void_p]
    big, codes = m.DeviceBuffer(2 * rows * cols), m.DeviceBuffer(rows * cols)
    ex, back = m.DeviceBuffer(rows * cols // 32), m.DeviceBuffer(2 * rows * cols)
    m._check(L.mcke_fill_u32_async(big.ptr, 0x3F803F80, rows * cols // 2, None))
    last, _, _ = _draw(1, cols, BF16, BF16, 5)
    raw = last.view(torch.int16).numpy()
    at = (rows - 1) * cols
    m._check(L.mcke_rt_memcpy_async(big.ptr + 2 * at, raw.ctypes.data, raw.nbytes, 0, None))
    m.device_synchronize()
    m.launch_bias_act_checkpoint8(big, None, None, codes, ex, BF16, BF16, rows, cols,
                                  NONE).throw_if_error()
    m.launch_bias_act_checkpoint8_backward(None, codes, ex, None, back, None, BF16, BF16, rows, cols,
                                           NONE).throw_if_error()
    m.device_synchronize()
    got = np.empty((2, cols), np.int16)
    m._check(L.mcke_rt_memcpy_async(got.ctypes.data, back.ptr + 2 * (at - cols), got.nbytes, 1, None))
    m.device_synchronize()
    got = torch.from_numpy(got).view(torch.bfloat16)
    assert (got[0] == 1).all()
    assert torch.equal(got[1].double(), saved(last.float())[0][0])


@pytest.mark.parametrize("dt", DTYPES, ids=[ID[t] for t in DTYPES])
@pytest.mark.parametrize("act", [ERF, TANH])
def test_activation_is_zero_far_below(gpu, act, dt):
    """y = act(u) once more, of every code whose value is below -20, down to -2^128 (what a u from
    -248 2^120 on is rounded to): both GELUs are within 20 e^-200 of 0 there.  GELU_tanh's argument
    is held at -10, where q is below 2^-125 and y below 10 times that; the erfc's exponential is 0.
    (The forward pass gives -0 for all that are finite.)"""
    ex = torch.arange(1, 248, dtype=torch.uint8)[:, None].repeat(1, 8)
    code = torch.arange(256, dtype=torch.int32).to(torch.uint8)[None].repeat(247, 1)
    code[:, 127], code[:, 255] = 0, 0
    low = restored(code, ex) < -20
    assert low.any(dim=1).sum() > 100
    y = run_backward(gpu, None, code, ex, dt, dt, act, want=(False, True, False))[1]
    assert (y[low].double().abs() <= 10 * 2.0**-125).all()
    if dt != F16:                         # (their values are past fp16's)
        u = restored(code, ex).to(TORCH[dt])
        forward = run_forward(gpu, u, None, dt, dt, act)[0]
        assert not forward[low & u.isfinite()].any()
