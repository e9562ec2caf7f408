"""Embedding lookup and its gradient (mcke_launch_embedding, ..._backward) on the GPU against the
formulas in 64 bits.

Tolerances are counts of roundings (U is one in fp32).  Forward: the product and the output's.
Backward: a token's c rows are added up in at most c roundings, each relative to the sum of
absolute values, the product with scale and the addition to what was there take one each, and the
output its own.  With quarter multiples and a power of two for scale every sum is exact, and the
output is the exact value rounded once."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from tests.operator_util import (BF16, F16, F32, HALF, ID, TINY, TORCH, U, Captured, Dev, check,
                                 out, same_bits, workspace)

pytestmark = pytest.mark.gpu

PAIRS = [(BF16, BF16), (F16, F16), (F32, F32), (BF16, F32), (F16, F32)]     # table, out
PAIR_IDS = [f"{ID[t]}-{ID[o]}" for t, o in PAIRS]
# rows, vocab, cols: one of each, rows shorter than a 16-byte vector, odd widths, more than one
# round of lanes; more tokens than are added up without an order (512), than a run of the sort has
# (1024), and than are counted (16384: runs and three merges, four above 65536).
SHAPES = [(1, 1, 1), (3, 5, 3), (7, 2, 8), (64, 1000, 127), (5, 300, 2050), (1024, 513, 40),
          (1025, 70, 64), (4097, 1000, 9), (2000, 131072, 16), (300, 77, 4099), (20001, 4001, 24),
          (140001, 1021, 8)]


def _tokens(rows, vocab, seed, kind="text"):
    g = torch.Generator().manual_seed(seed)
    if kind == "text":          # a few tokens often, most of them rarely, some padding
        t = torch.exp(torch.rand(rows, generator=g, dtype=torch.float64) * np.log(vocab + 1)) - 1
        t = t.long().clamp(0, vocab - 1)
        t[torch.rand(rows, generator=g) < 0.1] = -100
        return t
    if kind == "one":
        return torch.full((rows,), vocab - 1)
    if kind == "none":
        return torch.full((rows,), -1)
    if kind == "outside":       # past the vocabulary, and at the ends of 64 bits
        t = torch.randint(vocab, (rows,), generator=g)
        t[::3] = vocab
        t[1::7] = torch.iinfo(torch.int64).max
        t[2::7] = torch.iinfo(torch.int64).min
        t[4::7] = (1 << 32) + 1
        return t
    return torch.arange(rows - 1, -1, -1) % vocab          # each once, descending


def _draw(shape, dt, seed, quarters=False):
    g = torch.Generator().manual_seed(seed)
    if quarters:
        return (torch.randint(-4, 5, shape, generator=g) / 4).to(TORCH[dt])
    return torch.randn(*shape, generator=g).to(TORCH[dt])


def run_forward(m, tokens, table, tt, ot, scale, shift=0, stream=None):
    rows, (vocab, cols) = len(tokens), table.shape
    o = out(m, (rows, cols), TORCH[ot], shift)
    m.launch_embedding(Dev(m, tokens), Dev(m, table, shift), o, tt, ot, rows, vocab, cols, scale,
                       stream).throw_if_error()
    m.device_synchronize()
    return o.get()


def run_backward(m, tokens, dout, vocab, tt, ot, scale, old=None, shift=0, stream=None):
    rows, cols = dout.shape
    d = Dev(m, old, shift) if old is not None else out(m, (vocab, cols), TORCH[tt], shift)
    n = m.embedding_backward_workspace_bytes(rows, vocab, cols)
    ws = workspace(m, n)
    m.launch_embedding_backward(Dev(m, tokens), Dev(m, dout, shift), d, ot, tt, rows, vocab, cols,
                                scale, old is not None, ws, n, stream).throw_if_error()
    m.device_synchronize()
    if ws is not None:
        ws.get()
    return d.get()


def forward_reference(tokens, table, ot, scale):
    vocab = table.shape[0]
    s = float(np.float32(scale))
    there = (tokens >= 0) & (tokens < vocab)
    want = table.double()[torch.where(there, tokens, 0)] * s
    want = torch.where(there[:, None], want, torch.where(tokens < 0, 0.0, torch.nan)[:, None])
    t = U * want.abs()
    return want, t + HALF[ot] * (want.abs() + t) + TINY[ot]


def backward_reference(tokens, dout, vocab, tt, scale, old=None):
    s = float(np.float32(scale))
    there = (tokens >= 0) & (tokens < vocab)
    t, d = tokens[there], dout.double()[there]
    sums, size = (torch.zeros(vocab, dout.shape[1], dtype=torch.float64).index_add_(0, t, v)
                  for v in (d, d.abs()))
    count = torch.bincount(t, minlength=vocab)[:, None]
    want, tol = s * sums, (count + 1) * U * abs(s) * size
    if old is not None:
        want = want + old.double()
        tol = tol + U * (want.abs() + tol)
    return want, tol + HALF[tt] * (want.abs() + tol) + TINY[tt]


@pytest.mark.parametrize("tt,ot", PAIRS, ids=PAIR_IDS)
@pytest.mark.parametrize("i,shape", enumerate(SHAPES), ids=[str(s) for s in SHAPES])
def test_forward(gpu, i, shape, tt, ot):
    rows, vocab, cols = shape
    tokens = _tokens(rows, vocab, i, ("text", "outside")[i % 2])
    table = _draw((vocab, cols), tt, i)
    got = run_forward(gpu, tokens, table, tt, ot, cols**0.5, shift=i % 3)
    check("out", got, *forward_reference(tokens, table, ot, cols**0.5))


@pytest.mark.parametrize("tt,ot", PAIRS, ids=PAIR_IDS)
@pytest.mark.parametrize("i,shape", enumerate(SHAPES), ids=[str(s) for s in SHAPES])
def test_backward(gpu, i, shape, tt, ot):
    rows, vocab, cols = shape
    tokens = _tokens(rows, vocab, i, ("text", "text", "outside")[i % 3])
    dout = _draw((rows, cols), ot, i)
    scale = 0.375 * cols**0.5
    got = run_backward(gpu, tokens, dout, vocab, tt, ot, scale, shift=i % 2)
    check("dtable", got, *backward_reference(tokens, dout, vocab, tt, scale))
    old = _draw((vocab, cols), tt, 100 + i)
    got = run_backward(gpu, tokens, dout, vocab, tt, ot, scale, old=old, shift=i % 2)
    check("added", got, *backward_reference(tokens, dout, vocab, tt, scale, old))
    # Rows whose token is not there are left as they were, to the bit.
    absent = torch.ones(vocab, dtype=torch.bool)
    absent[tokens[(tokens >= 0) & (tokens < vocab)]] = False
    assert same_bits(got[absent], old[absent])


@pytest.mark.parametrize("kind", ["one", "none", "outside", "each"])
@pytest.mark.parametrize("rows", [1, 5, 700, 1024, 5000, 16384, 16385, 132000])
def test_backward_exact(gpu, rows, kind):
    """Quarters: exact sums.  All tokens equal (a sum that crosses every chunk), none there, each
    once."""
    for vocab in (3, 40000) if rows < 10000 else (37,):
        cols = 12
        tokens = _tokens(rows, vocab, rows, kind)
        dout = _draw((rows, cols), F32, rows, quarters=True)
        got = run_backward(gpu, tokens, dout, vocab, F32, F32, 2.0)
        want, _ = backward_reference(tokens, dout, vocab, F32, 2.0)
        assert torch.equal(got.double(), want), (vocab, kind)


@pytest.mark.parametrize("tt,ot", [(BF16, BF16), (F16, F32), (F32, F32)], ids=["bf16", "f16-f32", "f32"])
@pytest.mark.parametrize("kind", ["text", "one"])
@pytest.mark.parametrize("rows,vocab,cols", [(512, 40, 64), (511, 600, 513), (513, 40, 64), (512, 5, 1030),
                                             (300, 9, 4096), (200, 100, 8200), (65, 3, 2049)])
def test_few_tokens(gpu, rows, vocab, cols, kind, tt, ot):
    """Around the most tokens and columns whose sums each take one workgroup's way, most of them of
    many rows."""
    tokens = _tokens(rows, vocab, rows, kind)
    dout = _draw((rows, cols), ot, rows)
    old = _draw((vocab, cols), tt, 7)
    for o in (None, old):
        got = run_backward(gpu, tokens, dout, vocab, tt, ot, 1.5, old=o)
        check("dtable", got, *backward_reference(tokens, dout, vocab, tt, 1.5, o))
        assert same_bits(got, run_backward(gpu, tokens, dout, vocab, tt, ot, 1.5, old=o))


def test_no_rows(gpu):
    """A table of zeros; with accumulate, the table as it was."""
    old = _draw((5, 9), BF16, 1)
    empty, none = torch.empty(0, 9, dtype=torch.bfloat16), torch.empty(0, dtype=torch.int64)
    assert not run_backward(gpu, none, empty, 5, BF16, BF16, 1.0).any()
    assert same_bits(run_backward(gpu, none, empty, 5, BF16, BF16, 1.0, old=old), old)


def test_masked_rows_are_not_read(gpu):
    """NaN and infinities in rows of dout whose token is padding."""
    tokens = _tokens(3000, 50, 3)
    dout = _draw((3000, 33), F16, 3)
    want = run_backward(gpu, tokens, dout, 50, F16, F16, 1.0)
    dout[tokens < 0] = torch.nan
    assert same_bits(run_backward(gpu, tokens, dout, 50, F16, F16, 1.0), want)


def test_gradient_against_differences(gpu):
    """<dout, out(table + h v) - out(table - h v)> / 2 h = <dtable, v>, out linear in the table: in
    fp32 each side is off by its roundings alone."""
    rows, vocab, cols, scale = 400, 90, 70, 3.0
    tokens, table = _tokens(rows, vocab, 5), _draw((vocab, cols), F32, 5)
    v, dout = _draw((vocab, cols), F32, 6), _draw((rows, cols), F32, 7)
    up = run_forward(gpu, tokens, table + v, F32, F32, scale).double()
    down = run_forward(gpu, tokens, table - v, F32, F32, scale).double()
    slope = (dout.double() * (up - down)).sum() / 2
    want, tol = backward_reference(tokens, dout, vocab, F32, scale)
    got = run_backward(gpu, tokens, dout, vocab, F32, F32, scale).double()
    # table +- v are rounded once and multiplied once.
    size = (dout.double().abs() * (up.abs() + down.abs())).sum()
    assert abs(slope - (got * v).sum()) <= 2 * U * size + (tol * v.abs()).sum()


@pytest.mark.parametrize("rows", [5003, 300])
def test_same_bits_capture_and_streams(gpu, rows):
    m = gpu
    vocab, cols = 2000, 250
    tokens, dout = _tokens(rows, vocab, 11), _draw((rows, cols), BF16, 11)
    table = _draw((vocab, cols), BF16, 12)
    fwd = run_forward(m, tokens, table, BF16, BF16, 2.0)
    bwd = run_backward(m, tokens, dout, vocab, BF16, BF16, 2.0)
    dt, dd, dtab = Dev(m, tokens), Dev(m, dout), Dev(m, table)
    o, d = out(m, (rows, cols), torch.bfloat16), out(m, (vocab, cols), torch.bfloat16)
    n = m.embedding_backward_workspace_bytes(rows, vocab, cols)
    ws = workspace(m, n)

    def launch(stream):
        m.launch_embedding(dt, dtab, o, BF16, BF16, rows, vocab, cols, 2.0, stream).throw_if_error()
        m.launch_embedding_backward(dt, dd, d, BF16, BF16, rows, vocab, cols, 2.0, False, ws, n,
                                    stream).throw_if_error()

    graph = Captured(m, launch)
    try:
        for _ in range(3):
            graph.replay()
            assert same_bits(o.get(), fwd) and same_bits(d.get(), bwd)
            d.buf.upload(np.full(d.buf.nbytes, 0xA5, np.uint8))
            assert same_bits(run_backward(m, tokens, dout, vocab, BF16, BF16, 2.0), bwd)
    finally:
        graph.close()
    st = m.Stream()
    try:
        assert same_bits(run_forward(m, tokens, table, BF16, BF16, 2.0, stream=st), fwd)
        assert same_bits(run_backward(m, tokens, dout, vocab, BF16, BF16, 2.0, stream=st), bwd)
    finally:
        st.close()


def test_offsets_past_32_bits(gpu):
    """A table of more than 2^31 values: its last rows are read and written where they are."""
    m = gpu
    import ctypes as C
    cols = 8192
    vocab = (1 << 31) // cols + 5
    L = m.lib()
    L.mcke_fill_u32_async.argtypes = [C.c_void_p, C.c_uint32, C.c_size_t, C.c_void_p]
    big = m.DeviceBuffer(2 * vocab * cols)
    m._check(L.mcke_fill_u32_async(big.ptr, 0x3F803F80, vocab * cols // 2, None))
    last = _draw((3, cols), BF16, 4)
    raw = last.view(torch.int16).numpy()
    at = (vocab - 3) * cols * 2
    m._check(L.mcke_rt_memcpy_async(big.ptr + at, raw.ctypes.data, raw.nbytes, 0, None))
    m.device_synchronize()
    tokens = torch.tensor([vocab - 1, 0, vocab - 3, vocab - 2, vocab - 1, -1])
    o = out(m, (6, cols), torch.bfloat16)
    m.launch_embedding(Dev(m, tokens), big, o, BF16, BF16, 6, vocab, cols, 1.0).throw_if_error()
    m.device_synchronize()
    got = o.get()
    one, zero = torch.ones(cols, dtype=torch.bfloat16), torch.zeros(cols, dtype=torch.bfloat16)
    for g, w in zip(got, (last[2], one, last[0], last[1], last[2], zero)):
        assert same_bits(g, w)
    dout = _draw((6, cols), BF16, 5, quarters=True)
    for padding in (0, 600):             # few tokens, and more of them in order
        rows = 6 + padding
        t = torch.cat([tokens, torch.full((padding,), -1)])
        d = torch.cat([dout, torch.full((padding, cols), torch.nan, dtype=torch.bfloat16)])
        m._check(L.mcke_fill_u32_async(big.ptr, 0x3F803F80, vocab * cols // 2, None))
        n = m.embedding_backward_workspace_bytes(rows, vocab, cols)
        m.launch_embedding_backward(Dev(m, t), Dev(m, d), big, BF16, BF16, rows, vocab, cols, 1.0,
                                    False, workspace(m, n), n).throw_if_error()
        m.device_synchronize()
        tail = np.empty((4, cols), np.int16)
        m._check(L.mcke_rt_memcpy_async(tail.ctypes.data, big.ptr + at - 2 * cols, tail.nbytes, 1,
                                        None))
        m.device_synchronize()
        tail = torch.from_numpy(tail).view(torch.bfloat16)
        for g, w in zip(tail, (zero, dout[2], dout[3], dout[0] + dout[4])):
            assert same_bits(g, w)


@pytest.mark.parametrize("tt,ot", [(BF16, BF16), (F16, F32), (F32, F32)], ids=["bf16", "f16-f32", "f32"])
@pytest.mark.parametrize("rows,vocab,cols", [(700, 300, 509), (1500, 97, 1003), (9000, 700, 264),
                                             (16500, 3000, 512), (20001, 500, 517), (140001, 1021, 260)])
def test_wide_rows_of_many_tokens(gpu, rows, vocab, cols, tt, ot):
    """Rows of whole waves whose tokens are put in order: cut and whole vectors, tokens counted and
    merged, chunks of 4, 8, 16 and 128 positions (more than one round of loads in flight, and more
    than a wave's 64)."""
    tokens = _tokens(rows, vocab, rows)
    dout = _draw((rows, cols), ot, rows)
    old = _draw((vocab, cols), tt, 7)
    for o in (None, old):
        got = run_backward(gpu, tokens, dout, vocab, tt, ot, 1.5, old=o)
        check("dtable", got, *backward_reference(tokens, dout, vocab, tt, 1.5, o))


@pytest.mark.parametrize("kind", ["text", "one", "outside"])
@pytest.mark.parametrize("rows,cols", [(700, 509), (16500, 512), (20001, 517), (140001, 260)])
def test_wide_rows_exact(gpu, rows, cols, kind):
    """Quarters: exact sums, a token that crosses every chunk among them."""
    vocab = 37
    tokens = _tokens(rows, vocab, rows, kind)
    dout = _draw((rows, cols), BF16, rows, quarters=True)
    got = run_backward(gpu, tokens, dout.float(), vocab, F32, F32, 2.0)
    want, _ = backward_reference(tokens, dout, vocab, F32, 2.0)
    assert torch.equal(got.double(), want)
    got = run_backward(gpu, tokens, dout, vocab, BF16, BF16, 2.0)
    assert same_bits(got, want.to(torch.bfloat16))
