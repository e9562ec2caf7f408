"""Embedding, bias + activation kept in 8 bits and the cross entropy of hidden states, without a
GPU: workspace sizes, calls that launch nothing, and what is refused.  The calls pass fake device
addresses, so they run only where no GPU is visible."""
from __future__ import annotations

import pytest


@pytest.fixture()
def cpu_only(mcke):
    try:
        gpus = mcke.device_count()
    except Exception:
        gpus = 0
    if gpus:
        pytest.skip("a GPU is visible: these calls pass fake device addresses, so they run only "
                    "where a missed rejection cannot launch a kernel on them")
    return mcke


# Fake, 16 MiB apart.
A, B, Cc, D, E, F, G, H, W = (0x1000000 * i for i in range(1, 10))
BIG = 1 << 40
NAN, INF = float("nan"), float("inf")


def _refused(m, st, part):
    assert st.code == m.StatusCode.kInvalidArgument, st
    assert part in st.message, st.message


def test_host_tensors_are_refused(mcke):
    import torch
    x, t, b = torch.zeros(4, 64), torch.zeros(4, dtype=torch.int64), torch.zeros(4, dtype=torch.uint8)
    for call in (lambda: mcke.launch_embedding(t, x, x, 0, 0, 4, 4, 64),
                 lambda: mcke.launch_embedding_backward(t, x, x, 0, 0, 4, 4, 64),
                 lambda: mcke.launch_bias_act_checkpoint8(x, None, x, b, b, 0, 0, 4, 64, 0),
                 lambda: mcke.launch_bias_act_checkpoint8_backward(x, b, b, x, None, None, 0, 0, 4, 64, 0),
                 lambda: mcke.launch_linear_cross_entropy(x, x, t, x, x, 2, 4, 4, 64),
                 lambda: mcke.launch_linear_cross_entropy_backward(x, x, t, x, x, None, x, x, 2, 4, 4,
                                                                   64)):
        with pytest.raises(ValueError, match="host memory"):
            call()


# ---------------------------------------------------------------------------
# Embedding
# ---------------------------------------------------------------------------
def _fwd(m, tok=A, table=B, out=Cc, tt=2, ot=2, rows=4, vocab=100, cols=64, scale=1.0):
    return m.launch_embedding(tok, table, out, tt, ot, rows, vocab, cols, scale)


def test_embedding_refusals(cpu_only):
    m = cpu_only
    assert _fwd(m, rows=0).ok() and _fwd(m, cols=0).ok()
    assert _fwd(m, None, None, None, rows=0).ok()
    for name in ("tok", "table", "out"):
        _refused(m, _fwd(m, **{name: None}), "null")
    for name in ("rows", "vocab", "cols"):
        _refused(m, _fwd(m, **{name: -1}), "negative")
    _refused(m, _fwd(m, rows=1 << 31), "too large")
    _refused(m, _fwd(m, vocab=(1 << 31) - 1), "too large")
    _refused(m, _fwd(m, cols=(1 << 24) + 1), "too large")
    _refused(m, _fwd(m, tt=3), "table_dtype")
    _refused(m, _fwd(m, tt=2, ot=1), "out_dtype")
    _refused(m, _fwd(m, tt=0, ot=2), "out_dtype")
    for s in (NAN, INF, -INF):
        _refused(m, _fwd(m, scale=s), "scale")
    _refused(m, _fwd(m, tok=A + 4), "aligned")
    _refused(m, _fwd(m, table=B + 1), "aligned")
    _refused(m, _fwd(m, out=Cc + 2, ot=0), "aligned")
    _refused(m, _fwd(m, out=B + 2 * 100 * 64 - 2), "overlaps")
    _refused(m, _fwd(m, out=A), "overlaps")


def _bwd(m, tok=A, dout=B, dtable=Cc, ot=2, tt=2, rows=4, vocab=100, cols=64, scale=1.0, acc=False,
         ws=W, nbytes=BIG):
    return m.launch_embedding_backward(tok, dout, dtable, ot, tt, rows, vocab, cols, scale, acc, ws,
                                       nbytes)


def test_embedding_backward_refusals(cpu_only):
    m = cpu_only
    assert _bwd(m, vocab=0).ok() and _bwd(m, cols=0).ok()
    for name in ("tok", "dout", "dtable"):
        _refused(m, _bwd(m, **{name: None}), "null")
    _refused(m, _bwd(m, rows=-1), "negative")
    _refused(m, _bwd(m, rows=1 << 31), "too large")
    _refused(m, _bwd(m, tt=7), "table_dtype")
    _refused(m, _bwd(m, tt=1, ot=2), "dout_dtype")
    _refused(m, _bwd(m, scale=NAN), "scale")
    _refused(m, _bwd(m, dtable=Cc + 1), "aligned")
    need = m.embedding_backward_workspace_bytes(4, 100, 64)
    assert need > 0
    _refused(m, _bwd(m, ws=None), str(need))
    _refused(m, _bwd(m, nbytes=need - 1), str(need))
    _refused(m, _bwd(m, ws=W + 8), "16-byte")
    _refused(m, _bwd(m, dtable=B), "overlaps")
    _refused(m, _bwd(m, dtable=A - 2), "overlaps")
    for at in (A, B, Cc + 64):
        _refused(m, _bwd(m, ws=at), "overlaps")


def test_embedding_workspace(mcke):
    f = mcke.embedding_backward_workspace_bytes
    assert f(0, 100, 64) == 0 and f(4, 0, 64) == 0 and f(4, 100, 0) == 0 and f(-1, 100, 64) == 0
    assert f(1 << 31, 100, 64) == 0 and f(4, 100, 1 << 25) == 0
    for rows in (1, 1000, 16384, 16385, 1 << 20):
        # Positions and tokens, twice where runs are merged, and sums of two rows a chunk: at most
        # 1024 of 2048 columns, or as many narrow ones.
        assert 8 * rows <= f(rows, 100, 64) <= 16 * (rows + 16) + 1024 * 2048 * 4


# ---------------------------------------------------------------------------
# Bias + activation kept in 8 bits
# ---------------------------------------------------------------------------
def _save(m, x=A, b=B, y=Cc, codes=D, ex=E, dt=2, bt=0, rows=4, cols=100, act=3):
    return m.launch_bias_act_checkpoint8(x, b, y, codes, ex, dt, bt, rows, cols, act)


def test_checkpoint8_refusals(cpu_only):
    m = cpu_only
    assert _save(m, rows=0).ok() and _save(m, cols=0).ok()
    for name in ("x", "codes", "ex"):
        _refused(m, _save(m, **{name: None}), "null")
    _refused(m, _save(m, rows=-1), "negative")
    _refused(m, _save(m, cols=-1), "negative")
    _refused(m, _save(m, rows=1 << 31), "too large")
    _refused(m, _save(m, cols=(1 << 24) + 1), "too large")
    _refused(m, _save(m, dt=3), "dtype")
    _refused(m, _save(m, dt=2, bt=1), "bias_dtype")
    for act in (-1, 4):
        _refused(m, _save(m, act=act), "Activation")
    _refused(m, _save(m, x=A + 1), "aligned")
    _refused(m, _save(m, b=B + 2), "aligned")
    _refused(m, _save(m, y=A), "overlaps")
    _refused(m, _save(m, y=None, codes=A + 799), "overlaps")
    _refused(m, _save(m, ex=D + 399), "overlaps")
    _refused(m, _save(m, ex=B + 1), "overlaps")


def _use(m, dy=A, codes=B, ex=Cc, dx=D, y=E, db=F, dt=2, bt=0, rows=4, cols=100, act=3, ws=W,
         nbytes=BIG):
    return m.launch_bias_act_checkpoint8_backward(dy, codes, ex, dx, y, db, dt, bt, rows, cols, act, ws,
                                                  nbytes)


def test_checkpoint8_backward_refusals(cpu_only):
    m = cpu_only
    assert _use(m, cols=0).ok()
    assert _use(m, None, None, None, D, E, None, rows=0).ok()
    _refused(m, _use(m, dx=None, y=None, db=None), "no output")
    _refused(m, _use(m, codes=None), "null")
    _refused(m, _use(m, ex=None), "null")
    _refused(m, _use(m, dy=None), "need dy")
    _refused(m, _use(m, dy=None, dx=None), "need dy")
    _refused(m, _use(m, dt=-1), "dtype")
    _refused(m, _use(m, bt=1), "bias_dtype")
    _refused(m, _use(m, act=9), "Activation")
    _refused(m, _use(m, dx=D + 1), "aligned")
    _refused(m, _use(m, db=F + 2), "aligned")
    need = m.bias_act_checkpoint8_backward_workspace_bytes(4, 100)
    assert need > 0
    _refused(m, _use(m, ws=None), str(need))
    _refused(m, _use(m, nbytes=need - 1), str(need))
    _refused(m, _use(m, ws=W + 4), "16-byte")
    for name in ("dx", "y", "db"):
        for at in (A, B, Cc):
            _refused(m, _use(m, **{name: at}), "overlaps")
    _refused(m, _use(m, y=D + 2), "overlaps")
    _refused(m, _use(m, ws=D), "overlaps")


def test_checkpoint8_workspace(mcke):
    f = mcke.bias_act_checkpoint8_backward_workspace_bytes
    assert f(0, 64) == 0 and f(4, 0) == 0 and f(-1, 64) == 0 and f(1 << 31, 64) == 0
    for rows in (1, 5, 4096, 1 << 20):
        for cols in (1, 2048, 16384, 1 << 20):
            n = f(rows, cols)
            assert n > 0 and n % (4 * cols) == 0 and n // (4 * cols) <= min(rows, 1024)


# ---------------------------------------------------------------------------
# Cross entropy of hidden states
# ---------------------------------------------------------------------------
def _lce(m, h=A, w=B, t=Cc, loss=D, lse=E, dt=2, rows=4, vocab=100, dim=64, scale=1.0, ws=W,
         nbytes=BIG):
    return m.launch_linear_cross_entropy(h, w, t, loss, lse, dt, rows, vocab, dim, scale, ws, nbytes)


def test_linear_cross_entropy_refusals(cpu_only):
    m = cpu_only
    assert _lce(m, rows=0).ok()
    for name in ("h", "w", "t"):
        _refused(m, _lce(m, **{name: None}), "null")
    _refused(m, _lce(m, loss=None, lse=None), "no output")
    for name in ("rows", "vocab", "dim"):
        _refused(m, _lce(m, **{name: -1}), "negative")
    for name in ("vocab", "dim"):
        _refused(m, _lce(m, **{name: 0}), "> 0")
    for name, most in (("rows", 1 << 24), ("vocab", 1 << 24), ("dim", 1 << 16)):
        _refused(m, _lce(m, **{name: most + 1}), "too large")
    _refused(m, _lce(m, rows=1 << 24, vocab=1 << 24), "32-bit work size")
    for dt in (0, 3):
        _refused(m, _lce(m, dt=dt), "dtype")
    for s in (0.0, -1.0, NAN, INF, 3e38):
        _refused(m, _lce(m, scale=s), "scale")
    _refused(m, _lce(m, h=A + 1), "aligned")
    _refused(m, _lce(m, t=Cc + 4), "aligned")
    _refused(m, _lce(m, lse=E + 2), "aligned")
    _refused(m, _lce(m, w=B + 2), "4-byte")
    need = m.linear_cross_entropy_workspace_bytes(4, 100, 64)
    _refused(m, _lce(m, ws=None), str(need))
    _refused(m, _lce(m, nbytes=need - 1), str(need))
    _refused(m, _lce(m, ws=W + 8), "16-byte")
    _refused(m, _lce(m, loss=A), "overlaps")
    _refused(m, _lce(m, lse=D + 12), "overlaps")
    _refused(m, _lce(m, ws=B), "overlaps")


def _lceb(m, h=A, w=B, t=Cc, lse=D, dl=E, dz=F, dh=G, dw=H, dt=2, rows=4, vocab=100, dim=64, scale=1.0,
          ws=W, nbytes=BIG):
    return m.launch_linear_cross_entropy_backward(h, w, t, lse, dl, dz, dh, dw, dt, rows, vocab, dim,
                                                  scale, ws, nbytes)


def test_linear_cross_entropy_backward_refusals(cpu_only):
    m = cpu_only
    assert _lceb(m, rows=0, dw=None).ok() and _lceb(m, rows=0, vocab=0).ok()
    for name in ("h", "w", "t", "lse"):
        _refused(m, _lceb(m, **{name: None}), "null")
    _refused(m, _lceb(m, dh=None, dw=None), "no gradient is asked")
    _refused(m, _lceb(m, dl=None, dz=None), "no gradient is given")
    _refused(m, _lceb(m, dim=0), "> 0")
    _refused(m, _lceb(m, dt=0), "dtype")
    _refused(m, _lceb(m, scale=0.0), "scale")
    _refused(m, _lceb(m, dh=G + 1), "aligned")
    _refused(m, _lceb(m, w=B + 2), "4-byte")
    need = m.linear_cross_entropy_backward_workspace_bytes(4, 100, 64)
    _refused(m, _lceb(m, ws=None), str(need))
    _refused(m, _lceb(m, nbytes=need - 1), str(need))
    for name in ("dh", "dw", "ws"):
        for at in (A, B, Cc, D, E, F):
            _refused(m, _lceb(m, **{name: at}), "overlaps")
    _refused(m, _lceb(m, dw=G), "overlaps")


def test_linear_cross_entropy_workspace(mcke):
    for f in (mcke.linear_cross_entropy_workspace_bytes,
              mcke.linear_cross_entropy_backward_workspace_bytes):
        assert f(0, 100, 64) == 0 and f(4, 0, 64) == 0 and f(4, 100, 0) == 0 and f(-1, 100, 64) == 0
        assert f((1 << 24) + 1, 100, 64) == 0 and f(4, 100, (1 << 16) + 1) == 0
    # A training batch: far below its logits (2 GiB in 16 bits), its copy of the rows included.
    assert mcke.linear_cross_entropy_workspace_bytes(8192, 131072, 4096) < 192 << 20
    assert mcke.linear_cross_entropy_backward_workspace_bytes(8192, 131072, 4096) < 384 << 20


def test_linear_cross_entropy_of_many_logits(cpu_only):
    """More logits than one launch has 128 x 128 tiles for are not refused (what is missing here is
    the workspace): the forward pass takes 256 x 256 ones, up to 2^23 of them, and the backward pass
    goes by pieces of the vocabulary."""
    m = cpu_only
    for dim in (64, 65, 128, 4096):
        for rows, vocab in ((1 << 19, 1 << 18), (1 << 24, (1 << 15) - 256), (1 << 15, 1 << 24)):
            rows -= 256 if rows == 1 << 15 else 0
            need = m.linear_cross_entropy_workspace_bytes(rows, vocab, dim)
            _refused(m, _lce(m, 1 << 50, 1 << 51, 1 << 52, 1 << 53, 1 << 54, rows=rows, vocab=vocab,
                             dim=dim, ws=None), str(need))
        for rows, vocab in ((1 << 19, 1 << 18), (1 << 24, 1 << 24)):
            need = m.linear_cross_entropy_backward_workspace_bytes(rows, vocab, dim)
            _refused(m, _lceb(m, 1 << 50, 1 << 51, 1 << 52, 1 << 53, 1 << 54, 1 << 55, 1 << 56, 1 << 57,
                              rows=rows, vocab=vocab, dim=dim, ws=None), str(need))
    _refused(m, _lce(m, rows=1 << 24, vocab=1 << 15, ws=None), "32-bit work size")
