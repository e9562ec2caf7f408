"""Layer norm, token log probabilities and the 16-bit product's epilogue, without a GPU:
workspace sizes, calls that launch nothing, and what is refused.  The calls pass fake device
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


# Fake, 1 MiB apart.
A, B, Cc, D, E, F, G, H, W = (0x100000 * i for i in range(1, 10))
BIG = 1 << 40


def _refused(m, st, part):
    assert st.code == m.StatusCode.kInvalidArgument, st
    assert part in st.message, st.message


def test_host_tensors_are_refused(mcke):
    """A tensor that a kernel could not read is refused before its address is taken."""
    import torch
    x = torch.zeros(4, 8)
    with pytest.raises(ValueError, match="host memory"):
        mcke.launch_layer_norm(x, None, None, x, None, None, 0, 0, 4, 8, 1e-5)
    with pytest.raises(ValueError, match="host memory"):
        mcke.launch_row_softmax_f32(x, x, 4, 8, mcke.SoftmaxVariant.kOnlineOnePass)


def test_host_tensors_that_no_kernel_reads(mcke):
    """The query of an address's vector width takes any tensor, and a launch of nothing empty
    ones."""
    import torch
    x = torch.zeros(64)
    for t in (x, x[1:], x[2:]):
        assert mcke.max_vector_width_f32(t, 64) == mcke.max_vector_width_f32(t.data_ptr(), 64)
    e = torch.empty(0, 8)
    assert mcke.launch_row_softmax_f32(e, e, 0, 8, mcke.SoftmaxVariant.kOnlineOnePass).ok()
    assert mcke.launch_layer_norm(e, None, None, e, None, None, 0, 0, 0, 8, 1e-5).ok()


# ---------------------------------------------------------------------------
# Layer norm
# ---------------------------------------------------------------------------
def _ln(m, x=A, w=B, b=Cc, y=D, mean=E, rstd=F, dt=2, pt=2, rows=4, cols=64, eps=1e-5):
    return m.launch_layer_norm(x, w, b, y, mean, rstd, dt, pt, rows, cols, eps)


def test_layer_norm_refusals(cpu_only):
    m = cpu_only
    assert _ln(m, rows=0).ok() and _ln(m, cols=0).ok()
    assert _ln(m, None, None, None, None, None, None, rows=0).ok()
    _refused(m, _ln(m, x=None), "null")
    _refused(m, _ln(m, y=None), "null")
    _refused(m, _ln(m, rows=-1), "negative")
    _refused(m, _ln(m, cols=-1), "negative")
    _refused(m, _ln(m, cols=(1 << 30) + 1), "too large")
    _refused(m, _ln(m, rows=1 << 60), "too large")
    _refused(m, _ln(m, dt=3), "dtype")
    _refused(m, _ln(m, dt=2, pt=1), "param_dtype")
    _refused(m, _ln(m, dt=0, pt=2), "param_dtype")
    for eps in (-1e-5, float("nan"), float("inf")):
        _refused(m, _ln(m, eps=eps), "eps")
    _refused(m, _ln(m, x=A + 1), "aligned")
    _refused(m, _ln(m, w=B + 2, pt=0), "aligned")
    _refused(m, _ln(m, mean=E + 2), "aligned")
    _refused(m, _ln(m, y=A), "overlaps")
    _refused(m, _ln(m, y=A + 2 * 4 * 64 - 2), "overlaps")
    _refused(m, _ln(m, y=A - 2 * 4 * 64 + 2), "overlaps")
    _refused(m, _ln(m, mean=D + 4), "overlaps")
    _refused(m, _ln(m, rstd=E + 12), "overlaps")
    _refused(m, _ln(m, rstd=B), "overlaps")


def _lnb(m, dy=A, x=B, w=Cc, mean=D, rstd=E, dx=F, dw=G, db=H, dt=2, pt=0, rows=4, cols=64, ws=W,
         nbytes=BIG):
    return m.launch_layer_norm_backward(dy, x, w, mean, rstd, dx, dw, db, dt, pt, rows, cols, ws,
                                        nbytes)


def test_layer_norm_backward_refusals(cpu_only):
    m = cpu_only
    assert _lnb(m, cols=0).ok()
    assert _lnb(m, rows=0, dw=None, db=None).ok()
    for name in ("dy", "x", "mean", "rstd"):
        _refused(m, _lnb(m, **{name: None}), "null")
    _refused(m, _lnb(m, dx=None, dw=None, db=None), "no gradient")
    _refused(m, _lnb(m, rows=-1), "negative")
    _refused(m, _lnb(m, dt=7), "dtype")
    _refused(m, _lnb(m, dt=1, pt=2), "param_dtype")
    _refused(m, _lnb(m, dx=F + 1), "aligned")
    _refused(m, _lnb(m, dw=G + 2), "aligned")
    need = m.layer_norm_backward_workspace_bytes(4, 64)
    assert need > 0
    _refused(m, _lnb(m, ws=None), str(need))
    _refused(m, _lnb(m, nbytes=need - 1), str(need))
    _refused(m, _lnb(m, ws=W + 8), "16-byte")
    _refused(m, _lnb(m, dx=A), "overlaps")
    _refused(m, _lnb(m, dx=B + 2), "overlaps")
    _refused(m, _lnb(m, dw=Cc), "overlaps")
    _refused(m, _lnb(m, db=G + 4), "overlaps")
    _refused(m, _lnb(m, ws=F), "overlaps")
    _refused(m, _lnb(m, ws=A), "overlaps")


def test_layer_norm_workspace(mcke):
    f = mcke.layer_norm_backward_workspace_bytes
    assert f(0, 64) == 0 and f(4, 0) == 0 and f(-1, 64) == 0 and f(4, -1) == 0
    for rows in (1, 5, 100, 4096, 1 << 20, 1 << 40):
        for cols in (1, 8, 1000, 4096, 65536, 1 << 20):
            n = f(rows, cols)
            assert n > 0 and n % (8 * cols) == 0 and n // (8 * cols) <= min(rows, 1024)


# ---------------------------------------------------------------------------
# Token log probabilities
# ---------------------------------------------------------------------------
def _lp(m, x=A, tok=B, lp=Cc, ent=D, lse=E, tl=F, ti=G, dt=2, rows=4, vocab=100, stride=128,
        scale=1.0, k=5, ws=W, nbytes=BIG):
    return m.launch_token_logprobs(x, tok, lp, ent, lse, tl, ti, dt, rows, vocab, stride, scale, k,
                                   ws, nbytes)


def test_token_logprobs_refusals(cpu_only):
    m = cpu_only
    assert _lp(m, rows=0).ok() and _lp(m, vocab=0, k=0).ok()
    _refused(m, _lp(m, x=None), "null")
    _refused(m, _lp(m, tok=None), "tokens")
    _refused(m, _lp(m, tl=None, ti=None), "top_k")
    _refused(m, _lp(m, lp=None, ent=None, lse=None, k=0), "no output")
    _refused(m, _lp(m, rows=-1), "negative")
    _refused(m, _lp(m, vocab=-1), "negative")
    _refused(m, _lp(m, stride=99), "row_stride")
    _refused(m, _lp(m, vocab=1 << 31, stride=1 << 31), "vocab")
    _refused(m, _lp(m, rows=1 << 60), "too large")
    _refused(m, _lp(m, rows=1 << 25), "32-bit work size")
    _refused(m, _lp(m, dt=3), "dtype")
    for scale in (0.0, -1.0, float("nan"), float("inf"), 3e38):
        _refused(m, _lp(m, scale=scale), "scale")
    for k in (-1, 65):
        _refused(m, _lp(m, k=k), "top_k")
    _refused(m, _lp(m, vocab=4, k=5), "top_k")
    _refused(m, _lp(m, x=A + 1), "aligned")
    _refused(m, _lp(m, tok=B + 4), "aligned")
    _refused(m, _lp(m, ti=G + 4), "aligned")
    _refused(m, _lp(m, lse=E + 2), "aligned")
    need = m.token_logprobs_workspace_bytes(1, 100000, 5)
    assert need > 0
    one = dict(rows=1, vocab=100000, stride=100000)
    _refused(m, _lp(m, **one, ws=None), str(need))
    _refused(m, _lp(m, **one, nbytes=need - 1), str(need))
    _refused(m, _lp(m, **one, ws=W + 8), "16-byte")
    _refused(m, _lp(m, **one, ws=A), "overlaps")
    _refused(m, _lp(m, lp=A + 2 * (3 * 128 + 100) - 4), "overlaps")
    _refused(m, _lp(m, ent=Cc + 12), "overlaps")
    _refused(m, _lp(m, lse=B), "overlaps")
    _refused(m, _lp(m, ti=F), "overlaps")


def test_token_logprobs_backward_refusals(cpu_only):
    m = cpu_only

    def f(x=A, tok=B, lse=Cc, ent=D, g=E, h=F, dx=G, dt=2, rows=4, vocab=100, stride=128, scale=1.0):
        return m.launch_token_logprobs_backward(x, tok, lse, ent, g, h, dx, dt, rows, vocab, stride,
                                                scale)

    assert f(rows=0).ok() and f(vocab=0).ok()
    for name in ("x", "lse", "dx"):
        _refused(m, f(**{name: None}), "null")
    _refused(m, f(g=None, h=None), "no gradient")
    _refused(m, f(tok=None), "tokens")
    _refused(m, f(ent=None), "entropies")
    _refused(m, f(stride=99), "row_stride")
    _refused(m, f(scale=0.0), "scale")
    _refused(m, f(dt=-1), "dtype")
    _refused(m, f(rows=1 << 25, dx=BIG), "32-bit work size")
    _refused(m, f(dx=G + 1), "aligned")
    _refused(m, f(dx=A), "overlaps")
    _refused(m, f(dx=Cc), "overlaps")


def test_token_logprobs_workspace(mcke):
    f = mcke.token_logprobs_workspace_bytes
    assert f(0, 1000, 5) == 0 and f(1, 0, 0) == 0 and f(1, 1000, 65) == 0 and f(1, 1000, -1) == 0
    assert f(4096, 131072, 20) == 0                   # enough rows to fill the GPU
    assert f(1, 100, 20) == 0                         # too few logits to share
    assert f(1, 131072, 20) > f(1, 131072, 0) > 0


# ---------------------------------------------------------------------------
# The 16-bit product's epilogue
# ---------------------------------------------------------------------------
def test_gemm_lp_bias_act_refusals(cpu_only):
    m = cpu_only
    good = m.LP_TILES[0]

    def f(a=A, b=B, bias=Cc, res=D, y=E, ab=2, yt=2, bt=0, M=8, N=8, K=8, act=3, tile=good):
        return m.launch_gemm_lp_bias_act(a, b, bias, res, y, ab, yt, bt, M, N, K, 1.0, act, tile)

    assert f(M=0).ok() and f(N=0).ok()
    for name in ("a", "b", "y"):
        _refused(m, f(**{name: None}), "null")
    for name in ("M", "N", "K"):
        _refused(m, f(**{name: -8}), "negative")
        _refused(m, f(**{name: 1 << 31}), "INT32_MAX")
    _refused(m, f(ab=0), "ab_dtype")
    _refused(m, f(ab=2, yt=1), "y_dtype")
    _refused(m, f(ab=2, bt=1), "bias_dtype")
    for act in (-1, 4):
        _refused(m, f(act=act), "Activation")
    _refused(m, f(tile=m.GemmTile(256, 256, 32, 16, 16)), "no fallback")
    _refused(m, f(y=E + 1), "aligned")
    _refused(m, f(bias=Cc + 2), "aligned")
    _refused(m, f(res=D + 2, yt=0), "aligned")
    for out in (A, B + 2, Cc - 2):
        _refused(m, f(y=out, res=None), "overlaps")
    _refused(m, f(res=E + 2), "without being it")
    _refused(m, f(M=1 << 18, N=1 << 18, K=64, res=None, bias=None, y=BIG, a=BIG >> 2, b=BIG >> 3,
                  tile=m.GemmTile(64, 64, 64, 4, 4)), "32-bit work size")


@pytest.mark.parametrize("M,N", [(1, (1 << 31) - 1), ((1 << 31) - 1, 1)])
def test_gemm_lp_bias_act_grid_at_int32_max(cpu_only, M, N):
    m = cpu_only
    _refused(m, m.launch_gemm_lp_bias_act(BIG >> 2, BIG >> 3, None, None, BIG, 2, 2, 0, M, N, 1, 1.0,
                                          3, m.LP_TILES[0]), "32-bit work size")
