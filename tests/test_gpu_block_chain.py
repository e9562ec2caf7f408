"""A transformer block's MLP and scoring head as a program chains them, without a wait between
the launches: layer norm, the up product with GELU, the down product onto the residual
stream, layer norm, the logits' product, log probabilities; then back through the
log probabilities and the last norm.  Each stage is checked against its formula in 64 bits from
the values that the stage before it gave, and a capture of the whole chain replays to its bits."""
from __future__ import annotations

import pytest
import torch

from tests import test_gpu_gemm_lp_epilogue as gemm
from tests import test_gpu_layer_norm as norm
from tests import test_gpu_token_logprobs as lps
from tests.operator_util import (BF16, F32, TORCH, Captured, Dev, check, out, same_bits, workspace)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("tokens,d,ff,vocab", [(1, 256, 1024, 5003), (37, 128, 512, 1000),
                                               (600, 512, 2048, 8200)])
def test_block_and_head(gpu, tokens, d, ff, vocab):
    m = gpu
    g = torch.Generator().manual_seed(tokens)

    def draw(*shape, scale=1.0, mean=0.0, dt=BF16):
        return (torch.randn(*shape, generator=g) * scale + mean).to(TORCH[dt])

    host = {"x": draw(tokens, d), "w1n": draw(d, scale=0.1, mean=1), "b1n": draw(d, scale=0.1),
            "up": draw(d, ff, scale=d**-0.5), "bup": draw(ff, scale=0.1),
            "down": draw(ff, d, scale=ff**-0.5), "bdown": draw(d, scale=0.1),
            "w2n": draw(d, scale=0.1, mean=1), "b2n": draw(d, scale=0.1),
            "head": draw(d, vocab, scale=3 * d**-0.5),
            "ids": torch.randint(vocab, (tokens,), generator=g), "dlp": torch.ones(tokens)}
    k = 5
    dev = {n: Dev(m, t) for n, t in host.items()}
    bf, f32 = torch.bfloat16, torch.float32
    res = {n: out(m, s, t) for n, s, t in (
        ("n1", (tokens, d), bf), ("h", (tokens, ff), bf), ("stream", (tokens, d), bf),
        ("n2", (tokens, d), bf), ("mean", (tokens,), f32), ("rstd", (tokens,), f32),
        ("logits", (tokens, vocab), f32), ("logprobs", (tokens,), f32), ("entropy", (tokens,), f32),
        ("lse", (tokens,), f32), ("top_logprobs", (tokens, k), f32), ("top_ids", (tokens, k),
                                                                    torch.int64),
        ("dlogits", (tokens, vocab), f32), ("dx", (tokens, d), bf), ("dw", (d,), bf),
        ("db", (d,), bf))}
    n_lp = m.token_logprobs_workspace_bytes(tokens, vocab, k)
    n_ln = m.layer_norm_backward_workspace_bytes(tokens, d)
    ws_lp, ws_ln = workspace(m, n_lp), workspace(m, n_ln)
    A = m.Activation

    def launch(stream):
        v = {**dev, **res}
        for st in (
            m.launch_layer_norm(v["x"], v["w1n"], v["b1n"], v["n1"], None, None, BF16, BF16,
                                tokens, d, 1e-5, stream),
            m.launch_gemm_lp_bias_act(v["n1"], v["up"], v["bup"], None, v["h"], BF16, BF16, BF16,
                                      tokens, ff, d, 1.0, A.kGeluTanh, None, stream),
            m.launch_gemm_lp_bias_act(v["h"], v["down"], v["bdown"], v["x"], v["stream"], BF16, BF16,
                                      BF16, tokens, d, ff, 1.0, A.kNone, None, stream),
            m.launch_layer_norm(v["stream"], v["w2n"], v["b2n"], v["n2"], v["mean"], v["rstd"],
                                BF16, BF16, tokens, d, 1e-5, stream),
            m.launch_gemm_lp_bias_act(v["n2"], v["head"], None, None, v["logits"], BF16, F32, F32,
                                      tokens, vocab, d, 1.0, A.kNone, None, stream),
            m.launch_token_logprobs(v["logits"], v["ids"], v["logprobs"], v["entropy"], v["lse"],
                                    v["top_logprobs"], v["top_ids"], F32, tokens, vocab, vocab, 1.0,
                                    k, ws_lp, n_lp, stream),
            m.launch_token_logprobs_backward(v["logits"], v["ids"], v["lse"], None, v["dlp"], None,
                                             v["dlogits"], F32, tokens, vocab, vocab, 1.0, stream),
            # n2 in the place of a gradient of itself: any values of its type do.
            m.launch_layer_norm_backward(v["n2"], v["stream"], v["w2n"], v["mean"], v["rstd"],
                                         v["dx"], v["dw"], v["db"], BF16, BF16, tokens, d, ws_ln,
                                         n_ln, stream),
        ):
            st.throw_if_error()

    launch(None)
    m.device_synchronize()
    got = {n: t.get() for n, t in res.items()}

    def stage(name, want_tol):
        check(name, got[name], *want_tol)

    y, t = norm._forward(host["x"], host["w1n"], host["b1n"], BF16)
    stage("n1", (y[0], t[0]))
    stage("h", gemm._want(got["n1"], host["up"], host["bup"], None, gemm.TANH, 1.0, BF16))
    stage("stream", gemm._want(got["h"], host["down"], host["bdown"], host["x"], gemm.NONE, 1.0,
                               BF16))
    for name, w, tol in zip(("n2", "mean", "rstd"), *norm._forward(got["stream"], host["w2n"],
                                                                   host["b2n"], BF16)):
        stage(name, (w, tol))
    stage("logits", gemm._want(got["n2"], host["head"], None, None, gemm.NONE, 1.0, F32))
    lps.compare(got, lps._reference(got["logits"], host["ids"], 1.0, k))
    stage("dlogits", lps._gradient(got["logits"], host["ids"], got["lse"], None, host["dlp"], None,
                                   1.0, F32))
    for name, w, tol in zip(("dx", "dw", "db"),
                            *norm._backward(got["n2"], got["stream"], host["w2n"], got["mean"],
                                            got["rstd"], BF16, BF16)):
        stage(name, (w, tol))

    graph = Captured(m, launch)
    try:
        for _ in range(3):
            graph.replay()
            assert all(same_bits(res[n].get(), got[n]) for n in res)
            launch(None)
            m.device_synchronize()
            assert all(same_bits(res[n].get(), got[n]) for n in res)
    finally:
        graph.close()
