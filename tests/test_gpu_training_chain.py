"""A training step from tokens to the gradients of every weight, as a program chains it, without a
wait between the launches: embedding, layer norm, the up product, bias + GELU with its input kept
in 8 bits, the down product onto the residual stream, layer norm, the cross entropy of the
hidden states against the embedding's own table; then back to that table: the loss's
gradients, the last norm's, GELU's from the 8 bits, the first norm's, and the embedding's added to
the loss's.  Each stage is checked against its formula in 64 bits from the values that the stage
before it gave, and a capture of the whole step replays to its bits.

(The products of the backward pass run on transposed copies of the weights, as a program keeps
them.)"""
from __future__ import annotations

import math

import pytest
import torch

from tests import test_gpu_bias_act_checkpoint8 as act8
from tests import test_gpu_embedding as emb
from tests import test_gpu_gemm_lp_epilogue as gemm
from tests import test_gpu_layer_norm as norm
from tests import test_gpu_linear_cross_entropy as lce
from tests.operator_util import (BF16, F32, TORCH, Captured, Dev, check, out, same_bits, workspace)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("tokens,d,ff,vocab", [(1, 256, 1024, 5003), (37, 128, 512, 1000),
                                               (600, 512, 2048, 8200)])
def test_step(gpu, tokens, d, ff, vocab):
    m = gpu
    g = torch.Generator().manual_seed(tokens)
    bf, f32, u8 = torch.bfloat16, torch.float32, torch.uint8

    def draw(*shape, scale=1.0, mean=0.0, dt=BF16):
        return (torch.randn(*shape, generator=g) * scale + mean).to(TORCH[dt])

    ids = torch.randint(vocab, (tokens,), generator=g)
    ids[torch.rand(tokens, generator=g) < 0.3] = ids[0]      # one of them often
    targets = torch.randint(vocab, (tokens,), generator=g)
    if tokens > 1:
        ids[-1], targets[-1], targets[0] = -1, -100, -100    # padding, and a prompt's token
    scale = math.sqrt(d)
    up, down = draw(d, ff, scale=d**-0.5), draw(ff, d, scale=ff**-0.5)
    host = {"ids": ids, "targets": targets, "table": draw(vocab, d, scale=1 / scale),
            "w1n": draw(d, scale=0.1, mean=1), "b1n": draw(d, scale=0.1), "up": up,
            "bup": draw(ff, scale=0.1), "down": down, "down_t": down.t().contiguous(),
            "up_t": up.t().contiguous(), "w2n": draw(d, scale=0.1, mean=1),
            "b2n": draw(d, scale=0.1), "dloss": torch.full((tokens,), 1.0 / tokens)}
    dev = {n: Dev(m, t) for n, t in host.items()}
    res = {n: out(m, s, t) for n, s, t in (
        ("x", (tokens, d), bf), ("n1", (tokens, d), bf), ("mean1", (tokens,), f32),
        ("rstd1", (tokens,), f32), ("pre", (tokens, ff), bf), ("h", (tokens, ff), bf),
        ("codes", (tokens, ff), u8), ("ex", (tokens, act8.blocks(ff)), u8),
        ("stream", (tokens, d), bf), ("n2", (tokens, d), bf), ("mean2", (tokens,), f32),
        ("rstd2", (tokens,), f32), ("loss", (tokens,), f32), ("lse", (tokens,), f32),
        ("dn2", (tokens, d), bf), ("dtable0", (vocab, d), bf), ("dstream", (tokens, d), bf),
        ("dw2n", (d,), bf), ("db2n", (d,), bf), ("dh", (tokens, ff), bf), ("dpre", (tokens, ff), bf),
        ("h_again", (tokens, ff), bf), ("dbup", (ff,), bf), ("dn1", (tokens, d), bf),
        ("dx", (tokens, d), bf), ("dw1n", (d,), bf), ("db1n", (d,), bf), ("dtable", (vocab, d), bf))}
    sizes = {"ln": m.layer_norm_backward_workspace_bytes(tokens, d),
             "act": m.bias_act_checkpoint8_backward_workspace_bytes(tokens, ff),
             "lce": m.linear_cross_entropy_workspace_bytes(tokens, vocab, d),
             "lceb": m.linear_cross_entropy_backward_workspace_bytes(tokens, vocab, d),
             "emb": m.embedding_backward_workspace_bytes(tokens, vocab, d)}
    ws = {n: (workspace(m, s), s) for n, s in sizes.items()}
    A = m.Activation
    L = m.lib()
    import ctypes as C
    vp = C.c_void_p
    L.mcke_launch_stream_copy_f32.argtypes = [vp, vp, C.c_int64, vp]

    def launch(stream):
        v = {**dev, **res}

        def product(a, b, bias, r, y, mm, n, k):
            return m.launch_gemm_lp_bias_act(a, b, bias, r, y, BF16, BF16, BF16, mm, n, k, 1.0,
                                             A.kNone, None, stream)

        def norm_of(x, w, b, y, mean, rstd):
            return m.launch_layer_norm(x, w, b, y, mean, rstd, BF16, BF16, tokens, d, 1e-5, stream)

        def norm_back(dy, x, w, mean, rstd, dx, dw, db):
            return m.launch_layer_norm_backward(dy, x, w, mean, rstd, dx, dw, db, BF16, BF16, tokens,
                                                d, *ws["ln"], stream)

        for st in (
            m.launch_embedding(v["ids"], v["table"], v["x"], BF16, BF16, tokens, vocab, d, scale,
                               stream),
            norm_of(v["x"], v["w1n"], v["b1n"], v["n1"], v["mean1"], v["rstd1"]),
            product(v["n1"], v["up"], None, None, v["pre"], tokens, ff, d),
            m.launch_bias_act_checkpoint8(v["pre"], v["bup"], v["h"], v["codes"], v["ex"], BF16, BF16,
                                          tokens, ff, A.kGeluTanh, stream),
            product(v["h"], v["down"], None, v["x"], v["stream"], tokens, d, ff),
            norm_of(v["stream"], v["w2n"], v["b2n"], v["n2"], v["mean2"], v["rstd2"]),
            m.launch_linear_cross_entropy(v["n2"], v["table"], v["targets"], v["loss"], v["lse"],
                                          BF16, tokens, vocab, d, 1.0, *ws["lce"], stream),
            m.launch_linear_cross_entropy_backward(v["n2"], v["table"], v["targets"], v["lse"],
                                                   v["dloss"], None, v["dn2"], v["dtable0"], BF16,
                                                   tokens, vocab, d, 1.0, *ws["lceb"], stream),
            norm_back(v["dn2"], v["stream"], v["w2n"], v["mean2"], v["rstd2"], v["dstream"], v["dw2n"],
                      v["db2n"]),
            product(v["dstream"], v["down_t"], None, None, v["dh"], tokens, ff, d),
            m.launch_bias_act_checkpoint8_backward(v["dh"], v["codes"], v["ex"], v["dpre"],
                                                   v["h_again"], v["dbup"], BF16, BF16, tokens, ff,
                                                   A.kGeluTanh, *ws["act"], stream),
            product(v["dpre"], v["up_t"], None, None, v["dn1"], tokens, d, ff),
            norm_back(v["dn1"], v["x"], v["w1n"], v["mean1"], v["rstd1"], v["dx"], v["dw1n"], v["db1n"]),
            # The tied table: the embedding's gradient onto (a copy of) the loss's.
            m._st(L.mcke_launch_stream_copy_f32(v["dtable0"].ptr, v["dtable"].ptr, vocab * d // 2,
                                                stream.handle if stream else None)),
            m.launch_embedding_backward(v["ids"], v["dx"], v["dtable"], BF16, BF16, tokens, vocab, d,
                                        scale, True, *ws["emb"], stream),
        ):
            st.throw_if_error()

    launch(None)
    m.device_synchronize()
    got = {n: t.get() for n, t in res.items()}

    def stage(name, want_tol):
        check(name, got[name], *want_tol)

    def stages(names, ref):
        for name, w, t in zip(names, *ref):
            stage(name, (w, t))

    stage("x", emb.forward_reference(ids, host["table"], BF16, scale))
    stages(("n1", "mean1", "rstd1"), norm._forward(got["x"], host["w1n"], host["b1n"], BF16))
    stage("pre", gemm._want(got["n1"], up, None, None, gemm.NONE, 1.0, BF16))
    u = got["pre"].float() + host["bup"].float()
    v, ex = act8.saved(u)
    assert torch.equal(got["ex"], ex) and torch.equal(act8.restored(got["codes"], got["ex"]), v)
    stage("h", act8.y_reference(got["pre"].double() + host["bup"].double(), act8.TANH, BF16))
    stage("stream", gemm._want(got["h"], down, None, got["x"], gemm.NONE, 1.0, BF16))
    stages(("n2", "mean2", "rstd2"), norm._forward(got["stream"], host["w2n"], host["b2n"], BF16))
    stages(("loss", "lse"), lce.forward_reference(got["n2"], host["table"], targets, 1.0))
    stages(("dn2", "dtable0"), lce.backward_reference(got["n2"], host["table"], targets, got["lse"],
                                                      host["dloss"], None, 1.0, BF16))
    stages(("dstream", "dw2n", "db2n"),
           norm._backward(got["dn2"], got["stream"], host["w2n"], got["mean2"], got["rstd2"], BF16,
                          BF16))
    stage("dh", gemm._want(got["dstream"], host["down_t"], None, None, gemm.NONE, 1.0, BF16))
    stages(("dpre", "h_again", "dbup"), act8.backward_reference(v, got["dh"], act8.TANH, BF16, BF16))
    stage("dn1", gemm._want(got["dpre"], host["up_t"], None, None, gemm.NONE, 1.0, BF16))
    stages(("dx", "dw1n", "db1n"),
           norm._backward(got["dn1"], got["x"], host["w1n"], got["mean1"], got["rstd1"], BF16, BF16))
    stage("dtable", emb.backward_reference(ids, got["dx"], vocab, BF16, scale, got["dtable0"]))

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
