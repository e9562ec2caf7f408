"""The 16-bit product with bias, activation and residual in its epilogue
(mcke_launch_gemm_lp_bias_act) on the GPU against the formula in 64 bits.

Bars:
  * quarter-multiple operands, bias and residual without an activation or with ReLU: every
    product and sum is exact in fp32, so the output is the exact value, rounded once;
  * seeded operands: k products, each exact in fp32, and their sum are off by k U sum |a b|; the
    activation carries that on with a slope below 1.2 and adds at most 1e-6 + 1e-6 |v| of its
    own (the approximations' documented bound), the additions 3 U of their terms, and the
    output its rounding.
"""
from __future__ import annotations

import math

import numpy as np
import pytest
import torch

from tests.operator_util import (BF16, F16, F32, HALF, ID, TINY, TORCH, U, Captured, Dev, check,
                                 out, same_bits)

pytestmark = pytest.mark.gpu

NONE, RELU, ERF, TANH = range(4)
# Every kernel of the launcher: whole tiles of 256 and 128, even shapes of either (EDGE), odd
# ones (WHOLE), split K at its four tiles, short K over many tiles, and what is narrower than 32
# columns; single tokens, K of 0 and 1.
SHAPES = [(1, 1, 1), (1, 4096, 512), (3, 40, 0), (5, 7, 3), (1, 31, 100), (17, 33, 65),
          (16, 256, 512), (31, 70, 1), (64, 64, 64), (100, 300, 77), (130, 514, 192),
          (256, 256, 256), (384, 512, 96), (1100, 3000, 40), (1000, 1501, 5), (300, 9000, 30),
          (2048, 2048, 128), (1700, 2002, 258), (1901, 2001, 131), (2050, 2046, 66)]


def _act(v, act):
    if act == RELU:
        return torch.clamp(v, min=0)
    if act == ERF:
        return 0.5 * v * torch.special.erfc(-v / math.sqrt(2))
    if act == TANH:
        return 0.5 * v * (1 + torch.tanh(math.sqrt(2 / math.pi) * (v + 0.044715 * v**3)))
    return v


def _operands(m_, n, k, ab, yt, bt, seed, quarters=False):
    g = torch.Generator().manual_seed(seed)

    def draw(*shape, scale=1.0):
        if quarters:
            return torch.randint(-8, 9, shape, generator=g).float() / 4
        return torch.randn(*shape, generator=g) * scale

    return (draw(m_, k).to(TORCH[ab]), draw(k, n, scale=1 / math.sqrt(max(k, 1))).to(TORCH[ab]),
            draw(n, scale=0.5).to(TORCH[bt]), draw(m_, n).to(TORCH[yt]))


def run(m, a, b, bias, res, ab, yt, bt, act, alpha=1.0, tile=None, shift=0, in_place=False,
        stream=None):
    M, K = a.shape
    N = b.shape[1]
    da, db = Dev(m, a, shift), Dev(m, b, shift)
    dbias = Dev(m, bias, shift) if bias is not None else None
    dres = Dev(m, res, shift) if res is not None else None
    y = dres if in_place else out(m, (M, N), TORCH[yt], shift)
    m.launch_gemm_lp_bias_act(da, db, dbias, dres, y, ab, yt, bt, M, N, K, alpha, act, tile,
                              stream).throw_if_error()
    m.device_synchronize()
    if dres is not None and not in_place:
        assert same_bits(dres.get(), res)
    return y.get()


def _want(a, b, bias, res, act, alpha, yt):
    ad, bd = a.double(), b.double()
    s = alpha * (ad @ bd)
    t = a.shape[1] * U * abs(alpha) * (ad.abs() @ bd.abs()) + 2 * U * s.abs()
    if bias is not None:
        s = s + bias.double()
    t = t + U * s.abs()
    y = _act(s, act)
    if act != NONE:
        t = 1.2 * t + 1e-6 + 1e-6 * s.abs()
    if res is not None:
        y = y + res.double()
    t = t + 3 * U * (y.abs() + s.abs())
    return y, t + HALF[yt] * (y.abs() + t) + TINY[yt]


def _types(i):
    ab = (BF16, F16)[i % 2]
    return ab, (ab, F32)[(i // 2) % 2], (F32, ab)[(i // 4) % 2]


@pytest.mark.parametrize("which", range(4), ids=["bf16", "f16", "bf16-f32", "f16-f32"])
@pytest.mark.parametrize("i,shape", enumerate(SHAPES), ids=[f"{s[0]}x{s[1]}x{s[2]}" for s in SHAPES])
def test_exact_sums(gpu, i, shape, which):
    """Quarter multiples: the exact value rounded once, with and without bias and residual, and
    with the residual updated in place, for every kernel and pair of types."""
    ab, yt = (BF16, F16)[which % 2], ((BF16, F16)[which % 2], F32)[which // 2]
    bt = (F32, ab)[i % 2]
    a, b, bias, res = _operands(*shape, ab, yt, bt, i, quarters=True)
    for act in (NONE, RELU):
        for bb, rr in ((bias, res), (None, res), (bias, None), (None, None)):
            y, _ = _want(a, b, bb, rr, act, 1.0, yt)
            got = run(gpu, a, b, bb, rr, ab, yt, bt, act)
            assert torch.equal(got, y.to(TORCH[yt])), (act, bb is None, rr is None)
    y, _ = _want(a, b, bias, res, RELU, 1.0, yt)
    assert torch.equal(run(gpu, a, b, bias, res, ab, yt, bt, RELU, in_place=True), y.to(TORCH[yt]))


# The kernels for few rows at each of their widths (up to 16, 32 and 64 rows; 4096, 8192 and 16384
# columns), with K chunks that the waves share unevenly; odd extents at 256 x 256, 128 x 128 with
# two stages ahead (K of two, three and four steps), 64 x 128 and 64 x 64.
MORE = [(1, 200, 2000), (2, 300, 4090), (16, 4096, 96), (3, 5001, 131), (2, 9000, 70),
        (1, 16400, 96), (20, 300, 200), (25, 5003, 77), (30, 8500, 64), (50, 130, 333),
        (64, 4100, 65), (33, 8300, 66), (3701, 3701, 65), (2100, 2301, 67), (2100, 2301, 131),
        (2101, 2303, 200), (900, 2101, 65), (900, 2101, 130), (1201, 1701, 69)]


@pytest.mark.parametrize("i,shape", enumerate(MORE), ids=[f"{s[0]}x{s[1]}x{s[2]}" for s in MORE])
def test_exact_sums_of_more_kernels(gpu, i, shape):
    for which in (i % 4, (i + 1) % 4):
        ab = (BF16, F16)[which % 2]
        yt, bt = (ab, F32)[which // 2], (F32, ab)[i % 2]
        a, b, bias, res = _operands(*shape, ab, yt, bt, i, quarters=True)
        for act, bb, rr in ((NONE, bias, res), (RELU, None, res), (RELU, bias, None)):
            y, _ = _want(a, b, bb, rr, act, 1.0, yt)
            assert torch.equal(run(gpu, a, b, bb, rr, ab, yt, bt, act), y.to(TORCH[yt])), act
        y, _ = _want(a, b, bias, res, NONE, 1.0, yt)
        got = run(gpu, a, b, bias, res, ab, yt, bt, NONE, shift=1, in_place=True)
        assert torch.equal(got, y.to(TORCH[yt]))


@pytest.mark.parametrize("i,shape", enumerate(MORE), ids=[f"{s[0]}x{s[1]}x{s[2]}" for s in MORE])
def test_exact_sums_of_more_kernels_in_the_other_types(gpu, i, shape):
    for which in ((i + 2) % 4, (i + 3) % 4):
        ab = (BF16, F16)[which % 2]
        yt, bt = (ab, F32)[which // 2], (F32, ab)[i % 2]
        a, b, bias, res = _operands(*shape, ab, yt, bt, i, quarters=True)
        y, _ = _want(a, b, bias, res, RELU, 1.0, yt)
        assert torch.equal(run(gpu, a, b, bias, res, ab, yt, bt, RELU), y.to(TORCH[yt]))


@pytest.mark.parametrize("i,shape", enumerate(MORE), ids=[f"{s[0]}x{s[1]}x{s[2]}" for s in MORE])
def test_activations_of_more_kernels(gpu, i, shape):
    ab, yt, bt = _types(i)
    a, b, bias, res = _operands(*shape, ab, yt, bt, 70 + i)
    for act in (ERF, TANH):
        check("y", run(gpu, a, b, bias, res, ab, yt, bt, act),
              *_want(a, b, bias, res, act, 1.0, yt))


# Up to 64 rows on either side of 16384 columns, even and odd widths.
WIDE = [(64, 16384, 96), (64, 16386, 130), (33, 16500, 70), (40, 16385, 77), (32, 16402, 66),
        (17, 16401, 300), (16, 16385, 65), (1, 20001, 67)]


@pytest.mark.parametrize("i,shape", enumerate(WIDE), ids=[f"{s[0]}x{s[1]}x{s[2]}" for s in WIDE])
def test_few_rows_over_many_columns(gpu, i, shape):
    for which in range(4):
        ab = (BF16, F16)[which % 2]
        yt, bt = (ab, F32)[which // 2], (F32, ab)[i % 2]
        a, b, bias, res = _operands(*shape, ab, yt, bt, 60 + i, quarters=True)
        y, _ = _want(a, b, bias, res, RELU, 1.0, yt)
        got = run(gpu, a, b, bias, res, ab, yt, bt, RELU, in_place=which > 1)
        assert torch.equal(got, y.to(TORCH[yt])), which


# (shape, tile): 192 tiles of 256 and more that are ragged in M, N, K or all of them, whole tiles of
# 256; short K over many tiles of 128, in vectors and not; narrower than 32 columns at tiles of 128
# and 256.
LARGE = [((3500, 3590, 66), 0), ((3585, 3584, 128), 0), ((3584, 3602, 64), 0), ((2048, 2048, 64), 0),
         ((2166, 3544, 40), 1), ((2166, 3543, 7), 1), ((300, 31, 100), 1), ((517, 9, 64), 0)]
LARGE_IDS = [f"{s[0]}x{s[1]}x{s[2]}" for s, _ in LARGE]


@pytest.mark.parametrize("which", range(4), ids=["bf16", "f16", "bf16-f32", "f16-f32"])
@pytest.mark.parametrize("i,case", enumerate(LARGE), ids=LARGE_IDS)
def test_exact_sums_of_large_tiles(gpu, i, case, which):
    shape, tile = case[0], gpu.LP_TILES[case[1]]
    ab = (BF16, F16)[which % 2]
    yt, bt = (ab, F32)[which // 2], (F32, ab)[(i + which) % 2]
    a, b, bias, res = _operands(*shape, ab, yt, bt, 90 + i, quarters=True)
    for act, bb, rr, in_place in ((RELU, bias, res, False), (NONE, bias, res, True),
                                  (NONE, None, None, False)):
        y, _ = _want(a, b, bb, rr, act, 1.0, yt)
        got = run(gpu, a, b, bb, rr, ab, yt, bt, act, tile=tile, in_place=in_place)
        assert torch.equal(got, y.to(TORCH[yt])), (act, in_place)


@pytest.mark.parametrize("i,case", enumerate(LARGE), ids=LARGE_IDS)
def test_activations_of_large_tiles(gpu, i, case):
    shape, tile = case[0], gpu.LP_TILES[case[1]]
    ab, yt, bt = _types(i)
    a, b, bias, res = _operands(*shape, ab, yt, bt, 80 + i)
    for act in (ERF, TANH):
        check("y", run(gpu, a, b, bias, res, ab, yt, bt, act, 0.7, tile, in_place=act == TANH),
              *_want(a, b, bias, res, act, 0.7, yt))


@pytest.mark.parametrize("act", [NONE, RELU, ERF, TANH])
@pytest.mark.parametrize("i,shape", enumerate(SHAPES), ids=[f"{s[0]}x{s[1]}x{s[2]}" for s in SHAPES])
def test_activations(gpu, i, shape, act):
    ab, yt, bt = _types(i + act)
    a, b, bias, res = _operands(*shape, ab, yt, bt, 50 + i)
    alpha = (1.0, 0.5)[i % 2]
    check("y", run(gpu, a, b, bias, res, ab, yt, bt, act, alpha),
          *_want(a, b, bias, res, act, alpha, yt))


@pytest.mark.parametrize("shape", [(1, 512, 300), (70, 64, 64), (300, 520, 130), (2048, 2048, 64)])
def test_tiles_and_alignment(gpu, shape):
    """Any tile and any element alignment give the exact sums' value."""
    for ab, yt in ((BF16, BF16), (F16, F32)):
        a, b, bias, res = _operands(*shape, ab, yt, ab, 9, quarters=True)
        y, _ = _want(a, b, bias, res, NONE, 1.0, yt)
        for tile in gpu.LP_TILES:
            for shift in (0, 1, 2):
                got = run(gpu, a, b, bias, res, ab, yt, ab, NONE, tile=tile, shift=shift)
                assert torch.equal(got, y.to(TORCH[yt])), (tile, shift)
        assert torch.equal(run(gpu, a, b, bias, res, ab, yt, ab, NONE, shift=1, in_place=True),
                           y.to(TORCH[yt]))


@pytest.mark.parametrize("shape", [(1, 4096, 512), (512, 512, 96), (2048, 2048, 128),
                                   (1901, 2001, 131)])
def test_bits_of_the_two_launches(gpu, shape):
    """To fp32, with fp32 bias: the bits of the plain product followed by the bias and
    activation."""
    m = gpu
    M, N, K = shape
    a, b, bias, _ = _operands(M, N, K, BF16, F32, F32, 4)
    da, db, dbias = Dev(m, a), Dev(m, b), Dev(m, bias)
    c, y = out(m, (M, N), torch.float32), out(m, (M, N), torch.float32)
    m.launch_gemm_lp(da, db, c, BF16, F32, M, N, K, 1.0, 0.0).throw_if_error()
    for act in (NONE, RELU, ERF, TANH):
        m.launch_bias_act_f32(c, dbias, y, M, N, act, 1).throw_if_error()
        m.device_synchronize()
        got = run(m, a, b, bias, None, BF16, F32, F32, act)
        assert torch.equal(got.nan_to_num(7.0), y.get().nan_to_num(7.0)), act


@pytest.mark.parametrize("alpha", [1.0, 0.7, -1.3])
@pytest.mark.parametrize("shape", [(1, 4096, 512), (512, 512, 96), (2048, 2048, 128),
                                   (1901, 2001, 131)])
def test_bits_of_the_two_launches_at_any_alpha(gpu, shape, alpha):
    """The product with alpha is rounded before the bias is added, as a launch that stores it
    does, and where there is no residual nothing is added: also the zeros keep their signs (of
    empty rows, and of GELU far below zero).  Without a bias too, the plain product's bits."""
    m = gpu
    M, N, K = shape
    a, b, bias, _ = _operands(M, N, K, BF16, F32, F32, 4)
    a[M // 2] = 0
    bias[::3] -= 40
    bias[1::3] = -0.0
    da, db, dbias = Dev(m, a), Dev(m, b), Dev(m, bias)
    c, y = out(m, (M, N), torch.float32), out(m, (M, N), torch.float32)
    m.launch_gemm_lp(da, db, c, BF16, F32, M, N, K, alpha, 0.0).throw_if_error()
    m.device_synchronize()
    assert same_bits(run(m, a, b, None, None, BF16, F32, F32, NONE, alpha), c.get())
    for act in (NONE, RELU, ERF, TANH):
        m.launch_bias_act_f32(c, dbias, y, M, N, act, 1).throw_if_error()
        m.device_synchronize()
        assert same_bits(run(m, a, b, bias, None, BF16, F32, F32, act, alpha), y.get()), act


@pytest.mark.parametrize("shape", [(4, 64, 128), (300, 520, 130), (2048, 2048, 64)])
def test_special_values(gpu, shape):
    """A NaN or infinity in a row of A spoils that row alone, one in the residual its element."""
    M, N, K = shape
    a, b, bias, res = _operands(M, N, K, BF16, BF16, F32, 3)
    clean = run(gpu, a, b, bias, res, BF16, BF16, F32, TANH)
    a[M - 1, K // 2] = float("nan")
    res[0, N - 1], res[1, 0] = float("inf"), float("nan")
    got = run(gpu, a, b, bias, res, BF16, BF16, F32, TANH)
    assert got[M - 1].isnan().all() and got[0, N - 1] == float("inf") and got[1, 0].isnan()
    got[0, N - 1], got[1, 0] = clean[0, N - 1], clean[1, 0]
    assert same_bits(got[:M - 1], clean[:M - 1])


@pytest.mark.parametrize("shape", [(1, 4096, 1024), (513, 514, 130)])
def test_captured(gpu, shape):
    m = gpu
    M, N, K = shape
    a, b, bias, res = _operands(M, N, K, F16, F16, F16, 5)
    eager = run(m, a, b, bias, res, F16, F16, F16, ERF)
    da, db, dbias, dres = (Dev(m, t) for t in (a, b, bias, res))
    y = out(m, (M, N), torch.float16)
    graph = Captured(m, lambda st: m.launch_gemm_lp_bias_act(
        da, db, dbias, dres, y, F16, F16, F16, M, N, K, 1.0, ERF, None, st).throw_if_error())
    try:
        for i in range(4):
            graph.replay()
            assert same_bits(y.get(), eager), i
            y.buf.upload(np.full(y.buf.nbytes, 0xA5, np.uint8))
            assert same_bits(run(m, a, b, bias, res, F16, F16, F16, ERF), eager)
    finally:
        graph.close()
