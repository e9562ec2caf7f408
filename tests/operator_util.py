"""Helpers of the operator tests: typed host tensors in guarded device buffers, and the
rounding units that their tolerances count.

A rounding to a type is off by at most half a step, `HALF[t]` relative to the value; a value
below a type's smallest normal number by at most half its smallest subnormal, `TINY[t]`."""
from __future__ import annotations

import numpy as np
import torch

F32, F16, BF16 = 0, 1, 2
DTYPES = [BF16, F16, F32]
ID = {F32: "f32", F16: "f16", BF16: "bf16"}
TORCH = {F32: torch.float32, F16: torch.float16, BF16: torch.bfloat16}
U = 2.0**-24                                    # one fp32 rounding
HALF = {F32: 2.0**-24, F16: 2.0**-11, BF16: 2.0**-8}
TINY = {F32: 2.0**-126, F16: 2.0**-25, BF16: 2.0**-126}   # fp32 and bf16: flushed at most
GUARD = 64                                      # bytes kept on either side of every buffer
PATTERN = 0xA5


def _bytes(t: torch.Tensor) -> np.ndarray:
    return t.contiguous().reshape(-1).view(torch.uint8).numpy()


class Dev:
    """A device copy of a host tensor, `shift` elements past a 256-byte boundary plus the
    guard, with a guard behind it."""

    def __init__(self, m, t: torch.Tensor, shift: int = 0):
        self.m, self.shape, self.dtype = m, tuple(t.shape), t.dtype
        raw = _bytes(t)
        self.at = GUARD + shift * t.element_size()
        self.nbytes = raw.size
        host = np.full(self.at + raw.size + GUARD, PATTERN, np.uint8)
        host[self.at:self.at + raw.size] = raw
        self.buf = m.DeviceBuffer.from_array(host)
        self.ptr = self.buf.ptr + self.at

    def data_ptr(self):
        return self.ptr

    def get(self) -> torch.Tensor:
        host = self.buf.download(self.buf.nbytes, np.uint8)
        assert (host[:self.at] == PATTERN).all(), "written before the buffer"
        assert (host[self.at + self.nbytes:] == PATTERN).all(), "written behind the buffer"
        raw = torch.from_numpy(host[self.at:self.at + self.nbytes].copy())
        return raw.view(self.dtype).reshape(self.shape)


def out(m, shape, dtype, shift: int = 0) -> Dev:
    """An output: every byte a pattern, so that what is not written shows."""
    t = torch.empty(shape, dtype=dtype)
    _bytes(t)[:] = 0x5A
    return Dev(m, t, shift)


def workspace(m, nbytes: int) -> Dev:
    """A workspace of exactly `nbytes`, guarded, its contents a pattern that reads as NaN in
    fp32 (0xFFFFFFFF); null where none is needed."""
    if nbytes == 0:
        return None
    return Dev(m, torch.full((nbytes,), 0xFF, dtype=torch.uint8))


def same_bits(a: torch.Tensor, b: torch.Tensor) -> bool:
    return bool((_bytes(a) == _bytes(b)).all())


def check(name: str, got: torch.Tensor, want: torch.Tensor, tol) -> None:
    """|got - want| <= tol elementwise in 64 bits; NaN and infinities in the same places."""
    got, want = got.double(), want.double()
    tol = torch.as_tensor(tol, dtype=torch.float64).expand_as(want)
    assert got.shape == want.shape, (name, got.shape, want.shape)
    assert torch.equal(got.isnan(), want.isnan()), f"{name}: NaN in other places"
    inf = want.isinf()
    assert torch.equal(got[inf], want[inf]) and not got[~inf].isinf().any(), f"{name}: infinities"
    fine = want.isfinite()
    over = ((got - want).abs() - tol)[fine]
    if over.numel() and over.max() > 0:
        i = int(over.argmax())
        raise AssertionError(f"{name}: {got[fine][i]} for {want[fine][i]}, off by "
                             f"{(got - want).abs()[fine][i]:.3g} with {tol[fine][i]:.3g} allowed")


class Captured:
    """Launches captured on a stream into a graph, for replays."""

    def __init__(self, m, launch):
        import ctypes as C
        self.m, self.stream, L = m, m.Stream(), m.lib()
        vp = C.c_void_p
        for name, args in (("mcke_rt_stream_begin_capture", [vp]),
                           ("mcke_rt_stream_end_capture", [vp, C.POINTER(vp)]),
                           ("mcke_rt_graph_launch", [vp, vp]), ("mcke_rt_graph_destroy", [vp])):
            getattr(L, name).argtypes, getattr(L, name).restype = args, C.c_int
        m._check(L.mcke_rt_stream_begin_capture(self.stream.handle))
        launch(self.stream)
        self.exe = vp()
        m._check(L.mcke_rt_stream_end_capture(self.stream.handle, C.byref(self.exe)))

    def replay(self):
        self.m._check(self.m.lib().mcke_rt_graph_launch(self.exe, self.stream.handle))
        self.stream.synchronize()

    def close(self):
        self.m.lib().mcke_rt_graph_destroy(self.exe)
        self.stream.close()
