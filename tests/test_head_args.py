"""Refusals of the 8-bit float and scoring entry points: checked before any CUDA work, so without a GPU."""
import ctypes as C

import numpy as np
import pytest

torch = pytest.importorskip("torch")

from dabnn_b200 import capi, ops  # noqa: E402
from dabnn_b200.build import build_library  # noqa: E402


@pytest.fixture(scope="module")
def lib():
    build_library()
    return capi.load()


ARG, SHAPE = 1, 2


def buffer(nbytes):
    raw = np.zeros(nbytes + 64, np.uint8)
    off = -raw.ctypes.data % 64
    return raw[off:off + nbytes], raw.ctypes.data + off


def test_quantize_refusals(lib):
    keep, p = buffer(4096)

    def call(src=p, kind=0, ld_in=128, out=p, ld_out=128, scales=p, rows=2, k=128, block_rows=1):
        return lib.dabnn_fp8_quantize(src, kind, ld_in, out, ld_out, scales, 1, 1, rows, k, block_rows, None)

    assert call(kind=3) == ARG and call(kind=-1) == ARG
    assert call(rows=-1) == ARG and call(k=-1) == ARG
    assert call(block_rows=64) == ARG and call(block_rows=0) == ARG
    assert call(src=None) == ARG and call(out=None) == ARG and call(scales=None) == ARG
    assert call(ld_in=127) == SHAPE and call(ld_out=127) == SHAPE
    assert call(src=p + 2) == ARG and call(src=p + 1, kind=2) == ARG and call(scales=p + 2) == ARG
    assert call(rows=0) == 0 and call(k=0, src=None, out=None, scales=None) == 0


def test_gemm_refusals(lib):
    keep, p = buffer(4096)

    def call(a=p, lda=128, sa=p, b=p, ldb=128, sb=p, bias=None, c=p, kind=0, ldc=4, m=2, n=4, k=128):
        return lib.dabnn_fp8_gemm(a, lda, sa, 1, 1, b, ldb, sb, 1, 1, bias, c, kind, ldc, m, n, k, None)

    assert call(kind=3) == ARG
    assert call(m=-1) == ARG and call(n=-1) == ARG and call(k=-1) == ARG
    for name in ("a", "sa", "b", "sb", "c"):
        assert call(**{name: None}) == ARG, name
    assert call(lda=112) == SHAPE and call(ldb=112) == SHAPE and call(ldc=3) == SHAPE
    assert call(lda=136) == SHAPE and call(ldb=136) == SHAPE            # pitches off 16 bytes
    assert b"16-byte" in lib.dabnn_last_error()
    assert call(a=p + 8) == SHAPE and call(b=p + 1) == SHAPE
    assert call(c=p + 2) == ARG and call(c=p + 1, kind=1) == ARG and call(sa=p + 1) == ARG and call(sb=p + 2) == ARG and call(bias=p + 2) == ARG
    assert call(m=0, a=None) == 0 and call(n=0, b=None) == 0


def test_logprobs_refusals(lib):
    keep, p = buffer(4096)

    def call(x=p, kind=0, ld=100, labels=p, rows=2, classes=100, lp=p, rank=p, ent=p, tlp=p, ti=p, top=2):
        return lib.dabnn_logprobs(x, kind, ld, labels, rows, classes, lp, rank, ent, tlp, ti, top, None)

    assert call(kind=3) == ARG and call(rows=-1) == ARG and call(classes=0) == ARG
    assert call(top=-1) == ARG and call(top=65) == ARG and call(top=5, classes=4) == ARG
    assert call(labels=None) == ARG                                       # a label's outputs without labels
    assert call(tlp=None) == ARG and call(ti=None) == ARG and call(x=None) == ARG
    assert call(ld=99) == SHAPE
    assert call(x=p + 2) == ARG and call(x=p + 1, kind=1) == ARG
    assert call(rows=0, x=None) == 0
    assert lib.dabnn_net_logprobs(None, b"x", None, None, None, None, None, None, 0) == ARG


def test_python_refusals():
    """Tensors that are not on the current device, and kinds that are not taken, never reach the library."""
    x = torch.zeros((2, 128))
    f8 = x.to(torch.float8_e4m3fn)
    for call in (lambda: ops.fp8_quantize(x), lambda: ops.fp8_quantize_weights(x), lambda: ops.fp8_gemm(f8, x, f8, x), lambda: ops.logprobs(x)):
        with pytest.raises((TypeError, RuntimeError, AssertionError)):
            call()


class _Cuda(torch.Tensor):
    """A CPU tensor that says it lies on device `at`."""
    at = 0

    @property
    def is_cuda(self):
        return True

    @property
    def device(self):
        return torch.device("cuda", self.at)

    def get_device(self):
        return self.at


@pytest.fixture
def pretend(monkeypatch):
    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: 0, raising=False)
    monkeypatch.setattr(capi, "load", lambda: pytest.fail("the call reached the library"))

    def tensor(t, at=0):
        t = t.as_subclass(_Cuda)
        t.at = at
        return t

    return tensor


def test_python_refusals_by_device_and_kind(pretend):
    f = torch.zeros((2, 128))
    good = {"a": pretend(f.to(torch.float8_e4m3fn)), "a_scales": pretend(torch.zeros((2, 1))), "b": pretend(torch.zeros((5, 128)).to(torch.float8_e4m3fn)),
            "b_scales": pretend(torch.zeros((1, 1)))}
    for x in (pretend(f, 1), pretend(f.double()), pretend(torch.zeros((128, 4)).t())):
        for call in (ops.fp8_quantize, ops.fp8_quantize_weights, ops.logprobs):
            with pytest.raises(TypeError):
                call(x)
    with pytest.raises(TypeError):
        ops.fp8_quantize_weights(pretend(torch.zeros((2, 3, 128))))
    bad = {"a": [f, pretend(f), pretend(good["a"], 0).view(torch.uint8)], "a_scales": [pretend(torch.zeros((2, 2))), pretend(torch.zeros((1, 2))), pretend(torch.zeros((2, 1)).half())],
           "b": [pretend(torch.zeros((5, 127)).to(torch.float8_e4m3fn)), pretend(torch.zeros((2, 5, 128)).to(torch.float8_e4m3fn))],
           "b_scales": [pretend(torch.zeros((5, 1))), torch.zeros((1, 1))], "bias": [pretend(torch.zeros(4)), pretend(torch.zeros(5).half()), pretend(torch.zeros(10))[::2]],
           "out_dtype": [torch.float64, torch.int32]}
    for name, values in bad.items():
        for v in values:
            with pytest.raises((TypeError, ValueError)):
                ops.fp8_gemm(**{**good, name: v})
    x = pretend(torch.zeros((4, 100)))
    for labels in (torch.zeros(4, dtype=torch.int64), pretend(torch.zeros(4, dtype=torch.int32)), pretend(torch.zeros(3, dtype=torch.int64)),
                   pretend(torch.zeros((4, 1), dtype=torch.int64)), pretend(torch.zeros(8, dtype=torch.int64))[::2], pretend(torch.zeros(4, dtype=torch.int64), 1)):
        with pytest.raises(TypeError):
            ops.logprobs(x, labels)


def test_collect_engine_status_refusals(lib):
    assert lib.dabnn_collect_engine_status(None) == ARG
    assert lib.dabnn_debug_fp8_give_up(-2, 0) == ARG and lib.dabnn_debug_fp8_give_up(0, 8) == ARG and lib.dabnn_debug_fp8_give_up(0, -1) == ARG
