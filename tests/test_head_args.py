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


# logits [..., classes] and labels [...] as a program slices them; None: refused
B = torch.zeros((4, 9, 30))
L = torch.zeros((4, 9), dtype=torch.int64)
SLICES = {
    "all but the last position": (B[:, :-1], L[:, 1:]),
    "the middle, a padded vocabulary": (B[:, 2:7, :25], L[:, 1:6]),
    "padded vocabulary": (B[..., :25], L),
    "padded vocabulary, labels of all but the first": (B[:, :8, 3:25].contiguous(), L[:, 1:]),
    "labels made whole": (B[:, :-1], L[:, 1:].contiguous()),
    "logits made whole": (B[:, :-1].contiguous(), L[:, 1:]),
    "no labels": (B[1:, 3:], None),
    "one position of each": (B[:, 4], L[:, 4].contiguous()),
    "one position of each, kept": (B[:, 4:5], L[:, 4:5].contiguous()),
    "two positions": (B[:, 3:4], L[:, 5:6]),
    "two positions, the same logits": (B[:1, 3:4].expand(4, 1, 30), L[:, 5:6]),
    "every other sequence": (B[::2, :-1], L[::2, 1:]),
    "one sequence": (B[1:2, :-1], L[2:3, 1:]),
    "one sequence, flat": (B[1, :-1], L[2, 1:]),
    "the same logits for each": (B[:1].expand(4, 9, 30)[:, 1:], L[:, 1:]),
    "four levels that are two": (torch.zeros((2, 3, 5, 7, 10))[:, 1:], torch.zeros((2, 2, 5, 7), dtype=torch.int64)),
    "one row": (B[2, 3, 4:], L[1, 2]),
    "none": (B[:0, :-1], L[:0, 1:]),
    "a gap in two dimensions": (torch.zeros((2, 3, 4, 5, 6))[:, :2, :3, :4], None),
    "classes apart": (B.transpose(1, 2)[:, :-1], None),
    "labels apart": (B[:, :-1], L.t().contiguous().t()[:, 1:]),
    "labels apart, flat": (B[:, 4], L[:, 4]),
    "groups of other sizes": (torch.zeros((3, 4, 5, 30))[:, :, 1:], torch.zeros((3, 5, 5), dtype=torch.int64)[:, 1:].view(3, 4, 5)),
}
REFUSED = {"a gap in two dimensions", "classes apart", "labels apart", "labels apart, flat", "groups of other sizes"}


@pytest.mark.parametrize("name", SLICES)
def test_where_rows_and_labels_are_read(name, monkeypatch):
    """The addresses a call hands over are those of its tensors' rows, in their order."""
    calls = []

    class Recorder:
        def __getattr__(self, function):
            return lambda *args: calls.append((function, args)) or 0

    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: 0, raising=False)
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda device: 0, raising=False)
    monkeypatch.setattr(capi, "load", Recorder)
    logits, labels = (None if t is None else t.as_subclass(_Cuda) for t in SLICES[name])
    if name in REFUSED:
        with pytest.raises(TypeError):
            ops.logprobs(logits, labels)
        assert not calls
        return
    lp, rank, entropy, _, _ = ops.logprobs(logits, labels)
    assert entropy.shape == logits.shape[:-1] and entropy.is_contiguous()
    assert labels is None or (lp.shape == rank.shape == labels.shape and lp.is_contiguous() and rank.is_contiguous())
    (function, args), = calls
    if function == "dabnn_logprobs":
        at, kind, ld, lab, rows, classes = args[:6]
        group_rows, ld_group, label_group = max(rows, 1), 0, 0
    else:
        assert function == "dabnn_logprobs_grouped"
        at, kind, ld, ld_group, lab, label_group, group_rows, rows, classes = args[:9]
    assert kind == 0 and classes == logits.shape[-1] and rows == logits.shape[:-1].numel()
    read = [(at + 4 * (r // group_rows * ld_group + r % group_rows * ld)) for r in range(rows)]
    index = [()] if logits.dim() == 1 else list(np.ndindex(*logits.shape[:-1]))
    assert read == [logits[i].data_ptr() for i in index]
    if labels is None:
        assert lab is None
    else:
        assert [lab + 8 * (r // group_rows * label_group + r % group_rows) for r in range(rows)] == [labels[i].data_ptr() for i in index]
    assert rows <= 1 or group_rows == 1 or ld >= classes


def test_rows_with_a_pitch():
    """Leading dimensions whose rows alone have a pitch are one matrix; others are refused."""
    x = torch.zeros((3, 5, 40)).as_subclass(_Cuda)
    assert ops._rows(x[..., 3:30], "x") == (15, 27, 40)
    assert ops._rows(x[:, 2:3, :30], "x") == (3, 30, 200)
    assert ops._rows(x[1:2, 1:3, :30], "x") == (2, 30, 40)
    for bad in (x[:, 1:], x.transpose(0, 1), x[..., ::2], x.expand(2, 3, 5, 40)[:, :, 1:]):
        with pytest.raises(TypeError):
            ops._rows(bad, "x")


def test_grouped_refusals(lib):
    keep, p = buffer(4096)

    def call(x=p, ld=100, ld_group=400, labels=p, label_group=3, group_rows=2, rows=4, lp=p, rank=p, top=0):
        return lib.dabnn_logprobs_grouped(x, 0, ld, ld_group, labels, label_group, group_rows, rows, 100, lp, rank, p, None, None, top, None)

    assert call(group_rows=0) == ARG and call(group_rows=-1) == ARG and call(rows=-1) == ARG
    assert call(ld=99) == SHAPE
    assert call(labels=None) == ARG and call(top=1) == ARG and call(x=None) == ARG
    assert call(rows=0, x=None) == 0
