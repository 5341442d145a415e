"""8-bit float matrices with a scale for each block of 128: quantiser and product against their 64-bit forms."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

import head_reference as R  # noqa: E402

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


@pytest.fixture(scope="module")
def ops():
    from dabnn_b200 import ops as o
    yield o
    assert o.engine_status() == 0


def values(t):
    return t.float().cpu().double().numpy()


def same(got, expected):
    np.testing.assert_array_equal(values(got), expected)


# ---------------------------------------------------------------------------------------------- quantiser
def check_quantize(ops, x, weights):
    q, s = ops.fp8_quantize_weights(x) if weights else ops.fp8_quantize(x)
    eq, es = R.quantize(values(x), 128 if weights else 1)
    assert q.dtype == torch.float8_e4m3fn and s.dtype == torch.float32 and q.shape == x.shape
    same(s, es)
    same(q, eq)
    assert x.shape[0] <= 1 or q.stride(0) % 16 == 0


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("weights", [False, True])
@pytest.mark.parametrize("rows,k", [(1, 1), (1, 4096), (3, 127), (5, 128), (130, 129), (64, 257), (129, 1000), (257, 512)])
def test_quantize(ops, rows, k, weights, kind):
    g = torch.Generator().manual_seed(rows * 7 + k)
    x = torch.randn((rows, k), generator=g) * torch.exp(3 * torch.randn((rows, 1), generator=g))
    check_quantize(ops, x.to(TYPES[kind]).cuda(), weights)


@pytest.mark.parametrize("weights", [False, True])
def test_quantize_borders(ops, weights):
    """Magnitudes at and next to 448 2^e, ties between e4m3 values, subnormal bytes, zero blocks, the ends of fp32."""
    x = torch.zeros((10, 640))
    x[0, :4] = torch.tensor([448.0, -447.99997, 1.0, 0.0])
    x[1, :3] = torch.tensor([448.00003, -1.0, 0.3])
    x[2, :6] = torch.tensor([256.0, 17.0, 19.0, -17.0, 21.0, 18.999998])             # ties between 16, 18, 20
    x[3, :6] = torch.tensor([300.0, 2.0 ** -9, 2.0 ** -10, 3 * 2.0 ** -10, -(2.0 ** -11), 1e-5])
    x[4, 128:132] = torch.tensor([3.4028235e38, -1.0, 1e30, 2.0 ** 118])
    x[5, 256:260] = torch.tensor([1.1754944e-38, 1e-45, -1e-45, 5e-39])
    x[6, 384:387] = torch.tensor([2.0 ** -117, -(2.0 ** -126), 2.0 ** -135])
    x[7, 639] = -1.75
    x[8, 500] = 1.7500001
    x[9, :640] = torch.arange(640) * 0.7 - 224
    check_quantize(ops, x.cuda(), weights)


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("weights", [False, True])
def test_quantize_not_finite(ops, weights, kind):
    """NaN and infinities become NaN; the scale and the other values of their block are those without them."""
    g = torch.Generator().manual_seed(3)
    x = torch.randn((140, 300), generator=g)
    for v, at in ((float("nan"), (3, 5)), (float("inf"), (3, 6)), (-float("inf"), (7, 299)), (float("nan"), (139, 128))):
        x[at] = v
    x[9, 128:256] = float("inf")      # nothing finite in the block
    check_quantize(ops, x.to(TYPES[kind]).cuda(), weights)


@pytest.mark.parametrize("kind", TYPES)
def test_quantize_strided_rows_and_offsets(ops, kind):
    """Rows with a pitch, bases off every vector boundary, leading dimensions."""
    g = torch.Generator().manual_seed(4)
    store = torch.randn((33, 1003), generator=g).to(TYPES[kind]).cuda()
    for first in (0, 1, 3, 8):
        for k in (130, 512, 900):
            x = store[:, first:first + k]
            for weights in (False, True):
                check_quantize(ops, x, weights)
    x = store[:24, :600].contiguous().view(2, 3, 4, 600)
    q, s = ops.fp8_quantize(x)
    assert q.shape == (2, 3, 4, 600) and s.shape == (2, 3, 4, 5)
    eq, es = R.quantize(values(x.view(24, 600)), 1)
    same(q.reshape(24, 600), eq)
    same(s.reshape(24, 5), es)
    q1, s1 = ops.fp8_quantize(store[2, :600])
    same(q1, eq[2])
    same(s1, es[2])


def test_quantize_leaves_the_rest_alone(ops):
    """Bytes behind a row's end, rows and scales behind the last: as they were; any strides of the scales."""
    from dabnn_b200 import capi
    x = torch.randn((5, 200), device="cuda")
    out = torch.full((8, 256), 0x55, dtype=torch.uint8, device="cuda")
    scales = torch.full((8, 9), -7.0, device="cuda")
    capi.check(capi.load().dabnn_fp8_quantize(x.data_ptr(), 0, 200, out.data_ptr(), 256, scales.data_ptr(), 9, 4, 5, 200, 1, ops._stream()))
    eq, es = R.quantize(values(x), 1)
    same(out[:5, :200].view(torch.float8_e4m3fn), eq)
    same(scales[:5, 0:5:4], es)
    assert (out[5:] == 0x55).all() and (out[:, 200:] == 0x55).all()
    scales[:5, 0:5:4] = -7
    assert (scales == -7).all()


def test_quantize_empty(ops):
    for shape in ((0, 256), (4, 0), (0, 0)):
        q, s = ops.fp8_quantize(torch.empty(shape, device="cuda"))
        assert q.shape == shape and s.shape == (shape[0], -(-shape[1] // 128))


# ---------------------------------------------------------------------------------------------- product
def operands(m, n, k, seed, powers=False):
    """Values of e4m3 bytes (every finite one occurs) and scales of either sign, as 64-bit arrays."""
    rng = np.random.default_rng(seed)
    table = torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn).double().numpy()
    table = table[np.isfinite(table)]
    a, b = rng.choice(table, (m, k)), rng.choice(table, (n, k))
    nk = -(-k // 128)

    def scales(rows):
        s = np.exp2(rng.integers(-6, 6, (rows, nk)).astype(np.float64))
        return s if powers else (s * rng.uniform(-1.5, 1.5, (rows, nk))).astype(np.float32).astype(np.float64)

    return a, scales(m), b, scales(-(-n // 128)), rng.normal(0, 100, n).astype(np.float32).astype(np.float64)


def dev(a):
    return torch.from_numpy(a).float().cuda()


def check_gemm(ops, m, n, k, out="f32", bias=True, seed=None):
    a, sa, b, sb, bv = operands(m, n, k, seed if seed is not None else m * 31 + n * 7 + k)
    if not bias:
        bv = None
    dt = TYPES[out]
    if out == "f16":                                                # keep the results inside the type
        sa, sb = sa * 2.0 ** -14, sb * 2.0 ** -6
    c, tol = R.gemm(a, sa, b, sb, bv, torch.finfo(dt).eps)
    got = ops.fp8_gemm(R.f8(a), dev(sa), R.f8(b), dev(sb), None if bv is None else dev(bv), dt)
    assert got.dtype == dt
    # fp16 results below its normal range step by 2^-24
    R.close(values(got), c, tol + (2.0 ** -25 if out == "f16" else 0.0))


@pytest.mark.parametrize("m,n,k", [(1, 1, 1), (1, 8, 16), (1, 128, 128), (2, 129, 144), (3, 1000, 512), (5, 17, 257), (8, 4100, 1300), (15, 257, 640),
                                   (16, 512, 2048), (17, 130, 129), (31, 640, 384), (33, 64, 4096), (37, 4100, 2064), (63, 1, 300), (64, 129, 1000)])
def test_gemm_few_rows(ops, m, n, k):
    check_gemm(ops, m, n, k)


@pytest.mark.parametrize("m,n,k", [(65, 128, 128), (100, 1000, 512), (127, 255, 257), (128, 128, 256), (129, 1, 128), (200, 2050, 96), (255, 300, 130),
                                   (256, 256, 1024), (257, 513, 1025), (1024, 1000, 512), (700, 1300, 64)])
def test_gemm_many_rows(ops, m, n, k):
    check_gemm(ops, m, n, k)


def test_gemm_large(ops):
    """More tiles than SMs in both directions, long K."""
    check_gemm(ops, 2300, 4200, 700)
    check_gemm(ops, 300, 520, 16400)


@pytest.mark.parametrize("out", TYPES)
@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("m,n,k", [(1, 1000, 512), (20, 131, 300), (150, 259, 384), (300, 1001, 200), (700, 1304, 200), (700, 1301, 200), (2300, 2104, 300), (1900, 2101, 300)])
def test_gemm_output_types(ops, m, n, k, out, bias):
    check_gemm(ops, m, n, k, out, bias)


def test_gemm_without_k_and_empty(ops):
    bias = torch.randn(9, device="cuda")
    a, b = torch.empty((4, 0), device="cuda").to(torch.float8_e4m3fn), torch.empty((9, 0), device="cuda").to(torch.float8_e4m3fn)
    e = torch.empty((4, 0), device="cuda")
    assert torch.equal(ops.fp8_gemm(a, e, b, torch.empty((1, 0), device="cuda"), bias), bias.expand(4, 9))
    assert torch.equal(ops.fp8_gemm(a, e, b, torch.empty((1, 0), device="cuda")), torch.zeros((4, 9), device="cuda"))
    a, s = ops.fp8_quantize(torch.randn((0, 256), device="cuda"))
    b, t = ops.fp8_quantize_weights(torch.randn((130, 256), device="cuda"))
    assert ops.fp8_gemm(a, s, b, t).shape == (0, 130)
    assert ops.fp8_gemm(b, t.repeat_interleave(128, 0)[:130], a, torch.empty((0, 2), device="cuda")).shape == (130, 0)


@pytest.mark.parametrize("m", [3, 40, 200])
def test_gemm_strides(ops, m):
    """Operands with row pitches, scales in either memory order, inside larger tensors, an output with a pitch."""
    from dabnn_b200 import capi
    n, k = 200, 272
    a, sa, b, sb, bias = operands(m, n, k, 5)
    c, tol = R.gemm(a, sa, b, sb, bias, torch.finfo(torch.float32).eps)
    wide_a, wide_b = torch.zeros((m, 336), dtype=torch.float8_e4m3fn, device="cuda"), torch.zeros((n, 400), dtype=torch.float8_e4m3fn, device="cuda")
    wide_a.view(torch.uint8).fill_(0x7f)   # NaN around the operands
    wide_b.view(torch.uint8).fill_(0x7f)
    wide_a[:, 16:16 + k] = R.f8(a)
    wide_b[:, 32:32 + k] = R.f8(b)
    va, vb = wide_a[:, 16:16 + k], wide_b[:, 32:32 + k]
    store = torch.full((m, 7), float("nan"), device="cuda")
    store[:, 1:7:2] = dev(sa)
    for s in (dev(sa), dev(sa).t().contiguous().t(), store[:, 1:7:2]):
        for t in (dev(sb), dev(sb).t().contiguous().t()):
            R.close(values(ops.fp8_gemm(va, s, vb, t, dev(bias))), c, tol)
    out = torch.full((m + 2, n + 13), -5.0, device="cuda")
    s, t = dev(sa), dev(sb)
    capi.check(capi.load().dabnn_fp8_gemm(va.data_ptr(), 336, s.data_ptr(), *s.stride(), vb.data_ptr(), 400, t.data_ptr(), *t.stride(), dev(bias).data_ptr(),
                                          out.data_ptr() + 4 * 5, 0, n + 13, m, n, k, ops._stream()))
    R.close(values(out[:m, 5:5 + n]), c, tol)
    out[:m, 5:5 + n] = -5
    assert (out == -5).all()


@pytest.mark.parametrize("m", [2, 70, 900])
def test_gemm_broadcast_scales(ops, m):
    """One scale for everything, one for each row, one for each block of K: strides of zero."""
    n, k = 1400, 300
    a, _, b, _, _ = operands(m, n, k, 31)
    row, block = np.arange(1.0, m + 1)[:, None] / 64, np.array([[0.5, -2.0, 3.0]])
    for one in (np.full((1, 1), 0.25), row, block):
        for other in (np.full((1, 1), 0.125), block):
            c, tol = R.gemm(a, np.broadcast_to(one, (m, 3)), b, np.broadcast_to(other, (11, 3)), None, torch.finfo(torch.float32).eps)
            R.close(values(ops.fp8_gemm(R.f8(a), dev(one).expand(m, 3), R.f8(b), dev(other).expand(11, 3))), c, tol)


@pytest.mark.parametrize("m,n,pitch,ldc", [(3, 300, 1 << 31, (1 << 31) + 16), (130, 2500, 1 << 25, (1 << 25) + 4), (130, 2500, 1 << 25, (1 << 25) + 1)])
def test_gemm_offsets_beyond_32_bits(ops, m, n, pitch, ldc):
    """Rows of the activations and of the output that begin beyond 2^32 bytes and elements of their bases."""
    from dabnn_b200 import capi
    k = 272
    a, sa, b, sb, bias = operands(m, n, k, 21)
    c, tol = R.gemm(a, sa, b, sb, bias, torch.finfo(torch.float32).eps)
    wide = torch.empty((m - 1) * pitch + k, dtype=torch.float8_e4m3fn, device="cuda").as_strided((m, k), (pitch, 1))
    wide.copy_(R.f8(a))
    s, t, q = dev(sa), dev(sb), R.f8(b)
    out = torch.empty((m - 1) * ldc + n, device="cuda").as_strided((m, n), (ldc, 1))
    capi.check(capi.load().dabnn_fp8_gemm(wide.data_ptr(), pitch, s.data_ptr(), *s.stride(), q.data_ptr(), q.stride(0), t.data_ptr(), *t.stride(),
                                          dev(bias).data_ptr(), out.data_ptr(), 0, ldc, m, n, k, ops._stream()))
    R.close(values(out), c, tol)


@pytest.mark.parametrize("m,n", [(4, 300), (90, 300), (300, 300)])
def test_gemm_special_values(ops, m, n):
    """NaN bytes reach the outputs of their row and column and no other; scales of zero; blocks of zeros."""
    k = 400
    a, sa, b, sb, _ = operands(m, n, k, 6, powers=True)
    a[m // 2, 130:250] = 0
    c, tol = R.gemm(a, sa, b, sb, None, torch.finfo(torch.float32).eps)
    qa, qb = R.f8(a), R.f8(b)
    qa[1, 399] = float("nan")
    qb[257, 3] = float("nan")
    got = values(ops.fp8_gemm(qa, dev(sa), qb, dev(sb)))
    expected = c.copy()
    expected[1, :] = np.nan
    expected[:, 257] = np.nan
    R.close(got, expected, tol)
    sz = sa.copy()
    sz[2, :] = 0
    got = values(ops.fp8_gemm(R.f8(a), dev(sz), R.f8(b), dev(sb)))
    assert (got[2] == 0).all()


@pytest.mark.parametrize("m,n,k", [(2, 1000, 4096), (40, 520, 2048), (300, 700, 512)])
def test_gemm_is_deterministic_and_row_independent(ops, m, n, k):
    """The same bits each time; a row's results do not depend on what the other rows hold."""
    a, sa, b, sb, bias = operands(m, n, k, 8)
    args = (R.f8(b), dev(sb), dev(bias))
    first = ops.fp8_gemm(R.f8(a), dev(sa), *args)
    for _ in range(3):
        assert torch.equal(ops.fp8_gemm(R.f8(a), dev(sa), *args), first)
    other, so, _, _, _ = operands(m, n, k, 9)
    other[1], so[1] = a[1], sa[1]
    assert torch.equal(ops.fp8_gemm(R.f8(other), dev(so), *args)[1], first[1])


def test_gemm_leading_dimensions_streams_and_graphs(ops):
    """[2, 3, K] activations; a side stream; capture and replay with new contents, two graphs in turn."""
    g = torch.Generator().manual_seed(1)
    x, w = torch.randn((2, 3, 320), generator=g).cuda(), torch.randn((150, 320), generator=g).cuda()
    q, s = ops.fp8_quantize(x)
    b, t = ops.fp8_quantize_weights(w)
    plain = ops.fp8_gemm(q, s, b, t)
    assert plain.shape == (2, 3, 150)
    assert torch.equal(ops.fp8_gemm(q[1, 2], s[1, 2], b, t), plain[1, 2])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = ops.fp8_gemm(q, s, b, t)
    side.synchronize()
    assert torch.equal(other, plain)
    graphs = []
    xs = [x.clone(), x.clone()]
    for xi in xs:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            qi, si = ops.fp8_quantize(xi)
            ci = ops.fp8_gemm(qi, si, b, t)
        graphs.append((graph, ci))
    for i in (0, 1, 0):
        xs[i].mul_(-2.0)
        expected = ops.fp8_gemm(*ops.fp8_quantize(xs[i]), b, t)
        graphs[i][0].replay()
        assert torch.equal(graphs[i][1], expected)


@pytest.mark.parametrize("m,n,k", [(5, 300, 2048), (100, 520, 512), (1000, 2600, 384)])
def test_gemm_scales_without_a_number(ops, m, n, k):
    """A scale that is NaN or infinite reaches the outputs of its row, or of its 128 columns, and no other."""
    a, sa, b, sb, bias = operands(m, n, k, 12, powers=True)
    c, tol = R.gemm(a, sa, b, sb, bias, torch.finfo(torch.float32).eps)
    da, db = dev(sa), dev(sb)
    da[m - 1, k // 128 - 1] = float("nan")
    db[1, 0] = float("nan")
    got = values(ops.fp8_gemm(R.f8(a), da, R.f8(b), db, dev(bias)))
    expected = c.copy()
    expected[m - 1] = np.nan
    expected[:, 128:256] = np.nan
    R.close(got, expected, tol)


@pytest.mark.parametrize("m", [4, 200, 3000])
def test_launches_one_after_the_other(ops, m):
    """Each call of a chain reads what the call before wrote, in memory that the allocator hands round, with nothing in between:
    the same bits as with a synchronisation after every call."""
    g = torch.Generator().manual_seed(m)
    w = [(torch.randn((384, 384), generator=g) * 384 ** -0.5).cuda() for _ in range(3)]
    x0 = torch.randn((m, 384), generator=g).cuda()

    def chain(wait):
        x, out = x0.clone(), []
        for i in range(24):
            wq, ws = ops.fp8_quantize_weights(w[i % 3])
            q, s = ops.fp8_quantize(x)
            x = ops.fp8_gemm(q, s, wq, ws)
            out.append(ops.logprobs(x, None, 3)[4])
            if wait:
                torch.cuda.synchronize()
        return x, torch.stack(out)

    for a, b in zip(chain(True), chain(False)):
        assert torch.equal(a, b)


def test_two_streams_at_once(ops):
    """Calls of every shape side by side: they share no memory."""
    shapes = [(1, 2000, 4096), (40, 1000, 2048), (300, 1500, 768), (1500, 2600, 512)]
    sets = []
    for m, n, k in shapes:
        a, sa, b, sb, bias = operands(m, n, k, m)
        args = (R.f8(a), dev(sa), R.f8(b), dev(sb), dev(bias))
        sets.append((args, ops.fp8_gemm(*args)))
    torch.cuda.synchronize()
    streams, results = [torch.cuda.Stream() for _ in range(2)], []
    for round_ in range(6):
        for j, st in enumerate(streams):
            with torch.cuda.stream(st):
                for i in range(len(sets)):
                    args, expected = sets[(i + j * 2 + round_) % len(sets)]
                    results.append((ops.fp8_gemm(*args), expected))
    torch.cuda.synchronize()
    for got, expected in results:
        assert torch.equal(got, expected)


def test_a_wait_that_gave_up_is_reported(ops):
    """The code is planted from the host; no kernel is made to stall."""
    from dabnn_b200 import capi
    lib = capi.load()
    assert ops.engine_status() == 0
    capi.check(lib.dabnn_debug_raise_engine_status(3, 54))
    assert ops.engine_status() == 54
    capi.check(lib.dabnn_debug_raise_engine_status(3, 0))
    assert ops.engine_status() == 0
    assert lib.dabnn_debug_raise_engine_status(4, 1) == 1


# ---------------------------------------------------------------------------------------------- the head as a whole
@pytest.mark.parametrize("m,classes,k", [(1, 1000, 512), (64, 1000, 512), (200, 365, 1100)])
def test_classifier_head(ops, m, classes, k):
    """Features -> bytes -> logits -> scores, each step against the 64-bit form of what went into it."""
    g = torch.Generator().manual_seed(m + classes)
    x, w, bias = torch.randn((m, k), generator=g).cuda(), (torch.randn((classes, k), generator=g) * 4 * k ** -0.5).cuda(), torch.randn(classes, generator=g).cuda()
    labels = torch.randint(0, classes, (m,), generator=g).cuda()
    wq, ws = ops.fp8_quantize_weights(w)
    q, s = ops.fp8_quantize(x)
    logits = ops.fp8_gemm(q, s, wq, ws, bias)
    lp, rank, entropy, tlp, ti = ops.logprobs(logits, labels, 5)
    c, tol = R.gemm(*R.quantize(values(x), 1), *R.quantize(values(w), 128), values(bias), torch.finfo(torch.float32).eps)
    R.close(values(logits), c, tol)
    expected, tols = R.logprobs(values(logits), labels.cpu().numpy(), 5)
    for got, e, t in zip((lp, entropy, tlp), (expected[0], expected[2], expected[3]), tols):
        R.close(got.cpu(), e, t)
    np.testing.assert_array_equal(rank.cpu(), expected[1])
    np.testing.assert_array_equal(ti.cpu(), expected[4])
    # the bytes cost little: rounding is off by at most 2^-4 of a value or half of 2^-9 of the block's scale
    exact = values(x) @ values(w).T + values(bias)
    ax, aw = np.abs(values(x)), np.abs(values(w))
    sx = np.repeat(R.quantize(values(x), 1)[1], 128, 1)[:, :k] * 2.0 ** -10
    sw = np.repeat(np.repeat(R.quantize(values(w), 128)[1], 128, 0)[:classes], 128, 1)[:, :k] * 2.0 ** -10
    ex, ew = np.maximum(ax * 2.0 ** -4, sx), np.maximum(aw * 2.0 ** -4, sw)
    R.close(values(logits), exact, tol + ex @ aw.T + ax @ ew.T + ex @ ew.T)


# ---------------------------------------------------------------------------------------------- results as another launch's constants
def test_results_as_parameters_of_the_next_launch(ops):
    """Factors, offsets, biases and weights that the launch just before computes (a product of few rows, which leaves most SMs
    free; a pooling): the same bits as with a synchronisation between the two."""
    g = torch.Generator().manual_seed(41)
    cout, k = 128, 16384
    x8 = ops.binarize_u8(torch.randn((2, 14, 14, 128), generator=g).cuda())
    bits = ops.pack_mat(torch.randn((cout, 3, 3, 128), generator=g).cuda())
    we = ops.bconv_u8_expand_weights(bits, cout, 18)
    image, stem = torch.randn((1, 224, 224, 3), generator=g).cuda(), torch.randn((64, 7, 7, 3), generator=g).cuda()
    assert ops.fconv_maxpool_supported(1, 224, 224, 3, 64, 7, 7, 3, 3, 2, 2)
    w = [ops.fp8_quantize_weights((torch.randn((n, k), generator=g) * k ** -0.5).cuda()) for n in (cout, 64, 64 * 7 * 7 * 3)]
    features = [ops.fp8_quantize(torch.randn((2, k), generator=g).cuda()) for _ in range(4)]
    thin = [ops.fp8_quantize(torch.randn((2, k), generator=g).cuda()) for _ in range(4)]
    maps = [torch.randn((1, 8, 8, cout), generator=g).cuda() for _ in range(4)]

    def chain(wait):
        out = []

        def sync(t):
            if wait:
                torch.cuda.synchronize()
            return t

        for i in range(12):
            f = features[i % 4]
            c = sync(ops.fp8_gemm(*f, *w[0]))
            out.append(ops.bconv_u8_block(x8, we, cout, 3, 3, 1, 1, 1, 1, c[0], c[1])[0])
            c = sync(ops.fp8_gemm(*f, *w[0]))
            out.append(ops.bconv_u8_block(x8, we, cout, 3, 3, 1, 1, 2, 2, c[1], c[0])[0])
            c = sync(ops.avepool(maps[i % 4], 8, 8, 0, 0, 8, 8)).view(cout)
            out.append(ops.bconv_u8_block(x8, we, cout, 3, 3, 1, 1, 1, 1, c, c)[0])
            c = sync(ops.fp8_gemm(*f, *w[1]))
            out.append(ops.fconv_maxpool(image, stem, c[1], 3, 3, 2, 2, c[0], c[1])[0])
            c = sync(ops.fp8_gemm(*f, *w[1]))
            out.append(ops.fconv(image, stem, c[0], 3, 3, 2, 2))
            c = sync(ops.fp8_gemm(*thin[i % 4], *w[2]))
            out.append(ops.fconv(image, c[0].view(64, 7, 7, 3), None, 3, 3, 2, 2))
            sync(None)
        return out

    for got, expected in zip(chain(False), chain(True)):
        assert torch.equal(got, expected)


@pytest.mark.parametrize("m,n,k,places", [
    (1, 300, 300, [(0, 0)]), (1, 8192, 4096, [(0, 0), (1, 3)]), (20, 700, 2048, [(0, 1)]), (50, 600, 4096, [(0, 0), (0, 7)]), (50, 600, 1280, [(2, 0)]),
    (200, 4100, 2048, [(0, 0), (2, 0)]), (1000, 2600, 4096, [(0, 0), (0, 1), (1, 1), (4, 0), (7, 1)]), (2300, 4200, 1100, [(1, 0), (3, 1), (4, 0), (5, 1)])])
def test_winding_down_after_a_wait_that_gave_up(ops, m, n, k, places):
    """Every kind of tile, either CTA of a pair, early and late: the call ends, its code is there to be read, and what follows
    it in the stream, at once, is as it always is.  (A wait is declared to have run out; nothing is made to stall.)"""
    from dabnn_b200 import capi
    lib = capi.load()
    a, sa, b, sb, bias = operands(m, n, k, 17)
    args = (R.f8(a), dev(sa), R.f8(b), dev(sb), dev(bias))
    expected = ops.fp8_gemm(*args)
    assert ops.engine_status() == 0
    try:
        for group, rank in places:
            for _ in range(3):
                capi.check(lib.dabnn_debug_fp8_give_up(group, rank))
                ops.fp8_gemm(*args)
                capi.check(lib.dabnn_debug_fp8_give_up(-1, 0))
                after = ops.fp8_gemm(*args)
                torch.cuda.synchronize()
                assert ops.engine_status() == 55, (group, rank)
                capi.check(lib.dabnn_debug_raise_engine_status(3, 0))
                assert torch.equal(after, expected), (group, rank)
    finally:
        capi.check(lib.dabnn_debug_fp8_give_up(-1, 0))
    assert lib.dabnn_debug_fp8_give_up(-2, 0) == 1 and lib.dabnn_debug_fp8_give_up(0, 8) == 1 and lib.dabnn_debug_fp8_give_up(0, -1) == 1


def test_collecting_the_code_of_a_wait_that_gave_up(ops):
    """Codes planted from the host: reading leaves them, collecting clears the words of every kernel, a Net's run only its own."""
    from dabnn_b200 import capi
    lib = capi.load()
    for which, code in ((0, 3), (1, 12), (2, 21), (3, 53)):
        capi.check(lib.dabnn_debug_raise_engine_status(which, code))
        assert ops.engine_status() == code and ops.engine_status() == code
        assert ops.engine_status(collect=True) == code
        assert ops.engine_status(collect=True) == 0 and ops.engine_status() == 0
    for which, code in ((0, 3), (3, 51)):
        capi.check(lib.dabnn_debug_raise_engine_status(which, code))
    assert ops.engine_status(collect=True) == 3 and ops.engine_status() == 0        # one answer for all that happened before it
    capi.check(lib.dabnn_debug_raise_engine_status(3, 52))
    from dabnn_b200.bireal import OUTPUT_BLOB, build_bireal18
    from dabnn_b200.dab_format import write_dab
    from dabnn_b200.net import Net
    net = Net.create()
    net.max_batch = 1
    net.read_buf(write_dab(build_bireal18(image_hw=32, num_classes=10)))
    net.run(torch.randn((1, 32, 32, 3), device="cuda")).get_blob(OUTPUT_BLOB)
    net.close()
    assert ops.engine_status(collect=True) == 52 and ops.engine_status() == 0
    # a code that a kernel itself has raised
    a, sa, b, sb, bias = operands(3, 300, 300, 18)
    capi.check(lib.dabnn_debug_fp8_give_up(0, 0))
    try:
        ops.fp8_gemm(R.f8(a), dev(sa), R.f8(b), dev(sb))
    finally:
        capi.check(lib.dabnn_debug_fp8_give_up(-1, 0))
    assert ops.engine_status(collect=True) == 55 and ops.engine_status() == 0


# ---------------------------------------------------------------------------------------------- paths of the product that other sizes do not reach
@pytest.mark.parametrize("m,n,k", [(1, 40001, 300), (20, 50000, 144), (64, 60000, 640), (33, 80000, 200), (2, 39000, 1700), (7, 76100, 1), (16, 38000, 2050)])
def test_gemm_few_rows_by_many_columns(ops, m, n, k):
    """More tiles than CTAs of few rows at once: stages, accumulators and factors go on from one tile to the next, with counts of
    blocks that are odd and no multiple of a group of factors."""
    check_gemm(ops, m, n, k)


@pytest.mark.parametrize("out", TYPES)
@pytest.mark.parametrize("m,n", [(130, 2501), (300, 1003), (900, 1301), (1900, 2502)])
def test_gemm_rows_that_end_inside_16_bytes(ops, m, n, out):
    """An output whose pitch is a multiple of 16 bytes and whose rows are not: nothing behind a row or the last row is written."""
    from dabnn_b200 import capi
    k, dt = 200, TYPES[out]
    a, sa, b, sb, bias = operands(m, n, k, 19)
    if out == "f16":
        sa, sb = sa * 2.0 ** -14, sb * 2.0 ** -6
    c, tol = R.gemm(a, sa, b, sb, bias, torch.finfo(dt).eps)
    ldc = (n + 15) // 16 * 16 + 16
    store = torch.full((m + 3, ldc), -5.0, dtype=dt, device="cuda")
    qa, qb, s, t, bv = R.f8(a), R.f8(b), dev(sa), dev(sb), dev(bias)
    capi.check(capi.load().dabnn_fp8_gemm(qa.data_ptr(), qa.stride(0), s.data_ptr(), *s.stride(), qb.data_ptr(), qb.stride(0), t.data_ptr(), *t.stride(),
                                          bv.data_ptr(), store.data_ptr(), {"f32": 0, "f16": 1, "bf16": 2}[out], ldc, m, n, k, ops._stream()))
    R.close(values(store[:m, :n]), c, tol + (2.0 ** -25 if out == "f16" else 0.0))
    store[:m, :n] = -5
    assert (store == -5).all()


@pytest.mark.parametrize("first", ["head", "bytes", "floats"])
def test_first_calls_of_a_process_inside_a_capture(first):
    """Nothing has to be called before a capture: each kind of tile and of scoring is captured by the first call it ever has, and so are
    the other kernels that load through tensor maps."""
    import subprocess
    import sys
    from pathlib import Path
    program = """
import torch
from dabnn_b200 import ops
g = torch.Generator(device="cuda").manual_seed(2)
sets = []
for m, n, k, c in ((1, 300, 300, 70), (1, 8192, 4096, 20000), (20, 700, 2048, 9000), (50, 600, 1280, 1000), (200, 4100, 512, 5000), (1000, 2600, 300, 300)):
    x, w = torch.randn((m, k), device="cuda", generator=g), torch.randn((n, k), device="cuda", generator=g)
    z = torch.randn((m, c), device="cuda", generator=g)
    labels = torch.randint(0, c, (m,), device="cuda", generator=g)
    sets.append((x, w, z, labels))
x8, we = torch.randint(0, 2, (1, 16, 16, 64), dtype=torch.uint8, device="cuda"), torch.zeros(1 << 20, dtype=torch.uint8, device="cuda")
image, weight = torch.randn((1, 16, 16, 64), device="cuda", generator=g), torch.randn((64, 3, 3, 64), device="cuda", generator=g)
torch.cuda.synchronize()
def run():
    if FIRST == "bytes":
        return [ops.bconv_u8_block(x8, we, 64, 3, 3, 1, 1, 1, 1)[0]]
    if FIRST == "floats":
        return [ops.fconv(image, weight, None, 1, 1, 1, 1)]
    out = []
    for x, w, z, labels in sets:
        q, s = ops.fp8_quantize(x)
        b, t = ops.fp8_quantize_weights(w)
        out += [s, t, ops.fp8_gemm(q, s, b, t), ops.fp8_gemm(q, s, b, t, None, torch.bfloat16), *ops.logprobs(z, labels, 5), *ops.logprobs(z, labels, 0)[:3]]
    return out
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    captured = run()
graph.replay()
for a, b in zip(captured, run()):
    assert torch.equal(a, b)
assert ops.engine_status() == 0
"""
    done = subprocess.run([sys.executable, "-c", f"FIRST = {first!r}\n" + program], cwd=Path(__file__).resolve().parent.parent, capture_output=True, text=True, timeout=300)
    assert done.returncode == 0, done.stdout[-2000:] + done.stderr[-4000:]


@pytest.mark.parametrize("m", [2, 30, 60, 200, 900])
@pytest.mark.parametrize("k", [1, 13, 100, 129, 257, 1100])
def test_gemm_reads_nothing_behind_a_row(ops, m, k):
    """Rows of a length that is no multiple of 16 bytes, NaN in all that lies behind them up to the pitch, behind the last row and
    in front of the first."""
    n = 2301
    a, sa, b, sb, bias = operands(m, n, k, 29)
    c, tol = R.gemm(a, sa, b, sb, bias, torch.finfo(torch.float32).eps)

    def surrounded(v):
        store = torch.full((v.shape[0] + 2, (k + 15) // 16 * 16), 0x7f, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn)
        store[1:-1, :k] = R.f8(v)
        return store[1:-1, :k]

    R.close(values(ops.fp8_gemm(surrounded(a), dev(sa), surrounded(b), dev(sb), dev(bias))), c, tol)


@pytest.mark.parametrize("k", [100, 256])
def test_gemm_of_slices_of_leading_dimensions(ops, k):
    """Slices of every dimension of quantised activations, whose rows begin on 16-byte boundaries whether they lie at equal steps or not."""
    g = torch.Generator().manual_seed(k)
    q, s = ops.fp8_quantize(torch.randn((3, 5, 4, k), generator=g).cuda())
    b, t = ops.fp8_quantize_weights(torch.randn((70, k), generator=g).cuda())
    whole = ops.fp8_gemm(q, s, b, t)
    for at in ((slice(None), slice(0, -1)), (slice(None), 2), (slice(None), slice(None), slice(1, 3)), (slice(1, 3), slice(1, 4), slice(0, 2)), (2, slice(1, 5, 2)),
               (slice(None), slice(0, 0)), (0, 1, 2)):
        assert torch.equal(ops.fp8_gemm(q[at], s[at], b, t), whole[at])
    assert torch.equal(ops.fp8_gemm(q.transpose(0, 2), s.transpose(0, 2), b, t), whole.transpose(0, 2))
