"""Scoring of logits against its 64-bit form: kernel level and on a Net's output."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

import head_reference as R  # noqa: E402

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
INF, NAN = float("inf"), float("nan")


@pytest.fixture(scope="module")
def ops():
    from dabnn_b200 import ops as o
    return o


def check(ops, logits, labels, top):
    """logits on the device, labels a list or None"""
    lab = None if labels is None else torch.tensor(labels, dtype=torch.int64)
    got = ops.logprobs(logits, None if lab is None else lab.cuda(), top)
    (lp, rank, ent, tlp, ti), (tol, etol, ttol) = R.logprobs(logits.float().cpu().numpy(), None if lab is None else lab.numpy(), top)
    if labels is None:
        assert got[0] is None and got[1] is None
    else:
        np.testing.assert_array_equal(got[1].cpu(), rank)
        R.close(got[0].cpu(), lp, tol)
    R.close(got[2].cpu(), ent, etol)
    if top:
        np.testing.assert_array_equal(got[4].cpu(), ti)
        R.close(got[3].cpu(), tlp, ttol)
    else:
        assert got[3] is None and got[4] is None


def rows_of(rows, classes, seed, kind, spread=3.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn((rows, classes), generator=g) * spread).to(TYPES[kind]).cuda(), torch.randint(0, classes, (rows,), generator=g).tolist()


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("classes", [1, 2, 7, 31, 32, 33, 100, 255, 1000, 1023, 1024, 1025, 2048, 4097, 8191, 8192, 8193])
def test_logprobs(ops, classes, kind):
    for rows in (1, 3, 40):
        x, labels = rows_of(rows, classes, classes + rows, kind)
        for top in sorted({0, 1, min(5, classes), min(20, classes), min(64, classes)}):
            check(ops, x, labels, top)
    check(ops, x, None, min(3, classes))


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("rows,classes,top", [(1, 131072, 20), (2, 50000, 5), (3, 262144, 64), (1, 65537, 32), (150, 20001, 8), (400, 12345, 5)])
def test_logprobs_wide(ops, rows, classes, top, kind):
    x, labels = rows_of(rows, classes, classes + rows, kind)
    check(ops, x, labels, top)


def test_logprobs_many_rows(ops):
    x, labels = rows_of(5000, 10, 1, "f32")
    check(ops, x, labels, 3)
    x, labels = rows_of(1024, 1000, 2, "f32")
    check(ops, x, labels, 5)


@pytest.mark.parametrize("kind,classes,top", [("bf16", 4500, 8), ("f32", 4200, 0), ("f16", 4301, 40)])
def test_logprobs_many_wide_rows(ops, kind, classes, top):
    """Enough rows for a warp each."""
    x, labels = rows_of(3700, classes, 5, kind)
    check(ops, x, labels, top)


def test_two_streams_at_once(ops):
    sets = []
    for rows, classes, top in ((1, 100000, 20), (700, 1000, 5), (3, 30000, 64), (150, 9000, 8)):
        x, labels = rows_of(rows, classes, rows, "bf16")
        lab = torch.tensor(labels).cuda()
        sets.append((x, lab, top, ops.logprobs(x, lab, top)))
    torch.cuda.synchronize()
    streams, results = [torch.cuda.Stream() for _ in range(2)], []
    for round_ in range(6):
        for j, st in enumerate(streams):
            with torch.cuda.stream(st):
                for i in range(len(sets)):
                    x, lab, top, expected = sets[(i + j * 2 + round_) % len(sets)]
                    results.append((ops.logprobs(x, lab, top), expected))
    torch.cuda.synchronize()
    for got, expected in results:
        for a, b in zip(got, expected):
            assert torch.equal(a, b)


@pytest.mark.parametrize("classes", [70, 1000, 9000, 40000])
@pytest.mark.parametrize("kind", TYPES)
def test_ties_and_orders(ops, classes, kind):
    """Constant rows, few distinct values, both zeros, rising and falling rows, everything large at the end."""
    x = torch.zeros((8, classes))
    x[1] = 3.0
    x[2] = torch.arange(classes) % 3
    x[3, 1::2] = -0.0
    x[4] = torch.arange(classes) / classes * 8
    x[5] = -torch.arange(classes) / classes * 8
    x[6, -5:] = 7.0
    x[7] = (torch.arange(classes) * 7919 % 101).float()
    for label in (0, classes // 2, classes - 1):
        check(ops, x.to(TYPES[kind]).cuda(), [label] * 8, 5)
    check(ops, x.to(TYPES[kind]).cuda(), [classes - 3] * 8, 64)


@pytest.mark.parametrize("classes", [70, 1000, 9000, 140000])
@pytest.mark.parametrize("kind", TYPES)
def test_barred_classes_and_special_values(ops, classes, kind):
    """-inf, the type's lowest value, +inf and NaN: rows with few classes left, one, none."""
    lowest = torch.finfo(TYPES[kind]).min
    g = torch.Generator().manual_seed(classes)
    x = (torch.randn((14, classes), generator=g) * 3).to(TYPES[kind])
    x[0] = -INF
    x[1] = -INF
    x[1, classes - 2] = 1.5
    x[2, 3:] = -INF
    x[3, ::2] = -INF
    x[4] = lowest
    x[5, 2:] = lowest
    x[6, classes // 3] = NAN
    x[7, classes // 3] = INF
    x[8] = NAN
    x[9] = -INF
    x[9, 5] = NAN
    x[10, 5], x[10, 6] = INF, -INF
    x[11] = torch.finfo(TYPES[kind]).max
    x[12, 1:] = lowest
    x[12, 0] = torch.finfo(TYPES[kind]).max
    x[13, 0::2], x[13, 1::2] = -NAN, NAN
    labels = [0, classes - 2, 1, 2, classes - 1, 7, 3, classes // 3, 4, 5, 6, 9, 1, 2]
    check(ops, x.cuda(), labels, 8)
    check(ops, x.cuda(), labels, 0)


@pytest.mark.parametrize("classes", [5, 1000, 20000])
def test_labels_outside(ops, classes):
    x, _ = rows_of(6, classes, 3, "f32")
    check(ops, x, [-1, -100, classes, classes + 7, 2**62, -2**63], 2)
    check(ops, x, [0, classes - 1, -1, classes, 1, 2], 0)


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("classes", [100, 1000, 9001])
def test_strided_rows_and_offsets(ops, kind, classes):
    """Row pitches and bases off every vector boundary; what lies around the rows is not read into them."""
    store = torch.full((9, classes + 37), NAN, dtype=TYPES[kind]).cuda()
    for first in (0, 1, 2, 4, 8, 13):
        x = store[:, first:first + classes]
        x.copy_(rows_of(9, classes, first, kind)[0])
        check(ops, x, list(range(9)), 6)
        x.fill_(NAN)


def test_shapes(ops):
    x, labels = rows_of(24, 50, 1, "bf16")
    lab = torch.tensor(labels).cuda()
    flat = ops.logprobs(x, lab, 4)
    deep = ops.logprobs(x.view(2, 3, 4, 50), lab.view(2, 3, 4), 4)
    for f, d in zip(flat, deep):
        assert d.shape[:3] == (2, 3, 4) and torch.equal(f, d.reshape(f.shape))
    one = ops.logprobs(x[5], lab[5], 4)
    for f, d in zip(flat, one):
        assert torch.equal(f[5], d)
    for t in ops.logprobs(torch.empty((0, 50), device="cuda"), torch.empty(0, dtype=torch.int64, device="cuda"), 4):
        assert t.shape[0] == 0


@pytest.mark.parametrize("rows,classes", [(2, 1000), (3, 30000)])
def test_same_bits_alone_and_in_a_batch(ops, rows, classes):
    x, labels = rows_of(rows, classes, 7, "f32")
    lab = torch.tensor(labels).cuda()
    first = ops.logprobs(x, lab, 5)
    for _ in range(3):
        for a, b in zip(first, ops.logprobs(x, lab, 5)):
            assert torch.equal(a, b)


@pytest.mark.parametrize("rows,classes", [(3, 1000), (2, 40000)])
def test_streams_and_graphs(ops, rows, classes):
    x, labels = rows_of(rows, classes, 9, "f32")
    lab = torch.tensor(labels).cuda()
    plain = ops.logprobs(x, lab, 5)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = ops.logprobs(x, lab, 5)
    side.synchronize()
    for a, b in zip(plain, other):
        assert torch.equal(a, b)
    xs, graphs = [x.clone(), x.clone()], []
    for xi in xs:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = ops.logprobs(xi, lab, 5)
        graphs.append((graph, out))
    for i in (0, 1, 0):
        xs[i].mul_(-0.5)
        graphs[i][0].replay()
        for a, b in zip(graphs[i][1], ops.logprobs(xs[i], lab, 5)):
            assert torch.equal(a, b)


def test_offsets_beyond_32_bits(ops):
    """Rows that begin beyond 2^32 elements of the base."""
    classes, pitch = 1000, 1 << 31
    store = torch.zeros((2 * pitch + classes) // 2 * 2, dtype=torch.bfloat16, device="cuda")
    x = store.as_strided((3, classes), (pitch, 1))
    x.copy_(rows_of(3, classes, 11, "bf16")[0])
    check(ops, x, [1, 2, 3], 5)


def test_net_logprobs(ops):
    """The scores of a Net's own logits: as the kernel-level call gives them, in either plan, batches of several sizes."""
    from dabnn_b200.bireal import OUTPUT_BLOB, build_bireal18
    from dabnn_b200.capi import DabnnError
    from dabnn_b200.dab_format import write_dab
    from dabnn_b200.net import Net
    rng = np.random.default_rng(0)
    model = write_dab(build_bireal18(image_hw=64, num_classes=100))
    for optimize in (True, False):
        net = Net.create()
        net.max_batch, net.optimize = 5, optimize
        net.read_buf(model)
        with pytest.raises(DabnnError):
            net.logprobs(OUTPUT_BLOB)                       # nothing has been run
        for batch in (2, 5, 1):
            net.run(rng.normal(0, 1, (batch, 64, 64, 3)).astype(np.float32))
            logits = net.get_blob(OUTPUT_BLOB).reshape(batch, 100)
            labels = rng.integers(0, 100, batch)
            lp, rank, ent, tlp, ti = net.logprobs(OUTPUT_BLOB, labels, top=5)
            for got, e in zip((lp, rank, ent, tlp, ti), ops.logprobs(torch.from_numpy(logits).cuda(), torch.from_numpy(labels).cuda(), 5)):
                np.testing.assert_array_equal(got, e.cpu().numpy())
            assert (ti[:, 0] == logits.argmax(1)).all()
            only = net.logprobs(OUTPUT_BLOB)
            assert only[0] is None and only[4] is None
            np.testing.assert_array_equal(only[2], ent)
        with pytest.raises(DabnnError):
            net.logprobs(OUTPUT_BLOB, top=65)
        with pytest.raises(KeyError):
            net.logprobs("no such blob")
        with pytest.raises(ValueError):
            net.logprobs(OUTPUT_BLOB, labels=[1, 2, 3])
        net.close()


def test_rows_of_hundreds_of_millions_of_classes(ops):
    """One class far above 4 10^8 equal ones, in the part of the row that is joined last: each part of the row before it holds
    a sum of e^0 of 5 10^7, whose product with the distance between the maxima is beyond fp32."""
    classes, top = 400_000_000, 7 * 1024 + 5
    x = torch.full((1, classes), -1e30, dtype=torch.bfloat16, device="cuda")
    x[0, top] = 1e30
    low, high = float(x[0, 0]), float(x[0, top])
    lp, rank, ent, tlp, ti = ops.logprobs(x, torch.tensor([top], device="cuda"), 2)
    assert lp.item() == 0 and rank.item() == 0 and ent.item() == 0
    assert ti.tolist() == [[top, 0]] and tlp[0, 0].item() == 0
    R.close(tlp[0, 1:].cpu(), [low - high], 2.0 ** -23 * (high - low))
    x[0, top] = -1e30                                                  # all alike
    lp, rank, ent, tlp, ti = ops.logprobs(x, torch.tensor([top], device="cuda"), 2)
    # 4e8 terms of 1: sums of whole numbers below 2^24 in a lane, 64 lanes' worth of roundings above; a logarithm
    expected = np.log(float(classes))
    tol = 72 * 2.0 ** -24 + expected * 2.0 ** -22
    R.close(lp.cpu(), [-expected], tol)
    R.close(ent.cpu(), [expected], tol)
    assert rank.item() == top and ti.tolist() == [[0, 1]]
    R.close(tlp.cpu(), [[-expected, -expected]], tol)


def test_net_logprobs_refuses_what_logprobs_refuses(ops):
    """A label's outputs without labels, alternatives without a place for them: refused, nothing is written; what may be left out
    is left out."""
    import ctypes as C
    from dabnn_b200 import capi
    from dabnn_b200.bireal import OUTPUT_BLOB, build_bireal18
    from dabnn_b200.dab_format import write_dab
    from dabnn_b200.net import Net
    lib = capi.load()
    net = Net.create()
    net.max_batch = 3
    net.read_buf(write_dab(build_bireal18(image_hw=32, num_classes=10)))
    net.run(torch.randn((3, 32, 32, 3), device="cuda"))
    logits = torch.from_numpy(net.get_blob(OUTPUT_BLOB).reshape(3, 10)).cuda()
    labels = np.array([1, 9, 4], np.int64)
    lab_dev = torch.from_numpy(labels).cuda()
    want = [t.cpu().numpy() for t in ops.logprobs(logits, torch.from_numpy(labels).cuda(), 2)]
    for given in range(64):
        lab, top = bool(given & 1), 2 if given & 2 else 0
        out = [np.full(3, -77.0, np.float32), np.full(3, -77, np.int64), np.full(3, -77.0, np.float32), np.full((3, 2), -77.0, np.float32), np.full((3, 2), -77, np.int64)]
        have = [bool(given & 4), bool(given & 8), True, bool(given & 16), bool(given & 32)]
        ptr = [o.ctypes.data_as(C.c_void_p) if h else None for o, h in zip(out, have)]
        rc = lib.dabnn_net_logprobs(net._h, OUTPUT_BLOB.encode(), labels.ctypes.data_as(C.c_void_p) if lab else None, *ptr, top)
        keep = [torch.from_numpy(o).cuda() for o in out]
        dev = [t.data_ptr() if h else None for t, h in zip(keep, have)]
        assert rc == lib.dabnn_logprobs(logits.data_ptr(), 0, 10, lab_dev.data_ptr() if lab else None, 3, 10, *dev, top, ops._stream())
        torch.cuda.synchronize()
        refused = (not lab and (have[0] or have[1])) or (top and not (have[3] and have[4]))
        assert (rc == 1) if refused else (rc == 0), given
        for i, o in enumerate(out):
            written = not refused and have[i] and (i < 3 or top)
            np.testing.assert_array_equal(o, want[i] if written else np.full_like(o, -77))
    net.close()


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("batch,length,classes,top", [(3, 5, 1000, 5), (2, 3, 40001, 20), (700, 3, 301, 3), (40, 60, 4100, 0), (1, 7, 50, 2), (5, 2, 9001, 64)])
def test_sequences_where_they_lie(ops, batch, length, classes, top, kind):
    """All positions but the last, of a vocabulary with padding, against the tokens that follow; what is not a row is NaN."""
    g = torch.Generator().manual_seed(batch * length + classes)
    store = torch.full((batch, length, classes + 3), NAN, dtype=TYPES[kind], device="cuda")
    tokens = torch.randint(0, classes, (batch, length), generator=g).cuda()
    x, labels = store[:, :-1, 1:classes + 1], tokens[:, 1:]
    x.copy_((torch.randn((batch, length - 1, classes), generator=g) * 3).cuda())
    tokens[:, 0] = 1 << 40
    (lp, rank, ent, tlp, ti), (tol, etol, ttol) = R.logprobs(x.float().cpu().numpy().reshape(-1, classes), labels.cpu().numpy().reshape(-1), top)
    lead = (batch, length - 1)
    for logits in (x, x.contiguous()):
        for lab in (labels, labels.contiguous()):
            got = ops.logprobs(logits, lab, top)
            assert got[0].shape == got[1].shape == got[2].shape == lead
            np.testing.assert_array_equal(got[1].cpu(), rank.reshape(lead))
            R.close(got[0].cpu(), lp.reshape(lead), tol.reshape(lead))
            R.close(got[2].cpu(), ent.reshape(lead), etol.reshape(lead))
            if top:
                np.testing.assert_array_equal(got[4].cpu(), ti.reshape(*lead, top))
                R.close(got[3].cpu(), tlp.reshape(*lead, top), ttol.reshape(*lead, top))
    R.close(ops.logprobs(x)[2].cpu(), ent.reshape(lead), etol.reshape(lead))


def test_groups_beyond_32_bits_and_groups_that_are_one(ops):
    """Groups that begin beyond 2^32 elements of the base; one sequence's logits for every sequence's tokens; refused shapes."""
    classes, pitch = 1000, 1 << 31
    store = torch.zeros(2 * pitch + 4 * classes, dtype=torch.bfloat16, device="cuda")
    x = store.as_strided((3, 2, classes), (pitch, classes + 8, 1))
    flat = rows_of(6, classes, 13, "bf16")[0]
    x.copy_(flat.view(3, 2, classes))
    tokens = torch.arange(12, device="cuda").view(3, 4) * 80
    got, want = ops.logprobs(x, tokens[:, 1:3], 5), R.logprobs(flat.float().cpu().numpy(), tokens[:, 1:3].reshape(-1).cpu().numpy(), 5)
    np.testing.assert_array_equal(got[1].cpu().reshape(-1), want[0][1])
    R.close(got[0].cpu().reshape(-1), want[0][0], want[1][0])
    np.testing.assert_array_equal(got[4].cpu().reshape(6, 5), want[0][4])
    one = flat[:4].view(1, 4, classes).expand(3, 4, classes)[:, :-1]
    got = ops.logprobs(one, tokens[:, 1:])
    for b in range(3):
        (lp, rank, _, _, _), (tol, _, _) = R.logprobs(flat[:3].float().cpu().numpy(), tokens[b, 1:].cpu().numpy(), 0)
        np.testing.assert_array_equal(got[1][b].cpu(), rank)
        R.close(got[0][b].cpu(), lp, tol)
    with pytest.raises(TypeError):
        ops.logprobs(x.transpose(1, 2))


def test_quantise_rows_with_a_pitch(ops):
    """Leading dimensions whose rows alone have a pitch: the same bytes as of a copy."""
    x = torch.randn((3, 5, 400), device="cuda")
    for part in (x[..., :300], x[..., 3:260], x[:, 2:3, 8:]):
        for a, b in zip(ops.fp8_quantize(part), ops.fp8_quantize(part.contiguous())):
            assert a.shape == b.shape and torch.equal(a.float(), b.float())


@pytest.mark.parametrize("kind,classes", [("bf16", 9000), ("f32", 9000), ("f16", 20000)])
def test_the_same_rows_alone_and_in_batches(ops, kind, classes):
    """A row scored by a cluster, by a CTA and by a warp, as the number of rows has it: the same ranks and classes, log
    probabilities and entropies within the bounds of each."""
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    x, labels = rows_of(16 * sms + 3, classes, 23, kind)
    x[5] = torch.arange(classes, device="cuda") % 7                     # ties everywhere
    lab = torch.tensor(labels).cuda()
    full = ops.logprobs(x, lab, 20)                                     # a warp a row
    (_, _, _, _, _), (tol, etol, ttol) = R.logprobs(x[:8].float().cpu().numpy(), np.array(labels[:8]), 20)
    for rows in (1, 3, 8, sms, 4 * sms):                                # eight CTAs a row, fewer, one
        part = ops.logprobs(x[:rows], lab[:rows], 20)
        assert torch.equal(part[1], full[1][:rows]) and torch.equal(part[4], full[4][:rows])
        n = min(rows, 8)
        for got, all_of_it, bound in ((part[0], full[0], tol), (part[2], full[2], etol), (part[3], full[3], ttol)):
            R.close(got[:n].cpu(), all_of_it[:n].cpu(), 2 * bound[:n])
        for r in (rows - 1, rows // 2):                                 # and alone
            one = ops.logprobs(x[r:r + 1], lab[r:r + 1], 20)
            assert torch.equal(one[1], full[1][r:r + 1]) and torch.equal(one[4], full[4][r:r + 1])


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("classes", [40, 1000, 9000])
def test_zeros_next_to_the_smallest_numbers(ops, classes, kind):
    """Both zeros are one value, the smallest subnormals of the type on either side are others: as labels, before and behind."""
    tiny = torch.finfo(TYPES[kind]).smallest_normal * torch.finfo(TYPES[kind]).eps
    few = torch.tensor([0.0, tiny, -0.0, -tiny, 2 * tiny, -2 * tiny, 0.0, -0.0]).to(TYPES[kind])
    assert few[1] > 0 and few[3] < 0 and (few.float()[1] / 2).to(TYPES[kind]) == 0
    x = few[torch.randint(0, 8, (24, classes), generator=torch.Generator().manual_seed(classes))]
    labels = [(i * classes) // 24 for i in range(24)]
    for i in range(8):
        x[3 * i, labels[3 * i]], x[3 * i + 1, labels[3 * i + 1]], x[3 * i + 2, labels[3 * i + 2]] = few[i], few[i], few[i]
    check(ops, x.cuda(), labels, 7)
    check(ops, x.cuda(), labels, 0)


def test_net_logprobs_of_pixels(ops):
    """A blob of several pixels an image: a row for each of them, labels and results in the blob's shape; labels that are no whole
    numbers are refused."""
    from dabnn_b200.bireal import OUTPUT_BLOB, build_bireal18
    from dabnn_b200.dab_format import write_dab
    from dabnn_b200.net import Net
    rng = np.random.default_rng(1)
    net = Net.create()
    net.max_batch, net.optimize = 3, False
    net.read_buf(write_dab(build_bireal18(image_hw=64, num_classes=10)))
    for batch in (3, 2):
        net.run(rng.normal(0, 1, (batch, 64, 64, 3)).astype(np.float32))
        for name in ("s1b1_add_out", "s3b4_add_out"):
            blob = net.get_blob(name)
            assert blob.shape[0] == batch and blob.shape[1] > 1
            labels = rng.integers(-1, blob.shape[3], blob.shape[:3])
            want = ops.logprobs(torch.from_numpy(blob).cuda(), torch.from_numpy(labels).cuda(), 3)
            for got, e in zip(net.logprobs(name, labels, 3), want):
                np.testing.assert_array_equal(got, e.cpu().numpy())
    for labels in ([0.0, 1.0], [True, False], ["1", "2"], [None, None]):
        with pytest.raises(TypeError):
            net.logprobs(OUTPUT_BLOB, labels)
    np.testing.assert_array_equal(net.logprobs(OUTPUT_BLOB, [1, 2])[1], net.logprobs(OUTPUT_BLOB, np.array([1, 2], np.uint8))[1])
    net.close()
