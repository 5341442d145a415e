"""Plain 64-bit forms of the 8-bit product with block scales and of the scoring of logits, with error bounds."""
import numpy as np
import torch

BLOCK = 128


def quantize(x, block_rows):
    """x [rows, k] (float64, CPU) -> (values of the e4m3 bytes, scales), from the definition; NaN where x is not finite."""
    x = np.asarray(x, np.float64)
    rows, k = x.shape
    nr, nk = -(-rows // block_rows), -(-k // BLOCK)
    q, scales = np.zeros_like(x), np.zeros((nr, nk))
    for i in range(nr):
        for j in range(nk):
            at = (slice(i * block_rows, (i + 1) * block_rows), slice(j * BLOCK, (j + 1) * BLOCK))
            b = x[at]
            finite = np.isfinite(b)
            top = np.abs(b[finite]).max(initial=0.0)
            e = -126
            while top > 448 * 2.0 ** e:
                e += 1
            v = np.where(finite, b, 0.0) / 2.0 ** e
            # e4m3: steps of 2^(p - 3) at 2^p, p >= -6
            step = 2.0 ** (np.maximum(np.frexp(v)[1] - 1, -6) - 3)
            q[at] = np.where(finite, np.rint(v / step) * step, np.nan)   # rint: ties to even
            scales[i, j] = 2.0 ** e
    return q, scales


def spread(q, scales, block_rows):
    """The values that bytes and scales stand for, float64."""
    rows, k = q.shape
    return q * np.repeat(np.repeat(scales, block_rows, 0)[:rows], BLOCK, 1)[:, :k]


def gemm(a, a_scales, b, b_scales, bias, out_eps):
    """float64 product and how far a kernel may be off.  a, b: values of the bytes; everything float64 numpy.

    Products of e4m3 values are exact in fp32.  A block's 128 products are added in fp32 (the tensor core truncates: a whole
    step of 2^-23 for each of at most 128 additions); then for each block the product of the scales and one fused
    multiply-add, each off by 2^-24; the bias and the rounding to the output's type (out_eps / 2 of the result)."""
    av, bv = spread(a, a_scales, 1), spread(b, b_scales, BLOCK)
    blocks = a_scales.shape[1]
    c = av @ bv.T
    size = np.abs(av) @ np.abs(bv).T
    tol = size * (128 * 2.0 ** -23 + (2 * blocks + 2) * 2.0 ** -24)
    if bias is not None:
        c = c + bias
        tol = tol + (np.abs(c) + size) * 2.0 ** -24
    return c, tol * (1 + out_eps) + np.abs(c) * out_eps / 2 + 2.0 ** -149


def logprobs(logits, labels, top):
    """float64 (logprob, rank, entropy, top logprob, top index) and bounds for the three float results.

    A kernel forms d = x - max (off by 2^-24 |d|), e = exp(d) (off by 2^-23 |d| for the product in its argument and 2^-22 for
    the function), sums of e and d e over at most n / 32 + 64 additions in a row, and a logarithm (2^-22)."""
    x = np.asarray(logits, np.float64)
    rows, n = x.shape
    lp, rank, ent = np.full(rows, np.nan), np.full(rows, -1, np.int64), np.full(rows, np.nan)
    tlp, ti = np.full((rows, top), np.nan), np.zeros((rows, top), np.int64)
    tol, etol, ttol = np.zeros(rows), np.zeros(rows), np.zeros((rows, top))
    u, depth = 2.0 ** -24, n / 32 + 64
    for r in range(rows):
        v = x[r]
        key = np.where(np.isnan(v), np.inf, v)
        order = np.lexsort((np.arange(n), -key, ~np.isnan(v)))      # NaN first, then by value, then by index
        m = v.max() if not np.isnan(v).any() else np.nan
        if m == -np.inf:
            p_log, ent[r] = np.full(n, -np.inf), 0.0
        elif not np.isfinite(m):
            p_log = np.full(n, np.nan)
        else:
            d = v - m
            e = np.exp(d)
            s, ls = e.sum(), np.log(e.sum())
            de = np.where(e > 0, np.where(e > 0, d, 0) * e, 0.0)
            p_log, w, w2 = d - ls, -de.sum() / s, (np.where(e > 0, d, 0) * de).sum() / s
            ent[r] = ls + w
            ls_tol = u * (depth + 8 + 3 * w + 4 * ls)
            with np.errstate(invalid="ignore"):
                all_tol = np.where(np.isfinite(d), ls_tol + 3 * u * np.abs(d), 0.0)
            etol[r] = ls_tol * (1 + w) + u * ((depth + 8) * w + 3 * w2 + 4 * ls)
            tol[r] = all_tol[labels[r]] if labels is not None and 0 <= labels[r] < n else 0.0
            ttol[r] = all_tol[order[:top]]
        # the results are fp32, in which the difference of the type's largest and lowest value, 2^129 - 2^105, is infinite
        p_log = np.where(p_log <= -(2.0 ** 128 - 2.0 ** 103), -np.inf, p_log)
        if labels is not None:
            if 0 <= labels[r] < n:
                lp[r], rank[r] = p_log[labels[r]], int(np.where(order == labels[r])[0][0])
            elif labels[r] < 0:
                lp[r] = 0.0
        ti[r], tlp[r] = order[:top], p_log[order[:top]]
    return (lp, rank, ent, tlp, ti), (tol, etol, ttol)


def close(got, expected, tol):
    """Equal where the expected value is not finite, within tol elsewhere."""
    got, expected = np.asarray(got, np.float64), np.asarray(expected, np.float64)
    assert got.shape == expected.shape
    fine = np.isfinite(expected)
    np.testing.assert_array_equal(got[~fine], expected[~fine])
    off = np.abs(got[fine] - expected[fine]) - np.broadcast_to(tol, expected.shape)[fine]
    assert off.size == 0 or off.max() <= 0, f"off by {off.max()} more than allowed, at {np.argmax(off)}"


def f8(values):
    """float64 numpy of e4m3 values -> torch tensor of the bytes whose rows begin on 16-byte boundaries."""
    rows, k = values.shape
    q = torch.zeros((rows, (k + 15) // 16 * 16), dtype=torch.float32)
    q[:, :k] = torch.from_numpy(values).float()
    return q.to(torch.float8_e4m3fn).cuda()[:, :k]
