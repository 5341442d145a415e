"""Kernel-level host API over torch CUDA tensors - the Python mirror of the reference's free
functions (`pack_mat`, `pad`, `im2col`, `fused_binarize_im2col`, `bgemm`, `baseline_bconv` /
`bconv_3x3`, the float layers), with the same names and argument meaning - and of what the reference has no
counterpart for: an 8-bit float product with block scales, and the scoring of logits.

torch is used for device memory and streams only; every function hands raw device pointers to the
C ABI (include/dabnn_b200.h) and enqueues on torch's current CUDA stream.  Bit tensors are
torch.int64 (a uint64 word per element; view as uint64 on the host).  All entry points accept a
leading batch dimension; 3-D inputs are treated as a batch of one like the reference.
"""
from __future__ import annotations

import ctypes as C

import torch

from . import capi
from .capi import ENGINES, check


# What follows is most of a small call's time: on one 56x56x64 image the two kernels of `binconv_forward` take 12 us and the call
# took 21 us, 3.4 of them to build the stream object whose handle is asked for here directly (0.2 us).
def _stream():
    """Handle of torch's current stream on the current device."""
    return torch._C._cuda_getCurrentRawStream(torch._C._cuda_getDevice())


def _ptr(t):
    return t.data_ptr() if t is not None else None


def _cuda(t, dtype):
    if not (isinstance(t, torch.Tensor) and t.is_cuda and t.dtype == dtype and t.is_contiguous()):
        raise TypeError(f"expected a contiguous CUDA tensor of dtype {dtype}")
    return t


def _b4(t):
    return t if t.dim() == 4 else t.unsqueeze(0)


def _eng(engine):
    return ENGINES[engine] if isinstance(engine, str) else int(engine)


def out_dim(i, pad, dil, k, stride):
    return (i + 2 * pad - (dil * (k - 1) + 1)) // stride + 1


def pack_mat(x):
    """fp32 [..., H, W, C] -> int64 bits [..., H, W, C/64]   (reference dabnn/bitpack.h:277)."""
    x4 = _b4(_cuda(x, torch.float32))
    n, h, w, c = x4.shape
    out = torch.empty((*x.shape[:-1], max(c // 64, 0)), dtype=torch.int64, device=x.device)
    check(capi.load().dabnn_pack_mat(_ptr(x4), _ptr(out), n, h, w, c, _stream()))
    return out


def pad(x, pad_h, pad_w, val=0.0):
    """Spatial padding of a bit (int64) or float tensor   (reference dabnn/pad.h:7)."""
    x4 = _b4(x)
    n, h, w, c = x4.shape
    out = torch.empty((n, h + 2 * pad_h, w + 2 * pad_w, c), dtype=x.dtype, device=x.device)
    lib = capi.load()
    if x.dtype == torch.int64:
        if val != 0.0:
            raise ValueError("val cannot be set for DataType::Bit")  # pad.h:12
        check(lib.dabnn_pad_bits(_ptr(_cuda(x4, torch.int64)), _ptr(out), n, h, w, c, pad_h, pad_w, _stream()))
    else:
        check(lib.dabnn_pad_f32(_ptr(_cuda(x4, torch.float32)), _ptr(out), n, h, w, c, pad_h, pad_w, float(val), _stream()))
    return out if x.dim() == 4 else out[0]


def im2col(x, kh, kw, pad_h, pad_w, stride_h, stride_w, dil_h=1, dil_w=1):
    """[.., H, W, C] (float or bits) -> [.., OH*OW, kh*kw*C]   (reference dabnn/im2col.h:14)."""
    x4 = _b4(x)
    n, h, w, c = x4.shape
    oh, ow = out_dim(h, pad_h, dil_h, kh, stride_h), out_dim(w, pad_w, dil_w, kw, stride_w)
    out = torch.empty((n, max(oh * ow, 0), kh * kw * c), dtype=x.dtype, device=x.device)
    check(capi.load().dabnn_im2col(_ptr(x4.contiguous()), _ptr(out), x.element_size(), n, h, w, c, kh, kw, pad_h, pad_w,
                                   stride_h, stride_w, dil_h, dil_w, _stream()))
    return out if x.dim() == 4 else out[0]


def fused_binarize_im2col(x, kh, kw, pad_h, pad_w, stride_h, stride_w, dil_h=1, dil_w=1):
    """fp32 -> bit rows of ceil(kh*kw*C/128)*2 words   (reference dabnn/fused_binarize_im2col.h:6)."""
    x4 = _b4(_cuda(x, torch.float32))
    n, h, w, c = x4.shape
    oh, ow = out_dim(h, pad_h, dil_h, kh, stride_h), out_dim(w, pad_w, dil_w, kw, stride_w)
    out = torch.empty((n, max(oh * ow, 0), (kh * kw * c + 127) // 128 * 2), dtype=torch.int64, device=x.device)
    check(capi.load().dabnn_fused_binarize_im2col(_ptr(x4), _ptr(out), n, h, w, c, kh, kw, pad_h, pad_w, stride_h,
                                                  stride_w, dil_h, dil_w, _stream()))
    return out if x.dim() == 4 else out[0]


def bgemm(m, n, k, a, lda, b, ldb, c, ldc, engine="auto"):
    """C(i,j) += sum_h popcount(A(i,h) ^ B(h,j)) with the reference's operand layout
    (reference dabnn/bgemm.h:22-24,46): a[h*lda+i], b[j*ldb+h], c[j*ldc+i]; c is updated in place."""
    check(capi.load().dabnn_bgemm(m, n, k, _ptr(_cuda(a, torch.int64)), lda, _ptr(_cuda(b, torch.int64)), ldb,
                                  _ptr(_cuda(c, torch.float32)), ldc, _eng(engine), _stream()))
    return c


def bconv(x_bits, weight, cout, kh, kw, pad_h, pad_w, stride_h, stride_w, engine="auto"):
    """Binary convolution on packed input: mismatch counts as fp32
    (reference common/baseline.h:77 baseline_bconv; dabnn/bconv.h:855 bconv_3x3 with pad 0)."""
    x4 = _b4(_cuda(x_bits, torch.int64))
    n, h, w, cw = x4.shape
    oh, ow = out_dim(h, pad_h, 1, kh, stride_h), out_dim(w, pad_w, 1, kw, stride_w)
    out = torch.empty((n, max(oh, 0), max(ow, 0), cout), dtype=torch.float32, device=x_bits.device)
    check(capi.load().dabnn_bconv(_ptr(x4), _ptr(_cuda(weight, torch.int64)), weight.numel(), _ptr(out), n, h, w, cw,
                                  cout, kh, kw, pad_h, pad_w, stride_h, stride_w, _eng(engine), _stream()))
    return out if x_bits.dim() == 4 else out[0]


def binconv_forward(x, weight, cout, kh, kw, pad_h, pad_w, stride_h, stride_w, engine="auto"):
    """The BinConv operator: fp32 in, fp32 mismatch counts out
    (reference dabnn/layers/BinConv.cpp:144 forward_impl)."""
    x4 = _b4(_cuda(x, torch.float32))
    n, h, w, c = x4.shape
    lib = capi.load()
    oh, ow = out_dim(h, pad_h, 1, kh, stride_h), out_dim(w, pad_w, 1, kw, stride_w)
    out = torch.empty((n, max(oh, 0), max(ow, 0), cout), dtype=torch.float32, device=x.device)
    # whole words of channels: the packed input (the library checks the size it is given)
    nbytes = n * h * w * c // 8 if c % 64 == 0 else lib.dabnn_binconv_workspace_bytes(n, h, w, c, kh, kw, pad_h, pad_w, stride_h, stride_w)
    ws = torch.empty(max(nbytes, 8), dtype=torch.uint8, device=x.device)
    check(lib.dabnn_binconv_forward(_ptr(x4), _ptr(_cuda(weight, torch.int64)), weight.numel(), _ptr(out), n, h, w, c,
                                    cout, kh, kw, pad_h, pad_w, stride_h, stride_w, _ptr(ws), nbytes, _eng(engine),
                                    _stream()))
    return out if x.dim() == 4 else out[0]


def binconv_forward_static(x, weight, cout, kh, kw, pad_h, pad_w, stride_h, stride_w, engine="auto"):
    """`binconv_forward` without any allocation inside the library: the packed intermediate lives
    in the library's built-in 16 MiB device buffer.  For hosts that own all device memory
    themselves or may not call cudaMalloc where they run inference.  `out` is still the caller's
    (here: a torch tensor allocated before the call).  Calls on one device must not overlap."""
    x4 = _b4(_cuda(x, torch.float32))
    n, h, w, c = x4.shape
    oh, ow = out_dim(h, pad_h, 1, kh, stride_h), out_dim(w, pad_w, 1, kw, stride_w)
    out = torch.empty((n, max(oh, 0), max(ow, 0), cout), dtype=torch.float32, device=x.device)
    check(capi.load().dabnn_binconv_forward_static(_ptr(x4), _ptr(_cuda(weight, torch.int64)), weight.numel(), _ptr(out),
                                                   n, h, w, c, cout, kh, kw, pad_h, pad_w, stride_h, stride_w,
                                                   _eng(engine), _stream()))
    return out if x.dim() == 4 else out[0]


def bconv_block(x_bits, weight, cout, kh, kw, pad_h, pad_w, stride_h, stride_w, a=None, b=None, shortcut=None,
                want_f32=True, want_bits=False, engine="auto"):
    """Fused BinConv -> Affine -> Add -> sign bits (see dabnn_bconv_block).  Returns (f32, bits)."""
    x4 = _b4(_cuda(x_bits, torch.int64))
    n, h, w, cw = x4.shape
    oh, ow = out_dim(h, pad_h, 1, kh, stride_h), out_dim(w, pad_w, 1, kw, stride_w)
    dev = x_bits.device
    out = torch.empty((n, oh, ow, cout), dtype=torch.float32, device=dev) if want_f32 else None
    bits = torch.empty((n, oh, ow, cout // 64), dtype=torch.int64, device=dev) if want_bits else None
    check(capi.load().dabnn_bconv_block(_ptr(x4), _ptr(_cuda(weight, torch.int64)), weight.numel(), _ptr(a), _ptr(b),
                                        _ptr(shortcut), _ptr(out), _ptr(bits), n, h, w, cw, cout, kh, kw, pad_h, pad_w,
                                        stride_h, stride_w, _eng(engine), _stream()))
    return out, bits


def binarize_u8(x):
    """fp32 -> {0,1} bytes, byte = x > 0: the byte-activation engine's counterpart of pack_mat (bitpack.h:277)."""
    x = _cuda(x, torch.float32)
    out = torch.empty(x.shape, dtype=torch.uint8, device=x.device)
    check(capi.load().dabnn_binarize_u8(_ptr(x), _ptr(out), x.numel(), _stream()))
    return out


def bconv_u8_supported(n, h, w, cin, cout, kh, kw, pad_h, pad_w, stride_h, stride_w):
    return bool(capi.load().dabnn_bconv_u8_supported(n, h, w, cin, cout, kh, kw, pad_h, pad_w, stride_h, stride_w))


def bconv_u8_expand_weights(weight, cout, kwords):
    """Packed filters (cout rows of kwords words) -> the byte-activation engine's weight buffer (a uint8 tensor)."""
    weight = _cuda(weight, torch.int64)
    buf = torch.empty(capi.load().dabnn_bconv_u8_weight_bytes(cout, kwords), dtype=torch.uint8, device=weight.device)
    check(capi.load().dabnn_bconv_u8_expand_weights(_ptr(weight), weight.numel(), cout, kwords, _ptr(buf), _stream()))
    return buf


def bconv_u8_block(x_u8, w_expanded, cout, kh, kw, pad_h, pad_w, stride_h, stride_w, a=None, b=None, shortcut=None,
                   want_f32=True, want_u8=False, want_bits=False):
    """The fused block of bconv_block on {0,1}-byte activations (see dabnn_bconv_u8_block).  Returns (f32, u8, bits)."""
    x4 = _cuda(x_u8, torch.uint8)
    n, h, w, cin = x4.shape
    oh, ow = out_dim(h, pad_h, 1, kh, stride_h), out_dim(w, pad_w, 1, kw, stride_w)
    dev = x4.device
    out = torch.empty((n, oh, ow, cout), dtype=torch.float32, device=dev) if want_f32 else None
    o8 = torch.empty((n, oh, ow, cout), dtype=torch.uint8, device=dev) if want_u8 else None
    bits = torch.empty((n, oh, ow, cout // 64), dtype=torch.int64, device=dev) if want_bits else None
    check(capi.load().dabnn_bconv_u8_block(_ptr(x4), _ptr(w_expanded), _ptr(a), _ptr(b), _ptr(shortcut), _ptr(out), _ptr(o8),
                                           _ptr(bits), n, h, w, cin, cout, kh, kw, pad_h, pad_w, stride_h, stride_w,
                                           _stream()))
    return out, o8, bits


def bconv_u8_block_pooled_supported(n, h, w, cin, cout, kh, kw, pad_h, pad_w, stride_h, stride_w):
    return bool(capi.load().dabnn_bconv_u8_block_pooled_supported(n, h, w, cin, cout, kh, kw, pad_h, pad_w, stride_h, stride_w))


def bconv_u8_block_pooled(x_u8, w_expanded, cout, kh, kw, pad_h, pad_w, stride_h, stride_w, a=None, b=None, shortcut=None,
                          want_u8=False):
    """bconv_u8_block that also returns the 2x2 stride-2 average pooling of its fp32 result (reference
    layers/AvePool.cpp:84 on the block's output).  Returns (f32, u8 or None, pooled f32)."""
    x4 = _cuda(x_u8, torch.uint8)
    n, h, w, cin = x4.shape
    oh, ow = out_dim(h, pad_h, 1, kh, stride_h), out_dim(w, pad_w, 1, kw, stride_w)
    dev = x4.device
    out = torch.empty((n, oh, ow, cout), dtype=torch.float32, device=dev)
    o8 = torch.empty((n, oh, ow, cout), dtype=torch.uint8, device=dev) if want_u8 else None
    pooled = torch.empty((n, oh // 2, ow // 2, cout), dtype=torch.float32, device=dev)
    check(capi.load().dabnn_bconv_u8_block_pooled(_ptr(x4), _ptr(w_expanded), _ptr(a), _ptr(b), _ptr(shortcut), _ptr(out), _ptr(o8), None,
                                                  _ptr(pooled), n, h, w, cin, cout, kh, kw, pad_h, pad_w, stride_h, stride_w, _stream()))
    return out, o8, pooled


def affine_(x, a, b):
    """In place x = a[c]*x + b[c]   (reference dabnn/layers/Affine.cpp:10)."""
    c = x.shape[-1]
    check(capi.load().dabnn_affine(_ptr(_cuda(x, torch.float32)), _ptr(_cuda(a, torch.float32)),
                                   _ptr(_cuda(b, torch.float32)), x.numel() // c, c, _stream()))
    return x


def add_(x, y):
    """In place x += y   (reference dabnn/layers/Add.cpp:7)."""
    if x.shape != y.shape:
        raise ValueError("add: shapes differ")
    check(capi.load().dabnn_add(_ptr(_cuda(x, torch.float32)), _ptr(_cuda(y, torch.float32)), x.numel(), _stream()))
    return x


def relu_(x):
    """In place max(x, 0)   (reference dabnn/layers/Relu.cpp:21)."""
    check(capi.load().dabnn_relu(_ptr(_cuda(x, torch.float32)), x.numel(), _stream()))
    return x


def prelu_(x, slope):
    """In place x<0 ? x*slope : x   (reference dabnn/layers/PRelu.cpp:6)."""
    c = x.shape[-1]
    check(capi.load().dabnn_prelu(_ptr(_cuda(x, torch.float32)), _ptr(_cuda(slope, torch.float32)), slope.numel(),
                                  x.numel() // c, c, _stream()))
    return x


def _pool(fn, x, kh, kw, pad_h, pad_w, stride_h, stride_w):
    x4 = _b4(_cuda(x, torch.float32))
    n, h, w, c = x4.shape
    oh, ow = (h + 2 * pad_h - kh) // stride_h + 1, (w + 2 * pad_w - kw) // stride_w + 1
    out = torch.empty((n, max(oh, 0), max(ow, 0), c), dtype=torch.float32, device=x.device)
    check(fn(_ptr(x4), _ptr(out), n, h, w, c, kh, kw, pad_h, pad_w, stride_h, stride_w, _stream()))
    return out if x.dim() == 4 else out[0]


def maxpool(x, kh, kw, pad_h, pad_w, stride_h, stride_w):
    """reference dabnn/layers/MaxPool.cpp:209 max_pool_fallback."""
    return _pool(capi.load().dabnn_maxpool, x, kh, kw, pad_h, pad_w, stride_h, stride_w)


def avepool(x, kh, kw, pad_h, pad_w, stride_h, stride_w):
    """reference dabnn/layers/AvePool.cpp:84 ave_pool_fallback."""
    return _pool(capi.load().dabnn_avepool, x, kh, kw, pad_h, pad_w, stride_h, stride_w)


def concat(x1, x2):
    """Channel concatenation   (reference dabnn/layers/Concat.cpp:7)."""
    out = torch.empty((*x1.shape[:-1], x1.shape[-1] + x2.shape[-1]), dtype=torch.float32, device=x1.device)
    check(capi.load().dabnn_concat(_ptr(_cuda(x1, torch.float32)), x1.shape[-1], _ptr(_cuda(x2, torch.float32)),
                                   x2.shape[-1], _ptr(out), x1.numel() // x1.shape[-1], _stream()))
    return out


def fconv(x, weight, bias, pad_h, pad_w, stride_h, stride_w, dil_h=1, dil_w=1):
    """Float convolution, weight [Cout][kh][kw][Cin]   (reference dabnn/fconv.h:14,44)."""
    x4 = _b4(_cuda(x, torch.float32))
    n, h, w, c = x4.shape
    cout, kh, kw, _ = weight.shape
    oh, ow = out_dim(h, pad_h, dil_h, kh, stride_h), out_dim(w, pad_w, dil_w, kw, stride_w)
    out = torch.empty((n, max(oh, 0), max(ow, 0), cout), dtype=torch.float32, device=x.device)
    check(capi.load().dabnn_fconv(_ptr(x4), _ptr(_cuda(weight, torch.float32)), _ptr(bias), _ptr(out), n, h, w, c, cout,
                                  kh, kw, pad_h, pad_w, stride_h, stride_w, dil_h, dil_w, _stream()))
    return out if x.dim() == 4 else out[0]


def fconv_maxpool_supported(n, h, w, cin, cout, kh, kw, pad_h, pad_w, stride_h, stride_w):
    return bool(capi.load().dabnn_fconv_maxpool_supported(n, h, w, cin, cout, kh, kw, pad_h, pad_w, stride_h, stride_w))


def fconv_maxpool(x, weight, bias, pad_h, pad_w, stride_h, stride_w, a=None, b=None, relu=False, want_u8=False):
    """Float convolution (+ bias, affine, relu) followed by a 3x3 stride-2 pad-1 max pooling, in one kernel (the stem of
    a ResNet: reference dabnn/fconv.h:14 -> Affine.cpp:10 -> Relu.cpp:21 -> MaxPool.cpp:209).  Returns (pooled fp32,
    sign bytes or None)."""
    x4 = _b4(_cuda(x, torch.float32))
    n, h, w, c = x4.shape
    cout, kh, kw, _ = weight.shape
    oh, ow = out_dim(h, pad_h, 1, kh, stride_h), out_dim(w, pad_w, 1, kw, stride_w)
    ph, pw = (oh - 1) // 2 + 1, (ow - 1) // 2 + 1
    out = torch.empty((n, ph, pw, cout), dtype=torch.float32, device=x.device)
    o8 = torch.empty((n, ph, pw, cout), dtype=torch.uint8, device=x.device) if want_u8 else None
    check(capi.load().dabnn_fconv_maxpool(_ptr(x4), _ptr(_cuda(weight, torch.float32)), _ptr(bias), _ptr(a), _ptr(b), int(relu), _ptr(out),
                                          _ptr(o8), n, h, w, c, cout, kh, kw, pad_h, pad_w, stride_h, stride_w, _stream()))
    return out, o8


# ---- 8-bit float matrices with a scale for each block of 128, and the scoring of logits -----------------------------------
FP8_BLOCK = 128
_FLOATS = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}   # DABNN_F32 / F16 / BF16


def _here(*tensors):
    """The kernels run on the current device, on its current stream."""
    device = torch._C._cuda_getDevice()
    for t in tensors:
        if t is not None and t.get_device() != device:
            raise TypeError("expected CUDA tensors on the current device")


def _levels(shape, strides):
    """Dimensions, outermost first, as (size, stride) levels: those that walk memory in equal steps are one."""
    levels = []
    for size, stride in zip(shape, strides):
        if size == 1:
            continue
        if levels and levels[-1][1] == size * stride:
            levels[-1] = (levels[-1][0] * size, stride)
        else:
            levels.append((size, stride))
    return levels


def _rows(t, what):
    """(rows, columns, pitch) of a tensor taken as rows along its last dimension, which lie at equal steps: a matrix with any row
    pitch, a contiguous tensor, one whose rows alone have a pitch."""
    if t.dim() == 2:
        rows, cols = t.shape
        if cols <= 1 or t.stride(1) == 1:
            if rows >= 1 << 31 or cols >= 1 << 31:
                raise ValueError(f"{what}: too large a matrix")
            return rows, cols, t.stride(0) if rows > 1 else cols
    elif t.dim() >= 1 and t.is_contiguous():
        rows, cols = t.shape[:-1].numel(), t.shape[-1]
        if rows >= 1 << 31 or cols >= 1 << 31:
            raise ValueError(f"{what}: too large a matrix")
        return rows, cols, cols
    elif t.dim() > 2 and (t.shape[-1] <= 1 or t.stride(-1) == 1):
        levels = _levels(t.shape[:-1], t.stride()[:-1])
        if len(levels) < 2:
            rows, cols = t.shape[:-1].numel(), t.shape[-1]
            if rows >= 1 << 31 or cols >= 1 << 31:
                raise ValueError(f"{what}: too large a matrix")
            return rows, cols, levels[0][1] if levels else cols
    raise TypeError(f"{what}: expected rows of unit stride that lie at equal steps")


def _fp8_quantize(x, block_rows):
    _here(x)
    kind = _FLOATS.get(x.dtype)
    if kind is None:
        raise TypeError("fp8_quantize: expected fp32, fp16 or bf16")
    rows, k, ld = _rows(x, "fp8_quantize")
    pitch, blocks = (k + 15) // 16 * 16, (k + FP8_BLOCK - 1) // FP8_BLOCK
    q = torch.empty_strided((rows, k), (pitch, 1), dtype=torch.float8_e4m3fn, device=x.device)
    if block_rows == 1:   # block by block: the order in which the product reads them
        scales = torch.empty_strided((rows, blocks), (1, rows), dtype=torch.float32, device=x.device)
        step, block_step = 1, rows
    else:
        scales = torch.empty((rows + block_rows - 1) // block_rows, blocks, dtype=torch.float32, device=x.device)
        step, block_step = blocks, 1
    check(capi.load().dabnn_fp8_quantize(x.data_ptr(), kind, ld, q.data_ptr(), pitch, scales.data_ptr(), step, block_step, rows, k, block_rows, _stream()))
    return q, scales


def fp8_quantize(x):
    """Activations [..., K] (fp32, fp16, bf16) -> (e4m3 [..., K], fp32 scales [..., ceil(K / 128)]): one scale, a power of two,
    for each 128 values of a row (see dabnn_fp8_quantize).  The rows lie at equal steps.  Rows of the result begin on 16-byte boundaries, as fp8_gemm wants
    them; the scales lie block by block in memory."""
    q, scales = _fp8_quantize(x, 1)
    return (q, scales) if x.dim() == 2 else (q.unflatten(0, x.shape[:-1]), scales.unflatten(0, x.shape[:-1])) if x.dim() > 2 else (q[0], scales[0])


def fp8_quantize_weights(w):
    """Weights [N, K] -> (e4m3 [N, K], fp32 scales [ceil(N / 128), ceil(K / 128)]), once per model."""
    if w.dim() != 2:
        raise TypeError("fp8_quantize_weights: expected a matrix")
    return _fp8_quantize(w, FP8_BLOCK)


def _byte_rows(t):
    """[..., K] as a matrix; rows that do not lie at equal steps (a slice of a middle dimension) are copied, each to a 16-byte boundary."""
    lead, k = t.shape[:-1], t.shape[-1]
    if len(_levels(lead, t.stride()[:-1])) < 2 or t.is_contiguous():
        return t.flatten(0, -2)
    rows = torch.empty_strided((lead.numel(), k), ((k + 15) // 16 * 16, 1), dtype=t.dtype, device=t.device)
    rows.unflatten(0, lead).copy_(t)
    return rows


def fp8_gemm(a, a_scales, b, b_scales, bias=None, out_dtype=torch.float32):
    """[..., K] e4m3 activations times [N, K] e4m3 weights -> [..., N] of out_dtype (fp32, fp16, bf16), + bias (fp32 [N]).
    Scales as fp8_quantize and fp8_quantize_weights give them, of any value and in any memory order (see dabnn_fp8_gemm)."""
    _here(a, a_scales, b, b_scales, bias)
    kind = _FLOATS.get(out_dtype)
    if kind is None:
        raise TypeError("fp8_gemm: the result is fp32, fp16 or bf16")
    if a.dtype != torch.float8_e4m3fn or b.dtype != torch.float8_e4m3fn or a_scales.dtype != torch.float32 or b_scales.dtype != torch.float32:
        raise TypeError("fp8_gemm: expected float8_e4m3fn operands and fp32 scales")
    lead = None
    if a.dim() != 2:
        lead = a.shape[:-1]
        a = a.unsqueeze(0) if a.dim() == 1 else _byte_rows(a)
        a_scales = a_scales.unsqueeze(0) if a_scales.dim() == 1 else a_scales.flatten(0, -2)
    if b.dim() != 2:
        raise TypeError("fp8_gemm: expected a matrix of weights")
    m, k, lda = _rows(a, "fp8_gemm")
    n, kb, ldb = _rows(b, "fp8_gemm")
    blocks = (k + FP8_BLOCK - 1) // FP8_BLOCK
    if kb != k or a_scales.shape != (m, blocks) or b_scales.shape != ((n + FP8_BLOCK - 1) // FP8_BLOCK, blocks):
        raise ValueError("fp8_gemm: shapes of the operands and their scales do not go together")
    if bias is not None and (bias.dtype != torch.float32 or bias.shape != (n,) or not bias.is_contiguous()):
        raise TypeError("fp8_gemm: expected a contiguous fp32 bias of N values")
    c = torch.empty(m, n, dtype=out_dtype, device=a.device)
    check(capi.load().dabnn_fp8_gemm(a.data_ptr(), lda, a_scales.data_ptr(), *a_scales.stride(), b.data_ptr(), ldb, b_scales.data_ptr(), *b_scales.stride(),
                                     _ptr(bias), c.data_ptr(), kind, n, m, n, k, _stream()))
    return c if lead is None else c.unflatten(0, lead) if lead else c[0]


def _grouped_rows(logits, labels):
    """(rows, classes, pitch of rows, rows of a group, pitch of groups, pitch of the groups' labels) of logits whose rows, or
    whose labels, do not all lie at equal steps."""
    lead, classes = logits.shape[:-1], logits.shape[-1]
    rows = lead.numel()
    if rows >= 1 << 31 or classes >= 1 << 31:
        raise ValueError("logprobs: too large a matrix")
    levels = _levels(lead, logits.stride()[:-1])
    if (classes > 1 and logits.stride(-1) != 1) or len(levels) > 2:
        raise TypeError("logprobs: expected rows of unit stride, in groups that lie at equal steps")
    # rows: groups of `size`, `ld` apart; labels: groups of `label_size`
    size, ld = levels[-1] if levels else (rows, classes)
    ld_group = levels[0][1] if len(levels) == 2 else 0
    label_size, label_group = rows, 0
    if labels is not None and not labels.is_contiguous():
        levels = _levels(labels.shape, labels.stride())
        if len(levels) == 1 and labels.dim() > 1 and labels.shape[-1] == 1:
            levels.append((1, 1))
        if len(levels) != 2 or levels[1][1] != 1:
            raise TypeError("logprobs: expected labels that lie side by side, or in groups that do")
        label_size, label_group = levels[1][0], levels[0][1]
    if size == rows:
        size, ld_group = label_size, label_size * ld
    elif label_size == rows:
        label_group = size
    elif size != label_size:
        raise TypeError("logprobs: the groups of rows and of labels differ")
    return rows, classes, ld, size, ld_group, label_group


def logprobs(logits, labels=None, top=0):
    """Scores rows of logits [..., classes] (fp32, fp16, bf16) -> (label_logprob, label_rank, entropy, top_logprob, top_index):
    ln softmax of the class in `labels` (int64 [...]) and how many classes come before it, the entropy, and the `top`
    likeliest classes with their ln softmax [..., top]; None for what was not asked.  Equal logits rank by index; a
    negative label is ignored (0 and -1).  Rows with -inf, NaN and other labels: see dabnn_logprobs.
    Rows may have a pitch, and so may groups of rows of one size, labels included (see dabnn_logprobs_grouped):
    logprobs(logits[:, :-1], tokens[:, 1:]) scores a batch of sequences where they lie."""
    _here(logits, labels)
    kind = _FLOATS.get(logits.dtype)
    if kind is None:
        raise TypeError("logprobs: expected fp32, fp16 or bf16")
    lead = logits.shape[:-1]
    lp = rank = tlp = ti = groups = None
    whole = labels is None or labels.is_contiguous()
    if whole and (logits.dim() == 2 or logits.is_contiguous()):
        rows, classes, ld = _rows(logits, "logprobs")
    else:
        rows, classes, ld, *groups = _grouped_rows(logits, labels)
    if labels is not None:
        if labels.dtype != torch.int64 or labels.shape != lead:
            raise TypeError("logprobs: expected int64 labels, one for each row")
        rank = torch.empty_like(labels) if whole else torch.empty_like(labels, memory_format=torch.contiguous_format)
        lp = torch.empty_like(rank, dtype=torch.float32)
        entropy = torch.empty_like(lp)
    else:
        entropy = logits.new_empty(lead, dtype=torch.float32)
    if top:
        tlp = torch.empty(*lead, max(top, 0), dtype=torch.float32, device=logits.device)
        ti = torch.empty_like(tlp, dtype=torch.int64)
    if groups:
        group_rows, ld_group, label_group = groups
        check(capi.load().dabnn_logprobs_grouped(logits.data_ptr(), kind, ld, ld_group, _ptr(labels), label_group, group_rows, rows, classes, _ptr(lp),
                                                 _ptr(rank), entropy.data_ptr(), _ptr(tlp), _ptr(ti), top, _stream()))
    else:
        check(capi.load().dabnn_logprobs(logits.data_ptr(), kind, ld, _ptr(labels), rows, classes, _ptr(lp), _ptr(rank), entropy.data_ptr(), _ptr(tlp),
                                         _ptr(ti), top, _stream()))
    return lp, rank, entropy, tlp, ti


def measure_engine_peak(engine):
    """Register-resident peak of one contraction instruction in bit-op/s."""
    v = C.c_double()
    check(capi.load().dabnn_measure_engine_peak(_eng(engine), C.byref(v)))
    return v.value


def measure_tf32_peak():
    """Issue-bound rate of tcgen05.mma kind::tf32 in FLOP/s (the float convolution's denominator)."""
    v = C.c_double()
    check(capi.load().dabnn_measure_tf32_peak(C.byref(v)))
    return v.value


def engine_status(collect=False):
    """0, or the code of the first bounded wait that gave up inside a tcgen05 kernel (synchronises).  collect: the codes are
    cleared as well, so that the next answer tells of later calls (see dabnn_collect_engine_status)."""
    v = C.c_int()
    lib = capi.load()
    check((lib.dabnn_collect_engine_status if collect else lib.dabnn_engine_status)(C.byref(v)))
    return v.value


def last_engine():
    """Name of the engine the most recent bgemm / bconv / bconv_block / binconv_forward call of this thread launched
    (a "tcgen05" request falls back to "imma" for shapes the tensor-memory kernel does not take)."""
    code = capi.load().dabnn_last_engine()
    return next(k for k, v in ENGINES.items() if v == code)
