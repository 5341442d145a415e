"""Timed operators of the quantised classifier head, in their plain form and through the public entry points.

    own               False: `run` computes the plain form in torch; True: `run` makes the framework's calls
    listed()          the standing cases
    draw(rng)         one more case of the same ranges
    prepare(case, s)  what a program holds before the call: inputs made from seed s
    run(state)        one pass, as a program calls it; returns its outputs
    work(case)        bytes and operations that the pass cannot do without
    exact(case, s)    what the pass returns for these inputs, from the definition in 64 bits

Kinds of a case:
    quantize   rows of activations to e4m3, one scale for each 128 values of a row
    weights    a weight matrix to e4m3, one scale for each block of 128 x 128
    gemm       the product of such activations and weights, with fp32 scales of any value
    logprobs   log probabilities and ranks of given classes, entropy and top alternatives of rows of logits
"""
import torch

own = False

BLOCK = 128
E4M3_MAX = 448.0
DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZES = {"f32": 4, "f16": 2, "bf16": 2}


def listed():
    return [
        # the features of one image or token on their way into a quantised layer: the smallest call
        {"name": "quantize_one", "kind": "quantize", "rows": 1, "k": 4096, "dtype": "bf16"},
        # a long prompt's or a large batch's activations
        {"name": "quantize_rows", "kind": "quantize", "rows": 8192, "k": 4096, "dtype": "bf16"},
        # fp32 features of a ragged batch whose rows end inside a block
        {"name": "quantize_ragged", "kind": "quantize", "rows": 1023, "k": 1100, "dtype": "f32"},
        # a weight matrix, once per model
        {"name": "weights", "kind": "weights", "rows": 8192, "k": 4096, "dtype": "f32"},
        # one row against a wide layer: the weights have to be read
        {"name": "gemm_one", "kind": "gemm", "m": 1, "n": 8192, "k": 4096, "out": "bf16", "bias": False},
        # a few rows, nothing a multiple of a tile
        {"name": "gemm_few", "kind": "gemm", "m": 37, "n": 4100, "k": 2064, "out": "f32", "bias": True},
        # the classifier of the 1024-image benchmark batch
        {"name": "gemm_classifier", "kind": "gemm", "m": 1024, "n": 1000, "k": 512, "out": "f32", "bias": True},
        # a large layer on a large batch: the tensor cores' rate counts
        {"name": "gemm_large", "kind": "gemm", "m": 8192, "n": 8192, "k": 4096, "out": "bf16", "bias": False},
        # one image's 1000 classes and its five best
        {"name": "logprobs_image", "kind": "logprobs", "rows": 1, "classes": 1000, "dtype": "f32", "top": 5, "barred": False},
        # the 1024-image batch's
        {"name": "logprobs_batch", "kind": "logprobs", "rows": 1024, "classes": 1000, "dtype": "f32", "top": 5, "barred": False},
        # one token over a large vocabulary of which a part is barred, twenty alternatives
        {"name": "logprobs_one_wide", "kind": "logprobs", "rows": 1, "classes": 131072, "dtype": "bf16", "top": 20, "barred": True},
        # the scoring of a long text
        {"name": "logprobs_rows_wide", "kind": "logprobs", "rows": 4096, "classes": 65536, "dtype": "bf16", "top": 8, "barred": False},
    ]


def _log_int(rng, lo, hi):
    """An integer of [lo, hi], spread evenly over its logarithm."""
    return max(lo, min(hi, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    kind = rng.choice(("quantize", "weights", "gemm", "gemm", "logprobs", "logprobs"))
    while True:
        if kind in ("quantize", "weights"):
            k = _log_int(rng, 64, 16384)
            k = k if rng.random() < 0.4 else max(64, k // 64 * 64)
            case = {"kind": kind, "rows": _log_int(rng, 1, 16384), "k": k, "dtype": rng.choice(("f32", "f16", "bf16", "bf16"))}
        elif kind == "gemm":
            k = _log_int(rng, 64, 16384)
            k = k if rng.random() < 0.3 else max(64, k // 64 * 64)
            n = _log_int(rng, 10, 16384)
            n = n if rng.random() < 0.4 else max(16, n // 16 * 16)
            case = {"kind": kind, "m": _log_int(rng, 1, 8192), "n": n, "k": k, "out": rng.choice(("f32", "bf16", "bf16", "f16")),
                    "bias": rng.random() < 0.5}
        else:
            classes = _log_int(rng, 2, 262144)
            classes = classes if rng.random() < 0.5 else max(2, classes // 8 * 8)
            top = min(classes, rng.choice((0, 1, 5, 5, 10, 20, 32)))
            case = {"kind": kind, "rows": _log_int(rng, 1, 8192), "classes": classes, "dtype": rng.choice(("f32", "f16", "bf16", "bf16")),
                    "top": top, "barred": classes >= 1024 and rng.random() < 0.3}
        need = work(case)
        if need["bytes"] <= 5.4e8 and need["flops"] <= 5.5e11:
            return case


# ---- what the program holds before the call --------------------------------------------------------------------
def _pitched(q):
    """Rows of bytes as the quantiser lays them out: each begins on a 16-byte boundary."""
    rows, k = q.shape
    store = torch.zeros((rows, (k + 15) // 16 * 16), device=q.device, dtype=q.dtype)
    store[:, :k] = q
    return store[:, :k]


def _activations(rows, k, gen):
    """Features as layers leave them: rows of different size, a few channels that are much larger than the rest."""
    x = torch.randn((rows, k), device="cuda", generator=gen)
    x *= torch.exp(torch.randn((rows, 1), device="cuda", generator=gen))
    return x * torch.where(torch.rand((1, k), device="cuda", generator=gen) < 0.01, 20.0, 1.0)


def _scaled(x, block_rows):
    """Operands of a product made elsewhere: scales of any value (largest / 448), not the quantiser's powers of two."""
    rows, k = x.shape
    nr, nk = -(-rows // block_rows), -(-k // BLOCK)
    full = torch.zeros((nr * block_rows, nk * BLOCK), device=x.device)
    full[:rows, :k] = x
    blocks = full.view(nr, block_rows, nk, BLOCK)
    scales = blocks.abs().amax((1, 3)).clamp_min(1e-20) / E4M3_MAX
    q = (blocks / scales[:, None, :, None]).clamp(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn)
    # the rows' scales lie block by block, as the quantiser writes them
    scales = scales.t().contiguous().t() if block_rows == 1 else scales
    return _pitched(q.view(full.shape)[:rows, :k]), scales


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    if case["kind"] == "quantize":
        return {"case": case, "x": _activations(case["rows"], case["k"], gen).to(DTYPES[case["dtype"]])}
    if case["kind"] == "weights":
        x = torch.randn((case["rows"], case["k"]), device="cuda", generator=gen) * case["k"] ** -0.5
        return {"case": case, "x": x.to(DTYPES[case["dtype"]])}
    if case["kind"] == "gemm":
        a, a_scales = _scaled(_activations(case["m"], case["k"], gen), 1)
        b, b_scales = _scaled(torch.randn((case["n"], case["k"]), device="cuda", generator=gen) * case["k"] ** -0.5, BLOCK)
        bias = torch.randn(case["n"], device="cuda", generator=gen) if case["bias"] else None
        return {"case": case, "a": a, "a_scales": a_scales, "b": b, "b_scales": b_scales, "bias": bias}
    rows, classes = case["rows"], case["classes"]
    # some rows are sure of their class, some are not
    spread = 1 + 3 * torch.rand((rows, 1), device="cuda", generator=gen)
    logits = (torch.randn((rows, classes), device="cuda", generator=gen) * spread).to(DTYPES[case["dtype"]])
    labels = torch.randint(0, classes, (rows,), device="cuda", generator=gen)
    # half of the given classes are the likeliest of eight, the others any
    few = torch.randint(0, classes, (rows, 8), device="cuda", generator=gen)
    likely = few.gather(1, logits.gather(1, few).float().argmax(1, keepdim=True))[:, 0]
    labels = torch.where(torch.rand(rows, device="cuda", generator=gen) < 0.5, likely, labels)
    if case["barred"]:   # one class in sixteen may not be taken; no given class is one of them
        logits[:, 7::16] = float("-inf")
        labels -= (labels % 16 == 7).long()
    return {"case": case, "logits": logits, "labels": labels}


# ---- one pass ---------------------------------------------------------------------------------------------------
def _plain_quantize(x, block_rows):
    """scale = the least power of two, not below 2^-126, with |x| <= 448 scale; x / scale rounded to e4m3."""
    rows, k = x.shape
    nr, nk = -(-rows // block_rows), -(-k // BLOCK)
    full = torch.zeros((nr * block_rows, nk * BLOCK), device=x.device, dtype=torch.float32)
    full[:rows, :k] = x
    blocks = full.view(nr, block_rows, nk, BLOCK)
    part, power = torch.frexp(blocks.abs().amax((1, 3)))       # largest = part 2^power, 448 = 0.875 2^9
    power = (power - 9 + (part > 0.875).int()).clamp_min(-126)
    one = torch.ones_like(part)
    q = (blocks * torch.ldexp(one, -power)[:, None, :, None]).to(torch.float8_e4m3fn)
    return q.view(full.shape)[:rows, :k], torch.ldexp(one, power)


def _plain_values(q, scales, block_rows):
    rows, k = q.shape
    spread = scales.repeat_interleave(block_rows, 0)[:rows] if block_rows > 1 else scales
    return q.float() * spread.repeat_interleave(BLOCK, 1)[:, :k]


def _plain_logprobs(logits, labels, top):
    x = logits.float()
    rows, classes = x.shape
    best = x.amax(1, keepdim=True)
    d = x - best
    e = torch.exp(d)
    total = e.sum(1)
    log_total = torch.log(total)
    weighted = torch.where(e > 0, d * e, torch.zeros_like(d)).sum(1)
    at = labels[:, None]
    mine = x.gather(1, at)
    index = torch.arange(classes, device=x.device)
    rank = ((x > mine) | ((x == mine) & (index < at))).sum(1)
    out = [d.gather(1, at)[:, 0] - log_total, rank, log_total - weighted / total]
    if top:
        left, values, indices = x.clone(), [], []
        taken = torch.zeros((rows, classes), device=x.device, dtype=torch.bool)
        for _ in range(top):
            value = left.masked_fill(taken, float("-inf")).amax(1, keepdim=True)
            where = torch.where((left == value) & ~taken, index, classes).amin(1, keepdim=True)
            taken.scatter_(1, where, True)
            values.append(value)
            indices.append(where)
        out += [torch.cat(values, 1) - best - log_total[:, None], torch.cat(indices, 1)]
    return tuple(out)


def run(state):
    case = state["case"]
    kind = case["kind"]
    if own:
        from dabnn_b200 import ops
        if kind == "quantize":
            return ops.fp8_quantize(state["x"])
        if kind == "weights":
            return ops.fp8_quantize_weights(state["x"])
        if kind == "gemm":
            return ops.fp8_gemm(state["a"], state["a_scales"], state["b"], state["b_scales"], state["bias"], DTYPES[case["out"]])
        return tuple(t for t in ops.logprobs(state["logits"], state["labels"], case["top"]) if t is not None)
    if kind in ("quantize", "weights"):
        return _plain_quantize(state["x"], BLOCK if kind == "weights" else 1)
    if kind == "gemm":
        c = _plain_values(state["a"], state["a_scales"], 1) @ _plain_values(state["b"], state["b_scales"], BLOCK).t()
        if state["bias"] is not None:
            c += state["bias"]
        return c.to(DTYPES[case["out"]])
    return _plain_logprobs(state["logits"], state["labels"], case["top"])


# ---- what a pass cannot do without -------------------------------------------------------------------------------
def work(case):
    """Bytes: every input and output once.  Operations: two for each multiply-accumulate; two for each value quantised
    (maximum, product); for each logit the maximum, difference, exponential, sum, weighted sum (two) and two comparisons."""
    if case["kind"] in ("quantize", "weights"):
        rows, k = case["rows"], case["k"]
        scales = (rows if case["kind"] == "quantize" else -(-rows // BLOCK)) * -(-k // BLOCK)
        return {"bytes": rows * k * (SIZES[case["dtype"]] + 1) + 4 * scales, "flops": 2 * rows * k}
    if case["kind"] == "gemm":
        m, n, k = case["m"], case["n"], case["k"]
        scales = (m + -(-n // BLOCK)) * -(-k // BLOCK)
        return {"bytes": (m + n) * k + 4 * scales + m * n * SIZES[case["out"]] + (4 * n if case["bias"] else 0), "flops": 2 * m * n * k}
    rows, classes = case["rows"], case["classes"]
    return {"bytes": rows * (classes * SIZES[case["dtype"]] + 8 + 4 + 8 + 4 + case["top"] * 12), "flops": 8 * rows * classes}


# ---- the definition in 64 bits -----------------------------------------------------------------------------------
def _exact_quantize(x, block_rows):
    x = x.double()
    rows, k = x.shape
    values, scales = torch.empty_like(x), torch.empty((-(-rows // block_rows), -(-k // BLOCK)), device=x.device, dtype=torch.float64)
    for j in range(scales.shape[1]):
        part = x[:, j * BLOCK:(j + 1) * BLOCK]
        largest = part.abs().amax(1)
        if block_rows > 1:
            largest = torch.stack([piece.amax() for piece in largest.split(block_rows)])
        scale = torch.exp2(torch.ceil(torch.log2(largest.clamp_min(2.0 ** -140) / E4M3_MAX)))
        scale = torch.where(largest > E4M3_MAX * scale, 2 * scale, scale)          # the logarithm may be off at a power of two
        scale = torch.where(largest <= E4M3_MAX * scale / 2, scale / 2, scale).clamp_min(2.0 ** -126)
        scales[:, j] = scale
        v = part / scale.repeat_interleave(block_rows)[:rows, None]
        # e4m3: four significant bits down to 2^-6, steps of 2^-9 below
        power = torch.frexp(v)[1].clamp_min(-5) - 4
        step = torch.ldexp(torch.ones_like(v), power)
        values[:, j * BLOCK:(j + 1) * BLOCK] = torch.round(v / step) * step
    return values, scales


def _exact_gemm(state):
    def values(q, scales, block_rows):
        v = q.float().double()
        for j in range(scales.shape[1]):
            v[:, j * BLOCK:(j + 1) * BLOCK] *= scales[:, j].double().repeat_interleave(block_rows)[:v.shape[0], None]
        return v

    c = torch.matmul(values(state["a"], state["a_scales"], 1), values(state["b"], state["b_scales"], BLOCK).transpose(0, 1))
    return c if state["bias"] is None else c + state["bias"].double()


def _exact_logprobs(logits, labels, top):
    out = []
    for x, label in zip(logits.split(256), labels.split(256)):
        x = x.double()
        lse = torch.logsumexp(x, 1, keepdim=True)
        logp = x - lse
        mine = x.gather(1, label[:, None])
        before = torch.arange(x.shape[1], device=x.device)[None] < label[:, None]
        rank = (x > mine).sum(1) + ((x == mine) & before).sum(1)
        entropy = -torch.special.xlogy(torch.exp(logp), torch.exp(logp)).sum(1)
        piece = [logp.gather(1, label[:, None])[:, 0], rank, entropy]
        if top:
            order = torch.sort(x, dim=1, descending=True, stable=True)[1][:, :top]
            piece += [logp.gather(1, order), order]
        out.append(piece)
    return tuple(torch.cat(parts) for parts in zip(*out))


def exact(case, seed):
    state = prepare(case, seed)
    if case["kind"] in ("quantize", "weights"):
        return _exact_quantize(state["x"], BLOCK if case["kind"] == "weights" else 1)
    if case["kind"] == "gemm":
        return _exact_gemm(state)
    return _exact_logprobs(state["logits"], state["labels"], case["top"])
