"""Cases of the 8-bit floating point operators (block quantiser, scaled product, linear training step, root-mean-square norm)
and of gradient clipping: their inputs, their plain forms in elementary torch operations, and the framework's own calls.

The 8-bit format: e4m3 codes with one scale for every block of 128 along the rows of a matrix ("row" blocks, 1 x 128) or for every
128 x 128 tile; made scales are powers of two, the smallest that brings the block's largest magnitude to 448 or less."""
import math

import torch

own = False
DEV = "cuda"
BLK = 128
_TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
_SIZE = {"fp32": 4, "bf16": 2, "fp16": 2}


# ------------------------------------------------------------------------------------------ cases

def listed():
    return [
        # a small batch of pooled features on its way into a linear layer
        dict(name="quantise features", op="quantise", rows=64, cols=1000, type="fp32", both=False),
        # gradients of a large layer, needed along both axes by the backward products
        dict(name="quantise gradients both ways", op="quantise", rows=8192, cols=8192, type="bf16", both=True),
        # serving: one token, and a ragged handful of them against a 1000-class head
        dict(name="product one token", op="product", m=1, n=4096, k=4096, tile=True, scales="pow2", out="bf16", bias=False),
        dict(name="product few tokens head", op="product", m=37, n=1000, k=2048, tile=True, scales="pow2", out="fp32", bias=True),
        # weights of another origin, whose scales are not powers of two
        dict(name="product any scales", op="product", m=1500, n=5000, k=2560, tile=True, scales="any", out="bf16", bias=False),
        # a prompt, or a training batch, through a wide layer
        dict(name="product large", op="product", m=8192, n=8192, k=8192, tile=True, scales="pow2", out="bf16", bias=False),
        # forward and all gradients of a linear layer with float32 weights, quantisation included
        dict(name="linear training step", op="linear_step", m=4096, n=4096, k=4096, type="bf16"),
        # serving: a few tokens through norm and quantiser
        dict(name="norm to 8 bits, four tokens", op="norm_quantise", rows=4, cols=4096, type="bf16", residual=True),
        # a long prompt through norm and quantiser
        dict(name="norm to 8 bits, prompt", op="norm_quantise", rows=16384, cols=8192, type="bf16", residual=True),
        # training: forward and gradients, with the gradient that arrives over the residual path
        dict(name="norm training", op="norm_train", rows=8192, cols=5120, type="bf16", residual=True),
        # the tensors of a small residual network
        dict(name="clip small network", op="clip", tensors=58, total=272_474, type="fp32", clipped=True),
        # a large model's gradients
        dict(name="clip large model", op="clip", tensors=48, total=400_000_000, type="fp32", clipped=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["quantise", "product", "product", "linear_step", "norm_quantise", "norm_train", "clip"])
    kind = rng.choice(["fp32", "bf16", "bf16", "fp16"])
    if op == "quantise":
        rows = _log(rng, 1, 16384)
        return dict(op=op, rows=rows, cols=_log(rng, 64, min(16384, (1 << 26) // rows)), type=kind, both=rng.random() < 0.5)
    if op == "product":
        m, n = _log(rng, 1, 8192), _log(rng, 64, 8192)
        k = 16 * _log(rng, 8, 512)
        return dict(op=op, m=m, n=n, k=k if rng.random() < 0.7 else k - rng.randrange(1, 16), tile=rng.random() < 0.7,
                    scales=rng.choice(["pow2", "pow2", "any"]), out=rng.choice(["bf16", "bf16", "fp32"]), bias=rng.random() < 0.4)
    if op == "linear_step":
        return dict(op=op, m=_log(rng, 64, 8192), n=_log(rng, 128, 4096), k=_log(rng, 128, 4096), type=rng.choice(["fp32", "bf16"]))
    if op == "norm_quantise":
        rows = _log(rng, 1, 16384)
        return dict(op=op, rows=rows, cols=_log(rng, 100, 8192), type=kind, residual=rng.random() < 0.7)
    if op == "norm_train":
        return dict(op=op, rows=_log(rng, 16, 8192), cols=_log(rng, 100, 8192), type=kind, residual=rng.random() < 0.7)
    return dict(op=op, tensors=rng.randrange(1, 60), total=_log(rng, 1000, 200_000_000), type=kind, clipped=rng.random() < 0.7)


def work(case):
    c, op = case, case["op"]
    if op == "quantise":  # x in; codes and scales, and the values they stand for, out: for each form
        n, forms = c["rows"] * c["cols"], 2 if c["both"] else 1
        return {"bytes": n * _SIZE[c["type"]] + forms * n * (1 + 2 + 1 / BLK), "flops": 0}
    if op == "product":
        m, n, k = c["m"], c["n"], c["k"]
        ss = 1 if c["scales"] == "pow2" else 4
        scales = ss * (m * k / BLK + n * k / BLK / (BLK if c["tile"] else 1))
        return {"bytes": (m + n) * k + scales + m * n * _SIZE[c["out"]] + 4 * n * c["bias"], "flops": 2.0 * m * n * k}
    if op == "linear_step":
        m, n, k, s = c["m"], c["n"], c["k"], _SIZE[c["type"]]
        return {"bytes": s * (2 * m * k + 2 * m * n) + 8 * n * k + 4 * n, "flops": 6.0 * m * n * k}
    if op == "norm_quantise":
        n, s = c["rows"] * c["cols"], _SIZE[c["type"]]
        return {"bytes": n * (s + (2 * s if c["residual"] else 0) + 1 + 2) + 4 * c["cols"], "flops": 0}
    if op == "norm_train":  # forward: x (r) in, y (h) out; backward: dy, h (dh) in, dx out
        n, s = c["rows"] * c["cols"], _SIZE[c["type"]]
        return {"bytes": n * s * (8 if c["residual"] else 5) + 8 * c["cols"], "flops": 0}
    return {"bytes": 2 * c["total"] * _SIZE[c["type"]], "flops": 0}


# ----------------------------------------------------------------------------------------- inputs

def _parts(case):
    """Sizes of the gradient tensors: uneven, odd ones among them, `total` elements together."""
    n, total = case["tensors"], case["total"]
    w = [1 + (i * i * 7) % 31 for i in range(n)]
    sizes = [max(1, total * v // sum(w)) for v in w]
    sizes[-1] = max(1, total - sum(sizes[:-1]))
    return sizes


def _activations(g, rows, cols, dtype):
    """Features with a spread of magnitudes along both axes and a few outlying channels."""
    x = torch.randn(rows, cols, device=DEV, generator=g)
    x *= torch.exp(0.5 * torch.randn(rows, 1, device=DEV, generator=g))
    s = torch.exp(0.5 * torch.randn(1, cols, device=DEV, generator=g))
    s[:, torch.randint(0, cols, (max(1, cols // 200),), device=DEV, generator=g)] *= 20.0
    return (x * s).to(dtype)


def _operand(g, rows, k, tile, pow2):
    """Codes with scales, in storage whose rows start at multiples of 16 bytes, as the quantiser lays them out."""
    x = torch.randn(rows, k, device=DEV, generator=g) * 0.02
    if tile:
        amax = torch.nn.functional.pad(x.abs(), (0, -k % BLK, 0, -rows % BLK))
        amax = amax.view(amax.shape[0] // BLK, BLK, -1, BLK).amax((1, 3))
    else:
        amax = torch.nn.functional.pad(x.abs(), (0, -k % BLK)).view(rows, -1, BLK).amax(2)
    scale = _pow2_scale(amax) if pow2 else torch.clamp(amax, min=1e-30) / 448.0
    full = _spread(scale, rows, k, BLK if tile else 1)
    data = torch.zeros(rows, k + (-k % 16), device=DEV, dtype=torch.float8_e4m3fn)
    data[:, :k].copy_((x / full).clamp(-448, 448).to(torch.float8_e4m3fn))
    return data[:, :k], scale.to(torch.float8_e8m0fnu) if pow2 else scale


def prepare(case, seed):
    c, op = case, case["op"]
    g = torch.Generator(device=DEV).manual_seed(seed)
    s = {"case": c}
    if op == "quantise":
        s["x"] = _activations(g, c["rows"], c["cols"], _TYPES[c["type"]])
    elif op == "product":
        s["a"], s["sa"] = _operand(g, c["m"], c["k"], False, c["scales"] == "pow2")
        s["b"], s["sb"] = _operand(g, c["n"], c["k"], c["tile"], c["scales"] == "pow2")
        s["bias"] = torch.randn(c["n"], device=DEV, generator=g) if c["bias"] else None
    elif op == "linear_step":
        t = _TYPES[c["type"]]
        s["x"] = _activations(g, c["m"], c["k"], t).requires_grad_(True)
        s["w"] = (torch.randn(c["k"], c["n"], device=DEV, generator=g) / math.sqrt(c["k"])).requires_grad_(True)
        s["bias"] = (0.1 * torch.randn(c["n"], device=DEV, generator=g)).requires_grad_(True)
        s["dy"] = (1e-3 * torch.randn(c["m"], c["n"], device=DEV, generator=g)).to(t)
    elif op in ("norm_quantise", "norm_train"):
        t = _TYPES[c["type"]]
        s["x"] = _activations(g, c["rows"], c["cols"], t)
        s["r"] = torch.randn(c["rows"], c["cols"], device=DEV, generator=g).to(t) if c["residual"] else None
        s["w"] = 1.0 + 0.2 * torch.randn(c["cols"], device=DEV, generator=g)
        if op == "norm_train":
            s["dy"] = (1e-2 * torch.randn(c["rows"], c["cols"], device=DEV, generator=g)).to(t)
            s["dh"] = (1e-2 * torch.randn(c["rows"], c["cols"], device=DEV, generator=g)).to(t) if c["residual"] else None
    else:
        s["g"] = [(torch.randn(n, device=DEV, generator=g) * 10.0 ** (i % 4 - 3)).to(_TYPES[c["type"]]) for i, n in enumerate(_parts(c))]
        s["out"] = [torch.empty_like(t) for t in s["g"]]
        # half, or twice, of what the norm of such tensors comes to
        about = math.sqrt(sum(n * 100.0 ** (i % 4 - 3) for i, n in enumerate(_parts(c))))
        s["max_norm"] = about * (0.5 if c["clipped"] else 2.0)
    return s


EPS = 1e-6


# ------------------------------------------------------------------------------------ plain forms

def _spread(scale, rows, cols, block_rows):
    """The scale of every element, from one of every block."""
    full = scale.repeat_interleave(BLK, 1)[:, :cols]
    return full if block_rows == 1 else full.repeat_interleave(block_rows, 0)[:rows]


def _pow2_scale(amax):
    m, e = torch.frexp(amax)  # amax = m 2^e with m in [1/2, 1); 448 = 0.875 * 2^9
    e = torch.where(m > 0.875, e - 8, e - 9).clamp(min=-126)
    return torch.where(amax > 0, torch.ldexp(torch.ones_like(amax), e), torch.ones_like(amax))


def _values(x, block_rows=1):
    """The values that the codes of x stand for, in float32."""
    rows, cols = x.shape
    x = x.float()
    a = torch.nn.functional.pad(x.abs(), (0, -cols % BLK, 0, -rows % block_rows))
    a = a.view(a.shape[0] // block_rows, block_rows, -1, BLK).amax((1, 3))
    full = _spread(_pow2_scale(a), rows, cols, block_rows)
    return (x / full).to(torch.float8_e4m3fn).float() * full


def _plain(s):
    c, op = s["case"], s["case"]["op"]
    if op == "quantise":
        rows = _values(s["x"]).bfloat16()
        return (rows, _values(s["x"].t().contiguous()).bfloat16()) if c["both"] else rows
    if op == "product":
        a = s["a"].float() * _spread(s["sa"].float(), c["m"], c["k"], 1)
        b = s["b"].float() * _spread(s["sb"].float(), c["n"], c["k"], BLK if c["tile"] else 1)
        y = a @ b.t()
        return (y + s["bias"] if c["bias"] else y).to(_TYPES[c["out"]])
    if op == "linear_step":
        x, w, dy = s["x"].detach(), s["w"].detach(), s["dy"]
        wq = _values(w, BLK)
        y = _values(x) @ wq + s["bias"].detach()
        dx = _values(dy) @ wq.t()
        dw = _values(x.t().contiguous()) @ _values(dy.t().contiguous()).t()
        return y.to(x.dtype), dx.to(x.dtype), dw, dy.double().sum(0).float()
    if op in ("norm_quantise", "norm_train"):
        x, w = s["x"], s["w"]
        h = (x.float() + s["r"].float()).to(x.dtype) if c["residual"] else x
        hf = h.float()
        rstd = torch.rsqrt(hf.double().square().mean(1, keepdim=True) + EPS).float()  # 64 bits: codes next to a border follow it
        n = hf * rstd
        if op == "norm_quantise":
            q = _values(n * w).bfloat16()
            return (q, h) if c["residual"] else q
        y = (n * w).to(x.dtype)
        dy = s["dy"].float()
        g = dy * w
        dx = rstd * (g - n * (g * n).mean(1, keepdim=True))
        if c["residual"]:
            dx = dx + s["dh"].float()
        dw = (dy * n).double().sum(0).float()
        return (y, h, dx.to(x.dtype), dw) if c["residual"] else (y, dx.to(x.dtype), dw)
    total = torch.stack([t.double().square().sum() for t in s["g"]]).sum().sqrt()
    coef = torch.clamp(s["max_norm"] / (total + EPS), max=1.0).float()
    return [total.float()] + [(t.float() * coef).to(t.dtype) for t in s["g"]]


# ------------------------------------------------------------------------- the framework's own calls

def _own(s):
    from quantized_cnn_amd import fp8, ops
    c, op = s["case"], s["case"]["op"]
    if op == "quantise":
        if c["both"]:
            q, qt = ops.fp8_quantize(s["x"], forms="both")
            return ops.fp8_dequantize(q), ops.fp8_dequantize(qt)
        return ops.fp8_dequantize(ops.fp8_quantize(s["x"]))
    if op == "product":
        return ops.fp8_matmul(ops.Fp8Blocks(s["a"], s["sa"]), ops.Fp8Blocks(s["b"], s["sb"], block_rows=BLK if c["tile"] else 1),
                              bias=s["bias"], out_dtype=_TYPES[c["out"]])
    if op == "linear_step":
        y = fp8.linear(s["x"], s["w"], s["bias"])
        return (y.detach(),) + torch.autograd.grad(y, (s["x"], s["w"], s["bias"]), s["dy"])
    if op == "norm_quantise":
        q, h, _ = ops.rms_norm_forward(s["x"], s["w"], residual=s["r"], eps=EPS, quantize=True)
        q = ops.fp8_dequantize(q)
        return (q, h) if c["residual"] else q
    if op == "norm_train":
        y, h, rstd = ops.rms_norm_forward(s["x"], s["w"], residual=s["r"], eps=EPS)
        dx, dw = ops.rms_norm_backward(s["dy"], h, s["w"], rstd, dh=s["dh"])
        return (y, h, dx, dw) if c["residual"] else (y, dx, dw)
    return [ops.clip_grad_norm(s["g"], s["max_norm"], out=s["out"])] + s["out"]


def run(state):
    return _own(state) if own else _plain(state)


# -------------------------------------------------------------------------------- exact, in 64 bits

def _exact_values(x):
    """Row blocks of 128: codes and scales from logarithms and rounding to the format's steps, in double."""
    x = x.double()
    out = torch.empty_like(x)
    for j in range(0, x.shape[1], BLK):
        b = x[:, j:j + BLK]
        top = b.abs().amax(1, keepdim=True)
        e = torch.ceil(torch.log2(torch.where(top > 0, top, torch.full_like(top, 448.0)) / 448.0)).clamp(min=-126)
        e = torch.where(top > 448.0 * torch.exp2(e), e + 1, e)  # the logarithm's own rounding next to a power of two
        e = torch.where(top <= 448.0 * torch.exp2(e - 1), e - 1, e).clamp(min=-126)
        v = b / torch.exp2(e)
        step = torch.exp2(torch.floor(torch.log2(v.abs().clamp(min=2.0 ** -6))) - 3)  # 3 bits of mantissa, subnormals below 2^-6
        out[:, j:j + BLK] = torch.round(v / step) * step * torch.exp2(e)
    return out


def _exact_tiles(w):
    w = w.double()
    out = torch.empty_like(w)
    for i in range(0, w.shape[0], BLK):
        for j in range(0, w.shape[1], BLK):
            t = w[i:i + BLK, j:j + BLK]
            out[i:i + BLK, j:j + BLK] = _exact_flat(t)
    return out


def _exact_flat(t):
    top = t.abs().max()
    top = torch.where(top > 0, top, torch.full_like(top, 448.0))
    e = torch.ceil(torch.log2(top / 448.0)).clamp(min=-126)
    e = torch.where(top > 448.0 * torch.exp2(e), e + 1, e)
    e = torch.where(top <= 448.0 * torch.exp2(e - 1), e - 1, e).clamp(min=-126)
    v = t / torch.exp2(e)
    step = torch.exp2(torch.floor(torch.log2(v.abs().clamp(min=2.0 ** -6))) - 3)
    return torch.round(v / step) * step * torch.exp2(e)


def exact(case, seed):
    c, op = case, case["op"]
    s = prepare(case, seed)
    if op == "quantise":
        rows = _exact_values(s["x"])
        return (rows, _exact_values(s["x"].t())) if c["both"] else rows
    if op == "product":
        y = torch.zeros(c["m"], c["n"], device=DEV, dtype=torch.float64)
        at = torch.arange(c["n"], device=DEV) // (BLK if c["tile"] else 1)
        for b, j in enumerate(range(0, c["k"], BLK)):
            p = s["a"][:, j:j + BLK].double() @ s["b"][:, j:j + BLK].double().t()
            y += p * s["sa"][:, b:b + 1].double() * s["sb"].double()[at, b][None]
        return y + s["bias"].double() if c["bias"] else y
    if op == "linear_step":
        x, w, dy = s["x"].detach(), s["w"].detach(), s["dy"]
        wq = _exact_tiles(w)
        return (_exact_values(x) @ wq + s["bias"].detach().double(), _exact_values(dy) @ wq.t(),
                _exact_values(x.t()) @ _exact_values(dy.t()).t(), dy.double().sum(0))
    if op in ("norm_quantise", "norm_train"):
        x, w = s["x"], s["w"].double()
        h = (x.double() + s["r"].double()).to(x.dtype).double() if c["residual"] else x.double()
        r = (h.square().sum(1, keepdim=True) / h.shape[1] + EPS) ** -0.5
        y = h * r * w
        if op == "norm_quantise":
            return (_exact_values(y), h) if c["residual"] else _exact_values(y)
        dy = s["dy"].double()
        dx = r * dy * w - h * r ** 3 * (dy * w * h).sum(1, keepdim=True) / h.shape[1]
        dw = (dy * h * r).sum(0)
        return (y, h, dx + s["dh"].double(), dw) if c["residual"] else (y, dx, dw)
    total = math.sqrt(sum(float(t.double().square().sum()) for t in s["g"]))
    coef = min(1.0, s["max_norm"] / (total + EPS))
    return [torch.tensor(total, dtype=torch.float64)] + [t.double() * coef for t in s["g"]]
