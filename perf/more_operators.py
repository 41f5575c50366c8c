"""What is measured of the operators of a low-precision Linear block: the root-mean-square norm in front of it and its products in 4 bits.

  norm      a residual's addition and the root-mean-square norm of the sum, with the statistics that the backward pass reads
  norm8     the same with its output in 8 bits (e4m3, a power-of-two scale for each 128 columns), as the 8-bit product takes it
  norm_bwd  its backward pass: the input's gradient, the residual stream's added, and the weight's; the input read as f32 or from an
            8-bit checkpoint
  save4     a matrix or its transpose in microscaled 4 bits (e2m1, a power-of-two scale for each 32 columns), written and restored
  product4  the Linear forward: a product of two such matrices, f32 out, bias and activation

`run` is either the plain form in elementary torch operations or, where `own` is true, the calls of rustorch_b200.
"""
import torch

own = False

EPS = 1e-5


def listed():
    return [
        # a few tokens of one generation step: latency
        {"name": "norm_step", "op": "norm", "rows": 16, "d": 1024, "residual": True},
        # a training batch of the MLP's hidden width
        {"name": "norm_batch", "op": "norm", "rows": 8192, "d": 4096, "residual": True},
        # a ragged batch of an odd width (rows that no 16-byte load fits), the first layer's: no residual yet
        {"name": "norm8_ragged", "op": "norm8", "rows": 1531, "d": 1001, "residual": False},
        # a training batch whose next product is in 8 bits
        {"name": "norm8_batch", "op": "norm8", "rows": 8192, "d": 4096, "residual": True},
        # a ragged batch of an odd width whose input was kept in 8 bits
        {"name": "norm_bwd_ragged", "op": "norm_bwd", "rows": 1531, "d": 1001, "saved": True, "residual": False},
        # a training batch's backward pass, the residual stream's gradient coming in beside
        {"name": "norm_bwd_batch", "op": "norm_bwd", "rows": 8192, "d": 4096, "saved": False, "residual": True},
        # a small ragged activation
        {"name": "save4_ragged", "op": "save4", "rows": 777, "d": 1000, "columns": False},
        # a training batch's gradient transposed, as the weight gradient's product takes it
        {"name": "save4_columns", "op": "save4", "rows": 8192, "d": 4096, "columns": True},
        # one token against a square layer: a stream over the weight
        {"name": "product4_token", "op": "product4", "m": 1, "n": 4096, "k": 4096, "act": 0},
        # ragged everything
        {"name": "product4_ragged", "op": "product4", "m": 333, "n": 1000, "k": 1000, "act": 1},
        # a batch of generation steps against a large layer
        {"name": "product4_steps", "op": "product4", "m": 48, "n": 8192, "k": 8192, "act": 0},
        # a large training batch
        {"name": "product4_batch", "op": "product4", "m": 8192, "n": 4096, "k": 8192, "act": 0},
    ]


def _size(rng, lo, hi):
    """A size spread over its logarithm; half of them are rounded to a multiple of 64, the others stay odd as they fall."""
    v = int(round(lo * (hi / lo) ** rng.random()))
    if rng.random() < 0.5 and v >= 64:
        v = v // 64 * 64
    return max(lo, min(hi, v))


def draw(rng):
    op = rng.choice(["norm", "norm8", "norm_bwd", "norm_bwd", "save4", "save4", "product4", "product4", "product4"])
    if op != "product4":
        case = {"op": op, "rows": _size(rng, 1, 16384), "d": _size(rng, 32, 16384)}
        while case["rows"] * case["d"] > 8192 * 4096:
            case["rows"] = max(1, case["rows"] // 2)
        if op == "save4":
            case["columns"] = rng.random() < 0.5
        else:
            case["residual"] = rng.random() < 0.7
        if op == "norm_bwd":
            case["saved"] = rng.random() < 0.5
        return case
    m, n, k = _size(rng, 1, 8192), _size(rng, 64, 8192), _size(rng, 64, 8192)
    while m * n * k > 8192 * 4096 * 8192:
        m = max(1, m // 2)
    return {"op": op, "m": m, "n": n, "k": k, "act": rng.choice([0, 0, 1, 2, 3])}


def _blocks(n, size):
    return -(-n // size)


def work(case):
    op = case["op"]
    if op == "product4":
        m, n, k = case["m"], case["n"], case["k"]
        held = _blocks(k, 2) + _blocks(k, 32)  # bytes of a row: codes and scales
        return {"bytes": (m + n) * held + 4 * n + 4 * m * n, "flops": 2 * m * n * k}
    r, d = case["rows"], case["d"]
    if op == "save4":
        # written and read back: 4 bytes a value and a half, each way
        rows, cols = (d, r) if case["columns"] else (r, d)
        return {"bytes": 8 * r * d + 2 * rows * (_blocks(cols, 2) + _blocks(cols, 32)), "flops": 4 * r * d}
    stream = 4 * r * d if case["residual"] else 0  # the residual, its sum, or its gradient
    if op == "norm":
        return {"bytes": 8 * r * d + 2 * stream + 4 * r + 4 * d, "flops": 5 * r * d}
    if op == "norm8":
        return {"bytes": 5 * r * d + 2 * stream + r * _blocks(d, 128) + 4 * r + 4 * d, "flops": 7 * r * d}
    x = r * d + r * _blocks(d, 128) if case["saved"] else 4 * r * d
    return {"bytes": x + 8 * r * d + stream + 4 * r + 8 * d, "flops": 11 * r * d}


# ------------------------------------------------------------------ inputs


def _activations(g, rows, d):
    """Values with a scale and an offset for each row and a few large columns, as the input of a norm has them."""
    x = torch.randn((rows, d), device="cuda", generator=g)
    x *= 0.25 + 2.0 * torch.rand((rows, 1), device="cuda", generator=g)
    x *= 1.0 + 15.0 * (torch.rand((1, d), device="cuda", generator=g) > 0.99)
    return x.add_(torch.randn((rows, 1), device="cuda", generator=g), alpha=0.5)


def _scaled(x, block, largest):
    """x's rows in blocks of `block` columns, each divided by the smallest power of two (2^-126 and more) that holds its largest
    magnitude within `largest` = 1.75 2^8 or 1.5 2^2: (the quotients, the exponents' bytes)."""
    rows, d = x.shape
    cb = _blocks(d, block)
    full = torch.zeros((rows, cb * block), device=x.device)
    full[:, :d] = x
    top = full.abs().view(rows, cb, block).amax(dim=2)
    bits = top.view(torch.int32)
    room, mantissa = (8, 0x600000) if largest == 448.0 else (2, 0x400000)
    byte = ((bits >> 23) - room + ((bits & 0x7FFFFF) > mantissa).int()).clamp_(min=1)
    byte = torch.where(top == 0, torch.full_like(byte, 127), byte)
    inverse = ((254 - byte) << 23).view(torch.float32)
    return full * inverse.repeat_interleave(block, 1), byte.to(torch.uint8).view(torch.float8_e8m0fnu)


def _saved8(x):
    """x as 8-bit blocks of a row's 128 columns: (e4m3 values, e8m0 scales)."""
    v, scale = _scaled(x, 128, 448.0)
    return v[:, :x.shape[1]].to(torch.float8_e4m3fn), scale


def _saved4(x):
    """x as 4-bit blocks of a row's 32 columns: (e2m1 codes, two in a byte, the first in its low bits; e8m0 scales)."""
    v, scale = _scaled(x, 32, 6.0)
    a = v.abs()
    half = torch.round(a * 2).clamp_(max=4)     # below 2 in steps of a half: codes 0..4
    whole = torch.round(a).clamp_(2, 4) + 2     # from 2 to 4 in steps of 1: codes 4..6
    double = torch.round(a * 0.5).clamp_(max=3) + 4  # from 4 to 6: codes 6, 7
    code = torch.where(a < 2, half, torch.where(a < 4, whole, double)).to(torch.uint8)
    code |= torch.signbit(v).to(torch.uint8) << 3
    held = _blocks(x.shape[1], 2)
    return (code[:, 0::2] | (code[:, 1::2] << 4))[:, :held].contiguous().view(torch.float4_e2m1fn_x2), scale


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    op = case["op"]
    s = {"case": case}
    if op == "product4":
        m, n, k = case["m"], case["n"], case["k"]
        s["a"], s["a_scale"] = _saved4(_activations(g, m, k))
        s["weight"], s["weight_scale"] = _saved4(torch.randn((n, k), device="cuda", generator=g) * k ** -0.5)
        s["bias"] = 0.1 * torch.randn(n, device="cuda", generator=g)
        return s
    rows, d = case["rows"], case["d"]
    x = _activations(g, rows, d)
    if op == "save4":
        return dict(s, x=x)
    s["w"] = 1.0 + 0.1 * torch.randn(d, device="cuda", generator=g)
    if op in ("norm", "norm8"):
        s["residual"] = 2.0 * torch.randn((rows, d), device="cuda", generator=g) if case["residual"] else None
        return dict(s, x=x)
    # what the forward pass left: the norm's input (as f32 or as a checkpoint) and the rows' statistic
    s["rstd"] = (x.double().square().mean(1) + EPS).rsqrt().float()
    s["grad"] = 1e-3 * torch.randn((rows, d), device="cuda", generator=g)
    s["grad_sum"] = 1e-3 * torch.randn((rows, d), device="cuda", generator=g) if case["residual"] else None
    s["x"], s["x_scale"] = _saved8(x) if case["saved"] else (x, None)
    return s


# ------------------------------------------------------------------ one pass


def _factors(scale, block, d):
    return (scale.view(torch.uint8).int() << 23).view(torch.float32).repeat_interleave(block, 1)[:, :d]


def _restored8(q, scale):
    """The f32 values that 8-bit blocks stand for."""
    return q.float() * _factors(scale, 128, q.shape[1])


def _restored4(q, scale, d):
    """The f32 values that 4-bit blocks stand for."""
    byte = q.view(torch.uint8)
    code = torch.stack((byte & 15, byte >> 4), dim=2).view(byte.shape[0], -1)[:, :d].int()
    c = (code & 7).float()
    a = torch.where(c < 4, c * 0.5, torch.where(c < 6, c - 2, c * 2 - 8))
    return torch.where(code > 7, -a, a) * _factors(scale, 32, d)


def _activated(z, act):
    if act == 1:
        return z.clamp(min=0)
    if act == 2:
        return 1 / (1 + torch.exp(-z))
    return torch.tanh(z) if act == 3 else z


def run(state):
    s, case = state, state["case"]
    op = case["op"]
    if own:
        import rustorch_b200 as rb
        if op == "norm":
            return rb.rms_norm_fwd(s["x"], s["w"], EPS, residual=s["residual"])
        if op == "norm8":
            return rb.rms_norm_fp8(s["x"], s["w"], EPS, residual=s["residual"])
        if op == "norm_bwd":
            return rb.rms_norm_backward(s["x"], s["rstd"], s["grad"], s["w"], grad_sum=s["grad_sum"], x_scale=s["x_scale"])
        if op == "save4":
            x = s["x"].t() if case["columns"] else s["x"]
            q, scale = rb.fp4_quantize(x)
            return rb.fp4_dequantize(q, scale, cols=x.shape[1])
        return rb.fp4_matmul(s["a"], s["a_scale"], s["weight"].t(), s["weight_scale"].t(), s["bias"], case["act"])
    if op in ("norm", "norm8"):
        total = s["x"] if s["residual"] is None else s["x"] + s["residual"]
        rstd = 1 / torch.sqrt((total * total).mean(1, keepdim=True) + EPS)
        y = total * rstd * s["w"]
        return (*((y,) if op == "norm" else _saved8(y)), total, rstd[:, 0])
    if op == "norm_bwd":
        x = _restored8(s["x"], s["x_scale"]) if case["saved"] else s["x"]
        rstd = s["rstd"][:, None]
        unit = x * rstd
        u = s["grad"] * s["w"]
        dx = rstd * (u - unit * (u * unit).mean(1, keepdim=True))
        if s["grad_sum"] is not None:
            dx = dx + s["grad_sum"]
        return dx, (s["grad"] * unit).sum(0)
    if op == "save4":
        x = s["x"].t() if case["columns"] else s["x"]
        return _restored4(*_saved4(x), x.shape[1])
    k = 2 * s["a"].shape[1]
    c = _restored4(s["a"], s["a_scale"], k) @ _restored4(s["weight"], s["weight_scale"], k).t()
    return _activated(c + s["bias"], case["act"])


# ------------------------------------------------------------------ the definition in 64 bits


def _power(e):
    """2^e for whole e, exactly: the power's bits are put together, since a computed one may be off in its last place."""
    return ((e.long() + 1023) << 52).view(torch.float64)


def _rounded64(x, block, largest, bits, low):
    """(values, exponents): x's rows by blocks of columns, v = x 2^-e with the smallest e >= -126 that holds the block's largest
    magnitude within `largest` (0 for a block of zeros), rounded to `bits` fraction bits, in steps of 2^(low - bits) below 2^low."""
    rows, d = x.shape
    cell = torch.arange(d, device=x.device) // block
    top = torch.zeros((rows, int(cell[-1]) + 1), dtype=torch.float64, device=x.device)
    top.scatter_reduce_(1, cell.expand(rows, d), x.abs(), "amax")
    mantissa, exponent = torch.frexp(top / largest)  # mantissa in [0.5, 1)
    exponent = exponent - (mantissa == 0.5).int()
    exponent = torch.where(top > 0, exponent.clamp(min=-126), torch.zeros_like(exponent))
    v = x * _power(-exponent[:, cell])
    step = torch.frexp(v).exponent - 1
    step = torch.where(v == 0, torch.full_like(step, low), step.clamp(min=low)) - bits
    return torch.round(v * _power(-step)) * _power(step), exponent


def _values8(q, scale):
    """sum over the code's fields: (-1)^s 2^(e-7) (1 + m/8), or (-1)^s 2^-6 m/8 where e = 0, times 2^(byte-127)."""
    code = q.view(torch.uint8).long()
    e, m = (code >> 3) & 15, (code & 7).double()
    v = torch.where(e > 0, 1 + m / 8, m / 8) * _power(e.clamp(min=1) - 7)
    exponent = scale.view(torch.uint8).long() - 127
    return torch.where(code > 127, -v, v) * _power(exponent[:, torch.arange(q.shape[1], device=q.device) // 128])


def _values4(q, scale):
    """The code's fields: (-1)^s 2^(e-1) (1 + m/2), or (-1)^s m/2 where e = 0, times 2^(byte-127)."""
    byte = q.view(torch.uint8).long()
    code = torch.empty((byte.shape[0], 2 * byte.shape[1]), dtype=torch.int64, device=byte.device)
    code[:, 0::2], code[:, 1::2] = byte & 15, byte >> 4
    e, m = (code >> 1) & 3, (code & 1).double()
    v = torch.where(e > 0, 1 + m / 2, m / 2) * _power(e.clamp(min=1) - 1)
    exponent = scale.view(torch.uint8).long() - 127
    return torch.where(code > 7, -v, v) * _power(exponent[:, torch.arange(code.shape[1], device=q.device) // 32])


def exact(case, seed):
    s, op = prepare(case, seed), case["op"]
    if op in ("norm", "norm8"):
        total = s["x"].double()
        if s["residual"] is not None:
            total = total + s["residual"].double()
        rstd = (torch.linalg.vector_norm(total, dim=1) ** 2 / case["d"] + EPS) ** -0.5
        y = total * (rstd[:, None] * s["w"].double())
        if op == "norm":
            return y, total, rstd
        v, exponent = _rounded64(y, 128, 448.0, 3, -6)
        return v, _power(exponent), total, rstd
    if op == "norm_bwd":
        x = _values8(s["x"], s["x_scale"]) if case["saved"] else s["x"].double()
        w, rstd, grad = s["w"].double(), s["rstd"].double(), s["grad"].double()
        unit = x * rstd[:, None]
        along = (grad * unit) @ w / case["d"]
        dx = rstd[:, None] * (grad * w - unit * along[:, None])
        if s["grad_sum"] is not None:
            dx += s["grad_sum"].double()
        return dx, torch.einsum("rd,rd->d", grad, unit)
    if op == "save4":
        x = s["x"].double()
        v, exponent = _rounded64(x.t().contiguous() if case["columns"] else x, 32, 6.0, 1, 0)
        return v * _power(exponent).repeat_interleave(32, 1)[:, :v.shape[1]]
    z = torch.einsum("mk,nk->mn", _values4(s["a"], s["a_scale"]), _values4(s["weight"], s["weight_scale"]))
    z += s["bias"].double()
    return (z, torch.relu(z), 0.5 + 0.5 * torch.tanh(0.5 * z), torch.tanh(z))[case["act"]]
