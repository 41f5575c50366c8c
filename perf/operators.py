"""What is measured of the operators of an 8-bit Linear + LayerNorm training block.

  norm_fwd   layer norm over the last dimension with the row statistics that its backward pass reads
  norm_bwd   its backward pass: the input's gradient and the reduced gradients of weight and bias, the input read as f32 or from
             an 8-bit checkpoint
  save       an 8-bit activation checkpoint written and restored (e4m3 with a power-of-two scale for each 1 x 128 or 128 x 128 block)
  product    the Linear forward: a product of two block-scaled 8-bit matrices, f32 out, bias and activation
  wgrad      the weight gradient of a product whose left operand was kept as an 8-bit checkpoint

`run` is either the plain form in elementary torch operations or, where `own` is true, the calls of rustorch_b200.
"""
import torch

own = False

EPS = 1e-5
BLOCK = 128
E4M3_MAX = 448.0


def listed():
    return [
        # a few tokens of one generation step: latency
        {"name": "norm_fwd_step", "op": "norm_fwd", "rows": 16, "d": 1024, "act": 0},
        # a training batch of the MLP's hidden width
        {"name": "norm_fwd_batch", "op": "norm_fwd", "rows": 8192, "d": 4096, "act": 0},
        # the same batch's backward pass
        {"name": "norm_bwd_batch", "op": "norm_bwd", "rows": 8192, "d": 4096, "act": 0, "saved": False},
        # a ragged batch of an odd width (rows that no 16-byte load fits), with the fused activation
        {"name": "norm_bwd_odd", "op": "norm_bwd", "rows": 1531, "d": 1001, "act": 3, "saved": False},
        # long sequences whose input was kept in 8 bits
        {"name": "norm_bwd_saved", "op": "norm_bwd", "rows": 16384, "d": 2048, "act": 0, "saved": True},
        # a small ragged activation kept and restored
        {"name": "save_ragged", "op": "save", "rows": 777, "d": 1000, "block_rows": 1},
        # a training batch's activations
        {"name": "save_batch", "op": "save", "rows": 16384, "d": 4096, "block_rows": 1},
        # one token against a square layer: a stream over the weight
        {"name": "product_token", "op": "product", "m": 1, "n": 4096, "k": 4096, "act": 0, "b_rows": 128},
        # ragged everything, a scale for each row block of both sides
        {"name": "product_ragged", "op": "product", "m": 333, "n": 1000, "k": 1000, "act": 1, "b_rows": 1},
        # a large training batch
        {"name": "product_batch", "op": "product", "m": 8192, "n": 4096, "k": 8192, "act": 0, "b_rows": 128},
        # a short ragged sequence's weight gradient
        {"name": "wgrad_ragged", "op": "wgrad", "m": 515, "n": 1000, "k": 520},
        # a training batch's weight gradient
        {"name": "wgrad_batch", "op": "wgrad", "m": 8192, "n": 4096, "k": 4096},
    ]


def _size(rng, lo, hi):
    """A size spread over its logarithm; half of them are rounded to a multiple of 64, the others stay odd as they fall."""
    v = int(round(lo * (hi / lo) ** rng.random()))
    if rng.random() < 0.5 and v >= 64:
        v = v // 64 * 64
    return max(lo, min(hi, v))


def draw(rng):
    op = rng.choice(["norm_fwd", "norm_bwd", "norm_bwd", "save", "product", "product", "wgrad", "wgrad"])
    if op in ("norm_fwd", "norm_bwd", "save"):
        case = {"op": op, "rows": _size(rng, 1, 16384), "d": _size(rng, 32, 16384)}
        while case["rows"] * case["d"] > 8192 * 4096:
            case["rows"] = max(1, case["rows"] // 2)
        if op == "save":
            case["block_rows"] = rng.choice([1, 1, 128])
        else:
            case["act"] = rng.choice([0, 0, 0, 2, 3])
        if op == "norm_bwd":
            case["saved"] = rng.random() < 0.5
        return case
    most = 8192 * 4096 * (8192 if op == "product" else 4096)
    m, n, k = _size(rng, 1, 8192), _size(rng, 64, 8192), _size(rng, 64, 8192)
    while m * n * k > most:
        m = max(1, m // 2)
    case = {"op": op, "m": m, "n": n, "k": k}
    if op == "product":
        case["act"] = rng.choice([0, 0, 1, 2, 3])
        case["b_rows"] = rng.choice([128, 128, 1])
    return case


def _blocks(n):
    return -(-n // BLOCK)


def work(case):
    op = case["op"]
    if op in ("norm_fwd", "norm_bwd", "save"):
        r, d = case["rows"], case["d"]
        if op == "norm_fwd":
            return {"bytes": 8 * r * d + 8 * r + 8 * d, "flops": 8 * r * d}
        if op == "norm_bwd":
            x = r * d + r * _blocks(d) if case["saved"] else 4 * r * d
            return {"bytes": x + 8 * r * d + 8 * r + 16 * d, "flops": 16 * r * d}
        scales = -(-r // case["block_rows"]) * _blocks(d)
        # written and read back: 4 + 1 bytes a value each way
        return {"bytes": 10 * r * d + 2 * scales, "flops": 4 * r * d}
    m, n, k = case["m"], case["n"], case["k"]
    if op == "product":
        scales = m * _blocks(k) + -(-n // case["b_rows"]) * _blocks(k)
        return {"bytes": m * k + n * k + scales + 4 * n + 4 * m * n, "flops": 2 * m * n * k}
    return {"bytes": m * k + m * _blocks(k) + 4 * m * n + 4 * k * n, "flops": 2 * m * n * k}


# ------------------------------------------------------------------ inputs


def _activations(g, rows, d):
    """Values with a scale and an offset for each row and a few large columns, as the input of a layer norm has them."""
    x = torch.randn((rows, d), device="cuda", generator=g)
    x *= 0.25 + 2.0 * torch.rand((rows, 1), device="cuda", generator=g)
    x *= 1.0 + 15.0 * (torch.rand((1, d), device="cuda", generator=g) > 0.99)
    return x.add_(torch.randn((rows, 1), device="cuda", generator=g), alpha=0.5)


def _saved(x, block_rows):
    """x as 8-bit blocks: (e4m3 values, e8m0 scales), by the format's rule."""
    rows, d = x.shape
    rb, cb = -(-rows // block_rows), _blocks(d)
    full = torch.zeros((rb * block_rows, cb * BLOCK), device=x.device)
    full[:rows, :d] = x
    top = full.abs().view(rb, block_rows, cb, BLOCK).amax(dim=(1, 3))
    bits = top.view(torch.int32)
    byte = ((bits >> 23) - 8 + ((bits & 0x7FFFFF) > 0x600000).int()).clamp_(min=1)
    byte = torch.where(top == 0, torch.full_like(byte, 127), byte)
    inverse = ((254 - byte) << 23).view(torch.float32)
    inverse = inverse.repeat_interleave(block_rows, 0)[:rows].repeat_interleave(BLOCK, 1)[:, :d]
    return (x * inverse).to(torch.float8_e4m3fn), byte.to(torch.uint8).view(torch.float8_e8m0fnu)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    op = case["op"]
    s = {"case": case}
    if op in ("norm_fwd", "norm_bwd", "save"):
        rows, d = case["rows"], case["d"]
        x = _activations(g, rows, d)
        if op == "save":
            return dict(s, x=x)
        s["w"] = 1.0 + 0.1 * torch.randn(d, device="cuda", generator=g)
        s["b"] = 0.1 * torch.randn(d, device="cuda", generator=g)
        if op == "norm_fwd":
            return dict(s, x=x)
        # what the forward pass left: its input (as f32 or as a checkpoint) and the rows' statistics
        s["mean"] = x.double().mean(1).float()
        s["rstd"] = (x.double().var(1, unbiased=False) + EPS).rsqrt().float()
        s["grad"] = 1e-3 * torch.randn((rows, d), device="cuda", generator=g)
        if case["saved"]:
            s["x"], s["x_scale"] = _saved(x, 1)
        else:
            s["x"], s["x_scale"] = x, None
        return s
    m, n, k = case["m"], case["n"], case["k"]
    s["a"], s["a_scale"] = _saved(_activations(g, m, k), 1)
    if op == "product":
        weight = torch.randn((n, k), device="cuda", generator=g) * k ** -0.5
        s["weight"], s["weight_scale"] = _saved(weight, case["b_rows"])
        s["bias"] = 0.1 * torch.randn(n, device="cuda", generator=g)
    else:
        s["grad"] = 1e-3 * torch.randn((m, n), device="cuda", generator=g)
    return s


# ------------------------------------------------------------------ one pass


def _restored(q, scale):
    """The f32 values that 8-bit blocks stand for."""
    rows, d = q.shape
    block_rows = 1 if scale.shape[0] == rows else BLOCK
    factor = (scale.view(torch.uint8).int() << 23).view(torch.float32)
    factor = factor.repeat_interleave(block_rows, 0)[:rows].repeat_interleave(BLOCK, 1)[:, :d]
    return q.float() * factor


def _activated(z, act):
    if act == 1:
        return z.clamp(min=0)
    if act == 2:
        return 1 / (1 + torch.exp(-z))
    return torch.tanh(z) if act == 3 else z


def _through_activation(grad, z, act):
    """grad times the activation's derivative at z."""
    if act == 1:
        return grad * (z > 0)
    if act == 2:
        y = 1 / (1 + torch.exp(-z))
        return grad * y * (1 - y)
    return grad * (1 - torch.tanh(z) ** 2) if act == 3 else grad


def run(state):
    s, case = state, state["case"]
    op = case["op"]
    if own:
        import rustorch_b200 as rb
        if op == "norm_fwd":
            return rb.layer_norm_fwd(s["x"], s["w"], s["b"], EPS, case["act"])
        if op == "norm_bwd":
            return rb.layer_norm_backward(s["x"], s["mean"], s["rstd"], s["grad"], s["w"], s["b"], case["act"],
                                          x_scale=s["x_scale"])
        if op == "save":
            return rb.fp8_dequantize(*rb.fp8_quantize(s["x"], case["block_rows"]))
        if op == "product":
            return rb.fp8_matmul(s["a"], s["a_scale"], s["weight"].t(), s["weight_scale"].t(), s["bias"], case["act"])
        return rb.matmul_backward_fp8(s["a"], s["a_scale"], None, s["grad"], need_a=False)[1]
    if op == "norm_fwd":
        x = s["x"]
        mean = x.mean(1, keepdim=True)
        centred = x - mean
        rstd = 1 / torch.sqrt((centred * centred).mean(1, keepdim=True) + EPS)
        return _activated(centred * rstd * s["w"] + s["b"], case["act"]), mean[:, 0], rstd[:, 0]
    if op == "norm_bwd":
        x = _restored(s["x"], s["x_scale"]) if case["saved"] else s["x"]
        rstd = s["rstd"][:, None]
        unit = (x - s["mean"][:, None]) * rstd
        dz = _through_activation(s["grad"], unit * s["w"] + s["b"], case["act"])
        u = dz * s["w"]
        dx = rstd * (u - u.mean(1, keepdim=True) - unit * (u * unit).mean(1, keepdim=True))
        return dx, (dz * unit).sum(0), dz.sum(0)
    if op == "save":
        return _restored(*_saved(s["x"], case["block_rows"]))
    if op == "product":
        c = _restored(s["a"], s["a_scale"]) @ _restored(s["weight"], s["weight_scale"]).t()
        return _activated(c + s["bias"], case["act"])
    return _restored(s["a"], s["a_scale"]).t() @ s["grad"]


# ------------------------------------------------------------------ the definition in 64 bits


def _times_power(v, e):
    """v 2^e for whole e, exactly: the power's bits are put together, since a computed one may be off in its last place."""
    return v * ((e.long() + 1023) << 52).view(torch.float64)


def _values64(q, scale):
    """sum over the code's fields: (-1)^s 2^(e-7) (1 + m/8), or (-1)^s 2^-6 m/8 where e = 0, times 2^(byte-127)."""
    code = q.view(torch.uint8).long()
    e, m = (code >> 3) & 15, (code & 7).double()
    mantissa = torch.where(e > 0, 1 + m / 8, m / 8)
    v = _times_power(mantissa, e.clamp(min=1) - 7)
    v = torch.where(code > 127, -v, v)
    exponent = scale.view(torch.uint8).long() - 127
    row = torch.arange(q.shape[0], device=q.device) // (1 if scale.shape[0] == q.shape[0] else BLOCK)
    col = torch.arange(q.shape[1], device=q.device) // BLOCK
    return _times_power(v, exponent[row][:, col])


def _sigmoid64(z):
    return 0.5 + 0.5 * torch.tanh(0.5 * z)


def exact(case, seed):
    s, op = prepare(case, seed), case["op"]
    act = case.get("act", 0)

    def activated(z):
        return (z, torch.relu(z), _sigmoid64(z), torch.tanh(z))[act] if act else z

    if op == "norm_fwd":
        x = s["x"].double()
        var, mean = torch.var_mean(x, 1, correction=0)
        rstd = (var + EPS) ** -0.5
        y = activated((x - mean[:, None]) * (rstd[:, None] * s["w"].double()) + s["b"].double())
        return y, mean, rstd
    if op == "norm_bwd":
        x = _values64(s["x"], s["x_scale"]) if case["saved"] else s["x"].double()
        w, b, rstd = s["w"].double(), s["b"].double(), s["rstd"].double()
        unit = (x - s["mean"].double()[:, None]) * rstd[:, None]
        z = unit * w + b
        slope = (1.0, (z > 0).double(), _sigmoid64(z) * _sigmoid64(-z), torch.cosh(z) ** -2)[act]
        dz = s["grad"].double() * slope
        d = case["d"]
        first = dz @ w / d
        second = (dz * unit) @ w / d
        dx = rstd[:, None] * (dz * w - first[:, None] - unit * second[:, None])
        return dx, torch.einsum("rd,rd->d", dz, unit), torch.einsum("rd->d", dz)
    if op == "save":
        x, br = s["x"].double(), case["block_rows"]
        rows, d = x.shape
        row = torch.arange(rows, device=x.device) // br
        col = torch.arange(d, device=x.device) // BLOCK
        cell = row[:, None] * _blocks(d) + col[None, :]
        top = torch.zeros(int(cell.max()) + 1, dtype=torch.float64, device=x.device)
        top.scatter_reduce_(0, cell.reshape(-1), x.abs().reshape(-1), "amax")
        mantissa, exponent = torch.frexp(top / E4M3_MAX)  # mantissa in [0.5, 1)
        exponent = exponent - (mantissa == 0.5).int()
        exponent = torch.where(top > 0, exponent.clamp(min=-126), torch.zeros_like(exponent))[cell]
        v = _times_power(x, -exponent)
        step = (torch.frexp(v).exponent - 1).clamp(min=-6) - 3
        step = torch.where(v == 0, torch.zeros_like(step), step)
        return _times_power(torch.round(_times_power(v, -step)), step + exponent)
    if op == "product":
        c = torch.einsum("mk,nk->mn", _values64(s["a"], s["a_scale"]), _values64(s["weight"], s["weight_scale"]))
        return activated(c + s["bias"].double())
    return torch.einsum("mk,mn->kn", _values64(s["a"], s["a_scale"]), s["grad"].double())
