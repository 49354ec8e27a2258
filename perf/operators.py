"""Cases that time the block-scaled float8, layer-norm and gradient-clipping operators.

`run` makes one pass through an operator: with `own` true as a user calls it through
`float8_experimental_b200`, otherwise in a plain form made of elementary torch operations in 32 bits.
`exact` restates the operators' definitions in 64 bits.

Definitions.  A block is 128 consecutive elements of a row (1 x 128), of a column (128 x 1) or a
128 x 128 square; the last block of a dimension may be shorter.  With a = max(max|x| over the block, 1e-12),
    s = 2^-e,  e the largest whole number with a * 2^e <= 448,     q = e4m3(x * 2^e)   (nearest, ties to even)
and the block stands for q * s.  A block-scaled product multiplies the values that two such matrices stand
for.  A block-scaled linear layer takes x by rows and W by squares for the output, the output's
gradient by rows and W for x's gradient, and both of them by columns for W's gradient.
"""
import math

import torch

own = False

_DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_BLOCK = 128
_E4M3_MAX = 448.0


# ---------------------------------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------------------------------
def listed():
    return [
        # one token through an attention projection of a 4096-wide model: launch latency and 16 MB of weights
        {"name": "infer_1x4096x4096", "op": "infer", "m": 1, "k": 4096, "n": 4096, "dtype": "bf16", "bias": False},
        # a decode batch through the widest projection of an 8192-wide model, with bias: weight bandwidth
        {"name": "infer_37x8192x28672", "op": "infer", "m": 37, "k": 8192, "n": 28672, "dtype": "bf16", "bias": True},
        # a prefill chunk against weights whose block scales came with a checkpoint (any fp32 value), an inner
        # size that ends inside a block
        {"name": "product_300x4104x4096", "op": "product", "m": 300, "k": 4104, "n": 4096, "dtype": "fp16",
         "bias": False},
        # a training step (output and both gradients) of the output projection of an 8192-wide model: tensor rate
        {"name": "train_16384x8192x8192", "op": "train", "m": 16384, "k": 8192, "n": 8192, "dtype": "bf16",
         "bias": False},
        # a training step of an up projection with a token count that fills no tile, with bias, in fp16
        {"name": "train_2039x4096x14336", "op": "train", "m": 2039, "k": 4096, "n": 14336, "dtype": "fp16",
         "bias": True},
        # the casts of a training step's activations, by rows and by columns: memory bandwidth
        {"name": "cast_16384x8192", "op": "cast", "rows": 16384, "cols": 8192, "dtype": "bf16"},
        # the same of an fp32 tensor that ends inside a block both ways
        {"name": "cast_1003x4100", "op": "cast", "rows": 1003, "cols": 4100, "dtype": "fp32"},
        # the norm of a few tokens while serving: launch latency
        {"name": "norm_8x8192", "op": "norm", "rows": 8, "cols": 8192, "dtype": "bf16", "affine": "bf16"},
        # forward and backward of the norm of a training step: memory bandwidth
        {"name": "norm_train_16384x8192", "op": "norm_train", "rows": 16384, "cols": 8192, "dtype": "bf16",
         "affine": "bf16"},
        # an odd width in fp32, rows that are not aligned to 16 bytes
        {"name": "norm_train_4099x1030", "op": "norm_train", "rows": 4099, "cols": 1030, "dtype": "fp32",
         "affine": "fp32"},
        # gradients of four 4096-wide decoder blocks, above the bound: every gradient is scaled
        {"name": "clip_blocks", "op": "clip", "tensors": 28, "largest": 14336 * 4096, "smallest": 1024 * 4096,
         "dtype": "bf16", "active": True},
        # many small gradients below the bound (norm weights, biases, adapters): nothing is scaled
        {"name": "clip_many_small", "op": "clip", "tensors": 400, "largest": 65537, "smallest": 33, "dtype": "fp32",
         "active": False},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """One more case of the same ranges; none costs more than the largest listed one."""
    op = rng.choice(["infer", "product", "train", "cast", "norm", "norm_train", "clip"])
    if op in ("infer", "product", "train"):
        m = _log_int(rng, 1, 512) if op != "train" else _log_int(rng, 16, 16384)
        k, n = _log_int(rng, 100, 28672), _log_int(rng, 100, 28672)
        while k * n > 28672 * 8192 or m * k * n > 16384 * 8192 * 8192:
            k, n = max(100, k * 3 // 4), max(100, n * 3 // 4)
        if rng.random() < 0.7:  # most layers have sizes of whole 16-byte rows
            k, n = (k + 15) // 16 * 16, (n + 15) // 16 * 16
        return {"op": op, "m": m, "k": k, "n": n, "dtype": rng.choice(["bf16", "fp16"]), "bias": rng.random() < 0.5}
    if op == "clip":
        largest = _log_int(rng, 1000, 14336 * 4096)
        tensors = rng.randint(1, 600)
        while tensors * largest > 14336 * 4096 * 24:
            tensors = max(1, tensors // 2)
        return {"op": op, "tensors": tensors, "largest": largest, "smallest": _log_int(rng, 1, largest),
                "dtype": rng.choice(["bf16", "fp16", "fp32"]), "active": rng.random() < 0.5}
    cols = _log_int(rng, 64, 16384)
    rows = _log_int(rng, 1, min(16384, 16384 * 8192 // cols))
    if rng.random() < 0.7:
        cols = (cols + 7) // 8 * 8
    dtype = rng.choice(["bf16", "fp16", "fp32"])
    case = {"op": op, "rows": rows, "cols": cols, "dtype": dtype}
    if op != "cast":
        case["affine"] = rng.choice([dtype, "fp32"])
    return case


# ---------------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------------
def _activations(gen, rows, cols, dtype, scale=1.0):
    """Normal values, a few columns thirty times larger, as the inputs of linear layers have them."""
    x = torch.randn(rows, cols, device="cuda", generator=gen) * scale
    hot = torch.randint(0, cols, (max(1, cols // 500),), device="cuda", generator=gen)
    x[:, hot] *= 30.0
    return x.to(dtype)


def _gradients(gen, rows, cols, dtype):
    """Small values whose size differs from row to row by three orders of magnitude."""
    size = torch.exp(torch.rand(rows, 1, device="cuda", generator=gen) * 6.9 - 9.2)
    return (torch.randn(rows, cols, device="cuda", generator=gen) * size).to(dtype)


def _clip_sizes(case):
    lo, hi, n = case["smallest"], case["largest"], case["tensors"]
    if n == 1:
        return [hi]
    # every size of the geometric range, the largest as often as the smallest
    return [max(1, int(lo * (hi / lo) ** (((i * 7) % n) / (n - 1)))) for i in range(n)]


def _inputs(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    op, dtype = case["op"], _DT[case["dtype"]]
    if op in ("infer", "train"):
        m, k, n = case["m"], case["k"], case["n"]
        t = {"x": _activations(gen, m, k, dtype),
             "w": (torch.randn(n, k, device="cuda", generator=gen) / math.sqrt(k)).to(dtype),
             "b": (torch.randn(n, device="cuda", generator=gen) * 0.1).to(dtype) if case["bias"] else None}
        if op == "train":
            t["g"] = _gradients(gen, m, n, dtype)
        return t
    if op == "product":
        m, k, n = case["m"], case["k"], case["n"]
        kb, nb = -(-k // _BLOCK), -(-n // _BLOCK)
        return {
            "a": (torch.randn(m, k, device="cuda", generator=gen) * 60.0).to(torch.float8_e4m3fn),
            "sa": torch.rand(m, kb, device="cuda", generator=gen) * 0.02 + 0.001,
            "w": (torch.randn(n, k, device="cuda", generator=gen) * 60.0).to(torch.float8_e4m3fn),
            "sw": (torch.rand(nb, kb, device="cuda", generator=gen) + 0.05) * 0.02 / math.sqrt(k),
            "b": (torch.randn(n, device="cuda", generator=gen) * 0.1).to(dtype) if case["bias"] else None,
        }
    if op == "clip":
        # one buffer that holds every gradient, each from a 256-byte boundary on, as a bucket of them does
        sizes, starts, at = _clip_sizes(case), [], 0
        for size in sizes:
            starts.append(at)
            at += (size + 127) // 128 * 128
        bucket = torch.zeros(at, dtype=dtype, device="cuda")
        for start, size in zip(starts, sizes):
            bucket[start:start + size] = torch.randn(size, device="cuda", generator=gen) * 1e-3
        norm = 1e-3 * math.sqrt(sum(sizes))
        return {"bucket": bucket, "spans": list(zip(starts, sizes)),
                "max_norm": norm * (0.25 if case["active"] else 4.0)}
    if op == "cast":
        return {"x": _activations(gen, case["rows"], case["cols"], dtype)}
    affine = _DT[case["affine"]]
    cols = case["cols"]
    t = {"x": _activations(gen, case["rows"], cols, dtype) + 0.25,
         "w": (1.0 + 0.1 * torch.randn(cols, device="cuda", generator=gen)).to(affine),
         "b": (0.1 * torch.randn(cols, device="cuda", generator=gen)).to(affine)}
    if op == "norm_train":
        t["g"] = _gradients(gen, case["rows"], cols, dtype)
    return t


def prepare(case, seed):
    """What a program holds before the call: tensors, and with `own` the layers made from them."""
    state = _inputs(case, seed)
    state["op"], state["dtype"] = case["op"], _DT[case["dtype"]]
    if case["op"] == "clip":
        # the backward pass writes the gradients anew before every clipping: `run` copies them from here
        state["fresh"] = state["bucket"]
        state["bucket"] = state["fresh"].clone()
        state["grads"] = [state["bucket"][at:at + size] for at, size in state["spans"]]
        if own:
            state["params"] = [torch.nn.Parameter(torch.empty_like(g)) for g in state["grads"]]
            for p, g in zip(state["params"], state["grads"]):
                p.grad = g
    if own and case["op"] in ("infer", "train"):
        state["layer"] = _layer(case, state)
    if own and case["op"] == "train":
        state["x"].requires_grad_()
    if own and case["op"] == "norm_train":
        for name in ("x", "w", "b"):
            state[name].requires_grad_()
    return state


def _layer(case, state):
    from float8_experimental_b200 import CastConfig, convert_to_float8_training, Float8LinearConfig, ScalingType
    from float8_experimental_b200.inference import ActivationCasting, quantize_to_float8, QuantConfig

    lin = torch.nn.Linear(case["k"], case["n"], bias=case["bias"], device="meta", dtype=state["dtype"])
    lin.weight = torch.nn.Parameter(state["w"])
    if case["bias"]:
        lin.bias = torch.nn.Parameter(state["b"])
    if case["op"] == "infer":
        return quantize_to_float8(lin, QuantConfig(ActivationCasting.BLOCKWISE))
    by_block = CastConfig(scaling_type=ScalingType.BLOCKWISE)
    config = Float8LinearConfig(cast_config_input=by_block, cast_config_weight=by_block,
                                cast_config_grad_output=by_block)
    return convert_to_float8_training(lin, config=config)


# ---------------------------------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------------------------------
def run(state):
    return _run_own(state) if own else _run_plain(state)


def _run_own(state):
    op = state["op"]
    if op == "infer":
        with torch.no_grad():
            return state["layer"](state["x"])
    if op == "train":
        layer, x = state["layer"], state["x"]
        leaves = [x, layer.weight] + ([layer.bias] if layer.bias is not None else [])
        y = layer(x)
        return [y.detach(), *torch.autograd.grad(y, leaves, state["g"])]
    if op == "product":
        from float8_experimental_b200.float8_blockwise import blockwise_mm, Float8BlockTensor

        a = Float8BlockTensor(state["a"], state["sa"], (1, 128))
        w = Float8BlockTensor(state["w"], state["sw"], (128, 128))
        return blockwise_mm(a, w.t(), out_dtype=state["dtype"], bias=state["b"])
    if op == "cast":
        from float8_experimental_b200.float8_blockwise import cast_to_float8_blockwise_both

        by_row, by_col = cast_to_float8_blockwise_both(state["x"])
        return [by_row.to_original_precision(), by_row.scale_inv, by_col.to_original_precision(), by_col.scale_inv]
    if op == "norm":
        from float8_experimental_b200.layer_norm import layer_norm

        with torch.no_grad():
            return layer_norm(state["x"], state["w"], state["b"], 1e-5)
    if op == "norm_train":
        from float8_experimental_b200.layer_norm import layer_norm

        leaves = [state["x"], state["w"], state["b"]]
        y = layer_norm(*leaves, 1e-5)
        return [y.detach(), *torch.autograd.grad(y, leaves, state["g"])]
    from float8_experimental_b200.grad_clip import clip_grad_norm_

    state["bucket"].copy_(state["fresh"])
    total = clip_grad_norm_(state["params"], state["max_norm"])
    return [total, state["bucket"]]


def _pow2(e):
    """2^e for a tensor of whole numbers, by its bits."""
    return ((e.to(torch.int32) + 127) << 23).view(torch.float32)


def _grouped_amax(x, block):
    rows, cols = x.shape
    br, bc = block
    padded = torch.nn.functional.pad(x.abs(), (0, -cols % bc, 0, -rows % br))
    return padded.view(-(-rows // br), br, -(-cols // bc), bc).amax(dim=(1, 3))


def _spread(s, block, shape):
    """One scale per block as one per element."""
    return s.repeat_interleave(block[0], 0)[: shape[0]].repeat_interleave(block[1], 1)[:, : shape[1]]


def _plain_cast(x, block):
    """(the values that the stored bytes stand for in fp32, the blocks' factors)"""
    x = x.float()
    mantissa, exponent = torch.frexp(_grouped_amax(x, block).clamp(min=1e-12))  # mantissa in [0.5, 1)
    e = torch.where(mantissa <= 0.875, 9 - exponent, 8 - exponent)
    s = _pow2(-e)
    up = _spread(_pow2(e), block, x.shape)
    q = (x * up).clamp(-_E4M3_MAX, _E4M3_MAX).to(torch.float8_e4m3fn).float()
    return q * _spread(s, block, x.shape), s


def _plain_mm(a, b, bias, dtype):
    y = a @ b
    if bias is not None:
        y = y + bias.float()
    return y.to(dtype)


def _plain_norm(x, w, b):
    x = x.float()
    mean = x.mean(dim=1, keepdim=True)
    rstd = torch.rsqrt(((x - mean) ** 2).mean(dim=1, keepdim=True) + 1e-5)
    n = (x - mean) * rstd
    return n * w.float() + b.float(), n, rstd


def _run_plain(state):
    op, dtype = state["op"], state["dtype"]
    if op == "infer":
        x, _ = _plain_cast(state["x"], (1, _BLOCK))
        w, _ = _plain_cast(state["w"], (_BLOCK, _BLOCK))
        return _plain_mm(x, w.t(), state["b"], dtype)
    if op == "train":
        w, _ = _plain_cast(state["w"], (_BLOCK, _BLOCK))
        x, _ = _plain_cast(state["x"], (1, _BLOCK))
        out = [_plain_mm(x, w.t(), state["b"], dtype)]
        g, _ = _plain_cast(state["g"], (1, _BLOCK))
        out.append(_plain_mm(g, w, None, dtype))
        x, _ = _plain_cast(state["x"], (_BLOCK, 1))
        g, _ = _plain_cast(state["g"], (_BLOCK, 1))
        out.append(_plain_mm(g.t(), x, None, dtype))
        if state["b"] is not None:
            out.append(state["g"].float().sum(dim=0).to(dtype))
        return out
    if op == "product":
        a = state["a"].float() * _spread(state["sa"], (1, _BLOCK), state["a"].shape)
        w = state["w"].float() * _spread(state["sw"], (_BLOCK, _BLOCK), state["w"].shape)
        return _plain_mm(a, w.t(), state["b"], dtype)
    if op == "cast":
        by_row, s_row = _plain_cast(state["x"], (1, _BLOCK))
        by_col, s_col = _plain_cast(state["x"], (_BLOCK, 1))
        return [by_row.to(dtype), s_row, by_col.to(dtype), s_col]
    if op == "norm":
        return _plain_norm(state["x"], state["w"], state["b"])[0].to(dtype)
    if op == "norm_train":
        y, n, rstd = _plain_norm(state["x"], state["w"], state["b"])
        g = state["g"].float()
        h = g * state["w"].float()
        dx = rstd * (h - h.mean(dim=1, keepdim=True) - n * (h * n).mean(dim=1, keepdim=True))
        dw = (g * n).sum(dim=0).to(state["w"].dtype)
        return [y.to(dtype), dx.to(dtype), dw, g.sum(dim=0).to(state["b"].dtype)]
    state["bucket"].copy_(state["fresh"])
    total = torch.stack([(g.float() ** 2).sum() for g in state["grads"]]).sum().sqrt()
    factor = (state["max_norm"] / (total + 1e-6)).clamp(max=1.0)
    for g in state["grads"]:
        g.copy_(g.float() * factor)
    return [total, state["bucket"]]


# ---------------------------------------------------------------------------------------------------
# the work that a pass cannot do without
# ---------------------------------------------------------------------------------------------------
def work(case):
    op = case["op"]
    size = 4 if case["dtype"] == "fp32" else 2
    if op in ("infer", "product", "train"):
        m, k, n = case["m"], case["k"], case["n"]
        bias = n * size if case["bias"] else 0
        if op == "train":  # x, W and g read; the output, both gradients and the bias' gradient written
            return {"bytes": size * 2 * (m * k + n * k + m * n) + 2 * bias, "flops": 6 * m * k * n}
        x_size = 1 if op == "product" else size
        scales = 4 * (-(-k // _BLOCK)) * (-(-n // _BLOCK) + (m if op == "product" else 0))
        return {"bytes": x_size * m * k + k * n + scales + bias + size * m * n, "flops": 2 * m * k * n}
    if op == "clip":
        numel = sum(_clip_sizes(case))
        return {"bytes": numel * size * 2 if case["active"] else numel * size, "flops": 3 * numel}
    numel = case["rows"] * case["cols"]
    if op == "cast":  # both casts' values are returned in the input's type
        return {"bytes": numel * size * 3 + 2 * 4 * numel // _BLOCK, "flops": 4 * numel}
    affine = case["cols"] * (4 if case["affine"] == "fp32" else 2)
    if op == "norm":
        return {"bytes": 2 * numel * size + 2 * affine, "flops": 8 * numel}
    return {"bytes": 4 * numel * size + 4 * affine, "flops": 22 * numel}


# ---------------------------------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------------------------------
def _exact_cast(x, block):
    """(the values that the stored bytes stand for, the blocks' factors), in doubles."""
    x = x.double()
    rows, cols = x.shape
    br, bc = block
    row_id = torch.arange(rows, device=x.device) // br
    col_id = torch.arange(cols, device=x.device) // bc
    top = torch.zeros(int(row_id[-1]) + 1, cols, dtype=torch.float64, device=x.device)
    top.index_reduce_(0, row_id, x.abs(), "amax")
    amax = torch.zeros(top.shape[0], int(col_id[-1]) + 1, dtype=torch.float64, device=x.device)
    amax.index_reduce_(1, col_id, top, "amax")
    floor = amax.clamp(min=1e-12)
    e = torch.floor(torch.log2(_E4M3_MAX / floor))
    # the logarithm may be off in its last bit next to a whole number
    e = torch.where(floor * _two_to(e) > _E4M3_MAX, e - 1, e)
    e = torch.where(floor * _two_to(e + 1) <= _E4M3_MAX, e + 1, e)
    per_element = _two_to(e)[row_id][:, col_id]
    v = x * per_element
    # e4m3: three bits behind the leading one, down to an exponent of -6; frexp's fraction lies in [0.5, 1)
    step = _two_to((torch.frexp(v)[1] - 1).clamp(min=-6) - 3)
    return torch.round(v / step) * step / per_element, _two_to(-e)


def _two_to(e):
    """2^e in doubles, by its bits: a power function may be off in the last one."""
    return ((e.to(torch.int64) + 1023) << 52).view(torch.float64)


def exact(case, seed):
    op = case["op"]
    t = _inputs(case, seed)
    if op in ("infer", "train"):
        w = _exact_cast(t["w"], (_BLOCK, _BLOCK))[0]
        y = _exact_cast(t["x"], (1, _BLOCK))[0] @ w.t()
        if t["b"] is not None:
            y += t["b"].double()
        if op == "infer":
            return y
        dx = _exact_cast(t["g"], (1, _BLOCK))[0] @ w
        dw = _exact_cast(t["g"], (_BLOCK, 1))[0].t() @ _exact_cast(t["x"], (_BLOCK, 1))[0]
        return [y, dx, dw] + ([t["g"].double().sum(dim=0)] if t["b"] is not None else [])
    if op == "product":
        m, k = t["a"].shape
        n = t["w"].shape[0]
        y = torch.zeros(m, n, dtype=torch.float64, device="cuda")
        row_block = torch.arange(n, device="cuda") // _BLOCK
        for j in range(0, k, _BLOCK):
            part = t["a"][:, j:j + _BLOCK].double() @ t["w"][:, j:j + _BLOCK].double().t()
            y += part * t["sa"][:, j // _BLOCK, None].double() * t["sw"][row_block, j // _BLOCK].double()
        return y if t["b"] is None else y + t["b"].double()
    if op == "cast":
        return [*_exact_cast(t["x"], (1, _BLOCK)), *_exact_cast(t["x"], (_BLOCK, 1))]
    if op == "clip":
        bucket = t["bucket"].double()
        total = math.sqrt(float((bucket * bucket).sum()))  # what lies between the gradients is zero
        factor = min(1.0, t["max_norm"] / (total + 1e-6))
        return [torch.tensor(total, dtype=torch.float64, device="cuda"), bucket * factor]
    x, w, b = t["x"].double(), t["w"].double(), t["b"].double()
    var, mean = torch.var_mean(x, dim=1, unbiased=False, keepdim=True)
    inv = 1.0 / torch.sqrt(var + 1e-5)
    n = (x - mean) * inv
    y = n * w + b
    if op == "norm":
        return y
    g = t["g"].double()
    h = g * w
    cols = x.shape[1]
    dx = inv / cols * (cols * h - h.sum(1, keepdim=True) - n * (h * n).sum(1, keepdim=True))
    return [y, dx, (g * n).sum(0), g.sum(0)]
