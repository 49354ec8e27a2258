"""64-bit restatements of the block-scaled casts and products, the layer norm and the gradient norm, for the tests."""
import torch

TOP = {torch.float8_e4m3fn: (448.0, 3, -6), torch.float8_e5m2: (57344.0, 2, -14)}  # maximum, fraction bits, least exponent


def two_to(e):
    return ((e.to(torch.int64) + 1023) << 52).view(torch.float64)


def spread(s, block, shape):
    return s.repeat_interleave(block[0], 0)[: shape[0]].repeat_interleave(block[1], 1)[:, : shape[1]]


def cast(x, block, fmt):
    """(stored values before scaling back, factors) in doubles: block by block, the exponent found by trying them."""
    top, bits, least = TOP[fmt]
    x = x.double()
    rows, cols = x.shape
    nb = (-(-rows // block[0]), -(-cols // block[1]))
    q = torch.empty_like(x)
    s = torch.empty(nb, dtype=torch.float64, device=x.device)
    tries = torch.arange(-130, 60, device=x.device)
    for i in range(nb[0]):
        for j in range(nb[1]):
            rs, cs = slice(i * block[0], (i + 1) * block[0]), slice(j * block[1], (j + 1) * block[1])
            b = x[rs, cs]
            if not bool(torch.isfinite(b).all()):
                q[rs, cs] = float("nan")
                s[i, j] = float("nan")
                continue
            a = max(float(b.abs().max()), 1e-12)
            e = int(tries[(a * two_to(tries) <= top).nonzero().max()])
            v = b * 2.0 ** e
            step = two_to((torch.frexp(v)[1] - 1).clamp(min=least) - bits)
            q[rs, cs] = torch.round(v / step) * step
            s[i, j] = 2.0 ** -e
    return q, s


def product(a, sa, a_block, b, sb, b_block, bias=None):
    """(a @ b^T in doubles, the same with every term's absolute value) of fp8 a [M, K], b [N, K] and their factors."""
    va = a.double() * spread(sa.double(), (a_block, 128), a.shape)
    vb = b.double() * spread(sb.double(), (b_block, 128), b.shape)
    ref, mag = va @ vb.t(), va.abs() @ vb.abs().t()
    if bias is not None:
        ref, mag = ref + bias.double(), mag + bias.double().abs()
    return ref, mag


def product_tolerance(ref, mag, k, dtype):
    """Half a step of the result's type, and for the fp32 sums: inside a block 32 products per MMA and 4 MMAs, each
    addition off by at most one step of the largest partial sum, then one FMA per block and two roundings of
    its factor; every one of these is at most 2^-23 of the sum of the terms' magnitudes."""
    blocks = -(-k // 128)
    tiny = torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps  # below the normal range a step is this wide
    return torch.finfo(dtype).eps / 2 * ref.abs() * (1 + 1e-6) + (blocks + 40) * 2.0 ** -23 * mag + tiny


def layer_norm(x, w, b, eps):
    x = x.double()
    mean = x.mean(-1, keepdim=True)
    d = x - mean
    rstd = 1 / torch.sqrt((d * d).mean(-1, keepdim=True) + eps)
    n = d * rstd
    y = n * (1.0 if w is None else w.double()) + (0.0 if b is None else b.double())
    return y, n, rstd, mean
