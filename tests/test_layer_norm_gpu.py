"""Layer norm, forward and backward, against a 64-bit restatement and against differences."""
import gc
import pytest
import torch

from blockwise_reference import layer_norm as reference
from float8_experimental_b200._ops import ops
from float8_experimental_b200.layer_norm import layer_norm, LayerNorm

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True, scope="module")
def leave_no_tensors():
    """What failed calls left in reference cycles (tracebacks hold their frames) goes now, not in the middle of another
    file's count of allocated bytes."""
    yield
    gc.collect()


BF, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32
EPS = 1e-5
U = 2.0 ** -24  # half a step of fp32


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def randn(*shape, seed=0):
    return torch.randn(*shape, device="cuda", generator=gen(seed))


def half_step(ref, dtype):
    f = torch.finfo(dtype)
    return f.eps / 2 * ref.abs() * (1 + 1e-6) + f.smallest_normal * f.eps


def depth(cols):
    """Additions one value goes through in a sum over a row: 256 threads (32 in narrow rows), then the tree."""
    return cols / 32 + 16 if cols <= 1024 else cols / 256 + 16


def check_forward(y, x, w, b, dtype):
    """The mean is off by d*U*mean|x| (d additions), so x - mean is off by that and half a step; the variance's relative
    error is twice d*U plus the mean's, rstd's half of that and two roundings; n is their product."""
    ref, n, rstd, mean = reference(x, w, b, EPS)
    xd = x.double()
    d = depth(x.shape[-1])
    off_mean = (d + 2) * U * xd.abs().mean(-1, keepdim=True)
    wabs = 1.0 if w is None else w.double().abs()
    tol = wabs * (rstd * (off_mean + 2 * U * (xd - mean).abs()) + n.abs() * (d + 8) * U) + 2 * U * ref.abs()
    err = (y.double() - ref).abs() - half_step(ref, dtype) - tol
    assert float(err.max()) <= 0, float(err.max())
    return n, rstd, d


SHAPES = [(1, 1), (1, 8), (5, 33), (3, 256), (7, 264), (40, 1000), (9, 1024), (6, 1032), (17, 2048), (5, 4096), (33, 4104),
          (3, 8192), (4, 16384), (2, 16392), (3, 20001), (700, 96)]


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("dtype,affine", [(BF, BF), (BF, FP32), (FP16, FP16), (FP16, FP32), (FP32, FP32)])
def test_forward_and_backward(shape, dtype, affine):
    rows, cols = shape
    x = (randn(*shape, seed=1) * 2 + 0.5).to(dtype).requires_grad_()
    w = (1 + 0.2 * randn(cols, seed=2)).to(affine).requires_grad_()
    b = (0.3 * randn(cols, seed=3)).to(affine).requires_grad_()
    g = randn(*shape, seed=4).to(dtype)
    y = layer_norm(x, w, b, EPS)
    assert y.dtype == dtype
    dx, dw, db = torch.autograd.grad(y, [x, w, b], g)
    n, rstd, d = check_forward(y.detach(), x.detach(), w.detach(), b.detach(), dtype)
    gd, wd = g.double(), w.detach().double()
    h = gd * wd
    ref = rstd * (h - h.mean(-1, keepdim=True) - n * (h * n).mean(-1, keepdim=True))
    # n is off by e_n (see check_forward); each of the three terms by its sum's error and e_n where it holds n
    xd = x.detach().double()
    mean_off = (d + 2) * U * xd.abs().mean(-1, keepdim=True)
    e_n = rstd * mean_off + n.abs() * (d + 10) * U
    hn = (h * n).abs().mean(-1, keepdim=True)
    tol = rstd * ((d + 8) * U * (h.abs() + h.abs().mean(-1, keepdim=True) + n.abs() * hn) + e_n * hn +
                  n.abs() * (h.abs() * e_n).mean(-1, keepdim=True)) + ref.abs() * (d + 8) * U
    err = (dx.double() - ref).abs() - half_step(ref, dtype) - tol
    assert float(err.max()) <= 0, float(err.max())
    # sums over rows: at most `rows` additions of fp32 values, n off by e_n in dw
    for got, terms, extra in ((dw, gd * n, (gd.abs() * e_n).sum(0)), (db, gd, 0.0)):
        ref = terms.sum(0)
        tol = (rows + 8) * U * terms.abs().sum(0) + extra
        err = (got.double() - ref).abs() - half_step(ref, affine) - tol
        assert got.dtype == affine and float(err.max()) <= 0, float(err.max())


def test_many_rows():
    x = randn(20000, 264, seed=1).to(BF).requires_grad_()
    w = torch.ones(264, device="cuda", dtype=FP32, requires_grad=True)
    g = randn(20000, 264, seed=2).to(BF)
    y = layer_norm(x, w)
    _, dw = torch.autograd.grad(y, [x, w], g)
    n, _, d = check_forward(y.detach(), x.detach(), w.detach(), None, BF)
    terms = g.double() * n
    tol = (20000 + 8) * U * terms.abs().sum(0) + (d + 40) * U * g.double().abs().sum(0) * 8
    assert float(((dw.double() - terms.sum(0)).abs() - tol).max()) <= 0


def test_large_mean_and_constant_rows():
    """The variance is taken about the mean: values near 1000 with a spread of 1e-2 keep fp32's digits."""
    x = 1000.0 + 1e-2 * randn(8, 2048, seed=1)
    x[3] = 7.25
    x[4] = 0.0
    y = layer_norm(x, None, None, EPS)
    check_forward(y, x, None, None, FP32)
    assert float(y[3:5].abs().max()) == 0.0


def test_nonfinite_rows_stay_their_own():
    x = randn(6, 500, seed=1).to(BF)
    want = layer_norm(x.clone())
    x[2, 7] = float("nan")
    x[4, 0] = float("inf")
    y = layer_norm(x)
    assert bool(torch.isnan(y[2]).all()) and bool(torch.isnan(y[4]).all())
    keep = [0, 1, 3, 5]
    assert torch.equal(y[keep], want[keep])


@pytest.mark.parametrize("have_w,have_b", [(True, False), (False, True), (False, False)])
@pytest.mark.parametrize("cols", [250, 512])
def test_missing_affine_parts(have_w, have_b, cols):
    x = randn(30, cols, seed=1).to(FP16).requires_grad_()
    w = (1 + 0.1 * randn(cols, seed=2)).to(FP16).requires_grad_() if have_w else None
    b = randn(cols, seed=3).to(FP16).requires_grad_() if have_b else None
    y = layer_norm(x, w, b, EPS)
    check_forward(y.detach(), x.detach(), w, b, FP16)
    g = randn(30, cols, seed=4).to(FP16)
    leaves = [t for t in (x, w, b) if t is not None]
    got = torch.autograd.grad(y, leaves, g)
    one = torch.ones(cols, device="cuda", dtype=FP16, requires_grad=True)
    zero = torch.zeros(cols, device="cuda", dtype=FP16, requires_grad=True)
    full_leaves = [x, w if have_w else one, b if have_b else zero]
    full = torch.autograd.grad(layer_norm(*full_leaves, EPS), full_leaves, g)
    assert torch.equal(got[0], full[0])
    if have_w:
        assert torch.equal(got[1], full[1])
    if have_b:
        assert torch.equal(got[-1], full[2])


def test_gradient_against_differences():
    """<dx, u> and the like against (f(x + hu) - f(x - hu)) / 2h with f = sum(y * g) in doubles of the fp32 forward:
    third-derivative error h^2/6 * |f'''| (|u| ~ 1, rstd ~ 1: below 50 h^2 * sum|g|/sqrt(C)), rounding 4 U sum|y g| / h."""
    rows, cols, h = 16, 300, 2.0 ** -7
    x, w, b, g = (randn(rows, cols, seed=1), 1 + 0.1 * randn(cols, seed=2), randn(cols, seed=3), randn(rows, cols, seed=4))
    leaves = [t.clone().requires_grad_() for t in (x, w, b)]
    y = layer_norm(*leaves, EPS)
    grads = torch.autograd.grad(y, leaves, g)

    def f(*t):
        return float((layer_norm(*t, EPS).double() * g.double()).sum())

    size = float((y.double() * g.double()).abs().sum())
    for i, grad in enumerate(grads):
        u = randn(*leaves[i].shape, seed=10 + i)
        plus, minus = [x, w, b], [x, w, b]
        plus[i], minus[i] = plus[i] + h * u, minus[i] - h * u
        slope = (f(*plus) - f(*minus)) / (2 * h)
        tol = 100 * U * size / h + 50 * h * h * float(g.abs().sum()) / cols ** 0.5
        assert abs(slope - float((grad.double() * u.double()).sum())) <= tol


def test_strides_and_broadcast_gradients():
    big = randn(64, 600, seed=1).to(BF)
    w = randn(256, seed=2).to(BF)
    for x in (big[:, :256], big[::2, 8:264], big[:, 1:257], randn(256, 64, seed=3).to(BF).t(), randn(2, 3, 4, 256, seed=4).to(BF)):
        a, b = layer_norm(x, w), layer_norm(x.contiguous().clone(), w)
        assert a.shape == x.shape and a.is_contiguous()
        tol = 2.0 ** -8 * b.double().abs() * 2 + 1e-5  # another split of the sums: one step of bf16 apart at most
        assert bool(((a.double() - b.double()).abs() <= tol).all())
    x = big[:, :256].clone().requires_grad_()
    d1, = torch.autograd.grad(layer_norm(x, w), [x], torch.ones(1, 1, device="cuda", dtype=BF).expand(64, 256))
    d2, = torch.autograd.grad(layer_norm(x, w), [x], torch.ones(64, 256, device="cuda", dtype=BF))
    assert torch.equal(d1, d2)


def test_no_rows_and_partial_gradients():
    w = torch.ones(64, device="cuda", requires_grad=True)
    b = torch.ones(64, device="cuda", requires_grad=True)
    x = torch.empty(0, 64, device="cuda", requires_grad=True)
    y = layer_norm(x, w, b)
    dx, dw, db = torch.autograd.grad(y, [x, w, b], torch.empty(0, 64, device="cuda"))
    assert y.shape == (0, 64) and dx.shape == (0, 64) and float(dw.abs().max()) == 0 and float(db.abs().max()) == 0
    x = randn(40, 64, seed=1).requires_grad_()
    g = randn(40, 64, seed=2)
    full = torch.autograd.grad(layer_norm(x, w, b), [x, w, b], g)
    for i, leaf in enumerate((x, w, b)):
        others = [t if t is leaf else t.detach() for t in (x, w, b)]
        only, = torch.autograd.grad(layer_norm(*others), [leaf], g)
        assert torch.equal(only, full[i])


def test_repeats_to_the_bit_and_graphs():
    m = LayerNorm(4096, device="cuda", dtype=BF)
    x = randn(300, 4096, seed=1).to(BF)
    g = randn(300, 4096, seed=2).to(BF)
    _, mean, rstd = ops.layer_norm(x, m.weight, m.bias, m.eps, True)
    args = (x, g, m.weight.detach(), mean, rstd, BF, True, True, True)
    first = ops.layer_norm_bwd(*args)
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(first, ops.layer_norm_bwd(*args)))
    graph = torch.cuda.CUDAGraph()
    with torch.no_grad(), torch.cuda.graph(graph):
        y = m(x)
        out = ops.layer_norm_bwd(*args)
    x.mul_(-2)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(y, m(x)) and all(torch.equal(a, b) for a, b in zip(out, ops.layer_norm_bwd(*args)))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        z = m(x)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(z, y)


def test_refusals_on_the_gpu():
    x = torch.zeros(4, 8, device="cuda", dtype=BF)
    with pytest.raises(RuntimeError, match="one element per column"):
        layer_norm(x, torch.ones(7, device="cuda", dtype=BF))
    with pytest.raises(RuntimeError, match="both float32"):
        layer_norm(x, torch.ones(8, device="cuda", dtype=FP16))
    with pytest.raises(RuntimeError, match="both float32"):
        layer_norm(x, torch.ones(8, device="cuda", dtype=BF), torch.ones(8, device="cuda"))
    with pytest.raises(RuntimeError, match="different devices"):
        layer_norm(x, torch.ones(8, dtype=BF))
    with pytest.raises(RuntimeError, match="at least one element"):
        layer_norm(torch.zeros(4, 0, device="cuda"))
    w = torch.ones(8, device="cuda", dtype=BF, requires_grad=True)
    g, = torch.autograd.grad(layer_norm(x, w).sum(), [w], create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(g.sum(), [w])
