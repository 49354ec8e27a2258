"""When calls go past the dispatcher, and the eager step's buffer read as tensors: nothing here needs a GPU."""
import pytest
import torch
from torch.fx.experimental.proxy_tensor import make_fx
from torch.utils._python_dispatch import TorchDispatchMode
from torch._subclasses.fake_tensor import FakeTensorMode

from float8_experimental_b200 import _native as N
from float8_experimental_b200._ops import nothing_watches


class Counter(TorchDispatchMode):
    def __torch_dispatch__(self, func, types, args=(), kwargs=None):
        return func(*args, **(kwargs or {}))


def in_mode(mode):
    def run(f, x):
        with mode:
            f(x)
    return run


WATCHERS = {
    "make_fx": lambda f, x: make_fx(f)(x),
    "make_fx symbolic": lambda f, x: make_fx(f, tracing_mode="symbolic")(x),
    "make_fx pre-dispatch": lambda f, x: make_fx(f, pre_dispatch=True)(x),
    "jit.trace": lambda f, x: torch.jit.trace(f, (x,), check_trace=False),
    "dispatch mode": in_mode(Counter()),
    "fake tensors": in_mode(FakeTensorMode(allow_non_fake_inputs=True)),
    "vmap": lambda f, x: torch.func.vmap(f)(x),
    "grad": lambda f, x: torch.func.grad(lambda a: f(a).sum())(x),
}


@pytest.mark.parametrize("name", WATCHERS)
def test_watchers_are_noticed(name):
    seen = []

    def f(x):
        seen.append(nothing_watches())
        return x + 1

    WATCHERS[name](f, torch.zeros(3))
    assert seen and not any(seen)
    assert nothing_watches()


def test_ordinary_code_is_not_watched():
    with torch.no_grad(), torch.device("cpu"), torch.autocast("cpu", torch.bfloat16):
        assert nothing_watches()
    with torch.inference_mode():
        assert nothing_watches()


@pytest.mark.parametrize("rows,cols", [(1, 1), (130, 264), (300, 1000), (257, 513)])
@pytest.mark.parametrize("by", ["row", "col", "square"])
def test_a_form_as_tensors(rows, cols, by):
    """Each part starts where the form's address says, has its shape and overlaps no other."""
    form = N.BlockForm(rows, cols, by)
    start = 512
    buf = torch.zeros(start + form.nbytes, dtype=torch.uint8)
    form.at(buf.data_ptr() + start)
    data, scale, exps = form.tensors(buf, start)
    kb, rb = -(-cols // 128), -(-rows // 128)
    assert data.shape == (rows, cols) and data.dtype == torch.float8_e4m3fn and data.stride() == (form.pitch, 1)
    assert scale.shape == {"row": (rows, kb), "col": (rb, cols), "square": (rb, kb)}[by] and scale.dtype == torch.float32
    operand = form.operand(transposed=by != "row")
    assert (data.data_ptr(), scale.data_ptr(), exps.data_ptr()) == (operand[0], operand[3], operand[7])
    as_operand = scale if by == "row" else scale.t()
    assert operand[4:6] == tuple(as_operand.stride())
    n, k = (rows, cols) if by == "row" else (cols, rows)
    assert exps.numel() == -(-n // 256) * 1024 * -(-k // 512) and exps.is_contiguous()
    data.view(torch.uint8).add_(1)
    scale.view(torch.int32).add_(0x01010101)
    exps.add_(1)
    assert int(buf.max()) == 1 and int(buf.sum()) == rows * cols + 4 * scale.numel() + exps.numel() and int(buf[:start].max()) == 0
