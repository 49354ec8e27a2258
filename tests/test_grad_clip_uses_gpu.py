"""Clipping of gradients that share memory."""
import pytest
import torch

from float8_experimental_b200 import clip_grad_norm_, clip_grads_with_norm_, get_total_norm
from float8_experimental_b200._ops import ops

pytestmark = pytest.mark.gpu


def params_of(grads):
    out = []
    for g in grads:
        p = torch.nn.Parameter(torch.empty_like(g))
        p.grad = g
        out.append(p)
    return out


@pytest.mark.parametrize("views", [lambda b: [b[:100].view(10, 10), b[:100].view(100)], lambda b: [b[:100], b[50:150], b[200:]],
                                   lambda b: [b[200:], b[50:150], b[:51]]])
def test_views_that_overlap_are_refused(views):
    buf = torch.ones(300, device="cuda")
    grads = views(buf)
    for call in (lambda: clip_grad_norm_(params_of(grads), 0.1), lambda: ops.multi_clip_(grads, buf.norm(), 0.1),
                 lambda: clip_grads_with_norm_(params_of(grads), 0.1, buf.norm())):
        with pytest.raises(RuntimeError, match="overlap in memory"):
            call()
    assert bool((buf == 1).all())
    # the norm alone counts what it is given
    want = sum(float((g * g).sum()) for g in grads) ** 0.5
    assert float(get_total_norm(grads)) == pytest.approx(want, rel=1e-6)


def test_views_that_lie_apart_are_scaled():
    buf = torch.ones(300, device="cuda")
    grads = [buf[200:], buf[:64], buf[64:128].view(8, 8).t()]
    total = clip_grad_norm_(params_of(grads), 1.0)
    assert float(total) == pytest.approx(228 ** 0.5, rel=1e-6)
    want = torch.ones(300, device="cuda")
    want[:128] = want[200:] = 1.0 / 228 ** 0.5
    assert torch.allclose(buf, want, rtol=1e-5)
