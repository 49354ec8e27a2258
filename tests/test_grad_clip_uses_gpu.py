"""Clipping of gradients that share memory, and of gradients that a later backward pass needs."""
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


CLIPS = {"clip_grad_norm_": lambda p, total: clip_grad_norm_([p], 0.1),
         "clip_grads_with_norm_": lambda p, total: clip_grads_with_norm_([p], 0.1, total),
         "the operator": lambda p, total: ops.multi_clip_([p.grad], total, 0.1)}


@pytest.mark.parametrize("name", CLIPS)
def test_a_gradient_that_backward_still_needs(name):
    """As with torch's own clipping, the second backward pass notices that its gradient has changed."""
    w = torch.nn.Parameter(torch.full((8,), 2.0, device="cuda"))
    g, = torch.autograd.grad((w ** 3).sum(), [w], create_graph=True)
    penalty = (g * g).sum()
    total = get_total_norm([g.detach()])
    w.grad = g
    before = g._version
    with torch.no_grad():
        CLIPS[name](w, total)
    assert g._version > before
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(penalty, [w])


def test_gradients_made_in_inference_mode():
    with torch.inference_mode():
        g = torch.full((8,), 2.0, device="cuda")
        p = torch.nn.Parameter(torch.zeros(8, device="cuda"))
        p.grad = g
        clip_grad_norm_([p], 1.0)
        clip_grads_with_norm_([p], 1.0, torch.ones((), device="cuda"))
        assert torch.allclose(g, torch.full((8,), 8 ** -0.5, device="cuda"))
