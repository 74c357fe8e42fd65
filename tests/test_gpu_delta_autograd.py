"""What the gated delta rule and the layer norm refuse of autograd, and calls of several threads."""

import threading

import pytest
import torch
import torch.autograd.forward_ad as fwd

from tops.ops.delta import gated_delta_rule, gated_delta_rule_step
from tops.ops.norm import layer_norm

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def inputs(T, K, seed=0, dt=torch.bfloat16):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=gen, device=DEV)   # noqa: E731
    return dict(q=r(1, T, 1, K).to(dt), k=r(1, T, 1, K).to(dt), v=r(1, T, 2, 40).to(dt),
                g=-r(1, T, 2).abs(), beta=torch.sigmoid(r(1, T, 2)))


@pytest.mark.parametrize("K", [5, 64])
def test_no_second_derivative(K):
    x = {n: t.requires_grad_() for n, t in inputs(20, K).items()}
    o, _ = gated_delta_rule(**x, qk_l2norm=True)
    g, = torch.autograd.grad(o.float().sum(), x["v"], create_graph=True)
    with pytest.raises(RuntimeError):
        g.float().sum().backward()


def test_no_second_derivative_of_the_norm():
    x, w = torch.randn(4, 16, device=DEV).requires_grad_(), torch.ones(16, device=DEV)
    g, = torch.autograd.grad(layer_norm(x, w).square().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()


def test_no_forward_mode():
    x = inputs(20, 64)
    with fwd.dual_level():
        for n in x:
            dual = {**x, n: fwd.make_dual(x[n], torch.ones_like(x[n]))}
            with pytest.raises((RuntimeError, NotImplementedError)):
                gated_delta_rule(**dual)
        y = torch.randn(4, 16, device=DEV)
        with pytest.raises((RuntimeError, NotImplementedError)):
            layer_norm(fwd.make_dual(y, torch.ones_like(y)))
        o, _ = gated_delta_rule(**x)   # nothing to differentiate
    assert torch.equal(o, gated_delta_rule(**x)[0])


def test_threads():
    """Threads with streams of their own: sequences, packed sequences, steps, norms, gradients."""
    def work(i):
        T = 300 + 70 * i
        x = {n: t.requires_grad_() for n, t in inputs(T, 64, i).items()}
        w = torch.linspace(0.5, 1.5, 40, device=DEV).requires_grad_()
        o, ht = gated_delta_rule(**x, qk_l2norm=True, output_final_state=True,
                                 cu_seqlens=None if i % 2 else [0, 10 * i + 5, T])
        y = layer_norm(o, w)
        grads = torch.autograd.grad(y.float().sum() + ht.square().sum(), [*x.values(), w])
        state = ht.detach().clone()
        with torch.no_grad():
            s = gated_delta_rule_step(state[:1], *(t[:, -1] for t in x.values()), qk_l2norm=True)
        return [o.detach(), ht.detach(), y.detach(), *grads, state, s]

    n = 4
    want = [work(i) for i in range(n)]
    torch.cuda.synchronize()
    got, wrong = [None] * n, []

    def run(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(5):
                    got[i] = work(i)
                torch.cuda.current_stream().synchronize()
        except Exception as e:   # noqa: BLE001
            wrong.append(e)

    threads = [threading.Thread(target=run, args=(i,)) for i in range(n)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong, wrong
    for a, b in zip(want, got):
        assert all(torch.equal(s, t) for s, t in zip(a, b))
