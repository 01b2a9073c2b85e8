"""The row operators' refusals at the C entry (no launch is reached, so no GPU is needed), their Python wrappers without a GPU, and the
oracle's own gradient against autograd."""
import numpy as np
import pytest
import torch

import row_oracle as ro

P = 1 << 20                # stands for a device pointer; a refused call never follows it


def lib():
    from elg_amd import _lib as L
    return L, L.lib()


def top(**o):
    L, c = lib()
    a = dict(z=P, stride=10, type=0, R=4, V=10, k=3, t=1.0, values=P, idx=P, tail=None, stream=None)
    a.update(o)
    return c.elg_top_logits(*a.values())


def distill(**o):
    L, c = lib()
    a = dict(z=P, stride=10, type=0, R=4, V=10, tv=P, ttype=0, ti=P, wide=0, k=3, tail=None, t=1.0, weight=None, cot=None, cs=0, scale=1.0,
             rows=P, total=None, grad=None, ws=None, n=0, stream=None)
    a.update(o)
    return c.elg_distill_loss_grad(*a.values())


def verify(**o):
    L, c = lib()
    a = dict(p=P, pb=30, ps=10, q=None, qb=0, qs=0, type=0, x=P, wide=0, xs=2, u=P, us=3, n=None, B=4, G=2, V=10, out=P, acc=P, ws=None, n_ws=0, stream=None)
    a.update(o)
    return c.elg_verify_draft(*a.values())


@pytest.mark.parametrize("call,bad", [
    (top, dict(type=3)), (top, dict(type=-1)), (top, dict(R=-1)), (top, dict(V=0)), (top, dict(V=(1 << 24) + 1)), (top, dict(V=1 << 33)),
    (top, dict(k=0)), (top, dict(k=11)), (top, dict(V=1000, k=257)), (top, dict(t=0.0)), (top, dict(t=-1.0)), (top, dict(t=float("nan"))),
    (top, dict(t=float("inf"))), (top, dict(z=None)), (top, dict(values=None)), (top, dict(idx=None)), (top, dict(z=P + 2)), (top, dict(values=P + 1)),
    (distill, dict(type=3)), (distill, dict(ttype=9)), (distill, dict(R=-1)), (distill, dict(V=0)), (distill, dict(V=1 << 33)), (distill, dict(k=0)),
    (distill, dict(k=257)), (distill, dict(t=0.0)), (distill, dict(t=float("inf"))), (distill, dict(cs=2)), (distill, dict(rows=None)),
    (distill, dict(z=None)), (distill, dict(tv=None)), (distill, dict(ti=None)), (distill, dict(total=P, R=4000)), (distill, dict(total=P, R=400, ws=P, n=7)),
    (distill, dict(total=P, R=400, ws=P + 4, n=1 << 20)), (distill, dict(grad=P + 1)), (distill, dict(z=P + 2)), (distill, dict(ti=P + 4, wide=1)),
    (verify, dict(type=7)), (verify, dict(B=-1)), (verify, dict(G=-1)), (verify, dict(G=1025)), (verify, dict(V=0)), (verify, dict(V=1 << 33)),
    (verify, dict(p=None)), (verify, dict(x=None)), (verify, dict(u=None)), (verify, dict(out=None)), (verify, dict(acc=None)), (verify, dict(p=P + 2)),
    (verify, dict(x=P + 4, wide=1)), (verify, dict(V=9000)), (verify, dict(V=9000, ws=P, n_ws=16)), (verify, dict(V=9000, ws=P + 8, n_ws=1 << 20)),
    (distill, dict(V=9000)), (distill, dict(V=200000, R=1000, ws=P, n=64))])
def test_refused_at_the_c_entry(call, bad):
    L, c = lib()
    assert call(**bad) == L.ELG_EINVAL
    assert c.elg_last_error()
    with pytest.raises(ValueError):
        L.check(L.ELG_EINVAL, "row operator")


def test_empty_calls_return_without_a_launch():
    L, c = lib()
    assert top(R=0) == L.ELG_OK and verify(B=0) == L.ELG_OK and distill(R=0) == L.ELG_OK


def test_no_host_path():
    from elg_amd import logits as lg
    z, v, i = torch.zeros(2, 5), torch.zeros(2, 2), torch.zeros(2, 2, dtype=torch.int32)
    for f in (lambda: lg.top_logits(z, 2), lambda: lg.distill_loss(z, v, i), lambda: lg.distill_loss_grad(z, v, i),
              lambda: lg.verify_draft(z.view(1, 2, 5), i[:1, :1], torch.zeros(1, 2))):
        with pytest.raises(RuntimeError):
            f()


def test_oracle_gradient_is_autograds():
    torch.manual_seed(0)
    z = (torch.randn(4, 30, dtype=torch.float64) * 3)
    z[:, 20:24] = -np.inf
    x = z.clone().requires_grad_(True)
    tv, ti = torch.randn(4, 6).double(), torch.stack([torch.randperm(20)[:6] for _ in range(4)])
    a, w, tau = torch.tensor([0.1, 0.3, 0.0, 0.9]).double(), torch.tensor([1.0, 2.0, 0.5, 1.0]).double(), 1.7
    q = (1 - a)[:, None] * torch.softmax(tv / tau, -1)
    lp = torch.log_softmax(x / tau, -1)
    rest = torch.logsumexp(lp.scatter(1, ti, -np.inf), -1)
    loss = tau * tau * w * ((q * (q.log() - lp.gather(1, ti))).sum(-1) + torch.xlogy(a, a) - a * rest)
    (g,) = torch.autograd.grad(loss.sum(), x)
    rl, rg, _, _ = ro.distill(z.numpy(), tv.numpy(), ti.numpy(), a.numpy(), tau, w.numpy())
    np.testing.assert_allclose(rl, loss.detach().numpy(), rtol=1e-12)
    np.testing.assert_allclose(rg, g.numpy(), rtol=1e-10, atol=1e-14)


def test_oracle_order_and_draws():
    v, i = ro.top(np.array([[1.0, np.nan, 2.0, -0.0, 0.0, 2.0, -np.inf, np.inf]]), 8)
    assert i.tolist() == [[1, 7, 2, 5, 0, 3, 4, 6]]
    tok, acc = ro.verify(np.array([[[0.25, 0.75], [1.0, 0.0]]]), np.array([[1]]), np.array([[0.74, 0.5]]))
    assert tok.tolist() == [[1, 0]] and acc.tolist() == [1]
