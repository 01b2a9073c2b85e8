"""Row operators (elg_amd/logits.py) at the edges of what their documentation allows, against the definitions in 64 bits (row_oracle.py)."""
import numpy as np
import pytest
import torch

import row_oracle as ro

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
TYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}


def lg():
    from elg_amd import logits
    return logits


def rng(seed):
    return torch.Generator(device="cpu").manual_seed(seed)


def host(t):
    return t.detach().cpu().double().numpy()


# ------------------------------------------------------------------------------------------------------------- top_logits
@pytest.mark.parametrize("V,k,dtype", [(2049, 1, "float32"), (3001, 64, "float32"), (5003, 256, "bfloat16"), (20001, 256, "float16"),
                                       (65536, 100, "float32"), (70001, 256, "float32"), (131075, 128, "bfloat16")])
def test_top_of_rows_with_thousands_of_nan(V, k, dtype):
    """A diverged policy's rows: all NaN, all but one, more NaN than candidates fit and fewer open nodes than k beside them.  The lowest
    indices of the NaN come first, then the best of the others."""
    g = rng(V)
    z = torch.randn(12, V, generator=g).to(TYPES[dtype])
    z[0] = float("nan")
    z[1, :-1] = float("nan")
    z[2, torch.randperm(V, generator=g)[:1100]] = float("nan")
    z[3, torch.randperm(V, generator=g)[:V - 7]] = float("nan")
    z[4] = torch.where(torch.arange(V) % 2 == 0, float("nan"), -np.inf)
    z[5, :max(1, k // 2)] = float("nan")
    z[6:9] = z[0]
    z[9, 1::2] = -float("nan")
    rv, ri = ro.top(host(z), k)
    for _ in range(3):
        values, idx, tail = lg().top_logits(z.to(DEV), k, with_tail=True)
        np.testing.assert_array_equal(idx.cpu().numpy(), ri)
        np.testing.assert_array_equal(host(values), rv)
        assert torch.isnan(tail[:10]).all() and torch.isfinite(tail[10:]).all()


@pytest.mark.parametrize("dtype", list(TYPES))
def test_top_tail_of_equal_logits_is_rounded_once(dtype):
    """V equal logits: every exponential is 1 and every sum a whole number below 2^24, so that the tail is (V - k) / V after one division, which
    is the f32 next to it."""
    for V in (*range(2, 257), 300, 511, 777, 1001, 1500, 2047, 2049, 3001, 9001, 70001):
        for k in sorted({1, 2, V // 3 + 1, min(V, 256) // 2 + 1}):
            if k > min(V, 256):
                continue
            tail = lg().top_logits(torch.full((3, V), 1.25, dtype=TYPES[dtype], device=DEV), k, with_tail=True)[2]
            assert (tail.cpu().numpy() == np.float32((V - k) / V)).all(), (V, k)


# ----------------------------------------------------------------------------------------------------------- distillation
def check_losses(z, tv, ti, a, tau=1.0, w=None, R=None):
    """Losses of the rows and their mean against the definition, within its bounds; the gradient too."""
    d = [None if t is None else t.to(DEV) for t in (z, tv, ti, a, w)]
    loss, grad = lg().distill_loss_grad(d[0], d[1], d[2], tail=d[3], temperature=tau, weight=d[4], reduction="none")
    rl, rg, lb, gb = ro.distill(host(z), host(tv), ti.numpy(), host(a), tau, None if w is None else host(w))
    got, fin = host(loss), np.isfinite(rl)
    assert (got[~fin] == rl[~fin]).all(), (got, rl)
    assert (np.abs(got[fin] - rl[fin]) <= lb[fin] + 1e-30).all(), (got, rl, lb)
    assert (np.abs(host(grad) - rg) <= gb + 4 * ro.U * np.abs(rg) + ro.TINY["float32"]).all()
    mean = lg().distill_loss(d[0], d[1], d[2], tail=d[3], temperature=tau, weight=d[4]).item()
    if fin.all():
        assert abs(mean - rl.mean()) <= lb.mean() + 2 * ro.U * abs(rl.mean()) + 1e-30
    else:
        assert mean == np.inf
    return got, rl


TINY_TAILS = [1e-45, 1e-40, 1.2e-38, 1e-37, 2e-36, 1e-35, 1e-33, 1e-30, 1e-25, 1e-19, 1.1e-18, 1e-10]


@pytest.mark.parametrize("V", [17, 250, 1001, 2048, 2049, 9001])
def test_distill_tiny_tail_over_a_flat_rest(V):
    """The teacher leaves next to nothing outside its entries and the student has hundreds of nodes there, all alike: tail S / p_rest lies below
    the smallest normal number, and its logarithm is still finite."""
    k, n = 5, len(TINY_TAILS)
    z = torch.full((n, V), -50.0)
    z[:, 0] = 50.0
    z[1::2, 0] = -49.0                                     # the best node inside the rest's reach as well
    tv, ti = torch.tensor([40.0, -48.0, -49.0, -49.5, -50.0]).expand(n, k).contiguous(), torch.arange(k).int().expand(n, k).contiguous()
    a = torch.tensor(TINY_TAILS, dtype=torch.float64).float()
    got, _ = check_losses(z, tv, ti, a)
    assert np.isfinite(got).all()


@pytest.mark.parametrize("V", [16, 17, 250, 257, 1001, 2048, 2049, 9001, 70001])
def test_distill_any_tail_over_a_closed_rest_is_infinite(V):
    """The student has closed every node that is no entry's, or the entries are all of its open nodes: any mass of the teacher there, however
    small, makes the loss +inf, in rows of every length; no mass makes none."""
    k = 9
    a = torch.tensor(TINY_TAILS + [0.25, 0.0], dtype=torch.float64).float()
    z = torch.full((len(a), V), -np.inf)
    z[:, :k] = torch.linspace(-3, 3, k)
    tv, ti = torch.zeros(len(a), k), torch.arange(k).int().expand(len(a), k).contiguous()
    got, _ = check_losses(z, tv, ti, a)
    assert (got[:-1] == np.inf).all() and np.isfinite(got[-1])


@pytest.mark.parametrize("k", [9, 20, 100, 200])
def test_distill_any_tail_where_the_entries_are_all_nodes(k):
    a = torch.tensor(TINY_TAILS + [0.25, 0.0], dtype=torch.float64).float()
    z = torch.linspace(-3, 3, k).expand(len(a), k).contiguous()
    got, _ = check_losses(z, torch.zeros(len(a), k), torch.arange(k).int().expand(len(a), k).contiguous(), a)
    assert (got[:-1] == np.inf).all() and np.isfinite(got[-1])


@pytest.mark.parametrize("V", [4, 20, 300, 2048, 2049, 9001, 70001])
def test_distill_entry_without_mass_keeps_its_node_out_of_the_rest(V):
    """V equal logits, all mass of the entries on node 0, an entry of -inf at node 1, tail 1/2: q_0 = 1/2 on p_0 = 1/V, the tail on the V - 2 nodes
    of no entry.  Padding with node -1 instead leaves V - 1 of them."""
    z, tv = torch.zeros(2, V), torch.tensor([[0.0, -np.inf], [0.0, -np.inf]])
    ti, a = torch.tensor([[0, 1], [0, -1]]).int(), torch.tensor([0.5, 0.5])
    got, _ = check_losses(z, tv, ti, a)
    grad = host(lg().distill_loss_grad(z.to(DEV), tv.to(DEV), ti.to(DEV), tail=a.to(DEV), reduction="none")[1])
    for r, rest in ((0, V - 2), (1, V - 1)):
        loss = 0.5 * np.log(0.5 * V) + 0.5 * np.log(0.5 * V / rest)
        assert got[r] == pytest.approx(loss, abs=1e-6)
        want = np.full(V, 1 / V - 0.5 / rest)
        want[0] = 1 / V - 0.5
        if r == 0:
            want[1] = 1 / V
        np.testing.assert_allclose(grad[r], want, atol=2e-7)


@pytest.mark.parametrize("V", [33, 101, 250, 1001, 2048, 2049, 9001, 70001])
def test_distill_non_finite_teachers_and_cotangents_reach_what_the_formula_says(V):
    """A NaN or +inf among the teacher's entries is in every q of its row and in no p: the entries' nodes get NaN, the others keep their gradient.
    An infinite cotangent makes infinite gradients of the formula's signs.  The same in rows of every length."""
    R, k = 6, 7
    g = rng(V)
    z = torch.randn(R, V, generator=g) * 2
    tv, ti = torch.randn(R, k, generator=g), torch.stack([torch.randperm(V, generator=g)[:k] for _ in range(R)]).int()
    a = torch.full((R,), 0.2)
    good = lg().distill_loss_grad(z.to(DEV), tv.to(DEV), ti.to(DEV), tail=a.to(DEV), reduction="none")
    bad = tv.clone()
    bad[1, 3], bad[4, 0] = float("nan"), float("inf")
    loss, grad = lg().distill_loss_grad(z.to(DEV), bad.to(DEV), ti.to(DEV), tail=a.to(DEV), reduction="none")
    entry = torch.zeros(R, V, dtype=torch.bool, device=DEV).scatter_(1, ti.long().to(DEV), True)
    odd = torch.zeros(R, 1, dtype=torch.bool, device=DEV)
    odd[[1, 4]] = True
    assert torch.equal(torch.isnan(grad), entry & odd) and torch.equal(grad[~(entry & odd)], good[1][~(entry & odd)])
    assert torch.isnan(loss[[1, 4]]).all() and torch.equal(loss[[0, 2, 3, 5]], good[0][[0, 2, 3, 5]])
    # the cotangent, with a row that has no gradient among them
    z[2] = -np.inf
    x = z.to(DEV).requires_grad_(True)
    cot = torch.tensor([1.0, np.inf, np.inf, -np.inf, 1.0, float("nan")], device=DEV)
    (gx,) = torch.autograd.grad(lg().distill_loss(x, tv.to(DEV), ti.to(DEV), tail=a.to(DEV), reduction="none"), x, cot)
    assert torch.equal(gx[[0, 4]], good[1][[0, 4]]) and (gx[2] == 0).all() and torch.isnan(gx[5]).all()
    for r, sign in ((1, 1.0), (3, -1.0)):
        assert torch.equal(gx[r], torch.sign(good[1][r]) * sign * np.inf)


@pytest.mark.parametrize("V", [12, 101, 1001, 2048, 2049, 9001, 70001])
@pytest.mark.parametrize("tau", [1e-3, 0.1, 1.0, 3.0])
def test_distill_mass_on_nodes_closed_by_the_lowest_value(V, tau):
    """A student that closes nodes by the lowest value of f32 instead of -inf, a teacher that does not: the loss is large and finite wherever f32
    holds it, T (mass there) 3.4e38, whether one entry lies there, most of them, or the rest."""
    low, k = torch.finfo(torch.float32).min, 6
    z = torch.linspace(-2, 2, V).expand(5, V).clone()
    z[0, 2] = low
    z[1, :4] = low
    z[2, k:] = low
    z[3, 1:] = low
    z[4] = low                                             # all alike: an ordinary row
    a = torch.tensor([0.0, 0.25, 0.25, 0.25, 0.25])
    w = torch.tensor([0.3, 0.3, 0.3, -0.3, 1.0])
    d = [t.to(DEV) for t in (z, torch.zeros(5, k), torch.arange(k).int().expand(5, k), a, w)]
    more = dict(tail=d[3], temperature=tau, weight=d[4])
    got = host(lg().distill_loss(d[0], d[1], d[2], reduction="none", **more))
    # log p there is (low - m) / T to 37 digits; a sum of six terms and a dozen products, each rounded by 2^-24
    want = -low * tau * w[:4].double().numpy() * np.array([1 / 6, 0.75 * 4 / 6, 0.25, 0.75 * 5 / 6 + 0.25])
    assert np.isfinite(got).all() and (np.abs(got[:4] - want) <= 20 * ro.U * np.abs(want)).all(), (got, want)
    assert abs(got[4]) < 20 * tau * tau and lg().distill_loss(d[0], d[1], d[2], **more).item() == pytest.approx(want.sum() / 5, rel=1e-5)


@pytest.mark.parametrize("V", [9, 40, 101, 1001, 2048, 2049, 9001, 70001])
@pytest.mark.parametrize("odd", [float("nan"), float("inf")])
def test_distill_nan_is_not_hidden_by_a_closed_rest(V, odd):
    """The entries hold no mass (tail 1) and the rest is closed: +inf, but NaN where the student's row has diverged."""
    k = 9
    z = torch.full((3, V), -np.inf)
    z[:, :k] = torch.linspace(-1, 1, k)
    z[1, 4] = odd
    a = torch.tensor([1.0, 1.0, 0.5])
    loss, grad = lg().distill_loss_grad(z.to(DEV), torch.zeros(3, k, device=DEV), torch.arange(k, device=DEV).int().expand(3, k), tail=a.to(DEV), reduction="none")
    assert torch.isnan(loss[1]) and torch.isnan(grad[1]).any() and (loss[[0, 2]] == np.inf).all()


@pytest.mark.parametrize("V", [33, 101, 1001, 2048, 2049, 9001, 70001])
def test_distill_rows_without_loss_have_none_beside_a_diverged_teacher(V):
    """Rows of weight 0 and rows whose every node is closed, with NaN in the teacher's logits, in its tail and in the cotangent: 0."""
    R, k = 9, 5
    g = rng(V)
    z = torch.randn(R, V, generator=g)
    tv, ti = torch.randn(R, k, generator=g), torch.stack([torch.randperm(V, generator=g)[:k] for _ in range(R)]).int()
    a, w, cot = torch.full((R,), 0.25), torch.ones(R), torch.ones(R)
    z[[1, 2, 3, 7]] = -np.inf
    w[[4, 5, 6, 7]] = 0.0
    tv[[1, 4, 7]], a[[2, 5]], cot[[3, 6]] = float("nan"), float("nan"), float("nan")
    x = z.to(DEV).requires_grad_(True)
    loss = lg().distill_loss(x, tv.to(DEV), ti.to(DEV), tail=a.to(DEV), weight=w.to(DEV), reduction="none")
    (grad,) = torch.autograd.grad(loss, x, cot.to(DEV))
    assert (loss[1:8] == 0).all() and (grad[1:8] == 0).all()
    assert torch.isfinite(loss).all() and (loss[[0, 8]] > 0).all() and torch.isfinite(grad).all()


@pytest.mark.parametrize("V", [101, 1001, 9001])
@pytest.mark.parametrize("tau", [0.7, 1.0, 2.0])
def test_distill_of_a_policy_from_itself_is_nothing(V, tau):
    """With the tail taken at the loss's temperature.  A tail of another temperature belongs to another teacher: a loss above 0."""
    z = torch.randn(5, V, generator=rng(V)) * 2
    values, idx, tail = (o.cpu() for o in lg().top_logits(z.to(DEV), 20, temperature=tau, with_tail=True))
    _, exact = check_losses(z, values, idx, tail, tau)
    assert np.abs(exact).max() < 1e-10                     # second order in the tail's rounding of 2^-24
    if tau != 1.0:
        other = lg().top_logits(z.to(DEV), 20, with_tail=True)[2].cpu()
        assert (check_losses(z, values, idx, other, tau)[1] > 1e-4).all()


@pytest.mark.parametrize("V", [101, 3000])
def test_distill_backward_reads_what_hooks_on_saved_tensors_give_back(V):
    """A hook that keeps saved tensors on the host: the backward reads the copies it gives back, and the teacher's own memory is free for as long
    as the loss waits for its backward."""
    import weakref
    g = rng(V)
    z = torch.randn(6, V, generator=g).to(DEV).requires_grad_(True)
    tv, ti = (torch.randn(6, 9, generator=g), torch.randint(0, V, (6, 9), generator=g).int())
    a, w = torch.rand(6, generator=g), torch.rand(6, generator=g)
    (want,) = torch.autograd.grad(lg().distill_loss(z, tv.to(DEV), ti.to(DEV), tail=a.to(DEV), weight=w.to(DEV)), z)
    teacher = [t.to(DEV) for t in (tv, ti, a, w)]
    alive = [weakref.ref(t) for t in teacher]
    seen = []

    def unpack(t):
        seen.append(tuple(t.shape))
        return t.to(DEV)

    with torch.autograd.graph.saved_tensors_hooks(lambda t: t.cpu(), unpack):
        loss = lg().distill_loss(z, teacher[0], teacher[1], tail=teacher[2], weight=teacher[3])
    del teacher
    assert not any(r() is not None for r in alive)
    (got,) = torch.autograd.grad(loss, z)
    assert torch.equal(got, want) and sorted(seen) == sorted([(6, V), (6, 9), (6, 9), (6,), (6,)])
    # what a hook gives back is what is read: another teacher, another gradient
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t, lambda t: t.flip(0) if t.shape == (6,) else t):
        loss = lg().distill_loss(z, tv.to(DEV), ti.to(DEV), tail=a.to(DEV), weight=w.to(DEV))
    (got,) = torch.autograd.grad(loss, z)
    (want,) = torch.autograd.grad(lg().distill_loss(z, tv.to(DEV), ti.to(DEV), tail=a.flip(0).to(DEV), weight=w.flip(0).to(DEV)), z)
    assert torch.equal(got, want)


@pytest.mark.parametrize("which", ["logits", "values", "idx", "tail", "weight"])
@pytest.mark.parametrize("how", [lambda t: t.cpu(), lambda t: t[:-1], lambda t: t.double()], ids=["host", "shape", "type"])
def test_distill_refuses_what_else_a_hook_gives_back(which, how):
    R, V, k = 4, 60, 3
    tensors = dict(logits=torch.randn(R, V, device=DEV, requires_grad=True), values=torch.randn(R, k, device=DEV), tail=torch.rand(R, device=DEV),
                   idx=torch.zeros(R, k, device=DEV, dtype=torch.int32), weight=torch.rand(R, device=DEV) + 1)
    place = list(("logits", "values", "idx", "tail", "weight")).index(which)
    packed = []
    with torch.autograd.graph.saved_tensors_hooks(lambda t: (packed.append(t), len(packed) - 1)[1], lambda i: how(packed[i].detach()) if i == place else packed[i]):
        loss = lg().distill_loss(tensors["logits"], tensors["values"], tensors["idx"], tail=tensors["tail"], weight=tensors["weight"])
    with pytest.raises(RuntimeError):
        torch.autograd.grad(loss, tensors["logits"])


def test_distill_teacher_is_freed_with_the_graph():
    import weakref
    z, ti = torch.randn(4, 50, device=DEV, requires_grad=True), torch.zeros(4, 3, device=DEV, dtype=torch.int32)
    tv = torch.randn(4, 3, device=DEV)
    alive = weakref.ref(tv)
    loss = lg().distill_loss(z, tv, ti)
    del tv
    loss.backward()
    assert alive() is None and z.grad is not None


def test_distill_of_more_segments_than_one_launch_takes():
    """One row over and over as an expanded view: 990 000 rows of 17 segments are over 2^32 threads."""
    V, R, n = 65600, 990_000, 1000
    g = rng(3)
    z = torch.randn(1, V, generator=g)
    tv, ti, a, w = torch.randn(n, 2, generator=g), torch.randint(0, V, (n, 2), generator=g).int(), torch.rand(n, generator=g), torch.rand(n, generator=g)
    few = lg().distill_loss(z.expand(n, V).to(DEV), tv.to(DEV), ti.to(DEV), tail=a.to(DEV), weight=w.to(DEV), reduction="none")
    rl, _, lb, _ = ro.distill(host(z.expand(20, V)), host(tv[:20]), ti[:20].numpy(), host(a[:20]), 1.0, host(w[:20]))
    assert (np.abs(host(few)[:20] - rl) <= lb + 1e-30).all()
    tile = lambda t: t.repeat(R // n, *[1] * (t.dim() - 1)).to(DEV)  # noqa: E731
    more = dict(tail=tile(a), weight=tile(w))
    many = lg().distill_loss(z.to(DEV).expand(R, V), tile(tv), tile(ti), reduction="none", **more)
    assert torch.equal(many.view(-1, n), few.expand(R // n, n))
    total = lg().distill_loss(z.to(DEV).expand(R, V), tile(tv), tile(ti), reduction="sum", **more)
    assert total.item() == pytest.approx(many.double().sum().item(), rel=1e-6)


# ----------------------------------------------------------------------------------------------------------- verification
def test_verify_of_more_sequences_than_one_launch_takes():
    """2^26 and a few short sequences, one wave each: over 2^32 threads."""
    B, V = 2 ** 26 + 5, 2
    g = torch.Generator(device=DEV).manual_seed(1)
    p = torch.rand(B, 2, V, device=DEV, generator=g, dtype=torch.bfloat16)
    u = torch.rand(B, 2, device=DEV, generator=g)
    x = torch.randint(0, V, (B, 1), device=DEV, generator=g, dtype=torch.int32)
    tok, acc = lg().verify_draft(p, x, u)
    kept = u[:, 0].double() < p[:, 0].gather(1, x.long())[:, 0].double()
    assert torch.equal(acc, kept.int())
    row = torch.where(kept[:, None], p[:, 1], p[:, 0])
    left = row.masked_fill(~kept[:, None] & (torch.arange(V, device=DEV) == x), 0.0)
    row = torch.where((left.sum(1) > 0)[:, None], left, row).double()
    drawn = torch.where(row[:, 0] > u[:, 1].double() * row.sum(1), 0, 1).int()
    drawn[row.sum(1) == 0] = -1
    assert torch.equal(tok[:, 0], torch.where(kept, x[:, 0], drawn)) and torch.equal(tok[:, 1], torch.where(kept, drawn, -1))


@pytest.mark.parametrize("B,V", [(2 ** 24 + 8, 1100), (5_600_000, 8300)])
def test_verify_of_more_long_rows_than_one_launch_takes(B, V):
    """One target and one draft over and over as expanded views, a workgroup or three to a sequence."""
    n, G = 1000, 2
    g = rng(V)
    p, q = torch.softmax(torch.randn(1, G + 1, V, generator=g) * 3, -1), torch.softmax(torch.randn(1, G, V, generator=g) * 3, -1)
    x, u = torch.multinomial(q[0], n, replacement=True, generator=g).T.contiguous().int(), torch.rand(n, G + 1, generator=g)
    lengths = torch.randint(0, G + 1, (n,), generator=g).int()
    rt, ra = ro.verify(host(p.expand(n, G + 1, V))[:50], x[:50].numpy(), host(u)[:50], host(q.expand(n, G, V))[:50], lengths[:50].numpy())
    P, Q = p.to(DEV), q.to(DEV)
    few = lg().verify_draft(P.expand(n, G + 1, V), x.to(DEV), u.to(DEV), draft_probs=Q.expand(n, G, V), lengths=lengths.to(DEV))
    np.testing.assert_array_equal(few[0][:50].cpu().numpy(), rt)
    np.testing.assert_array_equal(few[1][:50].cpu().numpy(), ra)
    tile = lambda t: t.repeat(-(-B // n), *[1] * (t.dim() - 1))[:B].to(DEV)  # noqa: E731
    many = lg().verify_draft(P.expand(B, G + 1, V), tile(x), tile(u), draft_probs=Q.expand(B, G, V), lengths=tile(lengths))
    assert torch.equal(many[0], tile(few[0])) and torch.equal(many[1], tile(few[1]))


# ------------------------------------------------------------------------------------------------- ranges the documentation names
@pytest.mark.parametrize("tau", [1e-15, 1e-6, 0.05, 20.0, 1e6, 1e15])
@pytest.mark.parametrize("V", [17, 101, 300, 1500, 3000, 9001, 70001])
def test_temperatures_to_both_ends(V, tau):
    g = rng(V)
    z = torch.randn(5, V, generator=g) * 4
    z[1, 1::2] = -np.inf
    t = z + torch.randn(5, V, generator=g)
    k = min(V, 33) - 5
    values, idx, tail = (o.cpu() for o in lg().top_logits(t.to(DEV), k, temperature=tau, with_tail=True))
    rv, ri = ro.top(host(t), k)
    ref, err = ro.tail(host(t), ri, tau)
    np.testing.assert_array_equal(idx.numpy(), ri)
    # v_exp_f32 gives 0 for what lies below 2^-126: each of up to V - k terms of a sum that is divided by at least 1 can lose that much, and the
    # bound above allows it once
    assert (np.abs(host(tail) - ref) <= err + V * 2.0 ** -126).all()
    check_losses(z, values, idx, tail, tau)


def test_rows_beyond_32_bits_of_elements_and_bytes():
    """22 million rows of 101: 2.2e9 logits.  Row r is row r mod 1000 of a table with a shift of its own: the same order, tail, loss and gradient."""
    R, V, k, n = 22_000_000, 101, 6, 1000
    g = rng(1)
    base = torch.randn(n, V, generator=g).to(DEV)
    v0, i0, t0 = lg().top_logits(base, k, with_tail=True)
    z = torch.empty(R, V, dtype=torch.bfloat16, device=DEV)
    z.view(-1, n, V).copy_(base.bfloat16().expand(R // n, n, V))
    vb, ib, tb = lg().top_logits(base.bfloat16(), k, with_tail=True)
    values, idx, tail = lg().top_logits(z, k, with_tail=True)
    assert all(torch.equal(a.view(-1, *b.shape), b.expand(R // n, *b.shape)) for a, b in ((values, vb), (idx, ib), (tail, tb)))
    lb, gb = lg().distill_loss_grad(base.bfloat16(), v0, i0, tail=t0, reduction="none")
    tile = lambda t: t.repeat(R // n, *[1] * (t.dim() - 1))  # noqa: E731
    loss, grad = lg().distill_loss_grad(z, tile(v0), tile(i0), tail=tile(t0), reduction="none")
    assert torch.equal(loss.view(-1, n), lb.expand(R // n, n)) and torch.equal(grad.view(-1, n, V), gb.expand(R // n, n, V))
    # verification of rows behind the 2^31st probability
    p = torch.softmax(z.view(-1, 2, V)[-4000:].float(), -1)
    x, u = torch.randint(0, V, (R // 2, 1), device=DEV, dtype=torch.int32), torch.rand(R // 2, 2, device=DEV)
    z.view(-1, 2, V)[-4000:].copy_(p)
    tok, acc = lg().verify_draft(z.view(-1, 2, V), x, u)
    t2, a2 = lg().verify_draft(z.view(-1, 2, V)[-4000:].contiguous(), x[-4000:], u[-4000:])
    assert torch.equal(tok[-4000:], t2) and torch.equal(acc[-4000:], a2)
