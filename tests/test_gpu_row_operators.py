"""Row operators over node logits (elg_amd/logits.py) against their definitions in 64 bits (row_oracle.py): every kernel by size, the masks
and values a row can hold, strides, streams, captures, and the three together on a rollout's own rows."""
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


def rows(kind, R, V, seed, dtype=torch.float32):
    """Rows of logits on the host, rounded to dtype."""
    g = rng(seed)
    z = torch.randn(R, V, generator=g) * 6
    if kind == "closed":                                   # half of the nodes closed, the share rising over the rows
        share = torch.linspace(0, 1, R)[:, None] if R > 1 else torch.full((1, 1), 0.5)
        z = z.masked_fill(torch.rand(R, V, generator=g) < share, -np.inf)
        z[::3, 0] = 1.5                                    # some rows keep one open node, the others may be empty
    elif kind == "ties":
        z = torch.randint(-2, 3, (R, V), generator=g).float()
    elif kind == "equal":
        z = torch.full((R, V), 3.25)
    elif kind == "up":
        z = torch.arange(V, dtype=torch.float32).expand(R, V) / max(V, 1) * 9 - 4
    elif kind == "down":
        z = -torch.arange(V, dtype=torch.float32).expand(R, V) / max(V, 1) * 9
    elif kind == "lowest":                                 # closed by the type's lowest value instead of -inf
        z = z.masked_fill(torch.rand(R, V, generator=g) < 0.6, torch.finfo(dtype).min)
        z[-1] = torch.finfo(dtype).min
    elif kind == "empty":
        z = torch.full((R, V), -np.inf)
    elif kind == "spread":                                 # the decoder's clip: 50 tanh
        z = 50 * torch.tanh(torch.randn(R, V, generator=g) * 2)
    return z.to(dtype)


# ------------------------------------------------------------------------------------------------------------- top_logits
SIZES = [(1, 1), (2, 1), (2, 2), (7, 3), (64, 64), (101, 40), (121, 121), (122, 5), (125, 125), (126, 16), (128, 128), (129, 64), (249, 40),
         (253, 253), (254, 200), (1001, 63), (1021, 256), (1022, 256), (2045, 1), (2046, 33), (4099, 256), (8189, 100), (8190, 64), (16389, 128)]


def check_top(z, k, tau=1.0):
    """z on the host, of the type tested."""
    zd = z.to(DEV)
    values, idx, tail = lg().top_logits(zd, k, temperature=tau, with_tail=True)
    v2, i2 = lg().top_logits(zd, k, temperature=tau)
    rv, ri = ro.top(host(z).reshape(-1, z.shape[-1]), k)
    assert values.dtype == z.dtype and idx.dtype == torch.int32 and values.shape == (*z.shape[:-1], k) == idx.shape
    np.testing.assert_array_equal(idx.cpu().numpy().reshape(ri.shape), ri)
    np.testing.assert_array_equal(host(values).reshape(rv.shape), rv)
    assert torch.equal(i2, idx) and torch.equal(v2.isnan(), values.isnan()) and torch.equal(v2.nan_to_num(), values.nan_to_num())
    return host(tail).reshape(-1), ri


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("V,k", SIZES)
def test_top_sizes(V, k, dtype):
    for kind in ("plain", "closed", "ties"):
        R = 37 if V < 3000 else 3
        z = rows(kind, R, V, V + k, TYPES[dtype])
        tail, ri = check_top(z, k, 0.7)
        ref, err = ro.tail(host(z), ri, 0.7)
        assert (np.abs(tail - ref) <= err).all(), (kind, np.abs(tail - ref).max())


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("V,k", [(101, 40), (101, 101), (200, 77), (1001, 63), (2500, 256), (9001, 256), (33000, 64), (70001, 256), (131072, 128)])
@pytest.mark.parametrize("kind", ["equal", "up", "down", "lowest", "empty", "spread", "ties"])
def test_top_values(V, k, kind, dtype):
    z = rows(kind, 5 if V < 3000 else 2, V, 3, TYPES[dtype])
    tail, ri = check_top(z, k, 2.0)
    ref, err = ro.tail(host(z), ri, 2.0)
    assert (np.abs(tail - ref) <= err).all(), (np.abs(tail - ref).max(), err.max())


@pytest.mark.parametrize("V,k", [(64, 9), (101, 40), (300, 20), (1001, 63), (3001, 64), (40001, 200)])
def test_top_nan_infinities_and_signed_zeros(V, k):
    z = rows("closed", 9, V, 5)
    z[1, 1:V:7] = float("nan")
    z[2, V // 2] = float("inf")
    z[3] = torch.where(torch.arange(V) % 2 == 0, 0.0, -0.0)
    z[4, 1:] = float("nan")
    z[5, -1] = -float("nan")
    z[6] = float("inf")
    tail, ri = check_top(z, k)
    assert np.isfinite(tail[3]) and tail[3] == pytest.approx((V - k) / V, rel=1e-5)


def test_top_one_row_per_open_node_count():
    """0 ... V open nodes at random places: the closed ones fill up the rest, lowest index first."""
    for V, k in ((101, 40), (257, 64), (1001, 256), (5000, 256)):
        g = rng(V)
        counts = sorted({0, 1, 2, k - 1, k, k + 1, V // 2, V - 1, V})
        z = torch.full((len(counts), V), -np.inf)
        for r, n in enumerate(counts):
            z[r, torch.randperm(V, generator=g)[:n]] = torch.randn(n, generator=g)
        tail, _ = check_top(z, k)
        assert (tail[[i for i, n in enumerate(counts) if n <= k]] == 0).all()


@pytest.mark.parametrize("dtype", list(TYPES))
def test_top_strides_offsets_and_leading_dimensions(dtype):
    big = rows("plain", 24, 231, 1, TYPES[dtype])
    d = big.to(DEV)
    for view in (lambda t: t[:, 1:102], lambda t: t[1::2, 3:204], lambda t: t.view(4, 6, 231)[:, ::2, 5:130], lambda t: t[:, ::2],
                 lambda t: t[0], lambda t: t[:1].expand(7, 231)):
        z = view(big)
        k = min(40, z.shape[-1])
        values, idx = lg().top_logits(view(d), k)
        rv, ri = ro.top(host(z).reshape(-1, z.shape[-1]), k)
        np.testing.assert_array_equal(idx.cpu().numpy().reshape(ri.shape), ri)
        assert idx.shape == (*z.shape[:-1], k)


def test_top_many_rows():
    z = rows("closed", 70001, 33, 9)
    values, idx, tail = lg().top_logits(z.to(DEV), 5, with_tail=True)
    order = torch.sort(z, dim=-1, descending=True, stable=True)
    assert torch.equal(idx.cpu().long(), order.indices[:, :5]) and torch.equal(values.cpu(), order.values[:, :5])
    e = order.values.double().exp()
    ref = torch.where(e.sum(-1) > 0, e[:, 5:].sum(-1) / e.sum(-1), torch.zeros(()).double())
    assert (tail.cpu().double() - ref).abs().max() < 2e-5


# ----------------------------------------------------------------------------------------------------------- distillation
def teacher_of(z, k, seed, top_dtype=torch.float32, tail=True, tau=1.0):
    """A teacher near z over the same closed nodes, its k best entries in a scrambled order, and its mass outside them."""
    g = rng(seed)
    t = z.double() + torch.randn(z.shape, generator=g).double() * 1.5
    k = min(k, z.shape[1])
    v, i = t.topk(k, dim=1)
    perm = torch.randperm(k, generator=g)
    p = torch.softmax(torch.nan_to_num(t / tau, neginf=-1e9), 1)
    a = (1 - p.gather(1, i).sum(1)).clamp(0, 1).float() if tail else None
    return v[:, perm].to(top_dtype), i[:, perm].to(torch.int32), a


def compare(got_loss, got_grad, z, tv, ti, a, tau, w, scale_rows, dtype, mean=False):
    loss, grad, lb, gb = ro.distill(host(z), host(tv), ti.cpu().numpy(), None if a is None else host(a), tau, None if w is None else host(w))
    s = np.broadcast_to(np.asarray(scale_rows, np.float64), loss.shape)
    gl = host(got_loss)
    if mean:
        R = len(loss)
        if np.isfinite(loss).all():
            assert abs(gl - loss.sum() / R) <= lb.sum() / R + 2 * ro.U * abs(loss.sum() / R) + 1e-30
    else:
        fin = np.isfinite(loss)
        assert (gl[~fin] == loss[~fin]).all()
        assert (np.abs(gl - loss)[fin] <= lb[fin] + 1e-30).all(), (np.abs(gl - loss)[fin] / (lb[fin] + 1e-30)).max()
    gg = host(got_grad)
    bound = (gb + 4 * ro.U * np.abs(grad)) * np.abs(s)[:, None]
    bound = bound + ro.HALF_STEP[dtype] * (np.abs(grad * s[:, None]) + bound) + ro.TINY[dtype]
    bad = np.abs(gg - grad * s[:, None]) - bound
    assert (bad <= 0).all(), (np.unravel_index(bad.argmax(), bad.shape), bad.max(), (np.abs(gg - grad * s[:, None]) / bound).max())
    return loss, grad


def check_distill(z, tv, ti, a, tau, w, dtype):
    d = [None if t is None else t.to(DEV) for t in (z, tv, ti, a, w)]
    more = dict(tail=d[3], temperature=tau, weight=d[4])
    loss, grad = lg().distill_loss_grad(d[0], d[1], d[2], reduction="none", **more)
    compare(loss, grad, z, tv, ti, a, tau, w, 1.0, dtype)
    l2, g2 = lg().distill_loss_grad(d[0], d[1], d[2], reduction="none", **more)
    assert torch.equal(loss.nan_to_num(), l2.nan_to_num()) and torch.equal(grad, g2)                # the same bits again
    x = d[0].clone().requires_grad_(True)
    rows_loss = lg().distill_loss(x, d[1], d[2], reduction="none", **more)
    cot = torch.linspace(-2, 2, z.shape[0], device=DEV)
    (gr,) = torch.autograd.grad(rows_loss, x, cot)
    compare(rows_loss, gr, z, tv, ti, a, tau, w, host(cot), dtype)
    mean = lg().distill_loss(x, d[1], d[2], reduction="mean", **more)
    if torch.isfinite(mean):
        (gm,) = torch.autograd.grad(mean * 3.0, x)
        compare(mean, gm, z, tv, ti, a, tau, w, 3.0 / z.shape[0], dtype, mean=True)
        lm, gm1 = lg().distill_loss_grad(d[0], d[1], d[2], reduction="mean", **more)
        compare(lm, gm1, z, tv, ti, a, tau, w, 1.0 / z.shape[0], dtype, mean=True)
        ls, _ = lg().distill_loss_grad(d[0], d[1], d[2], reduction="sum", **more)
        assert ls.item() == pytest.approx(mean.item() * z.shape[0], rel=1e-6)


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("V,k", SIZES + [(24579, 200), (33000, 64), (70001, 100)])
def test_distill_sizes(V, k, dtype):
    R = 21 if V < 3000 else 3
    for n, (kind, tail, tau) in enumerate([("plain", True, 1.0), ("closed", False, 2.0), ("closed", True, 0.7)]):
        z = rows(kind, R, V, V + n, TYPES[dtype])
        tv, ti, a = teacher_of(z, k, n, tail=tail, tau=tau, top_dtype=TYPES[dtype])
        check_distill(z, tv, ti, a, tau, None, dtype)


@pytest.mark.parametrize("dtype,V", [("float32", 4099), ("float32", 8191), ("float32", 12001), ("float32", 16384), ("float32", 30011), ("float32", 65536),
                                     ("float32", 65533), ("bfloat16", 9001), ("bfloat16", 16001), ("bfloat16", 32768), ("float16", 60001),
                                     ("bfloat16", 131072), ("float16", 131071)])
def test_distill_long_rows_by_the_dozen(dtype, V):
    """Enough long rows for a workgroup each: every size of workgroup, rows that start at every alignment, weights and repeated nodes."""
    R, k = 70, 100
    z = rows("closed", R, V, V, TYPES[dtype])
    z[:, 5] = 2.0
    tv, ti, a = teacher_of(z, k, 7)
    ti[::3, 40:44] = ti[::3, :1]
    ti[1::3, -3:] = -1
    tv = torch.where(torch.isfinite(tv), tv, torch.full_like(tv, -np.inf))
    open_ = torch.isfinite(z.gather(1, ti.clamp(0, V - 1).long())) & (ti >= 0)
    tv = torch.where(open_, tv, torch.full_like(tv, -np.inf))
    w = torch.ones(R)
    w[4::9] = 0.0
    d = [t.to(DEV) for t in (z, tv, ti, a, w)]
    loss, grad = lg().distill_loss_grad(d[0], d[1], d[2], tail=d[3], weight=d[4], reduction="none")
    some = [0, 1, 2, 4, 33, 68, 69]
    compare(loss[some], grad[some], z[some], tv[some], ti[some], a[some], 1.0, w[some], 1.0, dtype)
    # the same rows a few at a time go another way
    for at in range(0, R, 35):
        l2, g2 = lg().distill_loss_grad(*(t[at:at + 35] for t in d[:3]), tail=d[3][at:at + 35], weight=d[4][at:at + 35], reduction="none")
        assert torch.allclose(l2, loss[at:at + 35], rtol=1e-5, atol=1e-6)
        assert (g2.double() - grad[at:at + 35].double()).norm() <= (2 * ro.HALF_STEP[dtype] + 1e-6) * g2.double().norm()
    mean, gm = lg().distill_loss_grad(d[0], d[1], d[2], tail=d[3], weight=d[4])
    assert mean.item() == pytest.approx(loss.double().mean().item(), rel=1e-6)
    # a strided view: rows and gradient lie differently in memory
    wide = torch.zeros(R, V + 3, dtype=TYPES[dtype], device=DEV)
    wide[:, 1:V + 1] = d[0]
    l3, g3 = lg().distill_loss_grad(wide[:, 1:V + 1], d[1], d[2], tail=d[3], weight=d[4], reduction="none")
    compare(l3[some], g3[some], z[some], tv[some], ti[some], a[some], 1.0, w[some], 1.0, dtype)
    assert torch.allclose(l3, loss, rtol=1e-5, atol=1e-6)


@pytest.mark.parametrize("V,k", [(101, 40), (500, 40), (1500, 64), (3000, 100), (20011, 256)])
@pytest.mark.parametrize("kind", ["spread", "lowest", "empty", "ties"])
def test_distill_values_and_weights(V, k, kind):
    z = rows(kind, 6, V, 11)
    tv, ti, a = teacher_of(z, k, 2)
    w = torch.tensor([1.0, 0.0, 0.25, 3.0, 0.0, 1.0])
    check_distill(z, tv, ti, a, 1.0, w, "float32")


@pytest.mark.parametrize("V,k", [(33, 12), (101, 40), (700, 100), (3000, 100), (40001, 256)])
@pytest.mark.parametrize("top_dtype,idx_dtype", [("float32", torch.int64), ("bfloat16", torch.int32), ("float16", torch.int64)])
def test_distill_padded_repeated_and_outside_entries(V, k, top_dtype, idx_dtype):
    z = rows("closed", 8, V, 4)
    z[:, 1:4] = torch.tensor([0.5, 1.0, -1.0])
    tv, ti, a = teacher_of(z, k, 3)
    ti[0, 5:] = -1                                         # padding
    ti[1, :4] = torch.tensor([V, V + 70000, -(2 ** 31), 2 ** 31 - 1])
    ti[2, :] = -1                                          # no entry at all
    ti[3, 1:4] = ti[3, 0]                                  # one node four times
    ti[4, :] = 2                                           # only one node, every time
    tv[5, :] = -np.inf                                     # entries, none of them open
    tv[6, ::2] = -np.inf
    ti[7, -2:] = ti[7, :2]                                 # two nodes twice
    ti = ti.to(idx_dtype)
    if idx_dtype == torch.int64:
        ti[1, 0] = 2 ** 40 + 1                             # its low half is a node
    tv = torch.where(torch.isfinite(tv), tv, torch.full_like(tv, -np.inf)).to(TYPES[top_dtype])
    ok = (ti >= 0) & (ti < V)
    open_ = torch.isfinite(z.gather(1, ti.clamp(0, V - 1).long())) & ok
    tv = torch.where(open_ | ~ok, tv, torch.full_like(tv, -np.inf))        # no mass on closed nodes here
    for tail in (a, None):
        check_distill(z, tv, ti, tail, 1.5, None, "float32")


def test_distill_mass_on_a_closed_node_and_an_empty_rest():
    z = torch.zeros(3, 50)
    z[0, 7] = -np.inf
    z[1, 10:] = -np.inf
    tv, ti = torch.zeros(3, 10), torch.arange(10).int().expand(3, 10).contiguous()
    a = torch.tensor([0.25, 0.25, 0.25])
    loss, grad = lg().distill_loss_grad(z.to(DEV), tv.to(DEV), ti.to(DEV), tail=a.to(DEV), reduction="none")
    assert loss[0] == np.inf and loss[1] == np.inf and torch.isfinite(loss[2])
    ref = ro.distill(z.numpy(), tv.numpy(), ti.numpy(), a.numpy(), 1.0, None)[1]
    np.testing.assert_allclose(grad.cpu().numpy(), ref, atol=1e-6)
    total = lg().distill_loss(z.to(DEV), tv.to(DEV), ti.to(DEV), tail=a.to(DEV))
    assert total.item() == np.inf


@pytest.mark.parametrize("V", [50, 700, 3001, 40001])
def test_distill_when_the_entries_hold_nothing(V):
    """tail = 1: the entries' masses are 0, also where the student has closed one of their nodes; tail above 1 is taken as 1, below 0 as 0."""
    z = rows("plain", 4, V, 5)
    z[0, 3] = -np.inf
    tv, ti = torch.zeros(4, 10), torch.arange(10).int().expand(4, 10).contiguous()
    for a in (torch.ones(4), torch.tensor([1.0, 1.5, -0.25, 0.0])):
        check_distill(z if a.min() == 1 else z.masked_fill(torch.isinf(z), -9.0), tv, ti, a, 1.3, None, "float32")


@pytest.mark.parametrize("V", [40, 900, 5000])
def test_distill_nan_is_not_hidden(V):
    z = rows("plain", 4, V, 1)
    tv, ti, a = teacher_of(z, 10, 1)
    z[1, V - 1] = float("nan")
    tv[2, 0] = float("nan")
    loss, grad = lg().distill_loss_grad(z.to(DEV), tv.to(DEV), ti.to(DEV), tail=a.to(DEV), reduction="none")
    assert torch.isnan(loss[1]) and torch.isnan(loss[2]) and torch.isnan(grad[1]).any() and torch.isnan(grad[2]).any()
    assert torch.isfinite(loss[[0, 3]]).all() and torch.isfinite(grad[[0, 3]]).all()


@pytest.mark.parametrize("V,k,tail", [(23, 5, True), (101, 40, True), (101, 40, False), (1300, 30, True), (3000, 20, True)])
def test_distill_gradient_against_differences(V, k, tail):
    """Central differences of the definition's loss in 64 bits, step h: off by h^2 times a third derivative (<= 2 for a softmax row with
    weights <= 1) and by rounding of 2^-53 |L| / h."""
    z = rows("plain", 2, V, 8) / 4
    tv, ti, a = teacher_of(z, k, 5, tail=tail)
    x = z.to(DEV).requires_grad_(True)
    loss = lg().distill_loss(x, tv.to(DEV), ti.to(DEV), tail=None if a is None else a.to(DEV), reduction="sum")
    (g,) = torch.autograd.grad(loss, x)
    h = 1e-4
    f = lambda zz: ro.distill(zz, host(tv), ti.numpy(), None if a is None else host(a), 1.0, None)[0].sum()  # noqa: E731
    for r, n in [(0, 0), (0, int(ti[0, 0])), (0, int(ti[0, k - 1])), (1, V - 1), (1, V // 2), (1, int(ti[1, 1]))]:
        zp, zm = host(z).copy(), host(z).copy()
        zp[r, n] += h
        zm[r, n] -= h
        assert abs((f(zp) - f(zm)) / (2 * h) - g[r, n].item()) < 2 * h * h + 1e-10 + 1e-5 * abs(g[r, n].item()) + 200 * ro.U


@pytest.mark.parametrize("dtype", list(TYPES))
def test_distill_views_and_untouched_neighbours(dtype):
    """Strided logits; the gradient of a view through autograd lands in the view's elements and nowhere else."""
    T = TYPES[dtype]
    big = rows("plain", 12, 333, 6, T)
    leaf = big.to(DEV).requires_grad_(True)
    for view in (lambda t: t[:, 3:104], lambda t: t[::3, 1:302], lambda t: t.view(3, 4, 333)[:, 1:3, 7:], lambda t: t[:, ::3]):
        z = view(big)
        flat = z.reshape(-1, z.shape[-1])
        tv, ti, a = teacher_of(flat, 20, 2)
        lead = z.shape[:-1]
        loss = lg().distill_loss(view(leaf), tv.view(*lead, 20).to(DEV), ti.view(*lead, 20).to(DEV), tail=a.view(lead).to(DEV), reduction="none")
        assert loss.shape == lead
        (g,) = torch.autograd.grad(loss, leaf, torch.ones_like(loss))
        compare(loss.reshape(-1), view(g).reshape(flat.shape), flat, tv, ti, a, 1.0, None, 1.0, dtype)
        outside = torch.ones_like(g, dtype=torch.bool)
        view(outside).fill_(False)
        assert (g[outside] == 0).all()


@pytest.mark.parametrize("V", [101, 515, 2100, 9000])
def test_distill_writes_inside_its_rows_only(V):
    """Through the C ABI: a gradient in the middle of a larger buffer, at an odd element, leaves what is around it."""
    from elg_amd import _lib as L
    z = rows("plain", 5, V, 2)
    tv, ti, a = teacher_of(z, 9, 2)
    d = [t.to(DEV) for t in (z, tv, ti, a)]
    ws = torch.empty(L.lib().elg_distill_ws_bytes(5, V, L.F32), dtype=torch.uint8, device=DEV)
    for off in (1, 2, 3, 64):
        buf = torch.full((off + 5 * V + 70,), 7.0, device=DEV)
        rc = L.lib().elg_distill_loss_grad(d[0].data_ptr(), V, L.F32, 5, V, d[1].data_ptr(), L.F32, d[2].data_ptr(), 0, 9, d[3].data_ptr(),
                                           1.0, None, None, 0, 1.0, None, None, buf.data_ptr() + 4 * off, ws.data_ptr(), ws.numel(),
                                           torch.cuda.current_stream().cuda_stream)
        assert rc == 0
        _, ref = lg().distill_loss_grad(*d[:3], tail=d[3], reduction="none")
        assert torch.equal(buf[off:off + 5 * V].view(5, V), ref)
        assert (buf[:off] == 7).all() and (buf[off + 5 * V:] == 7).all()


def test_distill_of_no_rows_and_of_many():
    z = torch.empty(0, 17, device=DEV, requires_grad=True)
    tv, ti = torch.empty(0, 3, device=DEV), torch.empty(0, 3, device=DEV, dtype=torch.int32)
    for red in ("sum", "mean", "none"):
        loss = lg().distill_loss(z, tv, ti, reduction=red)
        assert loss.sum().item() == 0
        assert torch.autograd.grad(loss.sum(), z)[0].shape == (0, 17)
    assert lg().top_logits(z.detach(), 3)[1].shape == (0, 3)
    z = rows("closed", 50021, 21, 3)
    z[:, 2] = 0.25
    tv, ti, a = teacher_of(z, 6, 4)
    loss, grad = lg().distill_loss_grad(z.to(DEV), tv.to(DEV), ti.to(DEV), tail=a.to(DEV))
    rl, rg, lb, gb = ro.distill(z[:300].numpy(), tv[:300].numpy(), ti[:300].numpy(), a[:300].numpy(), 1.0, None)
    each, _ = lg().distill_loss_grad(z.to(DEV), tv.to(DEV), ti.to(DEV), tail=a.to(DEV), reduction="none")
    assert (np.abs(host(each)[:300] - rl) <= lb + 1e-30).all()
    assert loss.item() == pytest.approx(host(each).sum() / 50021, rel=1e-6)
    assert (np.abs(host(grad)[:300] * 50021 - rg) <= gb + 1e-5 * np.abs(rg) + 1e-30).all()


# ----------------------------------------------------------------------------------------------------------- verification
def drafts(B, G, V, seed, dtype=torch.float32, closed=0.4):
    g = rng(seed)
    z = torch.randn(B, G + 1, V, generator=g) * 3
    z = z.masked_fill(torch.rand(B, G + 1, V, generator=g) < closed, -np.inf)
    z[..., 0] = 0.0
    p = torch.softmax(z, -1)
    q = torch.softmax(z[:, :G] + torch.randn(B, G, V, generator=g), -1)
    x = torch.stack([torch.multinomial(q[:, i], 1, generator=g)[:, 0] for i in range(G)], 1) if G else torch.zeros(B, 0, dtype=torch.int64)
    return p.to(dtype), q.to(dtype), x.to(torch.int32), torch.rand(B, G + 1, generator=g)


def check_verify(p, x, u, q=None, n=None):
    d = [None if t is None else t.to(DEV) for t in (p, x, u, q, n)]
    tok, acc = lg().verify_draft(d[0], d[1], d[2], draft_probs=d[3], lengths=d[4])
    rt, ra = ro.verify(host(p), x.numpy(), host(u), None if q is None else host(q), None if n is None else n.numpy())
    np.testing.assert_array_equal(acc.cpu().numpy(), ra)
    np.testing.assert_array_equal(tok.cpu().numpy(), rt)
    return ra


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("V", [1, 2, 5, 63, 64, 65, 101, 129, 255, 256, 1001, 2047, 2048, 4100, 20001, 70003])
def test_verify_sizes(V, dtype):
    B, G = (60, 5) if V < 3000 else (7, 3)
    p, q, x, u = drafts(B, G, V, V, TYPES[dtype])
    n = torch.arange(B).int() % (G + 2) - (torch.arange(B) % 11 == 0).int()              # -1 ... G + 1: clamped
    seen = set(check_verify(p, x, u, q, n).tolist()) | set(check_verify(p, x, u, q).tolist())
    assert len(seen) > 1
    check_verify(p, x, u)                                                                 # certain drafts
    check_verify(p, x.long(), u, None, n.long())


def test_verify_lengths_beyond_32_bits_are_clamped():
    p, q, x, u = drafts(6, 3, 40, 5)
    n = torch.tensor([2 ** 32, 2 ** 32 + 1, -2 ** 32, 2 ** 40, 3, 2 ** 31])
    got = lg().verify_draft(p.to(DEV), x.to(DEV), u.to(DEV), draft_probs=q.to(DEV), lengths=n.to(DEV))
    want = lg().verify_draft(p.to(DEV), x.to(DEV), u.to(DEV), draft_probs=q.to(DEV), lengths=n.clamp(0, 3).int().to(DEV))
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_verify_borders_are_exact():
    p = torch.tensor([[[0.25, 0.25, 0.5], [0.5, 0.0, 0.5]]]).repeat(7, 1, 1)
    q = torch.tensor([[[0.5, 0.25, 0.25]]]).repeat(7, 1, 1)
    x = torch.tensor([[0], [0], [1], [2], [0], [0], [1]], dtype=torch.int32)
    below, one = np.float32(0.5) - np.float32(2.0 ** -25), 1 - 2.0 ** -24
    u = torch.tensor([[0.5, 0.0], [float(below), 0.5], [one, float(below)], [one, one], [0.9, one], [one, 0.999], [0.0, 0.0]])
    tok, acc = lg().verify_draft(p.to(DEV), x.to(DEV), u.to(DEV), draft_probs=q.to(DEV))
    # 0.5 x 0.5 < 0.25 is false: refused; just below: accepted; q <= p: always accepted
    assert acc.tolist() == [0, 1, 1, 1, 0, 0, 1]
    assert tok.tolist() == [[2, -1], [0, 2], [1, 0], [2, 2], [2, -1], [2, -1], [1, 0]]
    check_verify(p, x, u, q)


def test_verify_nothing_left_and_empty_rows():
    V = 37
    p = torch.zeros(4, 3, V)
    p[0, :, 5] = 1.0                                       # the target equals the draft: nothing is left over it
    p[1, 0, 3] = 0.5                                       # a row that is empty where the draw falls
    p[2] = 0.0                                             # all empty
    p[3, 0, 7], p[3, 0, 8] = -0.5, float("nan")            # entries that are no probabilities count as 0
    p[3, 0, 9] = 0.125
    q = torch.zeros(4, 2, V)
    q[0, :, 5] = 1.0
    q[1, :, 3] = 0.5
    q[2, :, 1] = 1.0
    q[3, :, 9] = 1.0
    x = torch.tensor([[4, 5], [3, 3], [1, 1], [9, 9]], dtype=torch.int32)
    u = torch.full((4, 3), 0.5)
    tok, acc = lg().verify_draft(p.to(DEV), x.to(DEV), u.to(DEV), draft_probs=q.to(DEV))
    assert acc.tolist() == [0, 1, 0, 0]
    assert tok.tolist() == [[5, -1, -1], [3, -1, -1], [-1, -1, -1], [9, -1, -1]]


def test_verify_tokens_outside_the_row_and_long_drafts():
    p, q, x, u = drafts(9, 4, 50, 3)
    x[0, 0], x[1, 1], x[2, 0], x[3, 2] = -1, 50, 2 ** 31 - 1, -(2 ** 31)
    check_verify(p, x, u * 0.01, q)
    check_verify(p, x, u * 0.01)
    p, q, x, u = drafts(3, 200, 11, 4, closed=0.0)
    u[:, :150] = 0.0                                       # more than a wave's drafts accepted
    u[1, :] = 0.0
    check_verify(p, x, u, p[:, :200])
    tok, acc = lg().verify_draft(p[:, :1].to(DEV), torch.zeros(3, 0, dtype=torch.int32, device=DEV), u[:, :1].contiguous().to(DEV))
    assert tok.shape == (3, 1) and acc.tolist() == [0, 0, 0]


def test_verify_strided_views_and_empty_batches():
    p, q, x, u = drafts(24, 6, 64, 9)
    P, Q = p.to(DEV), q.to(DEV)
    # steps 1 ... 4 of longer records, (4, 6) leading dimensions, an odd part of the nodes
    view = lambda t, s: t.view(4, 6, *t.shape[1:])[:, :, 1:1 + s, 3:60]  # noqa: E731
    x4 = (x.view(4, 6, 6)[:, :, 1:5] - 3).clamp(0, 56)
    u4 = u.view(4, 6, 7)[:, :, 1:6]
    tok, acc = lg().verify_draft(view(P, 5), x4.to(DEV), u4.to(DEV), draft_probs=view(Q, 4))
    rt, ra = ro.verify(host(view(p, 5)).reshape(24, 5, 57), x4.reshape(24, 4).numpy(), host(u4).reshape(24, 5), host(view(q, 4)).reshape(24, 4, 57))
    np.testing.assert_array_equal(tok.cpu().numpy().reshape(24, 5), rt)
    np.testing.assert_array_equal(acc.cpu().numpy().reshape(24), ra)
    tok, acc = lg().verify_draft(P[:0], x[:0].to(DEV), u[:0].to(DEV), draft_probs=Q[:0])
    assert tok.shape == (0, 7) and acc.shape == (0,)


def test_verified_answers_follow_the_target():
    """Accepted and replaced first choices together are distributed as the target's row: 40 000 sequences, each frequency within six
    standard deviations of its probability."""
    B, V = 40000, 8
    g = rng(0)
    p = torch.softmax(torch.randn(1, 1, V, generator=g), -1)
    q = torch.softmax(torch.randn(1, 1, V, generator=g), -1)
    x = torch.multinomial(q[0, 0], B, replacement=True, generator=g).view(B, 1).int()
    u = torch.rand(B, 2, generator=g)
    tok, acc = lg().verify_draft(p.expand(B, 2, V).to(DEV), x.to(DEV), u.to(DEV), draft_probs=q.expand(B, 1, V).to(DEV))
    freq = torch.bincount(tok[:, 0].cpu().long(), minlength=V).double() / B
    pr = p[0, 0].double()
    assert ((freq - pr).abs() < 6 * (pr * (1 - pr) / B).sqrt()).all()
    assert abs(acc.double().mean().item() - torch.minimum(p, q).sum().item()) < 6 * 0.5 / B ** 0.5


# --------------------------------------------------------------------------------------- streams, captures, refusals, together
def test_other_streams_and_calls_in_flight():
    z = rows("plain", 300, 1001, 1).to(DEV)
    tv, ti, tail = lg().top_logits(z + 0.5 * torch.randn_like(z), 50, with_tail=True)
    p, q, x, u = (t.to(DEV) for t in drafts(64, 4, 9001, 2))
    ref = (lg().distill_loss_grad(z, tv, ti, tail=tail), lg().verify_draft(p, x, u, draft_probs=q))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    got = []
    for s in streams * 3:
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            got.append((lg().distill_loss_grad(z, tv, ti, tail=tail), lg().verify_draft(p, x, u, draft_probs=q)))
    torch.cuda.synchronize()
    for (l, g), (t, a) in got:
        assert torch.equal(l, ref[0][0]) and torch.equal(g, ref[0][1]) and torch.equal(t, ref[1][0]) and torch.equal(a, ref[1][1])


@pytest.mark.parametrize("R,V", [(64, 101), (40, 1001), (20, 5000), (3, 70001)])
def test_captured_and_replayed(R, V):
    """Two captured graphs of the whole set, replayed in turn with new inputs and eager calls between."""
    k = 20

    def inputs(seed):
        z = rows("plain", R, V, seed).to(DEV)
        p, q, x, u = (t.to(DEV) for t in drafts(8, 3, V, seed))
        return [z, z + 0.3 * rows("plain", R, V, seed + 50).to(DEV), p, q, x, u]

    def work(z, t, p, q, x, u):
        tv, ti, tail = lg().top_logits(t, k, with_tail=True)
        leaf = z.detach().requires_grad_(True)
        loss = lg().distill_loss(leaf, tv, ti, tail=tail, temperature=2.0)
        (g,) = torch.autograd.grad(loss, leaf)
        l2, g2 = lg().distill_loss_grad(z, tv, ti, tail=tail)
        tok, acc = lg().verify_draft(p, x, u, draft_probs=q)
        return [tv, ti, tail, loss.detach(), g, l2, g2, tok, acc]

    side = torch.cuda.Stream()
    graphs = []
    for s in (1, 2):
        held = inputs(s)
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            work(*held)
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = work(*held)
        graphs.append((graph, held, out))
    for i in range(6):
        graph, held, out = graphs[i % 2]
        new = inputs(10 + i)
        for h, n in zip(held, new):
            h.copy_(n)
        graph.replay()
        want = work(*new)
        torch.cuda.synchronize()
        for o, w in zip(out, want):
            assert torch.equal(o, w)


def test_refusals():
    z = torch.randn(4, 10, device=DEV)
    v, i = lg().top_logits(z, 3)
    u, x, p = torch.rand(4, 3, device=DEV), torch.zeros(4, 2, device=DEV, dtype=torch.int32), torch.rand(4, 3, 10, device=DEV)
    bad = [lambda: lg().top_logits(z, 0), lambda: lg().top_logits(z, 11), lambda: lg().top_logits(z.double(), 3), lambda: lg().top_logits(z.int(), 3),
           lambda: lg().top_logits(torch.randn(2, 300, device=DEV), 257), lambda: lg().top_logits(z, 3, temperature=0.0),
           lambda: lg().top_logits(z, 3, temperature=float("nan")), lambda: lg().top_logits(z, 3, temperature=float("inf")),
           lambda: lg().top_logits(z[:, :0], 1), lambda: lg().top_logits(z[0, 0], 1),
           lambda: lg().distill_loss(z, v, i.float()), lambda: lg().distill_loss(z, v[:3], i[:3]), lambda: lg().distill_loss(z, v[:, :2], i),
           lambda: lg().distill_loss(z, v, i, temperature=-1.0), lambda: lg().distill_loss(z, v, i, reduction="batchmean"),
           lambda: lg().distill_loss(z, v, i, tail=torch.zeros(3, device=DEV)), lambda: lg().distill_loss(z, v, i, weight=torch.ones(4, device=DEV).double()),
           lambda: lg().distill_loss(z, v[:, :0], i[:, :0]), lambda: lg().distill_loss(z, v.clone().requires_grad_(True), i),
           lambda: lg().distill_loss(z, v.double(), i), lambda: lg().distill_loss_grad(z, v, i, reduction="max"),
           lambda: lg().verify_draft(p, x.float(), u), lambda: lg().verify_draft(p, x, u[:, :2]), lambda: lg().verify_draft(p[:, :2], x, u),
           lambda: lg().verify_draft(p, x, u.double()), lambda: lg().verify_draft(p, x, u, draft_probs=p),
           lambda: lg().verify_draft(p, x, u, draft_probs=p[:, :2].half()), lambda: lg().verify_draft(p, x, u, lengths=torch.zeros(3, device=DEV, dtype=torch.int32)),
           lambda: lg().verify_draft(p.double(), x, u), lambda: lg().verify_draft(p[..., :0], x, u)]
    for n, f in enumerate(bad):
        with pytest.raises(ValueError):
            f()
            pytest.fail(f"call {n} was not refused")
    for f in (lambda: lg().top_logits(z.cpu(), 3), lambda: lg().distill_loss(z, v.cpu(), i), lambda: lg().distill_loss(z, v, i.cpu()),
              lambda: lg().verify_draft(p, x.cpu(), u), lambda: lg().verify_draft(p, x, u.cpu())):
        with pytest.raises(RuntimeError):
            f()
    leaf = z.clone().requires_grad_(True)
    (g,) = torch.autograd.grad(lg().distill_loss(leaf, v, i), leaf, create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()                                 # once, not twice
    loss = lg().distill_loss(leaf, v, i)
    v.add_(1.0)                                            # the teacher was overwritten before the backward
    with pytest.raises(RuntimeError):
        loss.backward()


def test_together_on_a_rollout():
    """A policy's rollout dumps its logits: it teaches a second one on its best ones, and checks nodes the second one drafts."""
    import gpu_common as gc
    from elg_amd import _lib as L
    from elg_amd import engine as eng
    from oracle import elg_oracle as orc
    fx, cfg, P, xy, dem, B, N, M = gc.cvrp_fixture("n50")
    acts = torch.from_numpy(fx["actions"].astype(np.int64))
    T = acts.shape[2]
    enc = orc.encoder_forward(P, cfg, xy, dem)
    prob = gc.make_problem(xy, dem, L.PROBLEM_CVRP)
    pol = gc.make_policy(P, cfg, enc.to(gc.DEV), L.PROBLEM_CVRP)
    other = gc.make_policy(P, cfg, (enc + 0.2 * torch.randn_like(enc)).to(gc.DEV), L.PROBLEM_CVRP)

    def dump(policy, what):
        return eng.rollout_forward(prob, policy, M, acts[0, :, 1], L.MODE_FORCED, forced=acts, dump_T=T, dump=what).full_probs

    # rows of steps that are not decoded (first moves, finished trajectories) are left zero by the rollout: weight 0
    teacher, student = dump(pol, "logits"), dump(other, "logits")
    tp, sp = dump(pol, "probs"), dump(other, "probs")
    decoded = (tp.sum(-1) > 0.5).float()
    assert 0 < decoded.mean() < 1
    values, idx, tail = lg().top_logits(teacher, cfg.local_size, with_tail=True)
    leaf = student.clone().requires_grad_(True)
    loss = lg().distill_loss(leaf, values, idx, tail=tail, weight=decoded, reduction="sum")
    (grad,) = torch.autograd.grad(loss, leaf)
    flat = lambda t: t.reshape(-1, *t.shape[3:]).cpu()  # noqa: E731
    rl, rg, lb, gb = ro.distill(flat(student).numpy(), flat(values).numpy(), flat(idx).numpy(), flat(tail).numpy(), 1.0, flat(decoded).numpy())
    assert abs(loss.item() - rl.sum()) <= lb.sum() + 2 * ro.U * abs(rl.sum())
    assert (np.abs(host(flat(grad)) - rg) <= gb + 4 * ro.U * np.abs(rg) + 1e-30).all()
    # a small step against the gradient lowers the sum by |grad|^2 per unit step, to first order
    step = 1e-3
    lower = lg().distill_loss(torch.where(torch.isfinite(student), student - step * grad, student), values, idx, tail=tail, weight=decoded, reduction="sum")
    drop = (loss - lower).item()
    assert drop == pytest.approx(step * grad.double().square().sum().item(), rel=0.05)
    # four nodes drafted from the second policy from step 6 on, checked against the first
    G, t0 = 4, 6
    x = acts[:, :, t0:t0 + G].to(gc.DEV)
    u = torch.rand(B, M, G + 1, generator=rng(3)).to(gc.DEV)
    tok, acc = lg().verify_draft(tp[:, :, t0:t0 + G + 1], x, u, draft_probs=sp[:, :, t0:t0 + G])
    rt, ra = ro.verify(host(tp[:, :, t0:t0 + G + 1]).reshape(-1, G + 1, N + 1), x.cpu().numpy().reshape(-1, G), host(u).reshape(-1, G + 1),
                       host(sp[:, :, t0:t0 + G]).reshape(-1, G, N + 1))
    np.testing.assert_array_equal(tok.cpu().numpy().reshape(rt.shape), rt)
    assert (tp[:, :, t0:t0 + G + 1].reshape(-1, G + 1, N + 1).cpu()[np.arange(len(ra)), ra, rt[np.arange(len(ra)), ra]] > 0).all()   # never a closed node
