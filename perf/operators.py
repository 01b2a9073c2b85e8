"""What the row operators over node logits cost: the k best logits of a row, the distillation loss on a teacher's best logits with its
gradient, and the verification of drafted choices.  `own = False` computes each in plain torch; `own = True` calls elg_amd.logits."""
import math

import torch

own = False

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
BYTES = {"f32": 4, "bf16": 2, "f16": 2}


def listed():
    return [
        # one decode step of one instance's POMO trajectories at CVRP-100 (100 rows of 101 nodes): a launch's latency
        dict(name="top_step", op="top", R=100, V=101, k=20, type="f32", tau=1.0, tail=False, closed=0.5),
        # a teacher's whole CVRP-100 training rollout, 64 instances x 100 trajectories x 140 steps; k = local_size = 40
        dict(name="top_rollout", op="top", R=896000, V=101, k=40, type="f32", tau=1.0, tail=True, closed=0.5),
        # one step of 8 augmented 1000-customer instances x 1000 trajectories, at the largest local_size
        dict(name="top_large", op="top", R=8000, V=1001, k=63, type="f16", tau=2.0, tail=True, closed=0.3),
        # long rows: a generic vocabulary, few rows of it per compute unit
        dict(name="top_vocab", op="top", R=512, V=131072, k=128, type="bf16", tau=2.0, tail=True, closed=0.0),
        # the loss of one decode step, forward and backward through autograd: latency
        dict(name="distill_step", op="distill", R=100, V=101, k=20, type="f32", tau=1.0, tail=False, closed=0.5, live=1.0, way="mean"),
        # the loss and its gradient in one call over a whole CVRP-100 training rollout, finished trajectories weighted 0
        dict(name="distill_rollout", op="distill", R=896000, V=101, k=40, type="f32", tau=1.0, tail=True, closed=0.5, live=0.85, way="one_call"),
        # forward and backward with one cotangent per row, half precision, ragged masks
        dict(name="distill_large", op="distill", R=8000, V=1001, k=63, type="f16", tau=2.0, tail=True, closed=0.3, live=1.0, way="rows"),
        # long rows, many of them
        dict(name="distill_vocab", op="distill", R=2048, V=131072, k=64, type="bf16", tau=2.0, tail=True, closed=0.0, live=1.0, way="one_call"),
        # a handful of long rows of odd length: fewer rows than compute units
        dict(name="distill_few", op="distill", R=6, V=100003, k=50, type="f32", tau=1.0, tail=True, closed=0.0, live=1.0, way="mean"),
        # the drafts of one instance's 100 trajectories at CVRP-100: latency
        dict(name="verify_step", op="verify", B=100, G=4, V=101, type="f32", closed=0.5, ragged=False),
        # a batch of 64 instances x 100 trajectories, drafts of different lengths
        dict(name="verify_batch", op="verify", B=6400, G=8, V=101, type="f32", closed=0.5, ragged=True),
        # a few sequences over a long vocabulary
        dict(name="verify_vocab", op="verify", B=48, G=5, V=131072, type="bf16", closed=0.0, ragged=True),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["top", "distill", "distill", "verify"])
    kind = rng.choice(["f32", "f32", "bf16", "f16"])
    closed = rng.choice([0.0, 0.3, 0.5, 0.9])
    if op == "verify":
        V = _log_int(rng, 2, 131072)
        G = rng.randint(1, 10)
        B = _log_int(rng, 1, max(1, min(20000, 30000000 // (V * (G + 1)))))
        return dict(op=op, B=B, G=G, V=V, type=kind, closed=closed, ragged=rng.random() < 0.5)
    V = _log_int(rng, 2, 131072)
    R = _log_int(rng, 1, max(1, min(800000, 60000000 // V)))
    c = dict(op=op, R=R, V=V, k=min(V, _log_int(rng, 1, 128)), type=kind, tau=rng.choice([1.0, 2.0, 0.7]), tail=rng.random() < 0.6, closed=closed)
    if op == "distill":
        c.update(live=rng.choice([1.0, 0.8]), way=rng.choice(["mean", "rows", "one_call"]))
    return c


def _logits(R, V, closed, g):
    """Rows as the decoder makes them: clipped at +-50, a part of the nodes closed (more of them in later steps), the first one open."""
    z = torch.randn(R, V, device="cuda", generator=g).mul_(0.12).tanh_().mul_(50.0)
    if closed:
        share = torch.rand(R, 1, device="cuda", generator=g).mul_(2 * closed).clamp_(max=1.0)
        shut = torch.rand(R, V, device="cuda", generator=g) < share
        shut[:, 0] = False
        z.masked_fill_(shut, -math.inf)
    return z


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    kind = TYPES[case["type"]]
    V = case["V"]
    if case["op"] == "verify":
        B, G = case["B"], case["G"]
        z = _logits(B * (G + 1), V, case["closed"], g).view(B, G + 1, V)
        target = torch.softmax(z * 0.5, -1)
        noisy = z[:, :G] * 0.5 + torch.randn(B, G, V, device="cuda", generator=g) * 0.7
        draft = torch.softmax(noisy, -1)
        at = torch.rand(B, G, 1, device="cuda", generator=g, dtype=torch.float64)
        sums = draft.double().cumsum(-1)
        tokens = (sums <= at * sums[..., -1:]).sum(-1).clamp_(max=V - 1).to(torch.int32)
        lengths = torch.randint(0, G + 1, (B,), device="cuda", generator=g, dtype=torch.int32) if case["ragged"] else None
        return dict(case=case, target=target.to(kind), draft=draft.to(kind), tokens=tokens, lengths=lengths, u=torch.rand(B, G + 1, device="cuda", generator=g))
    R, k = case["R"], case["k"]
    z = _logits(R, V, case["closed"], g)
    if case["op"] == "top":
        return dict(case=case, z=z.to(kind))
    # the teacher is near the student and sees the same closed nodes
    teacher = z.add(torch.randn(R, V, device="cuda", generator=g))
    values, idx = teacher.topk(k, dim=-1)
    tail = None
    if case["tail"]:
        e = torch.exp((teacher - values[:, :1]) / case["tau"])
        total = e.sum(-1)
        tail = e.scatter_(1, idx, 0.0).sum(-1).div_(total)
        del e
    del teacher
    state = dict(case=case, z=z.to(kind), values=values.to(kind), idx=idx.to(torch.int32), tail=tail, weight=None, cot=None)
    if case["live"] < 1.0:
        state["weight"] = torch.rand(R, device="cuda", generator=g).add_(0.5) * (torch.rand(R, device="cuda", generator=g) < case["live"])
    if case["way"] == "rows":
        state["cot"] = torch.randn(R, device="cuda", generator=g)
    if case["way"] != "one_call":
        state["z"].requires_grad_(True)
    return state


def _top_plain(z, k, tau, with_tail):
    """Order: larger first, equal ones by the lower index.  One 64-bit key per element carries both."""
    R, V = z.shape
    f = z.float() + 0.0
    b = f.view(torch.int32).long()
    key = torch.where(b < 0, -1 - (b & 0x7FFFFFFF), b)
    key = key * (1 << 21) + (V - 1 - torch.arange(V, device=z.device))
    idx = V - 1 - (key.topk(k, dim=-1).values & ((1 << 21) - 1))
    out = dict(values=z.gather(1, idx), idx=idx.to(torch.int32))
    if with_tail:
        m = f.gather(1, idx[:, :1])
        e = torch.exp((f - torch.where(m == -math.inf, torch.zeros_like(m), m)) / tau)
        total = e.sum(-1)
        rest = e.scatter(1, idx, 0.0).sum(-1)
        out["tail"] = torch.where(total > 0, rest / total, torch.zeros_like(total))
    return out


def _distill_plain(s, kind):
    """Losses of the rows and d(sum of the losses)/d(logits), every step in `kind`."""
    c, tau = s["case"], s["case"]["tau"]
    z, t = s["z"].detach().to(kind), s["values"].to(kind)
    idx = s["idx"].long()
    zero = torch.zeros((), device=z.device, dtype=kind)
    a = s["tail"].to(kind) if s["tail"] is not None else torch.zeros(z.shape[0], device=z.device, dtype=kind)
    m = z.amax(-1, keepdim=True)
    m = torch.where(m == -math.inf, zero, m)
    e = torch.exp((z - m) / tau)
    total = e.sum(-1, keepdim=True)
    tm = t.amax(-1, keepdim=True)
    tm = torch.where(tm == -math.inf, zero, tm)
    et = torch.exp((t - tm) / tau)
    st = et.sum(-1, keepdim=True)
    live = (total > 0) & (st > 0)
    q = torch.where(live, (1 - a[:, None]) * et / st, zero)
    logq = torch.log1p(-a[:, None]) + (t - tm) / tau - torch.log(st)
    logp = (z.gather(1, idx) - m) / tau - torch.log(total)
    loss = torch.where(q > 0, q * (logq - logp), zero).sum(-1)
    rest = e.scatter(1, idx, 0.0)
    rest_sum = rest.sum(-1, keepdim=True)
    p = e / total
    del e
    if s["tail"] is not None:
        prest = rest_sum / total
        loss = loss + torch.where(a > 0, a * (torch.log(a) - torch.log(prest[:, 0])), zero)
        g = p.sub_(torch.where(rest_sum > 0, a[:, None] / rest_sum, zero) * rest)
    else:
        g = p
    del rest
    g.scatter_add_(1, idx, -q)
    w = tau * (s["weight"].to(kind) if s["weight"] is not None else torch.ones(z.shape[0], device=z.device, dtype=kind))
    on = live[:, 0] & (w != 0)
    loss = torch.where(on, tau * w * loss, zero)
    g = torch.where(on[:, None], g.mul_(w[:, None]), zero)
    if c["way"] == "rows":
        return loss, g.mul_(s["cot"].to(kind)[:, None])
    return loss.mean(), g.div_(z.shape[0])


def _verify_plain(s):
    P, u = s["target"], s["u"].double()
    Q, x = s["draft"], s["tokens"].long()
    B, G = x.shape
    px = P[:, :G].gather(2, x[..., None])[..., 0].double()
    qx = Q.gather(2, x[..., None])[..., 0].double()
    n = s["lengths"].long() if s["lengths"] is not None else torch.full((B,), G, device=x.device)
    step = torch.arange(G + 1, device=x.device)
    ok = (u[:, :G] * qx < px) & (step[:G] < n[:, None])
    a = ok.to(torch.int64).cumprod(-1).sum(-1)
    row = torch.arange(B, device=x.device)
    p = P[row, a].double()
    q = Q[row, a.clamp(max=G - 1)].double()
    r = torch.where((a < n)[:, None], (p - q).clamp(min=0.0), p)
    r = torch.where(r.sum(-1, keepdim=True) > 0, r, p)
    sums = r.cumsum(-1)
    drawn = (sums <= u[:, G:] * sums[:, -1:]).sum(-1).clamp(max=P.shape[2] - 1)
    drawn = torch.where(sums[:, -1] > 0, drawn, torch.full_like(drawn, -1))
    out = torch.where(step < a[:, None], torch.cat([x, x[:, :1]], 1), torch.full_like(step, -1))
    out = torch.where(step == a[:, None], drawn[:, None], out)
    return dict(tokens=out.to(torch.int32), accepted=a.to(torch.int32))


def _run_own(s):
    from elg_amd import logits as lg

    c = s["case"]
    if c["op"] == "top":
        got = lg.top_logits(s["z"], c["k"], temperature=c["tau"], with_tail=c["tail"])
        return dict(zip(("values", "idx", "tail"), got))
    if c["op"] == "verify":
        tokens, accepted = lg.verify_draft(s["target"], s["tokens"], s["u"], draft_probs=s["draft"], lengths=s["lengths"])
        return dict(tokens=tokens, accepted=accepted)
    more = dict(tail=s["tail"], temperature=c["tau"], weight=s["weight"])
    if c["way"] == "one_call":
        loss, grad = lg.distill_loss_grad(s["z"], s["values"], s["idx"], **more)
        return dict(loss=loss, grad=grad)
    loss = lg.distill_loss(s["z"], s["values"], s["idx"], reduction="none" if c["way"] == "rows" else "mean", **more)
    (grad,) = torch.autograd.grad(loss, s["z"], s["cot"])
    return dict(loss=loss.detach(), grad=grad)


def run(state):
    if own:
        return _run_own(state)
    c = state["case"]
    if c["op"] == "top":
        return _top_plain(state["z"], c["k"], c["tau"], c["tail"])
    if c["op"] == "verify":
        return _verify_plain(state)
    loss, grad = _distill_plain(state, torch.float32)
    return dict(loss=loss, grad=grad.to(state["z"].dtype))


def exact(case, seed):
    """The definitions row by row in 64 bits: p and q as whole distributions, the loss as the divergence between the two when the nodes
    outside the teacher's best are one class."""
    if case["op"] == "verify":
        return None
    s = prepare(case, seed)
    tau, R = case["tau"], case["R"]
    step = max(1, 40000000 // case["V"])
    losses, grads, values, tails = [], [], [], []
    for r in range(0, R, step):
        z = s["z"].detach()[r:r + step].double()
        logp = torch.log_softmax(z / tau, -1)
        if case["op"] == "top":
            top = torch.sort(z, dim=-1, descending=True).values
            values.append(top[:, :case["k"]].clone())
            if case["tail"]:
                p = torch.softmax(top / tau, -1)
                tails.append(p[:, case["k"]:].sum(-1))
            continue
        i = s["idx"][r:r + step].long()
        a = s["tail"][r:r + step].double() if case["tail"] else torch.zeros(len(z), device=z.device, dtype=torch.float64)
        q = torch.softmax(s["values"][r:r + step].double() / tau, -1) * (1 - a)[:, None]
        inner = torch.xlogy(q, q) - torch.where(q > 0, q * logp.gather(1, i), 0.0)
        rest = logp.scatter(1, i, -math.inf)
        loss = inner.sum(-1)
        p = logp.exp()
        if case["tail"]:
            lrest = torch.logsumexp(rest, -1)
            loss = loss + torch.where(a > 0, torch.xlogy(a, a) - a * lrest, 0.0)
            within = torch.where(lrest[:, None] > -math.inf, (rest - lrest[:, None]).exp(), 0.0)
            p = p - a[:, None] * within
        g = p.scatter_add(1, i, -q)
        w = s["weight"][r:r + step].double() if s["weight"] is not None else torch.ones(len(z), device=z.device, dtype=torch.float64)
        losses.append(torch.where(w != 0, tau * tau * w * loss, 0.0))
        scale = tau * w * (s["cot"][r:r + step].double() if case["way"] == "rows" else 1.0 / R)
        grads.append(torch.where(w[:, None] != 0, scale[:, None] * g, 0.0))
    if case["op"] == "top":
        out = dict(values=torch.cat(values), idx=None)
        return dict(out, tail=torch.cat(tails)) if case["tail"] else out
    loss = torch.cat(losses)
    return dict(loss=loss if case["way"] == "rows" else loss.sum() / R, grad=torch.cat(grads))


def work(case):
    b = BYTES[case["type"]]
    V = case["V"]
    if case["op"] == "verify":
        B, G = case["B"], case["G"]
        # the drawn row of the target and, where a draft was refused, of the draft; one probability of each per drafted token
        return {"bytes": B * (2 * V * b + G * (2 * b + 8) + 4 + 4 * (G + 2)), "flops": B * (4 * V + 3 * G)}
    R, k = case["R"], case["k"]
    if case["op"] == "top":
        return {"bytes": R * (V * b + k * (b + 4) + (4 if case["tail"] else 0)), "flops": R * V * (4 if case["tail"] else 1)}
    live = case["live"]
    rows = R * (V * b * (1 + live) + k * (b + 4) * live + (4 if case["tail"] else 0) + (4 if live < 1.0 else 0))
    return {"bytes": rows + (8 * R if case["way"] == "rows" else 4), "flops": R * live * V * 8}
