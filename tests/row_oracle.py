"""The row operators over node logits from their definitions, in 64 bits on the host, with the f32 kernels' error bounds beside them.

U = 2^-24 is half a step of f32.  An exponential e^{-x} of a rounded product x' = x c (c rounded twice, the product once) is off by at
most 4 x U plus 2 U for v_exp itself; a sum of n positive terms in any order by n U.  With `n` the longest chain of additions the kernels
form (a thread's own elements, then the tree), every bound below is the first-order sum of these."""
import numpy as np

U = 2.0 ** -24
HALF_STEP = {"float32": 2.0 ** -24, "bfloat16": 2.0 ** -8, "float16": 2.0 ** -11}
TINY = {"float32": 2.0 ** -126, "bfloat16": 2.0 ** -126, "float16": 2.0 ** -24}     # f16 keeps subnormals: half of their step is 2^-25


def chain(V):
    """Additions on the longest path of a row's sum: at most V / 256 + 8 by one thread, 6 + 4 in the tree, a few joins."""
    return V / 256.0 + 32.0


def top(z, k):
    """(values, idx): larger first, equal ones by the lower index, NaN above +inf."""
    z = np.asarray(z, np.float64)
    key = np.where(np.isnan(z), np.inf, z) + 0.0
    nan_first = np.where(np.isnan(z), 0, 1)
    idx = np.stack([np.lexsort((np.arange(z.shape[1]), -key[r], nan_first[r]))[:k] for r in range(z.shape[0])])
    return np.take_along_axis(z, idx, 1), idx


def tail(z, idx, tau):
    """Mass outside idx and the bound on its f32 error."""
    z = np.asarray(z, np.float64)
    R, V = z.shape
    out, err = np.zeros(R), np.zeros(R)
    for r in range(R):
        m = z[r].max()
        if m == -np.inf:
            continue
        x = (m - z[r]) / tau
        e = np.exp(-x)
        slack = np.where(e > 0, e * (4 * np.where(np.isfinite(x), x, 0) + 2 + chain(V)) * U, 0)
        inside = np.zeros(V, bool)
        inside[idx[r]] = True
        S, rest = e.sum(), e[~inside].sum()
        out[r] = rest / S
        err[r] = slack[~inside].sum() / S + out[r] * (slack.sum() / S + 4 * U) + 2.0 ** -126
    return out, err


def distill(z, tv, ti, a, tau, w):
    """(loss, grad, loss bound, grad bound) per row; grad before any scale and cotangent."""
    z, tv = np.asarray(z, np.float64), np.asarray(tv, np.float64)
    R, V = z.shape
    loss, grad, lb, gb = np.zeros(R), np.zeros((R, V)), np.zeros(R), np.zeros((R, V))
    n = chain(V)
    for r in range(R):
        if w is not None and w[r] == 0:
            continue
        wr = 1.0 if w is None else float(w[r])
        ar = 0.0 if a is None else min(max(float(a[r]), 0.0), 1.0)
        ok = (ti[r] >= 0) & (ti[r] < V)
        i, t = ti[r][ok].astype(np.int64), tv[r][ok]
        m = z[r].max()
        if m == -np.inf or t.size == 0 or t.max() == -np.inf:
            continue
        y = (t.max() - t) / tau                                   # distance of a teacher entry from its best
        s = np.exp(-y)
        q = (1 - ar) * s / s.sum()
        x = (m - z[r]) / tau
        e = np.exp(-x)
        S = e.sum()
        p = e / S
        fx = np.where(np.isfinite(x), x, 0)
        top_set = np.zeros(V, bool)
        top_set[i] = True
        rest_max = z[r][~top_set].max() if (~top_set).any() else -np.inf
        live = q > 0
        logq = np.log(np.where(live, q, 1))
        with np.errstate(divide="ignore"):
            logp = -x[i] - np.log(S)
        term = np.where(live, q * (logq - np.where(live, logp, 0)), 0)
        L = term.sum()
        fy, fxi = np.where(np.isfinite(y), y, 0), fx[i]
        ok_t = live & np.isfinite(term)
        # q off by (4 y + n) U; the bracket (y' - x' + two logs of sums) by its own size and the sums' error
        b = (q * ((4 * fy + 2 * n) * (np.abs(np.where(ok_t, logq - np.where(live, logp, 0), 0))) + 4 * (fy + fxi) + 4 * n + 4 * np.abs(np.log(S))
                  + 4 * np.abs(np.log(s.sum())) + 8)).sum()
        g = p.copy()
        gbr = p * (8 * fx + 2 * n + 8)
        rest = (p * ~top_set).sum()
        if ar > 0:
            if rest > 0:
                xr = np.where(~top_set & np.isfinite(z[r]), (rest_max - z[r]) / tau, 0)
                er = np.where(~top_set, np.exp(-(np.where(np.isfinite(z[r]), (rest_max - z[r]) / tau, np.inf))), 0)
                Sr = er.sum()
                lrest = (rest_max - m) / tau + np.log(Sr) - np.log(S)
                L += ar * (np.log(ar) - lrest)
                b += ar * (4 * abs(np.log(ar)) + 4 * abs((rest_max - m) / tau) + 4 * np.log(Sr) + 4 * np.log(S) + 4 * n + 16)
                g = np.where(top_set, g, p - ar * er / Sr)
                gbr = gbr + np.where(top_set, 0, ar * er / Sr * (8 * xr + 2 * n + 8))
            else:
                L = np.inf
        np.subtract.at(g, i, q)
        np.add.at(gbr, i, q * (8 * fy + 2 * n + 8))
        loss[r], grad[r] = tau * tau * wr * L, tau * wr * g
        lb[r], gb[r] = tau * tau * abs(wr) * U * (b + 8 * abs(L) if np.isfinite(L) else 0), tau * abs(wr) * U * gbr
    return loss, grad, lb, gb


def verify(P, x, u, Q=None, lengths=None):
    P = np.asarray(P, np.float64)
    B, G1, V = P.shape
    G = G1 - 1
    out, acc = np.full((B, G1), -1, np.int64), np.zeros(B, np.int64)
    for b in range(B):
        n = G if lengths is None else int(min(max(lengths[b], 0), G))
        a = 0
        while a < n:
            t = int(x[b, a])
            if not 0 <= t < V:
                break
            q = 1.0 if Q is None else float(Q[b, a, t])
            if not float(u[b, a]) * q < P[b, a, t]:
                break
            a += 1
        own = np.where(P[b, a] > 0, P[b, a], 0)
        r = own
        if a < n:
            if Q is not None:
                d = P[b, a] - np.asarray(Q[b, a], np.float64)
                r = np.where(d > 0, d, 0)
            elif 0 <= int(x[b, a]) < V:
                r = own.copy()
                r[int(x[b, a])] = 0
            if r.sum() <= 0:
                r = own
        out[b, :a] = x[b, :a]
        c = np.cumsum(r)
        if c[-1] > 0:
            over = (c > float(u[b, G]) * c[-1]) & (r > 0)
            out[b, a] = int(np.argmax(over)) if over.any() else int(np.nonzero(r > 0)[0][-1])
        acc[b] = a
    return out, acc
