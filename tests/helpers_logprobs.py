"""Float64 references of the log-probability and distillation operators, and what a float evaluation of them may be off.

Error model (u = 2^-24, half a step of float32).  With x_c = (z_c - m) log2(e) / T an exponent carries at most 3 u |x_c|
(subtraction, product, the rounded constant), its power two half steps on top, and a sum over n classes at most
n / 64 + 16 half steps (64 or more partial sums, then a tree): the sum's relative error is
    kappa = u (16 + n / 64 + 4 E1),   E1 = sum p |x|   (3 ln 2 rounded up).
log p adds 4 u |log p|; the entropy's second term weighs every exponent once more, 4 u E2 with E2 = sum p x^2.  A stored
bf16 gradient is off by another half step, 2^-8 of its value."""
import numpy as np

U = 2.0 ** -24
HALF_STEP = {"f32": 2.0 ** -24, "bf16": 2.0 ** -8}


def softmax(z, T):
    """(log p, p, empty rows) of float64 rows; a row without any probability has log p = -inf, p = 0."""
    with np.errstate(all="ignore"):
        m = z.max(axis=1, keepdims=True)
        empty = (m == -np.inf)[:, 0]
        m = np.where(m == -np.inf, 0.0, m)
        d = (z - m) / T
        e = np.exp(d)
        s = e.sum(axis=1, keepdims=True)
        logp = np.where(empty[:, None], -np.inf, d - np.log(s))
        logp = np.where(logp < -np.finfo(np.float32).max, -np.inf, logp)  # (no float holds it)
        p = np.where(empty[:, None], 0.0, e / s)
    return logp, p, empty


def entropy(logp, p):
    with np.errstate(all="ignore"):
        return -np.where(p > 0, p * logp, 0.0).sum(axis=1)


def spread(z, T, p):
    """(E1, E2) of the error model."""
    with np.errstate(all="ignore"):
        m = z.max(axis=1, keepdims=True)
        x = np.where(p > 0, (z - np.where(np.isfinite(m), m, 0.0)) / T * np.log2(np.e), 0.0)
    return (p * np.abs(x)).sum(axis=1), (p * x * x).sum(axis=1)


def kappa(z, T, p):
    return U * (16 + z.shape[1] / 64 + 4 * spread(z, T, p)[0])


def token_logprobs(z, T, tokens=None, top=0):
    """dict of logprobs, entropy, top_logprobs, top_classes and the bounds of their errors ("logprobs_tol" ...)."""
    logp, p, _ = softmax(z, T)
    k = kappa(z, T, p)
    out = {"entropy": entropy(logp, p)}
    out["entropy_tol"] = k * (1 + out["entropy"]) + 4 * U * (spread(z, T, p)[1] + out["entropy"])
    n = np.arange(z.shape[0])
    tol = lambda lp: k.reshape([-1] + [1] * (lp.ndim - 1)) + 4 * U * np.where(np.isfinite(lp), np.abs(lp), 0.0)
    if tokens is not None:
        inside = (tokens >= 0) & (tokens < z.shape[1])
        out["logprobs"] = np.where(inside, logp[n, np.where(inside, tokens, 0)], np.nan)
        out["logprobs_tol"] = tol(out["logprobs"])
    if top:
        out["top_classes"] = np.argsort(-z, axis=1, kind="stable")[:, :top]
        out["top_logprobs"] = np.take_along_axis(logp, out["top_classes"], axis=1)
        out["top_logprobs_tol"] = tol(out["top_logprobs"])
    return out


def token_logprobs_grad(z, T, tokens, top_classes, g_logp, g_ent, g_top, dtype):
    """(gradient of the logits, bound of its error); any of the three incoming gradients may be None."""
    logp, p, empty = softmax(z, T)
    H = entropy(logp, p)
    rows = z.shape[0]
    n = np.arange(rows)
    lp = np.where(p > 0, logp, 0.0)
    g = np.zeros([rows])
    own = np.zeros_like(z)
    if g_logp is not None:
        g += g_logp
        ok = (tokens >= 0) & (tokens < z.shape[1])  # (a row whose token it does not have is the caller's to check)
        np.add.at(own, (n[ok], tokens[ok]), g_logp[ok])
    if g_top is not None:
        g += g_top.sum(axis=1)
        for j in range(g_top.shape[1]):
            np.add.at(own, (n, top_classes[:, j]), g_top[:, j])
    gh = np.zeros([rows]) if g_ent is None else g_ent
    dz = (own - p * (g[:, None] + gh[:, None] * (lp + H[:, None]))) / T
    k = kappa(z, T, p)[:, None] + 4 * U * np.abs(lp)
    sum_g = np.abs(g) if g_top is None else np.abs(g_top).sum(axis=1) + (0 if g_logp is None else np.abs(g_logp))
    inner = sum_g[:, None] + np.abs(gh)[:, None] * (np.abs(lp) + H[:, None])
    err_h = token_logprobs(z, T)["entropy_tol"][:, None] + k
    # (an exponential below the smallest normal float comes out as 0: 2^-126 of p, times what p is multiplied by)
    bound = (p * (inner * (k + 8 * U) + np.abs(gh)[:, None] * err_h) + 2.0 ** -126 * inner + 4 * U * np.abs(own)) / T
    dz[empty], bound[empty] = 0.0, 0.0
    return dz, bound + HALF_STEP[dtype] * np.abs(dz) + 1e-37


def teacher(values, classes, T, tail):
    """(log q, q, q_rest) of the entries; a negative class is none."""
    entry = classes >= 0
    with np.errstate(all="ignore"):
        if tail:
            logq = np.where(entry, values, -np.inf)
        else:
            v = np.where(entry, values, -np.inf) / T
            m = v.max(axis=1, keepdims=True)
            none = m == -np.inf
            v = v - np.where(none, 0.0, m)
            logq = np.where(none, -np.inf, v - np.log(np.exp(v).sum(axis=1, keepdims=True)))
        q = np.exp(logq)
    rest = np.maximum(0.0, 1.0 - q.sum(axis=1)) if tail else np.zeros([values.shape[0]])
    return logq, q, rest


def distill(z, values, classes, T, tail, g=None, dtype="f32"):
    """dict of loss, its bound and, with the gradient ``g`` of the rows, dlogits and its bound."""
    logp, p, empty = softmax(z, T)
    logq, q, rest = teacher(values, classes, T, tail)
    rows, n = z.shape
    k_entries = values.shape[1]
    r = np.arange(rows)
    at = np.where((classes >= 0) & (classes < n), classes, 0)
    bad = (classes >= n).any(axis=1)
    kap = kappa(z, T, p)
    with np.errstate(all="ignore"):
        chosen = np.take_along_axis(logp, at, axis=1)
        loss = np.where(q > 0, q * (logq - chosen), 0.0).sum(axis=1)
        mag = np.where(q > 0, q * (np.abs(logq) + np.where(np.isfinite(chosen), np.abs(chosen), 0.0)), 0.0).sum(axis=1)
        # the entries' own sums: k / 64 partial sums each, exponents off by 4 u |log q|
        tol = (kap + U * (16 + k_entries / 64)) * (q.sum(axis=1) + 1) + 8 * U * mag
        inside = np.zeros_like(z, dtype=bool)
        for j in range(k_entries):
            inside[r[classes[:, j] >= 0], at[classes[:, j] >= 0, j]] = True
        x = np.where(inside, -np.inf, z)
        among_logp, among, none = softmax(x, T)
        finite_m = np.where(np.isfinite(z.max(axis=1)), z.max(axis=1), 0.0)
        log_mass = np.where(none, -np.inf, np.log(np.exp((x - finite_m[:, None]) / T).sum(axis=1)) -
                            np.log(np.exp((z - finite_m[:, None]) / T).sum(axis=1)))
        # (a mass too small for the difference above in 64 bits does not occur in the tests)
        d_rest = U * (8 + k_entries / 64 + 4 * np.where(q > 0, q * np.abs(logq), 0.0).sum(axis=1))
        rest = np.where(none & (rest <= 1e-5), 0.0, rest)  # (rounding's leftovers where no class is left for them)
        if tail:
            term = np.where(rest > 0, rest * (np.log(rest) - log_mass), 0.0)
            loss = loss + term
            fin = np.where(np.isfinite(log_mass), np.abs(log_mass), 0.0)
            kap_r = kappa(x, T, among)
            tol = tol + d_rest * (2 + np.abs(np.log(np.maximum(rest, d_rest))) + fin) + rest * (kap + kap_r + 8 * U * fin)
        else:
            kap_r = kap * 0
    loss = np.where(bad, np.nan, loss)
    out = {"loss": loss, "loss_tol": tol}
    if g is None:
        return out
    total = q.sum(axis=1) + rest
    target = np.zeros_like(z)
    qerr = np.zeros_like(z)
    with np.errstate(all="ignore"):
        for j in range(k_entries):
            ok = classes[:, j] >= 0
            np.add.at(target, (r[ok], at[ok, j]), q[ok, j])
            np.add.at(qerr, (r[ok], at[ok, j]),
                      q[ok, j] * U * (24 + k_entries / 64 + 8 * np.where(q[ok, j] > 0, np.abs(logq[ok, j]), 0.0)))
        lp = np.where(p > 0, np.abs(logp), 0.0)
        perr = p * (kap[:, None] + 4 * U * lp + 8 * U) * np.maximum(total, 1)[:, None] + p * d_rest[:, None]
        if tail:
            lr = np.where(among > 0, np.abs(among_logp), 0.0)
            target = target + among * rest[:, None]
            perr = perr + np.where(inside, 0.0, among * (d_rest + rest * (kap + kap_r + 8 * U))[:, None] +
                                   among * rest[:, None] * 4 * U * lr + p * (kap_r[:, None] + 4 * U * lr))
    dz = (p * total[:, None] - target) * (g / T)[:, None]
    # (exponentials below the smallest normal float come out as 0, as in the gradient above)
    bound = (perr + qerr + 2.0 ** -126 * np.maximum(total, 1)[:, None]) * np.abs(g / T)[:, None]
    dz[empty], bound[empty] = 0.0, 0.0
    dz[bad] = np.nan
    out["dlogits"], out["dlogits_tol"] = dz, bound + (HALF_STEP[dtype] + 4 * U) * np.abs(np.nan_to_num(dz)) + 1e-37
    return out


def close(got, want, tol):
    """Whether got is within tol of want, infinities and NaN in the same places; the message says where it is not."""
    got = np.asarray(got, np.float64)
    special = ~np.isfinite(want)
    same = np.where(special, (got == want) | (np.isnan(got) & np.isnan(want)), True)
    assert same.all(), "special values differ at %s" % (np.argwhere(~same)[:5].tolist(),)
    err = np.where(special, 0.0, np.abs(np.where(special, 0.0, got) - np.where(special, 0.0, want)))
    ratio = err / np.broadcast_to(tol, err.shape)
    worst = np.unravel_index(np.argmax(np.nan_to_num(ratio, nan=np.inf)), ratio.shape) if ratio.size else None
    assert ratio.size == 0 or ratio[worst] <= 1, "%s: got %.9g, want %.9g, bound %.3g" % (
        worst, got[worst], want[worst], np.broadcast_to(tol, err.shape)[worst])
