"""Plain numpy forms, in 64 bits and row by row, of the operators on a head's weights and logits."""
import numpy as np

NONE = 0xffffffff
U = 2.0 ** -24  # half a step of fp32
HALF_STEP = {"float32": 2.0 ** -24, "bfloat16": 2.0 ** -8, "float16": 2.0 ** -11}
TINY = {"float32": 2.0 ** -149, "bfloat16": 2.0 ** -133, "float16": 2.0 ** -24}  # the smallest number


def adds(vocab):
    """Roundings of one sum over a row in any order that a CTA of at least 128 threads and a tree may take."""
    return vocab / 128 + 40


def has_distribution(x):
    return not (np.isnan(x).any() or (x == np.inf).any())


def log_softmax(x, temperature):
    """(z, l) of z = (x - max) / T and l = ln sum exp z; (-inf, 0) for a row of -inf only."""
    m = x.max()
    if m == -np.inf:
        return np.full(x.shape, -np.inf), 0.0
    z = (x - m) / temperature
    return z, np.log(np.exp(z).sum())


def best(x, n):
    """The n largest by (value desc, id asc); -0 counts as +0."""
    return np.lexsort((np.arange(x.size), -(x + 0.0)))[:n]


def logprobs(x, target, temperature, top):
    """One row: dict of logprob, rank, entropy, stats, ids, top, and a bound of fp32 arithmetic's error of the three kinds of results."""
    v = x.size
    has, none = target < v, target == NONE
    if not has_distribution(x):
        return dict(logprob=0.0 if none else np.nan, rank=0, entropy=np.nan, stats=(np.nan, np.nan), ids=[NONE] * top, top=[np.nan] * top, tol=0.0,
                    tol_h=0.0)
    z, l = log_softmax(x, temperature)
    p = np.exp(z - l)
    live = p > 0
    mean = float((p[live] * -z[live]).sum())
    order = best(x, top)
    ids = list(order) + [NONE] * (top - len(order))
    lp = list(z[order] - l) + [-np.inf] * (top - len(order))
    # an argument's error is 3 roundings of z (difference, 1 / T, product), an exponential's 2 more, a sum's `adds`, the logarithm's and the
    # last difference's one each of their results
    tol = U * (3 * mean + 2 + adds(v) + 2 * abs(l))
    return dict(logprob=0.0 if none else (z[target] - l) if has else np.nan, rank=0 if not has else 1 + int((x > x[target]).sum()),
                entropy=l + mean, stats=(x.max(), l), ids=ids, top=lp, tol=tol,
                tol_h=tol + U * ((2 * adds(v) + 8) * mean + 2 * (l + mean)) + U * 3 * float((p[live] * z[live] ** 2).sum()))


def logprob_grad(x, target, temperature, stats, entropy, g_lp, g_h, dtype):
    """(gradient, bound of its error) of one row from the forward call's fp32 results."""
    v = x.size
    zero = np.zeros(v)
    g_lp = g_lp if target < v else 0.0
    if (g_lp == 0 and g_h == 0) or stats[0] == -np.inf:
        return zero, zero
    if np.isnan(stats[0]):
        return np.full(v, np.nan), zero
    z = (x - stats[0]) / temperature
    lp = z - stats[1]
    p = np.exp(lp)
    one = zero.copy()
    if target < v:
        one[target] = 1.0
    lp0 = np.where(p > 0, lp, 0.0)
    z0 = np.where(p > 0, z, 0.0)
    d = (g_lp * (one - p) - g_h * p * (lp0 + entropy)) / temperature
    rel_p = U * (3 * np.abs(z0) + 2 * np.abs(lp0) + 4)
    tol = (abs(g_lp) * (p * rel_p + 4 * U * np.abs(one - p)) + abs(g_h) * p * ((rel_p + 6 * U) * np.abs(lp0 + entropy) + rel_p + U * 4 * (np.abs(lp0) + entropy))) / temperature
    return d, tol + HALF_STEP[dtype] * np.abs(d) * 1.001 + TINY[dtype]


def distill(x, ids, teacher, temperature, t_temperature, rest, target, g_kl, g_ce, dtype):
    """One row: dict of kl, ce, grad and bounds of their errors."""
    v = x.size
    there = ids < v
    q = np.where(there, teacher / t_temperature, -np.inf)
    r = 0.0
    with np.errstate(all="ignore"):
        if rest:
            t, log_t = np.exp(q), q
            r = max(1.0 - t.sum(), 0.0) if there.any() else 0.0
        else:
            m = q.max()
            e = np.exp(q - m) if m > -np.inf else np.zeros(q.shape)
            t = e / e.sum() if e.sum() > 0 else e
            log_t = q - m - (np.log(e.sum()) if e.sum() > 0 else 0.0)
        has = target < v
        w_ce = g_ce if has else 0.0
        none = np.zeros(v)
        zero_grad = g_kl == 0 and w_ce == 0
        if not has_distribution(x):
            return dict(kl=np.nan, ce=0.0 if target == NONE else np.nan, grad=none if zero_grad else np.full(v, np.nan), tol=0.0, tol_ce=0.0, tol_g=none)
        z, l = log_softmax(x, temperature)
        z1, l1 = log_softmax(x, 1.0)
        empty = x.max() == -np.inf
        lp = z - l
        # ln p is held in fp32: the lowest fp32 logit at a temperature of 0.7 has -3.4028e38 / 0.7 = -4.9e38, beyond fp32's range, and so -inf
        lp = np.where(lp < -3.4028236e38, -np.inf, lp)
        p = np.exp(lp)
        listed = np.zeros(v, bool)
        listed[ids[there].astype(int)] = True
        t_at = np.zeros(v)
        np.add.at(t_at, ids[there].astype(int), t[there])
        terms = [ti * (lti - lp[int(i)]) for i, ti, lti in zip(ids, t, log_t) if i < v and ti > 0]
        kl = float(np.sum(terms)) if terms else 0.0
        lse_rest = np.logaddexp.reduce(lp[~listed]) if (~listed).any() else -np.inf
        if r > 0:
            kl += r * (np.log(r) - lse_rest)
        mass = t.sum() + r
        d = mass * p - t_at
        inside = np.where(listed | (lse_rest == -np.inf), 0.0, np.exp(lp - lse_rest) if lse_rest > -np.inf else 0.0)
        d = d - r * inside if rest else d
        ce = 0.0 if target == NONE else np.nan if not has else np.inf if empty else l1 - z1[target]
        d = g_kl * d / temperature
        if w_ce:
            e1 = np.exp(z1 - l1)
            e1[target] -= 1.0
            d = d + w_ce * e1
        if empty or zero_grad:
            d = none
        mean = float((p * -np.where(p > 0, z, 0.0)).sum()) if not empty else 0.0
        base = U * (3 * mean + 6 + adds(v) + 2 * abs(l))  # of ln sum exp, absolute; of a probability's normaliser, relative
        span = sum(ti * (abs(lti) + abs(lp[int(i)])) for i, ti, lti in zip(ids, t, log_t) if i < v and ti > 0 and lp[int(i)] > -np.inf)
        q_span = float(np.abs(q[there & (q > -np.inf)]).max()) if (there & (q > -np.inf)).any() else 0.0
        rel_t = U * (6 * q_span + 300)  # softmax or exp of the entries, and sums of up to 256 of them
        finite_rest = abs(lse_rest) if np.isfinite(lse_rest) else 0.0
        tol = (mass + 1) * base + (rel_t + 8 * U) * (span + 1) + (U * 8 + base) * r * (finite_rest + abs(np.log(r)) + 1 if r > 0 else 0)
        rel_p = U * (3 * np.abs(np.where(p > 0, z, 0.0)) + 8) + 2 * base
        # r is a difference of numbers near 1: its error is of their size
        tol_g = abs(g_kl) / temperature * (p * mass * rel_p + t_at * (rel_t + 8 * U) + inside * (r * rel_p + rel_t + 4 * U)) + abs(w_ce) * (np.exp(z1 - l1) * 1.0 + (np.arange(v) == target)) * (
            U * (3 * np.abs(np.where(np.isfinite(z1), z1, 0.0)) + 10 + adds(v)))
        tol_g = np.where(np.isfinite(tol_g), tol_g, 0.0) + HALF_STEP[dtype] * np.abs(d) * 1.001 + TINY[dtype]
        tol_ce = 0.0 if not has or empty else U * (3 * float((np.exp(z1 - l1) * -np.where(np.isfinite(z1), z1, 0.0)).sum()) + 3 * abs(z1[target] if np.isfinite(z1[target]) else 0.0) + 6 + adds(v) + 2 * abs(l1))
        return dict(kl=kl, ce=ce, grad=d, tol=tol, tol_ce=tol_ce, tol_g=tol_g)


def quantize(w, group, zeros, scale_dtype):
    """(codes [n, k], scales, zeros) of an fp32 matrix; the same fp32 operations in the same order."""
    import torch
    n, k = w.shape
    groups = -(-k // group)
    codes, scales, zs = np.zeros((n, k), np.uint8), torch.zeros(n, groups, dtype=getattr(torch, scale_dtype)), np.zeros((n, groups), np.uint8)
    top = torch.finfo(scales.dtype).max
    for i in range(n):
        for g in range(groups):
            a = w[i, g * group:(g + 1) * group].astype(np.float32)
            with np.errstate(all="ignore"):
                lo, hi = np.float32(min(a.min(), 0.0)), np.float32(max(a.max(), 0.0))
                step = np.float32(hi - lo) / np.float32(15) if zeros else np.float32(max(hi, -lo)) / np.float32(7)
            step = np.float32(min(step, np.float32(top)))
            if not np.isfinite(a).all():
                step = np.float32(np.nan)
            s = torch.tensor(step).to(scales.dtype)
            scales[i, g] = s
            step = np.float32(s.float().item())
            zero = 8.0
            if zeros:
                zero = float(np.clip(np.rint(-lo / step), 0, 15)) if step > 0 else 0.0
                zs[i, g] = int(zero)
            codes[i, g * group:(g + 1) * group] = np.clip(np.rint(a / step) + np.float32(zero), 0, 15) if step > 0 else int(zero)
    return codes, scales, zs if zeros else None


def pack(codes):
    return (codes[:, ::2] | (codes[:, 1::2] << 4)).astype(np.uint8)


def dequantize(codes, scales, zeros, group):
    """The matrix in 64 bits."""
    at = np.arange(codes.shape[1]) // group
    zero = 8.0 if zeros is None else zeros.astype(np.float64)[:, at]
    return (codes.astype(np.float64) - zero) * scales.double().numpy()[:, at]
