"""What is timed of the operators on a head's weights and its logits: products with 4-bit weights, log probabilities of given tokens
and their gradient, and distillation from a teacher's top logits.

A case is a dict of plain values. `op` says which call it is:

  logprobs  the log probability, rank and entropy of every row's target, and the `top` best alternatives
  grad      the gradient of those log probabilities and entropies with respect to the logits
  distill   divergence from a teacher's `k` best ids (`rest`: with the mass of all other ids; `ce`: with a target's cross entropy),
            and its gradient with respect to the logits, in one call
  gemv      `rows` vectors times a matrix [n, k] held as 4-bit codes with a scale for each `group` of weights (`zeros`: and a zero)
  quantize  a matrix into that form

`type` is the type of the logits, or of the vectors and the result (of the matrix, for quantize); `scale` that of the group scales.
Vocabularies and widths are those of the small, mid and base models of `cases.py` and round or odd ones around them.
"""
import math

import torch

own = False

NONE = -1  # as an int32: the id that stands for no token
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SIZE = {"f32": 4, "bf16": 2, "f16": 2}


def listed():
    return [
        # a chat step of the base model: the chosen token's log probability and 20 alternatives to show beside it
        dict(name="logprobs_chat", op="logprobs", rows=1, vocab=16384, top=20, temperature=1.0, type="f32"),
        # one decode step of 256 streams, sampled at a temperature, five alternatives each
        dict(name="logprobs_decode", op="logprobs", rows=256, vocab=16384, top=5, temperature=0.7, type="f32"),
        # scoring long texts under a model with a large vocabulary; no alternatives
        dict(name="logprobs_score", op="logprobs", rows=4096, vocab=131072, top=0, temperature=1.0, type="bf16"),
        # a policy step on short answers of the mid model, whose vocabulary is odd: no row but the first starts aligned
        dict(name="grad_odd", op="grad", rows=700, vocab=5003, temperature=1.0, type="f32", entropy=True),
        # a policy step on a long batch with a large vocabulary
        dict(name="grad_large", op="grad", rows=4096, vocab=65536, temperature=0.9, type="bf16", entropy=True),
        # distilling the base model from 32 stored alternatives of each token
        dict(name="distill_base", op="distill", rows=2048, vocab=16384, k=32, temperature=2.0, rest=False, ce=True, type="f32"),
        # the same for a large vocabulary, with the mass that the teacher gave to all other ids
        dict(name="distill_large", op="distill", rows=2048, vocab=131072, k=64, temperature=1.0, rest=True, ce=False, type="bf16"),
        # the head of the base model for one stream
        dict(name="gemv_head", op="gemv", rows=1, n=16384, k=768, group=64, zeros=False, type="f32", scale="f32"),
        # a wide layer for one stream: nothing but the codes' way from memory
        dict(name="gemv_wide", op="gemv", rows=1, n=32768, k=8192, group=128, zeros=False, type="bf16", scale="bf16"),
        # a layer for a batch of streams, codes with zeros as other tools write them
        dict(name="gemv_batch", op="gemv", rows=48, n=16384, k=4096, group=128, zeros=True, type="f16", scale="f16"),
        # the head of the base model into 4 bits
        dict(name="quantize_head", op="quantize", n=16384, k=768, group=64, zeros=False, type="f32", scale="f32"),
        # a wide layer into 4 bits
        dict(name="quantize_wide", op="quantize", n=16384, k=8192, group=128, zeros=True, type="bf16", scale="f16"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("logprobs", "logprobs", "grad", "distill", "gemv", "gemv", "quantize"))
    t = rng.choice(("f32", "bf16", "f16"))
    if op in ("logprobs", "grad", "distill"):
        vocab = rng.choice((8192, 16384, 5003, _log(rng, 300, 200000)))
        rows = _log(rng, 1, max(2, min(8192, (1 << 27) // vocab)))
        temperature = rng.choice((1.0, 1.0, 0.7, 2.0))
        if op == "logprobs":
            return dict(op=op, rows=rows, vocab=vocab, top=rng.choice((0, 1, 5, 20, rng.randint(1, 64))), temperature=temperature, type=t)
        if op == "grad":
            return dict(op=op, rows=rows, vocab=vocab, temperature=temperature, type=t, entropy=rng.random() < 0.5)
        rest = rng.random() < 0.5
        return dict(op=op, rows=rows, vocab=vocab, k=_log(rng, 1, 128), temperature=temperature, rest=rest, ce=rng.random() < 0.5, type=t)
    n, k = rng.choice((192, 768, 5003, _log(rng, 32, 32768))), rng.choice((192, 384, 768, 32 * _log(rng, 1, 256)))
    group, zeros, scale = rng.choice((32, 64, 128, 128, 256)), rng.random() < 0.5, rng.choice(("f32", "bf16", "f16"))
    if op == "quantize":
        return dict(op=op, n=n, k=min(k, max(32, (1 << 27) // n // 32 * 32)), group=group, zeros=zeros, type=t, scale=scale)
    rows = rng.choice((1, 1, _log(rng, 1, min(256, max(2, (1 << 33) // (n * k))))))
    return dict(op=op, rows=rows, n=n, k=k, group=group, zeros=zeros, type=t, scale=scale)


# ---- inputs

def _logits(gen, case):
    """Logits as a head gives them: a broad bulk, a few ids far above it, one row in sixteen with most ids masked (a grammar), and,
    in a batch, one row of padding with every id masked."""
    rows, vocab = case["rows"], case["vocab"]
    x = torch.randn(rows, vocab, device="cuda", generator=gen) * 2.5
    peaks = torch.randint(0, vocab, (rows, 8), device="cuda", generator=gen)
    x.scatter_add_(1, peaks, torch.rand(rows, 8, device="cuda", generator=gen) * 10)
    if rows >= 16:
        some = x[5::16]
        some[torch.rand(some.shape, device="cuda", generator=gen) < 0.95] = -math.inf
        x[rows - 1] = -math.inf
    return x.to(TYPES[case["type"]]), peaks


def _targets(gen, case, peaks):
    """The id that was chosen: mostly one of the likely ones; in a batch, rows that have none."""
    rows, vocab = case["rows"], case["vocab"]
    t = torch.where(torch.rand(rows, device="cuda", generator=gen) < 0.8, peaks[:, 0], torch.randint(0, vocab, (rows,), device="cuda", generator=gen))
    if rows >= 16:
        t[3::16] = NONE
    return t.to(torch.int32)


def _weights(gen, case):
    n, k = case["n"], case["k"]
    return (torch.randn(n, k, device="cuda", generator=gen) * (0.02 + 0.04 * torch.rand(n, 1, device="cuda", generator=gen)))


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    c, st = case, dict(case=case)
    if c["op"] in ("logprobs", "grad", "distill"):
        rows, vocab = c["rows"], c["vocab"]
        x, peaks = _logits(gen, c)
        st.update(x=x, targets=_targets(gen, c, peaks))
        per_row = lambda: torch.empty(rows, device="cuda")  # noqa: E731
        if c["op"] == "logprobs":
            n = c["top"]
            st.update(logprob=per_row(), rank=torch.empty(rows, dtype=torch.int32, device="cuda"), entropy=per_row(),
                      stats=torch.empty(rows, 2, device="cuda"), ids=torch.empty(rows, n, dtype=torch.int32, device="cuda"),
                      top=torch.empty(rows, n, device="cuda"))
        elif c["op"] == "grad":  # what the forward call left, and the weights of a policy step
            _, _, entropy, stats, _, _ = _plain_logprobs(x, st["targets"], c["temperature"], 0)
            g = torch.randn(rows, device="cuda", generator=gen) / rows
            if rows >= 16:
                g[3::16] = 0.0
            st.update(entropy=entropy, stats=stats, g_logprob=g, g_entropy=torch.full((rows,), 0.01 / rows, device="cuda") if c["entropy"] else None,
                      grad=torch.empty_like(x))
        else:  # a teacher that agrees with the student on about half of its best ids
            k = min(c["k"], vocab)
            ids = torch.argsort(torch.rand(rows, vocab, device="cuda", generator=gen), dim=1)[:, :k] if vocab <= 1024 else \
                (torch.randint(0, vocab, (rows, 1), device="cuda", generator=gen) + torch.arange(k, device="cuda") * (vocab // k)) % vocab
            teacher = torch.sort(torch.randn(rows, k, device="cuda", generator=gen) * 2, descending=True)[0]
            if c["rest"]:  # log probabilities: 85 to 99 % of the mass on the listed ids
                mass = 0.85 + 0.14 * torch.rand(rows, 1, device="cuda", generator=gen)
                teacher = torch.log_softmax(teacher, 1) + torch.log(mass)
            if rows >= 16 and k >= 4:
                ids[7::16, k // 2:] = NONE  # a shorter list
            g = torch.full((rows,), 1.0 / rows, device="cuda") * (0.5 + torch.rand(rows, device="cuda", generator=gen))
            st.update(ids=ids.to(torch.int32).contiguous(), teacher=teacher.contiguous(), g_kl=g, g_ce=0.5 * g if c["ce"] else None,
                      kl=per_row(), ce=per_row() if c["ce"] else None, grad=torch.empty_like(x))
        return st
    n, k, group, s = c["n"], c["k"], c["group"], TYPES[c["scale"]]
    groups = -(-k // group)
    w = _weights(gen, c)
    if c["op"] == "quantize":
        return dict(st, w=w.to(TYPES[c["type"]]), codes=torch.empty(n, k // 2, dtype=torch.uint8, device="cuda"),
                    scales=torch.empty(n, groups, dtype=s, device="cuda"),
                    zeros=torch.empty(n, groups, dtype=torch.uint8, device="cuda") if c["zeros"] else None)
    codes, scales, zeros = _plain_quantize(w, group, c["zeros"], s)
    x = torch.randn(c["rows"], k, device="cuda", generator=gen)
    return dict(st, codes=codes, scales=scales, zeros=zeros, x=x.to(TYPES[c["type"]]),
                out=torch.empty(c["rows"], n, dtype=TYPES[c["type"]], device="cuda"))


# ---- the operators in their plain form

def _plain_rows(x, temperature):
    """z = (x - max) / T with the masked ids of an empty row at -inf, the row's maximum and ln sum exp z (0 for an empty row)."""
    x = x.float()
    m = x.max(1, keepdim=True)[0]
    some = m > -math.inf
    z = torch.where(some, (x - m) / temperature, -math.inf)
    w = torch.exp(z)
    s = w.sum(1, keepdim=True)
    return x, z, w, s, m, torch.where(some, torch.log(s), 0.0)


def _plain_logprobs(x, targets, temperature, top):
    x, z, w, s, m, ls = _plain_rows(x, temperature)
    rows, vocab = x.shape
    has = targets >= 0
    at = targets.clamp(min=0).long()[:, None]
    logprob = torch.where(has, (z.gather(1, at) - ls)[:, 0], 0.0)
    rank = torch.where(has, 1 + (x > x.gather(1, at)).sum(1), 0).to(torch.int32)
    entropy = torch.where(m > -math.inf, ls - torch.where(w > 0, w * z, 0.0).sum(1, keepdim=True) / s, 0.0)[:, 0]
    stats = torch.cat([m, ls], 1)
    if top == 0:
        return logprob, rank, entropy, stats, None, None
    bits = (x + 0.0).view(torch.int32)  # an order of (value, lower id first) in one 64-bit number
    order = (bits ^ ((bits >> 31) & 0x7FFFFFFF)).long()
    key = (order << 32) + (0x7FFFFFFF - torch.arange(vocab, device=x.device))
    best = torch.topk(key, min(top, vocab), dim=1)[0]
    ids = 0x7FFFFFFF - (best & 0xFFFFFFFF)
    lp = z.gather(1, ids) - ls
    more = top - ids.shape[1]
    if more > 0:  # fewer ids than alternatives asked for
        ids = torch.cat([ids, ids.new_full((rows, more), NONE)], 1)
        lp = torch.cat([lp, lp.new_full((rows, more), -math.inf)], 1)
    return logprob, rank, entropy, stats, ids.to(torch.int32), lp


def _plain_grad(st):
    c, x, t = st["case"], st["x"].float(), st["targets"]
    m, ls = st["stats"][:, :1], st["stats"][:, 1:]
    some = m > -math.inf
    logp = torch.where(some, (x - m) / c["temperature"], -math.inf) - ls
    p = torch.exp(logp)
    has = (t >= 0)[:, None] & some
    g_lp = torch.where(has, st["g_logprob"][:, None], 0.0)
    one = torch.zeros_like(x).scatter_(1, t.clamp(min=0).long()[:, None], 1.0)
    d = g_lp * (one - p)
    if st["g_entropy"] is not None:
        d = d - st["g_entropy"][:, None] * torch.where(p > 0, p * (logp + st["entropy"][:, None]), 0.0)
    return (d / c["temperature"]).to(st["x"].dtype)


def _plain_distill(st):
    c, g_kl, g_ce = st["case"], st["g_kl"][:, None], st["g_ce"]
    x, z, w, s, m, ls = _plain_rows(st["x"], c["temperature"])
    some = m > -math.inf
    has = st["ids"] >= 0
    ids = st["ids"].clamp(min=0).long()
    q = torch.where(has, st["teacher"], -math.inf)
    listed = torch.zeros_like(x).scatter_add_(1, ids, has.float()) > 0
    logp = z - ls
    p = w / torch.where(some, s, 1.0)
    if c["rest"]:
        t = torch.exp(q)
        r = (1 - t.double().sum(1, keepdim=True)).clamp(min=0.0).float()
        log_t = q
    else:
        t = torch.softmax(q, 1)
        log_t = torch.log_softmax(q, 1)
    kl = torch.where(t > 0, t * (log_t - logp.gather(1, ids)), 0.0).sum(1)
    t_at = torch.zeros_like(x).scatter_add_(1, ids, t)
    if c["rest"]:
        unlisted = torch.where(listed, 0.0, w).sum(1, keepdim=True)
        log_rest = torch.log(unlisted) - ls
        kl = kl + torch.where(r > 0, r * (torch.log(r) - log_rest), 0.0)[:, 0]
        q_rest = torch.where(listed, 0.0, w / unlisted)
        d = torch.where(listed, p - t_at, torch.where(unlisted > 0, q_rest * (torch.exp(log_rest) - r), 0.0))
    else:
        d = p - t_at
    d = g_kl * d / c["temperature"]
    ce = None
    if c["ce"]:
        _, z1, w1, s1, _, ls1 = _plain_rows(x, 1.0)
        tgt = st["targets"]
        there = (tgt >= 0)[:, None]
        at = tgt.clamp(min=0).long()[:, None]
        ce = torch.where(there, ls1 - z1.gather(1, at), 0.0)[:, 0]
        d = d + torch.where(there, g_ce[:, None] * (w1 / s1 - torch.zeros_like(x).scatter_(1, at, 1.0)), 0.0)
    return kl, ce, torch.where(some, d, 0.0).to(st["x"].dtype)


def _plain_quantize(w, group, zeros, scale_type):
    w = w.float()
    n, k = w.shape
    groups = -(-k // group)
    g = torch.nn.functional.pad(w, (0, groups * group - k)).view(n, groups, group)
    if zeros:
        lo, hi = g.amin(2).clamp(max=0.0), g.amax(2).clamp(min=0.0)
        step = (hi - lo) / torch.full_like(lo, 15.0)
    else:
        step = g.abs().amax(2) / torch.full((n, groups), 7.0, device=w.device)
    scales = step.to(scale_type)
    step = scales.float()[:, :, None]
    live = step > 0
    if zeros:
        zero = torch.where(live[:, :, 0], torch.round(-lo / step[:, :, 0]).clamp(0, 15), 0.0)
        q = torch.where(live, (torch.round(g / step) + zero[:, :, None]).clamp(0, 15), zero[:, :, None])
    else:
        zero = None
        q = torch.where(live, torch.round(g / step).clamp(-8, 7), 0.0) + 8
    q = q.reshape(n, groups * group)[:, :k].to(torch.uint8)
    return q[:, ::2] | (q[:, 1::2] << 4), scales, zero.to(torch.uint8) if zeros else None


def _dequantize(st, to):
    """The matrix that codes, scales and zeros stand for, in type `to`."""
    codes, c = st["codes"], st["case"]
    n, k = codes.shape[0], c["k"]
    q = torch.stack([codes & 15, codes >> 4], 2).view(n, k).to(to)
    at = torch.arange(k, device=codes.device) // c["group"]
    zero = 8.0 if st["zeros"] is None else st["zeros"].to(to)[:, at]
    return (q - zero) * st["scales"].to(to)[:, at]


def _plain(st):
    c = st["case"]
    if c["op"] == "logprobs":
        return _plain_logprobs(st["x"], st["targets"], c["temperature"], c["top"])
    if c["op"] == "grad":
        return _plain_grad(st)
    if c["op"] == "distill":
        return _plain_distill(st)
    if c["op"] == "quantize":
        return _plain_quantize(st["w"], c["group"], c["zeros"], TYPES[c["scale"]])
    return (st["x"].float() @ _dequantize(st, torch.float32).T).to(st["x"].dtype)


# ---- the framework's calls

_context = []


def _gpu():
    """The context that a program makes once, on the stream that the program works on now (its number alone: an object for it would
    be 3 us of a call of 6)."""
    stream = torch._C._cuda_getCurrentRawStream(0)
    if not _context:
        import pssa_b200
        _context[:] = pssa_b200.B200Dispatch(0, stream), stream
    elif _context[1] != stream:
        _context[0].set_stream(stream)
        _context[1] = stream
    return _context[0]


def _own(st):
    c, gpu = st["case"], _gpu()
    if c["op"] == "logprobs":
        top = c["top"]
        gpu.token_logprobs_dev(st["x"], c["rows"], c["vocab"], st["targets"], logprob=st["logprob"], rank=st["rank"], entropy=st["entropy"],
                               stats=st["stats"], top_n=top, top_ids=st["ids"] if top else None, top_logprobs=st["top"] if top else None,
                               temperature=c["temperature"])
        return (st["logprob"], st["rank"], st["entropy"], st["stats"], st["ids"], st["top"]) if top else \
            (st["logprob"], st["rank"], st["entropy"], st["stats"], None, None)
    if c["op"] == "grad":
        gpu.token_logprobs_grad_dev(st["x"], c["rows"], c["vocab"], st["targets"], st["stats"], st["grad"], grad_logprob=st["g_logprob"],
                                    entropy=st["entropy"], grad_entropy=st["g_entropy"], temperature=c["temperature"])
        return st["grad"]
    if c["op"] == "distill":
        gpu.distill_topk_dev(st["x"], c["rows"], c["vocab"], st["ids"], st["teacher"], st["ids"].shape[1], kl=st["kl"], grad_kl=st["g_kl"],
                             targets=st["targets"] if c["ce"] else None, ce=st["ce"], grad_ce=st["g_ce"], grad_logits=st["grad"],
                             temperature=c["temperature"], rest=c["rest"])
        return st["kl"], st["ce"], st["grad"]
    group = min(c["group"], -(-c["k"] // 128) * 128)  # one group of a narrow matrix: no wider than the call takes it
    if c["op"] == "quantize":
        gpu.w4_quantize_dev(st["w"], c["n"], c["k"], group, st["codes"], st["scales"], st["zeros"])
        return st["codes"], st["scales"], st["zeros"]
    gpu.gemv_w4_dev(st["x"], c["rows"], st["codes"], st["scales"], st["zeros"], c["n"], c["k"], group, st["out"])
    return st["out"]


def run(state):
    return _own(state) if own else _plain(state)


# ---- the definitions in 64 bits

def _by_rows(f, x, *more):
    """f on pieces of at most 2^25 logits, its outputs joined."""
    step = max(1, (1 << 25) // x.shape[1])
    parts = [f(x[i:i + step].double(), *[None if a is None else a[i:i + step] for a in more]) for i in range(0, x.shape[0], step)]
    return [None if p[0] is None else torch.cat(p) for p in zip(*parts)]


def _exact_logprobs(x, targets, temperature, top):
    m = x.max(1)[0]
    empty = m == -math.inf
    y = x / temperature
    logp = torch.where(empty[:, None], -math.inf, y - torch.logsumexp(y, 1, keepdim=True))
    there = targets != NONE
    logprob = torch.where(there, logp[torch.arange(len(x), device=x.device), torch.where(there, targets, 0).long()], 0.0)
    entropy = torch.special.entr(torch.exp(logp)).sum(1)
    ls = torch.where(empty, 0.0, torch.logsumexp(y, 1) - m / temperature)
    lp = None
    if top:
        lp = torch.sort(logp, 1, descending=True)[0][:, :top]
        if lp.shape[1] < top:
            lp = torch.cat([lp, lp.new_full((len(x), top - lp.shape[1]), -math.inf)], 1)
    return logprob, entropy, torch.stack([m, ls], 1), lp


def _exact_grad(x, targets, stats, entropy, g_lp, g_h, temperature):
    stats = stats.double()
    empty = stats[:, 0] == -math.inf
    p = torch.where(empty[:, None], 0.0, torch.exp((x - stats[:, :1]) / temperature - stats[:, 1:]))
    g = torch.where((targets != NONE) & ~empty, g_lp.double(), 0.0)
    d = -g[:, None] * p
    d[torch.arange(len(x), device=x.device), torch.where(targets != NONE, targets, 0).long()] += g
    if g_h is not None:
        d += g_h.double()[:, None] * (torch.special.entr(p) - p * entropy.double()[:, None])
    return (d / temperature,)


def _exact_distill(x, ids, teacher, targets, g_kl, g_ce, temperature, rest):
    rows, vocab = x.shape
    empty = x.max(1)[0] == -math.inf
    logp = torch.log_softmax(x / temperature, 1)
    q = teacher.double().masked_fill(ids == NONE, -math.inf)
    if not rest:
        q = q - torch.logsumexp(q, 1, keepdim=True)
    t = torch.exp(q)
    wide = torch.zeros(rows, vocab + 1, dtype=torch.float64, device=x.device)  # a column of its own for absent ids
    at = torch.where(ids == NONE, vocab, ids.long())
    t_v = wide.scatter_add(1, at, t)[:, :vocab]
    named = wide.scatter_add(1, at, torch.ones_like(t))[:, :vocab] > 0
    kl = torch.special.xlogy(t, t).sum(1) - torch.where(t_v > 0, t_v * logp, 0.0).sum(1)
    p = torch.exp(logp)
    d = p * t.sum(1, keepdim=True) - t_v
    if rest:
        r = (1 - t.sum(1)).clamp(min=0)
        log_rest = torch.logsumexp(logp.masked_fill(named, -math.inf), 1)
        kl = kl + torch.where(r > 0, torch.special.xlogy(r, r) - r * log_rest, 0.0)
        inside = torch.exp(logp - log_rest[:, None]).masked_fill(named | (log_rest == -math.inf)[:, None], 0.0)
        d = d + r[:, None] * (p - inside)
    kl = torch.where(empty, torch.where(t.sum(1) > 0, math.inf, 0.0), kl)
    d = g_kl.double()[:, None] * d / temperature
    ce = None
    if g_ce is not None:
        there = targets != NONE
        col = torch.where(there, targets, 0).long()
        row = torch.arange(rows, device=x.device)
        logp1 = torch.log_softmax(x, 1)
        ce = torch.where(there, torch.where(empty, math.inf, -logp1[row, col]), 0.0)
        e = torch.exp(logp1)
        e[row, col] -= 1
        d = d + torch.where(there, g_ce.double(), 0.0)[:, None] * e
    return kl, ce, d.masked_fill(empty[:, None], 0.0)


def exact(case, seed):
    st, c = prepare(case, seed), case
    if c["op"] == "logprobs":
        logprob, entropy, stats, lp = _by_rows(lambda x, t: _exact_logprobs(x, t, c["temperature"], c["top"]), st["x"], st["targets"])
        return logprob, None, entropy, stats, None, lp
    if c["op"] == "grad":
        return _by_rows(lambda x, *a: _exact_grad(x, *a, c["temperature"]), st["x"], st["targets"], st["stats"], st["entropy"], st["g_logprob"],
                        st["g_entropy"])[0]
    if c["op"] == "distill":
        return tuple(_by_rows(lambda x, *a: _exact_distill(x, *a, c["temperature"], c["rest"]), st["x"], st["ids"], st["teacher"], st["targets"],
                              st["g_kl"], st["g_ce"]))
    if c["op"] == "quantize":
        g = torch.nn.functional.pad(st["w"].double(), (0, -c["k"] % c["group"])).view(c["n"], -1, c["group"])
        span = (g.amax(2).clamp(min=0) - g.amin(2).clamp(max=0)) / 15 if c["zeros"] else g.abs().amax(2) / 7
        return None, span, None
    x, parts = st["x"].double(), []
    for i in range(0, c["n"], 4096):  # the groups' sums of code * x, each times its scale
        q = st["codes"][i:i + 4096].int()
        q = torch.stack([q % 16, q // 16], -1).flatten(1).double()
        z = torch.full((len(q), st["scales"].shape[1]), 8.0, dtype=torch.float64, device="cuda") if st["zeros"] is None else st["zeros"][i:i + 4096].double()
        rep = lambda v: v.repeat_interleave(c["group"], 1)[:, :c["k"]]  # noqa: E731
        parts.append(x @ ((q - rep(z)) * rep(st["scales"][i:i + 4096].double())).T)
    return torch.cat(parts, 1)


# ---- what a pass cannot do without

def work(case):
    c = case
    if c["op"] in ("logprobs", "grad", "distill"):
        rows, cells, size = c["rows"], c["rows"] * c["vocab"], SIZE[c["type"]]
        if c["op"] == "logprobs":  # the logits in; id in, log probability, rank, entropy, stats and alternatives out
            return {"bytes": cells * size + rows * (24 + 8 * c["top"]), "flops": 7 * cells}
        if c["op"] == "grad":  # the logits in and their gradient out
            return {"bytes": 2 * cells * size + rows * 24, "flops": (7 if c["entropy"] else 5) * cells}
        return {"bytes": 2 * cells * size + rows * (8 * c["k"] + (20 if c["ce"] else 8)), "flops": (10 if c["ce"] else 7) * cells}
    n, k, s = c["n"], c["k"], SIZE[c["scale"]]
    held = n * k // 2 + n * -(-k // c["group"]) * (s + (1 if c["zeros"] else 0))
    if c["op"] == "quantize":
        return {"bytes": held + n * k * SIZE[c["type"]], "flops": 5 * n * k}
    return {"bytes": held + c["rows"] * (n + k) * SIZE[c["type"]], "flops": 2 * c["rows"] * n * k}
