"""Calls of the head's operators at the edges of what they take: a teacher that is no number, logits of a model that are none, rows
near 2^31 logits, products whose inputs pass through shared memory in several turns, texts whose logits take several tiles."""
import numpy as np
import pytest

import head_plain as P
from test_distill_gpu import distill
from test_token_logprobs_gpu import close, dev, logits_of

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def gpu():
    import torch

    import pssa_b200
    d = pssa_b200.B200Dispatch(0, torch.cuda.current_stream())
    yield d
    d.close()


@pytest.mark.parametrize("vocab", [1000, 16384, 400003])
@pytest.mark.parametrize("rest", [False, True])
@pytest.mark.parametrize("value", ["nan", "inf", "overflow"])
@pytest.mark.parametrize("temperature", [1.0, 2.0])
def test_a_teacher_that_is_no_number_leaves_the_cross_entropy(gpu, vocab, rest, value, temperature):
    """A present entry that is NaN, +inf or too large at the teacher's temperature: its row's divergence is NaN and so is the gradient
    of that; the cross entropy and its gradient do not depend on the teacher, nor do other rows."""
    import torch
    rng = np.random.default_rng(vocab)
    rows, k = 6, 5
    x = rng.standard_normal((rows, vocab))
    ids = np.stack([rng.permutation(vocab)[:k] for _ in range(rows)]).astype(np.uint32)
    x[np.arange(rows)[:, None], ids] += 6  # the listed ids carry most of the student's mass: losing them shows
    targets = ids[:, 0].copy()
    targets[5] = (ids[5].max() + 1) % vocab  # a target that is not listed
    view = torch.from_numpy(x.astype(np.float32)).cuda()
    x = view.double().cpu().numpy()
    fine = np.log(np.full((rows, k), 0.9 / k, np.float32))
    t_temperature = 0.5 if value == "overflow" and not rest else 1.0
    teacher = fine.copy()
    bad = [0, 2, 3, 5]
    teacher[bad, [0, 1, 4, 2]] = {"nan": np.nan, "inf": np.inf, "overflow": 3e38 if t_temperature != 1.0 else np.inf}[value]
    g_kl, g_ce = np.array([1.0, 1.0, 0.0, 0.5, 1.0, 0.0], np.float32), np.array([1.0, 1.0, 0.5, 0.0, 1.0, 1.0], np.float32)
    kl, ce, grad = distill(gpu, view, ids, teacher, targets, g_kl, g_ce, temperature, t_temperature, rest)
    grad = grad.double().cpu().numpy()
    for r in range(rows):
        w = P.distill(x[r], ids[r], fine[r].astype(np.float64), temperature, t_temperature, rest, int(targets[r]), float(g_kl[r]), float(g_ce[r]), "float32")
        close(ce[r], w["ce"], w["tol_ce"], f"ce {r}")
        if r not in bad:
            close(kl[r], w["kl"], w["tol"], f"kl {r}")
        else:
            assert np.isnan(kl[r])
        if r in bad and g_kl[r] != 0:
            assert np.isnan(grad[r]).all()
        else:
            close(grad[r], w["grad"], w["tol_g"], f"gradient {r}")
    # without a weight of the divergence
    _, ce2, grad2 = distill(gpu, view, ids, teacher, targets, None, g_ce, temperature, t_temperature, rest)
    assert np.array_equal(ce, ce2)
    for r in range(rows):
        w = P.distill(x[r], ids[r], fine[r].astype(np.float64), temperature, t_temperature, rest, int(targets[r]), 0.0, float(g_ce[r]), "float32")
        close(grad2[r].double().cpu().numpy(), w["grad"], w["tol_g"], f"gradient of the cross entropy {r}")


@pytest.mark.parametrize("shift,gshift", [(0, 0), (1, 1), (0, 1)])
def test_a_vocabulary_just_below_2_31(gpu, shift, gshift):
    """Every index of the last elements and of what lies behind them is near the end of 32 bits. The bulk is 0, so that its sums are
    whole numbers below 2^24 in every thread whose reference is 0. It is a peak's in the warps that start with one: the one with the
    elements behind the last vector, and the one at the row's middle, where a CTA starts. These are 64 of 8192 threads (8 CTAs of
    1024), and each rounds its 2^31 / 8192 / 2 sums of pairs by at most 2^-24 of a running sum that is half the last one on
    average: 2^17 / 2 * 64 / 8192 = 512 times 2^-24 of the whole. The joins are at most 40 roundings more, and the logarithm of
    2^31 has steps of 2^-19. An entropy is ls less ent / sum, of about 2: e from the first and 2 (e + e) from the second."""
    import torch
    v, top = (1 << 31) - 1, 5
    buf, out = torch.zeros(v + 80, dtype=torch.bfloat16, device="cuda"), torch.full((v + 80,), 5.0, dtype=torch.bfloat16, device="cuda")
    x, grad = buf[shift:shift + v].view(1, v), out[gshift:gshift + v].view(1, v)
    peaks = [v - 1, v - 2, v // 2, 1 << 30]
    x[0, peaks] = torch.tensor([2.0, 1.5, 1.0, 0.5], dtype=torch.bfloat16, device="cuda")
    buf[shift + v:] = 50.0  # behind the row
    target = dev(np.array([v - 1], np.uint32))
    lp, h, stats, rank = (torch.zeros(1, device="cuda"), torch.zeros(1, device="cuda"), torch.zeros(1, 2, device="cuda"),
                          torch.zeros(1, dtype=torch.int32, device="cuda"))
    ids, tops = torch.zeros(top + 2, dtype=torch.int32, device="cuda"), torch.full((top + 2,), 7.0, device="cuda")
    ids[-1] = 77
    gpu.token_logprobs_dev(x, 1, v, target, logprob=lp, rank=rank, entropy=h, stats=stats, top_n=top, top_ids=ids[:top], top_logprobs=tops[:top], ld=v)
    g = torch.ones(1, device="cuda")
    gpu.token_logprobs_grad_dev(x, 1, v, target, stats, grad, grad_logprob=g, ld=v, ld_grad=v)
    torch.cuda.synchronize()
    gpu.poll_status()
    w = np.exp(np.array([2.0, 1.5, 1.0, 0.5]))
    total = (v - 4) + w.sum()
    tol = (512 + 40) * P.U + 2.0 ** -19
    assert abs(float(lp) - (2.0 - np.log(total))) <= tol and int(rank) == 1
    assert abs(float(h) - (np.log(total) - (w * np.log(w)).sum() / total)) <= 5 * tol
    assert float(stats[0, 0]) == 2.0 and abs(float(stats[0, 1]) - (np.log(total) - 2.0)) <= tol
    assert ids.cpu().tolist() == peaks + [0, 0, 77] and float(tops[-1]) == 7.0
    # the gradient: -1 / total in the bulk, 1 - p at the target; what is behind the row stays
    for i, a in zip(peaks, w):
        want = float(i == v - 1) - a / total
        assert abs(float(grad[0, i]) - want) <= 2.0 ** -8 * abs(want) + tol * a / total
    grad[0, peaks] = float(grad[0, 0])
    assert abs(float(grad[0, 0]) + 1 / total) <= (2.0 ** -8 + tol) / total
    assert float(grad.min()) == float(grad.max()) == float(grad[0, 0])
    assert bool((out[:gshift] == 5.0).all()) and bool((out[gshift + v:] == 5.0).all())


def sure_rows(rng, rows, vocab, dtype):
    """Rows with one id far above the others, which share 1e-1 to 1e-12 of the mass; the id lies at a row's ends and between them."""
    import torch
    x = rng.standard_normal((rows, vocab)) * 2
    best = np.array([(0, vocab - 1, vocab // 2, 1, min(8, vocab - 1), vocab // 3, vocab - 2, (5 * vocab) // 7)[r % 8] for r in range(rows)])
    x[np.arange(rows), best] = np.log(np.exp(x).sum(1)) + rng.uniform(2.3, 28, rows)
    view = torch.from_numpy(x).to(getattr(torch, dtype)).cuda()
    return view, view.double().cpu().numpy(), best


@pytest.mark.parametrize("dtype", ["float32", "bfloat16", "float16"])
@pytest.mark.parametrize("rows,vocab,top", [(8, 40, 2), (16, 1000, 0), (1, 16384, 20), (8, 16384, 5), (16, 70001, 0), (1, 131072, 3), (200, 5003, 1), (1400, 600, 4)])
@pytest.mark.parametrize("temperature", [1.0, 0.7])
def test_a_row_that_is_sure_of_one_id_keeps_its_small_numbers(gpu, dtype, rows, vocab, top, temperature):
    """Entropy, log sum and the best id's log probability come from what the other ids leave, each of whose terms has an argument of
    3 roundings, an exponential of 2 more, `adds` sums and a logarithm or a quotient of 2: relative to the result, however small."""
    from test_token_logprobs_gpu import forward
    view, x, best = sure_rows(np.random.default_rng(vocab + rows), rows, vocab, dtype)
    got = forward(gpu, view, vocab, best.astype(np.uint32), top, temperature)
    for r in range(rows):
        z = (x[r] - x[r].max()) / temperature
        assert z.argmax() == best[r]
        others = np.delete(z, best[r])
        rest = np.exp(others).sum()
        l, h = np.log1p(rest), np.log1p(rest) + (np.exp(others) * -others).sum() / (1 + rest)
        tol = P.U * (3 * -others.min() + 2 * P.adds(vocab) + 20)
        for name, a, want in (("log sum", got["stats"][r, 1], l), ("log probability", got["logprob"][r], -l), ("entropy", got["entropy"][r], h),
                              *([("best", got["top"][r, 0], -l)] if top else [])):
            assert abs(float(a) - want) <= tol * abs(want) + 2.0 ** -149, (name, r, float(a), want)
        assert got["rank"][r] == 1


def test_a_model_whose_logits_are_no_numbers():
    """What the scorer refuses `score_logprobs` refuses too: a target's logit of -inf, and a position of nothing else. An id that is
    not the target may be one, in both."""
    import oracle as O
    import pssa_b200
    from helpers import fill_synthetic, upload
    from pssa_b200 import model as M
    gpu = pssa_b200.B200Dispatch(0)
    v, d = 203, 32
    om = fill_synthetic(O.Model.new(2, v, d, 16, 8, 16, tau_mem=0.1, seed=5), 5)
    m = pssa_b200.PSSAModel(gpu, 2, v, d, 16, 8, 16, tau_mem=0.1, precision=1)
    upload(om, m)
    start = m.copy_recurrent_state_to(0)
    head = np.random.default_rng(0).standard_normal((v, d)).astype(np.float32)

    def with_head(u, f):
        m.set_tensor(-1, M.UNEMBED, u)
        m.copy_recurrent_state_from(start, 0)
        return f()

    probe = head.copy()
    probe[:d] = np.eye(d, dtype=np.float32)
    features = with_head(probe, lambda: m.score([1], [0], want_logits=True))[2][0, :d] * np.sqrt(d)  # a head's scale is 1 / sqrt(d)
    assert np.abs(features).sum() > 1.01
    lowest = np.finfo(np.float32).min * np.sign(features)  # products of one sign: their sum is beyond fp32's range
    one = head.copy()
    one[7] = lowest
    _, loss, logits = with_head(one, lambda: m.score([1], [3], want_logits=True))
    assert logits[0, 7] == -np.inf and np.isfinite(np.delete(logits[0], 7)).all()
    for f in (lambda: m.score([1], [7]), lambda: m.score_logprobs([1], [7]), lambda: m.score_logprobs([1, 1], [3, 7], top=2)):
        with pytest.raises(pssa_b200.B200Error):
            with_head(one, f)
    got = with_head(one, lambda: m.score_logprobs([1], [3], top=4))
    w = P.logprobs(logits[0].astype(np.float64), 3, 1.0, 4)
    assert got["rank"][0] == w["rank"] and np.array_equal(got["top_ids"][0], w["ids"]) and abs(got["logprob"][0] - w["logprob"]) <= w["tol"] + P.U * 40
    none = np.tile(lowest, (v, 1))
    for f in (lambda: m.score([1], [3]), lambda: m.score_logprobs([1], [3]), lambda: m.score_logprobs([1]), lambda: m.score_logprobs([1], [-1], top=3)):
        with pytest.raises(pssa_b200.B200Error):
            with_head(none, f)
    m.close()
    gpu.close()


def test_a_text_whose_logits_take_two_tiles():
    """256 rows of 131072 logits are a tile: positions behind it, with their targets and alternatives."""
    import pssa_b200
    gpu = pssa_b200.B200Dispatch(0)
    v, n, top = 131072, 300, 5
    m = pssa_b200.PSSAModel(gpu, 1, v, 32, 16, 8, 16, tau_mem=0.1)
    m.init_random(3)
    m.set_max_rows(n)
    rng = np.random.default_rng(1)
    ids, targets = rng.integers(0, v, n), rng.integers(0, v, n)
    start = m.copy_recurrent_state_to(0)
    _, _, logits = m.score(ids, targets, want_logits=True)
    m.copy_recurrent_state_from(start, 0)
    got = m.score_logprobs(ids, targets, top=top)
    for r in (0, 1, 254, 255, 256, 257, 298, 299):
        w = P.logprobs(logits[r].astype(np.float64), int(targets[r]), 1.0, top)
        assert got["rank"][r] == w["rank"] and np.array_equal(got["top_ids"][r], w["ids"])
        assert abs(got["logprob"][r] - w["logprob"]) <= w["tol"] + P.U * 100 and abs(got["entropy"][r] - w["entropy"]) <= w["tol_h"]
        assert np.max(np.abs(got["top_logprobs"][r] - w["top"])) <= w["tol"] + P.U * 100
    m.close()
    gpu.close()


@pytest.mark.parametrize("vocab,top", [(1000, 48), (1000, 49), (1000, 64), (5000, 52), (5003, 64), (16384, 16), (16384, 17)])
def test_alternatives_of_many_rows_on_both_sides_of_the_choice(gpu, vocab, top):
    """More rows than the GPU has CTAs: the best ids in order and their log probabilities, whichever CTA takes a row."""
    from test_token_logprobs_gpu import check_forward, forward
    import torch
    rng = np.random.default_rng(top)
    view, x = logits_of(rng, 24, vocab, "float32")
    many = view.repeat(50, 1)
    targets = rng.integers(0, vocab, 24).astype(np.uint32)
    got = forward(gpu, many, vocab, np.tile(targets, 50), top, 1.0)
    check_forward({k: v[:24] for k, v in got.items()}, x, targets, top, 1.0)
    for k, v in got.items():
        v = torch.from_numpy(v.view(np.int32)).view(50, -1)
        assert bool((v == v[:1]).all()), k


@pytest.mark.parametrize("rows,vocab,allowed", [(40, 40, 40), (40, 64, 64), (24, 5003, 30), (6, 400003, 30)])
@pytest.mark.parametrize("temperature", [1.0, 2.0])
def test_a_teacher_that_lists_every_id_there_is(gpu, rows, vocab, allowed, temperature):
    """All ids of a small vocabulary, or all that a mask leaves, as `token_logprobs_dev` gives them: what rounding leaves of the
    teacher's mass belongs to no id, and is no infinite divergence. A mass that is left in earnest is one."""
    import torch
    from test_token_logprobs_gpu import forward
    rng = np.random.default_rng(vocab)
    x, y = rng.standard_normal((rows, vocab)) * 3, rng.standard_normal((rows, vocab)) * 3
    masked = np.stack([rng.permutation(vocab) >= allowed for _ in range(rows)])
    x[masked], y[masked] = -np.inf, -np.inf
    teacher, student = (torch.from_numpy(a.astype(np.float32)).cuda() for a in (x, y))
    x, y = teacher.double().cpu().numpy(), student.double().cpu().numpy()
    top = min(vocab, 64)
    got = forward(gpu, teacher, vocab, np.full(rows, P.NONE, np.uint32), top, 1.0)
    g = np.ones(rows, np.float32)
    kl, _, grad = distill(gpu, student, got["ids"], got["top"], None, g, None, temperature, 1.0, True)
    grad = grad.double().cpu().numpy()
    for r in range(rows):
        zt, lt = P.log_softmax(x[r], 1.0)
        zs, ls = P.log_softmax(y[r], temperature)
        live = ~masked[r]
        t = np.exp(zt[live] - lt)
        want = float((t * (zt[live] - lt - zs[live] + ls)).sum())
        # the entries' rounding, and the statistics' of both rows: of numbers of this size
        size = float((t * (np.abs(zt[live] - lt) + np.abs(zs[live] - ls))).sum()) + abs(ls) + 1
        tol = P.U * (2 * P.adds(vocab) + 60) * size
        assert abs(kl[r] - want) <= tol, (r, kl[r], want)
        d = np.zeros(vocab)
        d[live] = (np.exp(zs[live] - ls) - t) / temperature
        assert np.abs(grad[r] - d).max() <= P.U * (2 * P.adds(vocab) + 60) * (1 + np.abs(zs[live]).max()), r
    less = got["top"] - np.float32(0.01)  # 1 % of the mass is left, and no id for it
    kl, _, _ = distill(gpu, student, got["ids"], less, None, None, None, temperature, 1.0, True, grad=False)
    assert np.isposinf(kl).all()


@pytest.mark.parametrize("dtype,vocab", [("float32", 393216), ("float32", 393215), ("bfloat16", 786432), ("float32", 393217), ("bfloat16", 786433), ("float16", 1638400)])
def test_distillation_on_both_sides_of_what_a_cluster_holds(gpu, dtype, vocab):
    import pssa_b200
    from test_distill_gpu import check, teacher_of
    rng = np.random.default_rng(vocab)
    view, x = logits_of(rng, 2, vocab, dtype, 1, vocab + 1)
    ids, teacher = teacher_of(rng, x, 30, True)
    targets, g = np.array([vocab - 1, 5], np.uint32), np.array([1.0, -0.5], np.float32)
    check(distill(gpu, view, ids, teacher, targets, g, g, 2.0, 1.0, True), x, ids, teacher, targets, g, g, 2.0, 1.0, True, dtype)
    if vocab == 1638400:
        wide = view.new_zeros(2, vocab + 1)
        with pytest.raises(pssa_b200.B200Error):
            gpu.distill_topk_dev(wide, 2, vocab + 1, dev(ids), dev(teacher), 30, kl=dev(np.zeros(2, np.float32)), rest=True)


def test_rows_that_lie_between_each_other(gpu):
    """Logits and their gradient, inputs and results side by side in the rows of one buffer, as the same calls with an array of its own for the
    result (a row's bits may depend on how it is aligned)."""
    import torch
    rng = np.random.default_rng(2)
    view, x = logits_of(rng, 24, 1000, "float32")
    wide = torch.full((24, 2003), 8.0, device="cuda")
    left, right = wide[:, :1000], wide[:, 1002:2002]
    left.copy_(view)
    g, ids, teacher = np.ones(24, np.float32), np.tile(np.array([[5, 9, 700]], np.uint32), (24, 1)), np.log(np.full((24, 3), 0.3, np.float32))
    apart = distill(gpu, left, ids, teacher, None, g, None, 1.0, 1.0, True)
    beside = distill(gpu, left, ids, teacher, None, g, None, 1.0, 1.0, True, out=right)
    assert np.array_equal(apart[0], beside[0], equal_nan=True) and torch.equal(apart[2].nan_to_num(3.0), right.nan_to_num(3.0))
    assert torch.equal(left, view) and bool((wide[:, 1000:1002] == 8.0).all()) and bool((wide[:, 2002:] == 8.0).all())
    stats, targets = torch.zeros(24, 2, device="cuda"), dev(np.arange(24, dtype=np.uint32))
    gpu.token_logprobs_dev(left, 24, 1000, stats=stats, ld=2003)
    out = torch.zeros(24, 1000, device="cuda")
    gpu.token_logprobs_grad_dev(left, 24, 1000, targets, stats, out, grad_logprob=dev(g), ld=2003)
    gpu.token_logprobs_grad_dev(left, 24, 1000, targets, stats, right, grad_logprob=dev(g), ld=2003, ld_grad=2003)
    assert torch.equal(out.nan_to_num(3.0), right.nan_to_num(3.0)) and torch.equal(left, view)
    codes, scales = torch.randint(0, 256, (96, 128), dtype=torch.uint8, device="cuda"), torch.rand(96, 4, device="cuda")
    both = torch.randn(5, 360, device="cuda")
    before, x, y = both.clone(), both[:, :256], both[:, 260:356]
    out = torch.zeros(5, 96, device="cuda")
    gpu.gemv_w4_dev(before[:, :256].contiguous(), 5, codes, scales, None, 96, 256, 64, out)
    gpu.gemv_w4_dev(x, 5, codes, scales, None, 96, 256, 64, y, ldx=360, ldo=360)
    y_is, both[:, 260:356] = y.clone(), before[:, 260:356]
    assert torch.equal(out, y_is) and torch.equal(both, before)
