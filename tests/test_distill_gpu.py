"""Distillation from a teacher's best ids, loss and gradient, against the plain form in 64 bits."""
import numpy as np
import pytest

import head_plain as P
from test_token_logprobs_gpu import DTYPES, close, dev, logits_of, targets_of

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def gpu():
    import torch

    import pssa_b200
    d = pssa_b200.B200Dispatch(0, torch.cuda.current_stream())
    yield d
    d.close()


def teacher_of(rng, x, k, rest):
    """Entries of each row: likely and arbitrary ids, a shorter list, one id twice, a list of nothing, a mass of 0."""
    rows, v = x.shape
    ids = np.stack([np.concatenate([np.argsort(-x[r], kind="stable")[:k // 2], rng.permutation(v)[:k]])[:k] if v >= k else rng.integers(0, v, k)
                    for r in range(rows)]).astype(np.uint32)
    for r in range(rows):  # every id once
        seen = set()
        for i in range(k):
            while int(ids[r, i]) in seen and len(seen) < v:
                ids[r, i] = rng.integers(0, v)
            if int(ids[r, i]) in seen:
                ids[r, i] = P.NONE
            seen.add(int(ids[r, i]))
    teacher = rng.standard_normal((rows, k)).astype(np.float32) * 2
    if rest:
        lse = np.log(np.exp(teacher.astype(np.float64)).sum(1, keepdims=True))
        teacher = (teacher - lse + np.log(rng.uniform(0.2, 0.999, (rows, 1)))).astype(np.float32)
    for r in range(rows):
        if r % 7 == 3:
            ids[r, k // 2:] = P.NONE
            teacher[r, k // 2:] = np.nan  # what stands at an absent entry is not read
        elif r % 7 == 4 and k > 1 and not rest:
            ids[r, 1] = ids[r, 0]
        elif r % 7 == 5:
            ids[r] = P.NONE
        elif r % 7 == 6 and k > 1:
            teacher[r, 0] = -np.inf
    return ids, teacher


def distill(gpu, view, ids, teacher, targets, g_kl, g_ce, temperature, t_temperature, rest, grad=True, out=None):
    import torch
    rows, vocab = view.shape
    kl, ce = torch.full((rows,), 77.0, device="cuda"), torch.full((rows,), 77.0, device="cuda")
    g = out if out is not None else torch.full((rows, vocab), 99.0, dtype=view.dtype, device="cuda") if grad else None
    gpu.distill_topk_dev(view, rows, vocab, dev(ids), dev(teacher), ids.shape[1], kl=kl, targets=None if targets is None else dev(targets),
                         ce=None if targets is None else ce, grad_kl=dev(g_kl) if grad and g_kl is not None else None,
                         grad_ce=dev(g_ce) if grad and g_ce is not None else None, grad_logits=g, temperature=temperature,
                         teacher_temperature=t_temperature, rest=rest, ld=view.stride(0), ld_grad=g.stride(0) if grad else None)
    torch.cuda.synchronize()
    return kl.cpu().numpy(), ce.cpu().numpy(), g


def check(got, x, ids, teacher, targets, g_kl, g_ce, temperature, t_temperature, rest, dtype):
    kl, ce, grad = got
    grad = None if grad is None else grad.double().cpu().numpy()
    for r in range(len(x)):
        w = P.distill(x[r], ids[r], teacher[r].astype(np.float64), temperature, t_temperature, rest, P.NONE if targets is None else int(targets[r]),
                      0.0 if g_kl is None else float(g_kl[r]), 0.0 if g_ce is None else float(g_ce[r]), dtype)
        close(kl[r], w["kl"], w["tol"], f"kl {r}")
        if targets is not None:
            close(ce[r], w["ce"], w["tol_ce"], f"ce {r}")
        if grad is not None:
            close(grad[r], w["grad"], w["tol_g"], f"gradient {r}")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,vocab,k", [(1, 1, 1), (13, 5, 8), (14, 40, 40), (28, 1000, 1), (28, 1003, 17), (28, 5003, 64), (1, 16384, 32), (2, 16384, 256),
                                          (28, 131072, 64), (300, 2000, 8), (3, 200003, 20), (14, 400003, 40), (1300, 300, 8), (1300, 513, 256)])
@pytest.mark.parametrize("rest", [False, True])
def test_loss_and_gradient_match_the_plain_form(gpu, dtype, rows, vocab, k, rest):
    rng = np.random.default_rng(rows * 3 + vocab + k)
    view, x = logits_of(rng, rows, vocab, dtype)
    ids, teacher = teacher_of(rng, x, k, rest)
    targets = targets_of(rng, x)
    g_kl, g_ce = rng.standard_normal(rows).astype(np.float32), rng.standard_normal(rows).astype(np.float32)
    g_kl[8::9] = 0.0
    g_ce[7::9] = 0.0
    for t, tt, a, b, tgt in ((1.0, 1.0, g_kl, None, None), (2.0, 1.0 if rest else 2.0, g_kl, g_ce, targets), (0.7, 1.0, None, g_ce, targets)):
        check(distill(gpu, view, ids, teacher, tgt, a, b, t, tt, rest), x, ids, teacher, tgt, a, b, t, tt, rest, dtype)
    check(distill(gpu, view, ids, teacher, targets, None, None, 1.0, 1.0, rest, grad=False), x, ids, teacher, targets, None, None, 1.0, 1.0, rest, dtype)
    gpu.poll_status()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shift,pitch,gpitch", [(1, 1001, 1000), (4, 1008, 1001), (0, 1000, 1016), (3, 1003, 1003), (8, 1008, 1008)])
def test_rows_may_start_anywhere_and_what_lies_between_them_stays(gpu, dtype, shift, pitch, gpitch):
    import torch
    rng = np.random.default_rng(pitch)
    view, x = logits_of(rng, 28, 1000, dtype, shift, pitch)
    ids, teacher = teacher_of(rng, x, 12, True)
    g = rng.standard_normal(28).astype(np.float32)
    buf = torch.full((28 * gpitch + 40,), 55.0, dtype=view.dtype, device="cuda")
    out = buf[shift:shift + 28 * gpitch].view(28, gpitch)[:, :1000]
    check(distill(gpu, view, ids, teacher, None, g, None, 1.0, 1.0, True, out=out), x, ids, teacher, None, g, None, 1.0, 1.0, True, dtype)
    out.fill_(55.0)
    assert bool((buf == 55.0).all())


def test_in_place_padding_and_bad_ids(gpu):
    import torch

    import pssa_b200
    rng = np.random.default_rng(8)
    view, x = logits_of(rng, 28, 3000, "float32")
    ids, teacher = teacher_of(rng, x, 16, False)
    view[2, 9], view[3, 5] = float("nan"), float("nan")
    x = view.double().cpu().numpy()
    targets = targets_of(rng, x)
    g_kl, g_ce = rng.standard_normal(28).astype(np.float32), rng.standard_normal(28).astype(np.float32)
    g_kl[2] = g_ce[2] = 0.0  # padding with garbage
    apart = distill(gpu, view, ids, teacher, targets, g_kl, g_ce, 1.0, 1.0, False)
    check(apart, x, ids, teacher, targets, g_kl, g_ce, 1.0, 1.0, False, "float32")
    assert bool((apart[2][2] == 0).all()) and bool(torch.isnan(apart[2][3]).all())
    gpu.poll_status()
    placed = distill(gpu, view, ids, teacher, targets, g_kl, g_ce, 1.0, 1.0, False, out=view)
    assert torch.equal(placed[2].nan_to_num(3.0), apart[2].nan_to_num(3.0)) and np.array_equal(placed[0], apart[0], equal_nan=True)
    # an id outside the vocabulary counts as absent
    view, x = logits_of(rng, 4, 3000, "float32")
    ids, teacher = teacher_of(rng, x, 16, False)
    bad = ids.copy()
    ids[1, 3], bad[1, 3] = P.NONE, 3000
    one = distill(gpu, view, ids, teacher, None, g_kl[:4], None, 1.0, 1.0, False)
    gpu.poll_status()
    two = distill(gpu, view, bad, teacher, None, g_kl[:4], None, 1.0, 1.0, False)
    assert torch.equal(one[2], two[2]) and np.array_equal(one[0], two[0])
    with pytest.raises(pssa_b200.B200Error) as e:
        gpu.poll_status()
    assert e.value.status == 7
    far = np.full(4, 0xfffffff0, np.uint32)
    got = distill(gpu, view, ids, teacher, far, None, g_ce[:4], 1.0, 1.0, False)
    assert np.isnan(got[1]).all() and bool((got[2] == 0).all())
    with pytest.raises(pssa_b200.B200Error):
        gpu.poll_status()


def test_an_id_listed_twice_has_the_sum_of_its_entries(gpu):
    """Without and with the mass of the other ids: the split list gives the loss of the joined one less the entropy of the split, and
    its gradient."""
    rng = np.random.default_rng(3)
    view, x = logits_of(rng, 1, 4000, "float32")
    p = np.array([0.5, 0.3, 0.1], np.float64)
    g = np.ones(1, np.float32)
    for rest in (False, True):
        scale = 0.9 if rest else 1.0
        one_ids, one = np.array([[7, 900, 3999]], np.uint32), np.log(p / p.sum() * scale)[None].astype(np.float32)
        split = np.array([0.2, 0.3, 0.3, 0.1])
        two_ids, two = np.array([[7, 900, 7, 3999]], np.uint32), np.log(split / split.sum() * scale)[None].astype(np.float32)
        a = distill(gpu, view, one_ids, one, None, g, None, 1.0, 1.0, rest)
        b = distill(gpu, view, two_ids, two, None, g, None, 1.0, 1.0, rest)
        check(b, x, two_ids, two, None, g, None, 1.0, 1.0, rest, "float32")
        s = 0.5 / 0.9 * scale
        extra = s * (0.4 * np.log(0.4) + 0.6 * np.log(0.6))
        assert abs(float(b[0][0]) - float(a[0][0]) - extra) <= 1e-5  # the fp32 entries' own rounding, 2^-24 of numbers below 10 each
        assert float((a[2] - b[2]).abs().max()) <= 1e-6


@pytest.mark.parametrize("vocab", [1000, 16384, 400003])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_a_student_that_is_sure_of_the_listed_ids(gpu, vocab, dtype):
    """The other ids share a mass of e^-150 and less: below fp32's range as a probability, not as a log probability, and the
    gradient pushes it up relative to its own maximum."""
    import torch
    rng = np.random.default_rng(4)
    x = rng.standard_normal((3, vocab))
    ids = np.tile(np.array([[3, 500, 999]], np.uint32), (3, 1))
    x[0, [3, 500, 999]] += 150
    x[1, [3, 500, 999]] += 400
    x[2, [3, 500, 999]] += 20
    view = torch.from_numpy(x).to(getattr(torch, dtype)).cuda()
    x = view.double().cpu().numpy()
    teacher = np.log(np.array([[0.5, 0.3, 0.15]] * 3, np.float32))
    g = np.array([1.0, -2.0, 0.5], np.float32)
    check(distill(gpu, view, ids, teacher, None, g, None, 1.0, 1.0, True), x, ids, teacher, None, g, None, 1.0, 1.0, True, dtype)


def test_gradient_matches_differences(gpu):
    rng = np.random.default_rng(9)
    for rest in (False, True):
        view, x = logits_of(rng, 1, 30, "float32")
        ids = np.array([[3, 9, 29, 0]], np.uint32)
        teacher = np.log(np.array([[0.4, 0.3, 0.1, 0.05]], np.float32))
        targets = np.array([9], np.uint32)
        g_kl, g_ce = np.array([1.5], np.float32), np.array([0.75], np.float32)
        t = 1.7
        _, _, grad = distill(gpu, view, ids, teacher, targets, g_kl, g_ce, t, 1.0, rest)

        def f(a):
            w = P.distill(a, ids[0], teacher[0].astype(np.float64), t, 1.0, rest, 9, 1.5, 0.75, "float32")
            return 1.5 * w["kl"] + 0.75 * w["ce"]

        step = 1e-5
        for v in range(30):
            up, down = x[0].copy(), x[0].copy()
            up[v] += step
            down[v] -= step
            # truncation step^2 / 6 of a third derivative of order 10, and 64-bit rounding over the step
            assert abs(float(grad[0, v]) - (f(up) - f(down)) / (2 * step)) <= 2e-6


def test_captured_and_replayed_with_new_inputs(gpu):
    import torch
    rng = np.random.default_rng(6)
    view, _ = logits_of(rng, 28, 9000, "bfloat16")
    other, x2 = logits_of(np.random.default_rng(7), 28, 9000, "bfloat16")
    ids, teacher = teacher_of(rng, x2, 20, True)
    i, t, g = dev(ids), dev(teacher), torch.ones(28, device="cuda")
    kl, grad = torch.zeros(28, device="cuda"), torch.zeros_like(view)
    step = lambda: gpu.distill_topk_dev(view, 28, 9000, i, t, 20, kl=kl, grad_kl=g, grad_logits=grad, rest=True)  # noqa: E731
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    gpu.set_stream(side)
    try:
        with torch.cuda.stream(side):
            step()
            side.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=side, capture_error_mode="relaxed"):
                step()
            view.copy_(other)
            graph.replay()
            side.synchronize()
    finally:
        gpu.set_stream(torch.cuda.current_stream())
    want = distill(gpu, other, ids, teacher, None, np.ones(28, np.float32), None, 1.0, 1.0, True)
    assert np.array_equal(kl.cpu().numpy(), want[0], equal_nan=True) and torch.equal(grad.nan_to_num(3.0), want[2].nan_to_num(3.0))


def test_offsets_beyond_32_bits(gpu):
    import torch
    vocab, rows = 500, 3
    pitch = (1 << 31) + 8
    buf = torch.empty(2 * pitch + vocab, dtype=torch.bfloat16, device="cuda")
    rng = np.random.default_rng(1)
    x = torch.from_numpy(rng.standard_normal((rows, vocab))).to(torch.bfloat16)
    for r in range(rows):
        buf[r * pitch:r * pitch + vocab] = x[r].cuda()
    view = torch.as_strided(buf, (rows, vocab), (pitch, 1))
    ids, teacher = teacher_of(rng, x.double().numpy(), 9, True)
    g = np.ones(rows, np.float32)
    got = distill(gpu, view, ids, teacher, None, g, None, 1.0, 1.0, True, out=view)
    check(got, x.double().numpy(), ids, teacher, None, g, None, 1.0, 1.0, True, "bfloat16")
