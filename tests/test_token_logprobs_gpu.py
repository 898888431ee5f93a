"""Log probabilities of given tokens, their rank, entropy and alternatives, and the gradient, against the plain forms in 64 bits."""
import numpy as np
import pytest

import head_plain as P

pytestmark = pytest.mark.gpu
DTYPES = ("float32", "bfloat16", "float16")


@pytest.fixture(scope="module")
def gpu():
    import torch

    import pssa_b200
    d = pssa_b200.B200Dispatch(0, torch.cuda.current_stream())
    yield d
    d.close()


def logits_of(rng, rows, vocab, dtype, shift=0, pitch=None):
    """A device view [rows, vocab] of `dtype` that starts `shift` elements into its buffer, and its values in 64 bits. Bulk and peaks,
    and by row: masks, ties, the type's lowest value, a row of masks only."""
    import torch
    x = rng.standard_normal((rows, vocab)) * 3
    x[np.arange(rows), rng.integers(0, vocab, rows)] += 9
    for r in range(rows):
        kind = r % 12
        if kind == 1:
            x[r, rng.random(vocab) < 0.9] = -np.inf
        elif kind == 2:
            x[r] = np.round(x[r])  # many ties
        elif kind == 3:
            x[r] = 0.0
            x[r, ::3] = -0.0
        elif kind == 4:
            x[r, rng.random(vocab) < 0.5] = float(torch.finfo(getattr(torch, dtype)).min)
        elif kind == 5:
            x[r] = float(torch.finfo(getattr(torch, dtype)).min)
        elif kind == 6:
            x[r] = -np.inf
        elif kind == 7:
            x[r] = np.sort(x[r])  # ascending: every id is better than all before it
        elif kind == 8:
            x[r] = -np.inf
            x[r, vocab // 2] = 4.0
        elif kind == 9:
            x[r] = np.sort(x[r])[::-1]
        elif kind == 10:
            x[r] = x[r] * 0.01 + 300.0  # far from zero
    pitch = vocab if pitch is None else pitch
    buf = torch.full((shift + rows * pitch + 64,), 7.0, dtype=getattr(torch, dtype), device="cuda")
    view = buf[shift:shift + rows * pitch].view(rows, pitch)[:, :vocab]
    view.copy_(torch.from_numpy(x).to(view.dtype))
    return view, view.double().cpu().numpy()


def targets_of(rng, x):
    t = rng.integers(0, x.shape[1], x.shape[0]).astype(np.uint32)
    likely = rng.random(len(t)) < 0.5
    t[likely] = np.argmax(x, axis=1)[likely]
    t[9::11] = P.NONE
    return t


def dev(a):
    import torch
    return torch.from_numpy(a.view(np.int32) if a.dtype == np.uint32 else a).cuda()


def forward(gpu, view, vocab, targets, top, temperature, rank=True):
    import torch
    rows = view.shape[0]
    f = lambda *s: torch.full(s, 77.0, device="cuda")  # noqa: E731
    i = lambda *s: torch.full(s, 77, dtype=torch.int32, device="cuda")  # noqa: E731
    out = dict(logprob=f(rows), rank=i(rows), entropy=f(rows), stats=f(rows, 2), ids=i(rows, top), top=f(rows, top))
    gpu.token_logprobs_dev(view, rows, vocab, dev(targets), out["logprob"], out["rank"], out["entropy"], out["stats"], top,
                           out["ids"] if top else None, out["top"] if top else None, temperature=temperature, ld=view.stride(0))
    torch.cuda.synchronize()
    return {k: (v.cpu().numpy().view(np.uint32) if v.dtype == torch.int32 else v.cpu().numpy()) for k, v in out.items()}


def close(got, want, tol, what):
    """Equal where `want` is no number, within `tol` otherwise. No result is wider than fp32: a number beyond its range (a type's lowest
    value over a temperature of 0.7 is -4.9e38, fp32 ends at 3.4028236e38) rounds to infinity."""
    got, want, tol = np.asarray(got, np.float64), np.asarray(want, np.float64), np.broadcast_to(tol, np.shape(want))
    want = np.where(np.abs(want) > 3.4028236e38, np.copysign(np.inf, want), want)
    fine = np.isfinite(want)
    assert np.array_equal(got[~fine], want[~fine], equal_nan=True), (what, got[~fine][:5], want[~fine][:5])
    off = np.abs(got[fine] - want[fine]) - tol[fine]
    assert not off.size or off.max() <= 0, (what, float(off.max()), got[fine][off.argmax()], want[fine][off.argmax()])


def check_forward(got, x, targets, top, temperature):
    for r in range(len(x)):
        w = P.logprobs(x[r], int(targets[r]), temperature, top)
        z_t = 0.0
        if targets[r] < x.shape[1] and np.isfinite(x[r, targets[r]]) and P.has_distribution(x[r]):
            z_t = abs((x[r, targets[r]] - x[r].max()) / temperature)
        close(got["logprob"][r], w["logprob"], w["tol"] + P.U * (4 * z_t + 2 * abs(w["logprob"]) if np.isfinite(w["logprob"]) else 0), f"logprob {r}")
        assert got["rank"][r] == w["rank"], (r, got["rank"][r], w["rank"])
        close(got["entropy"][r], w["entropy"], w["tol_h"], f"entropy {r}")
        close(got["stats"][r, 0], w["stats"][0], 0.0, f"max {r}")
        close(got["stats"][r, 1], w["stats"][1], w["tol"], f"log sum {r}")
        assert np.array_equal(got["ids"][r], np.asarray(w["ids"], np.uint32)), (r, got["ids"][r][:8], w["ids"][:8])
        lp = np.asarray(w["top"], np.float64)
        close(got["top"][r], lp, w["tol"] + P.U * 6 * (np.abs(np.where(np.isfinite(lp), lp, 0.0)) + w["tol"] + abs(w["stats"][1]) if np.isfinite(w["stats"][1]) else 0), f"top {r}")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,vocab,top", [(1, 1, 1), (1, 2, 3), (13, 7, 8), (12, 33, 33), (24, 255, 0), (25, 1000, 20), (12, 5003, 64),
                                            (1, 8192, 5), (3, 16384, 20), (150, 4099, 5), (600, 1031, 10), (12, 131072, 20), (1, 200003, 64), (1300, 777, 10), (1300, 300, 64)])
def test_forward_matches_the_plain_form(gpu, dtype, rows, vocab, top):
    rng = np.random.default_rng(rows * 7 + vocab)
    view, x = logits_of(rng, rows, vocab, dtype)
    targets = targets_of(rng, x)
    for temperature in (1.0, 0.7):
        check_forward(forward(gpu, view, vocab, targets, top, temperature), x, targets, top, temperature)
    gpu.poll_status()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shift,pitch", [(0, 1003), (1, 1001), (3, 1024), (5, 1008), (8, 1000)])
def test_rows_may_start_anywhere(gpu, dtype, shift, pitch):
    rng = np.random.default_rng(pitch)
    view, x = logits_of(rng, 36, 1000, dtype, shift, pitch)
    targets = targets_of(rng, x)
    check_forward(forward(gpu, view, 1000, targets, 9, 1.3), x, targets, 9, 1.3)


def test_rows_without_a_distribution_and_bad_targets(gpu):
    import torch

    import pssa_b200
    rng = np.random.default_rng(2)
    view, x = logits_of(rng, 8, 700, "float32")
    view[0, 5], view[1, 699], view[2, 0], view[3, 650] = np.nan, np.inf, -np.nan, np.nan
    view[3, 1:600] = -np.inf
    x = view.double().cpu().numpy()
    targets = np.array([3, 699, 5, P.NONE, 700, 0xfffffffe, 1, 699], np.uint32)
    got = forward(gpu, view, 700, targets, 6, 1.0)
    check_forward(got, x, targets, 6, 1.0)
    assert np.isnan(got["logprob"][[0, 1, 2, 4, 5]]).all() and got["logprob"][3] == 0.0
    with pytest.raises(pssa_b200.B200Error) as e:
        gpu.poll_status()
    assert e.value.status == 7
    gpu.poll_status()  # once
    assert torch.isnan(view[0, 5])


@pytest.mark.parametrize("rows,vocab", [(1, 40000), (3, 70001), (200, 3000)])
def test_a_row_of_almost_no_numbers_fills_its_alternatives(gpu, rows, vocab):
    """Fewer logits that can be compared than alternatives asked for, in one CTA and in a cluster of them."""
    import torch
    view = torch.full((rows, vocab), float("nan"), device="cuda")
    view[:, 5:9] = 1.0
    got = forward(gpu, view, vocab, np.full(rows, 6, np.uint32), 20, 1.0)
    assert (got["ids"] == P.NONE).all() and np.isnan(got["top"]).all() and np.isnan(got["logprob"]).all() and not got["rank"].any()


@pytest.mark.parametrize("asked", ["logprob", "rank", "entropy", "stats", "top"])
def test_each_result_alone_has_the_same_bits(gpu, asked):
    import torch
    rng = np.random.default_rng(5)
    view, x = logits_of(rng, 24, 3001, "bfloat16")
    targets = targets_of(rng, x)
    whole = forward(gpu, view, 3001, targets, 7, 0.9)
    rows = 24
    if asked == "top":
        ids, top = torch.zeros(rows, 7, dtype=torch.int32, device="cuda"), torch.zeros(rows, 7, device="cuda")
        gpu.token_logprobs_dev(view, rows, 3001, top_n=7, top_ids=ids, top_logprobs=top, temperature=0.9)
        torch.cuda.synchronize()
        assert np.array_equal(ids.cpu().numpy().view(np.uint32), whole["ids"]) and np.array_equal(top.cpu().numpy(), whole["top"], equal_nan=True)
        return
    out = torch.zeros(whole[asked].shape, dtype=torch.int32 if asked == "rank" else torch.float32, device="cuda")
    gpu.token_logprobs_dev(view, rows, 3001, dev(targets) if asked in ("logprob", "rank") else None, temperature=0.9, **{asked: out})
    torch.cuda.synchronize()
    assert np.array_equal(out.cpu().numpy().view(np.uint32), whole[asked].view(np.uint32))


@pytest.mark.parametrize("vocab,top", [(70000, 64), (70000, 5), (16384, 64)])
def test_alternatives_that_lie_in_one_thread_s_share(gpu, vocab, top):
    """The best ids at every distance at which a CTA's threads may stride over a row: however ids are dealt out, some row here puts
    all of the best into one thread's hands, in ascending or descending order."""
    import torch
    strides = [1, 2, 4, 8, 32, 64, 128, 256, 512, 1024, 2048, 4096, 8192]
    for dtype in ("float32", "bfloat16"):
        x = np.full((2 * len(strides), vocab), -50.0)
        x += np.random.default_rng(1).standard_normal(vocab)
        for i, s in enumerate(strides):
            at = np.arange(3, vocab, s)[:2000]
            x[2 * i, at] = np.linspace(0, 30, len(at))
            x[2 * i + 1, at] = np.linspace(30, 0, len(at))
        view = torch.from_numpy(x).to(getattr(torch, dtype)).cuda()
        x = view.double().cpu().numpy()
        targets = np.full(len(x), 3, np.uint32)
        check_forward(forward(gpu, view, vocab, targets, top, 1.0), x, targets, top, 1.0)
        check_forward(forward(gpu, view[:1], vocab, targets[:1], top, 1.0), x[:1], targets[:1], top, 1.0)
        if vocab <= 16384:  # many short rows take smaller CTAs
            many = view.repeat(50, 1)
            got = forward(gpu, many, vocab, np.full(len(many), 3, np.uint32), top, 1.0)
            check_forward({k: v[:len(x)] for k, v in got.items()}, x, targets, top, 1.0)
            assert all(np.array_equal(v, np.tile(v[:len(x)], (50,) + (1,) * (v.ndim - 1))) for v in got.values())


# ---- gradient

def gradient(gpu, view, vocab, targets, temperature, g_lp, g_h, fwd=None, grad=None):
    import torch
    rows = view.shape[0]
    fwd = fwd or forward(gpu, view, vocab, targets, 0, temperature)
    grad = torch.full((rows, vocab), 99.0, dtype=view.dtype, device="cuda") if grad is None else grad
    gpu.token_logprobs_grad_dev(view, rows, vocab, dev(targets), dev(fwd["stats"]), grad, None if g_lp is None else dev(g_lp),
                                dev(fwd["entropy"]), None if g_h is None else dev(g_h), temperature=temperature, ld=view.stride(0),
                                ld_grad=grad.stride(0))
    torch.cuda.synchronize()
    return grad, fwd


def check_gradient(got, x, targets, temperature, g_lp, g_h, fwd, dtype):
    for r in range(len(x)):
        want, tol = P.logprob_grad(x[r], int(targets[r]), temperature, fwd["stats"][r].astype(np.float64), float(fwd["entropy"][r]),
                                   0.0 if g_lp is None else float(g_lp[r]), 0.0 if g_h is None else float(g_h[r]), dtype)
        close(got[r], want, tol, f"gradient {r}")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,vocab", [(1, 1), (13, 9), (24, 1000), (25, 1003), (12, 5003), (1, 16384), (3, 131072), (400, 2048)])
def test_gradient_matches_the_formula(gpu, dtype, rows, vocab):
    rng = np.random.default_rng(rows + vocab)
    view, x = logits_of(rng, rows, vocab, dtype)
    targets = targets_of(rng, x)
    g_lp, g_h = rng.standard_normal(rows).astype(np.float32), rng.standard_normal(rows).astype(np.float32)
    g_lp[2::7] = 0.0
    g_h[2::5] = 0.0
    for temperature, a, b in ((1.0, g_lp, g_h), (0.6, g_lp, None), (2.0, None, g_h)):
        grad, fwd = gradient(gpu, view, vocab, targets, temperature, a, b)
        check_gradient(grad.double().cpu().numpy(), x, targets, temperature, a, b, fwd, dtype)
    gpu.poll_status()


@pytest.mark.parametrize("shift,pitch,gpitch", [(1, 1001, 1000), (4, 1008, 1001), (0, 1000, 1016), (3, 1003, 1003)])
@pytest.mark.parametrize("dtype", DTYPES)
def test_gradient_of_rows_that_start_anywhere_leaves_what_lies_between_them(gpu, dtype, shift, pitch, gpitch):
    import torch
    rng = np.random.default_rng(pitch)
    view, x = logits_of(rng, 24, 1000, dtype, shift, pitch)
    targets = targets_of(rng, x)
    g = rng.standard_normal(24).astype(np.float32)
    buf = torch.full((24 * gpitch + 40,), 55.0, dtype=view.dtype, device="cuda")
    out = buf[shift:shift + 24 * gpitch].view(24, gpitch)[:, :1000]
    _, fwd = gradient(gpu, view, 1000, targets, 1.0, g, g, grad=out)
    check_gradient(out.double().cpu().numpy(), x, targets, 1.0, g, g, fwd, dtype)
    out.fill_(55.0)
    assert bool((buf == 55.0).all())


def test_gradient_in_place_and_rows_that_are_left_out(gpu):
    import torch
    rng = np.random.default_rng(8)
    view, x = logits_of(rng, 24, 1500, "bfloat16")
    view[4, 7] = float("nan")  # padding with garbage: its weights are zero
    targets = targets_of(rng, x)
    g_lp, g_h = rng.standard_normal(24).astype(np.float32), rng.standard_normal(24).astype(np.float32)
    g_lp[4] = g_h[4] = 0.0
    apart, fwd = gradient(gpu, view, 1500, targets, 1.0, g_lp, g_h)
    assert bool((apart[4] == 0).all()) and bool((apart[6] == 0).all())  # row 6: masked ids only
    gradient(gpu, view, 1500, targets, 1.0, g_lp, g_h, fwd=fwd, grad=view)
    assert torch.equal(view, apart)
    targets[0] = 1500
    _, _ = gradient(gpu, apart, 1500, targets, 1.0, g_lp, None, fwd=fwd)
    import pssa_b200
    with pytest.raises(pssa_b200.B200Error):
        gpu.poll_status()


def test_gradient_matches_differences(gpu):
    """Central differences of the 64-bit forward form: the gradient is of what the forward call computes."""
    rng = np.random.default_rng(3)
    view, x = logits_of(rng, 1, 40, "float32")
    targets, temperature = np.array([11], np.uint32), 0.8
    g_lp, g_h = np.array([1.25], np.float32), np.array([-0.5], np.float32)
    grad, _ = gradient(gpu, view, 40, targets, temperature, g_lp, g_h)
    f = lambda a: 1.25 * P.logprobs(a, 11, temperature, 0)["logprob"] - 0.5 * P.logprobs(a, 11, temperature, 0)["entropy"]  # noqa: E731
    step = 1e-5
    for v in range(40):
        up, down = x[0].copy(), x[0].copy()
        up[v] += step
        down[v] -= step
        # truncation step^2 / 6 of a third derivative of order 10, and 64-bit rounding over the step
        assert abs(float(grad[0, v]) - (f(up) - f(down)) / (2 * step)) <= 1e-6


# ---- how it is called

def test_offsets_beyond_32_bits(gpu):
    """A pitch that puts the last row more than 2^32 elements behind the first."""
    import torch
    vocab, rows = 500, 3
    pitch = (1 << 31) + 8
    buf = torch.empty(2 * pitch + vocab, dtype=torch.bfloat16, device="cuda")
    rng = np.random.default_rng(1)
    x = torch.from_numpy(rng.standard_normal((rows, vocab))).to(torch.bfloat16)
    for r in range(rows):
        buf[r * pitch:r * pitch + vocab] = x[r].cuda()
    view = torch.as_strided(buf, (rows, vocab), (pitch, 1))
    targets = np.array([1, 2, 3], np.uint32)
    got = forward(gpu, view, vocab, targets, 3, 1.0)
    check_forward(got, x.double().numpy(), targets, 3, 1.0)
    g = np.ones(rows, np.float32)
    gradient(gpu, view, vocab, targets, 1.0, g, None, fwd=got, grad=view)
    check_gradient(view.double().cpu().numpy(), x.double().numpy(), targets, 1.0, g, None, got, "bfloat16")


def test_captured_and_replayed_on_another_stream_with_new_inputs(gpu):
    import torch
    rng = np.random.default_rng(6)
    view, x = logits_of(rng, 24, 4000, "float32")
    other, x2 = logits_of(np.random.default_rng(7), 24, 4000, "float32")
    targets = targets_of(rng, x)
    t = dev(targets)
    out = dict(logprob=torch.zeros(24, device="cuda"), entropy=torch.zeros(24, device="cuda"), stats=torch.zeros(24, 2, device="cuda"),
               top_ids=torch.zeros(24, 8, dtype=torch.int32, device="cuda"), top_logprobs=torch.zeros(24, 8, device="cuda"))
    grad = torch.zeros_like(view)
    g = torch.ones(24, device="cuda")

    def step():
        gpu.token_logprobs_dev(view, 24, 4000, t, top_n=8, **out)
        gpu.token_logprobs_grad_dev(view, 24, 4000, t, out["stats"], grad, grad_logprob=g)

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
    want = forward(gpu, other, 4000, targets, 8, 1.0)
    for a, b in (("logprob", "logprob"), ("entropy", "entropy"), ("stats", "stats"), ("top_logprobs", "top")):
        assert np.array_equal(out[a].cpu().numpy(), want[b], equal_nan=True)
    again, _ = gradient(gpu, other, 4000, targets, 1.0, np.ones(24, np.float32), None, fwd=want)
    assert torch.equal(grad.nan_to_num(5.0), again.nan_to_num(5.0))


def test_two_contexts_on_two_streams_at_once(gpu):
    """Calls that overlap on the device share nothing."""
    import torch

    import pssa_b200
    streams = [torch.cuda.Stream() for _ in range(2)]
    ctx = [pssa_b200.B200Dispatch(0, s) for s in streams]
    try:
        rng = np.random.default_rng(4)
        data = [logits_of(rng, 48, 20000, "bfloat16") for _ in range(2)]
        targets = [targets_of(rng, x) for _, x in data]
        outs = [[torch.zeros(48, device="cuda") for _ in range(8)] for _ in range(2)]
        t = [dev(a) for a in targets]
        torch.cuda.synchronize()
        for i in range(8):
            for c in range(2):
                ctx[c].token_logprobs_dev(data[c][0], 48, 20000, t[c], logprob=outs[c][i])
        torch.cuda.synchronize()
        for c in range(2):
            for o in outs[c]:
                assert torch.equal(o.nan_to_num(9.0), outs[c][0].nan_to_num(9.0))
            got = forward(ctx[c], data[c][0], 20000, targets[c], 0, 1.0)
            assert np.array_equal(got["logprob"], outs[c][0].cpu().numpy(), equal_nan=True)
    finally:
        for c in ctx:
            c.close()


def test_model_scores_with_log_probabilities():
    """`PSSAModel.score_logprobs` beside `score` of the same text: the target's loss, and results of the logits that `score` returns;
    more positions than a pass holds, positions without a target, refusals."""
    import oracle as O
    import pssa_b200
    from helpers import fill_synthetic, upload
    gpu = pssa_b200.B200Dispatch(0)
    om = fill_synthetic(O.Model.new(2, 203, 32, 16, 8, 16, tau_mem=0.1, seed=5), 5)
    for precision in (0, 1):
        m = pssa_b200.PSSAModel(gpu, 2, 203, 32, 16, 8, 16, tau_mem=0.1, precision=precision)
        upload(om, m)
        m.set_max_rows(64)
        rng = np.random.default_rng(1)
        ids, targets = rng.integers(0, 203, 150), rng.integers(0, 203, 150)
        start = m.copy_recurrent_state_to(0)
        _, loss, logits = m.score(ids, targets, want_logits=True)
        end = m.copy_recurrent_state_to(0)
        m.copy_recurrent_state_from(start, 0)
        shown = targets.copy()
        shown[::10] = -1
        got = m.score_logprobs(ids, shown, top=6, temperature=1.0)
        assert np.array_equal(m.copy_recurrent_state_to(0), end)
        has = shown >= 0
        assert np.max(np.abs(got["logprob"][has] + loss[has])) <= 1e-5 * max(1.0, float(loss.max())) and not got["logprob"][~has].any()
        t = np.where(has, shown, 0xffffffff).astype(np.uint32)
        check = dict(got, ids=got["top_ids"].astype(np.uint32), top=got["top_logprobs"], stats=None)
        for r in range(150):
            w = P.logprobs(logits[r].astype(np.float64), int(t[r]), 1.0, 6)
            assert check["rank"][r] == w["rank"] and np.array_equal(check["ids"][r], np.asarray(w["ids"], np.uint32))
            assert abs(check["entropy"][r] - w["entropy"]) <= w["tol_h"]
            assert np.max(np.abs(check["top"][r] - w["top"])) <= w["tol"] + P.U * 40
        assert m.score_logprobs(ids[:5])["logprob"] is None
        wide = m.score_logprobs(ids[:3], top=64)
        assert wide["top_ids"].shape == (3, 64) and (np.diff(wide["top_logprobs"], axis=1) <= 0).all()
        for bad in (dict(ids=[203]), dict(ids=[1], targets=[203]), dict(ids=[]), dict(ids=[1], top=65), dict(ids=[1], temperature=0.0), dict(ids=[1], stream=3)):
            with pytest.raises(pssa_b200.B200Error):
                m.score_logprobs(**bad)
        m.close()
    gpu.close()
