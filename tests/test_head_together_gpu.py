"""A head in 4 bits, its answers and its distance from the full head, as they are used together: the full head's logits by the dense
product, their best ids with log probabilities, the head quantised, the student's logits by the 4-bit product, divergence and gradient,
and the student's own log probabilities with their gradient; on one stream with no wait between the calls, and as one captured graph."""
import numpy as np
import pytest

import head_plain as P
from test_token_logprobs_gpu import close, dev

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("vocab,d,rows,group", [(8192, 192, 6, 64), (5003, 384, 9, 128)])
@pytest.mark.parametrize("captured", [False, True])
def test_a_head_in_4_bits_against_the_full_one(vocab, d, rows, group, captured):
    import torch

    import pssa_b200
    from pssa_b200 import _native as N
    gpu = pssa_b200.B200Dispatch(0, torch.cuda.current_stream())
    rng = np.random.default_rng(vocab)
    w = torch.from_numpy(rng.standard_normal((vocab, d)).astype(np.float32) * 0.2).cuda()
    x = torch.from_numpy(rng.standard_normal((rows, d)).astype(np.float32)).cuda()
    k, groups = 12, -(-d // group)
    f = lambda *s: torch.zeros(*s, device="cuda")  # noqa: E731
    i = lambda *s: torch.zeros(*s, dtype=torch.int32, device="cuda")  # noqa: E731
    full, student, grad, policy = f(rows, vocab), f(rows, vocab), f(rows, vocab), f(rows, vocab)
    codes, scales = torch.zeros(vocab, d // 2, dtype=torch.uint8, device="cuda"), f(vocab, groups)
    ids, top, kl, ce, stats, lp, h = i(rows, k), f(rows, k), f(rows), f(rows), f(rows, 2), f(rows), f(rows)
    targets = dev(rng.integers(0, vocab, rows).astype(np.uint32))
    g = torch.full((rows,), 1.0 / rows, device="cuda")

    def run():
        gpu.gemm_xwt_dev(x, w, rows, vocab, d, full, precision=N.PRECISION_FP32_EXACT)
        gpu.token_logprobs_dev(full, rows, vocab, top_n=k, top_ids=ids, top_logprobs=top)
        gpu.w4_quantize_dev(w, vocab, d, group, codes, scales)
        gpu.gemv_w4_dev(x, rows, codes, scales, None, vocab, d, group, student)
        gpu.token_logprobs_dev(student, rows, vocab, targets, logprob=lp, entropy=h, stats=stats)
        gpu.token_logprobs_grad_dev(student, rows, vocab, targets, stats, policy, grad_logprob=g, entropy=h, grad_entropy=g)
        gpu.distill_topk_dev(student, rows, vocab, ids, top, k, kl=kl, grad_kl=g, targets=targets, ce=ce, grad_ce=g, grad_logits=grad, rest=True)

    if captured:
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        gpu.set_stream(side)
        with torch.cuda.stream(side):
            run()
            side.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=side, capture_error_mode="relaxed"):
                run()
            for t in (full, student, grad, policy, codes, scales, ids, top, kl, ce, stats, lp, h):
                t.zero_()
            graph.replay()
            side.synchronize()
        gpu.set_stream(torch.cuda.current_stream())
    else:
        run()
        torch.cuda.synchronize()
    gpu.poll_status()
    # each step from its own inputs
    q, s, _ = P.quantize(w.cpu().numpy()[:40], group, False, "float32")
    assert np.array_equal(codes[:40].cpu().numpy(), P.pack(q)) and torch.equal(scales[:40].cpu(), s)
    code = codes.cpu().numpy()
    unpacked = np.stack([code & 15, code >> 4], 2).reshape(vocab, d)
    w4, x64 = P.dequantize(unpacked, scales.cpu(), None, group), x.double().cpu().numpy()
    want = x64 @ w4.T
    close(student.double().cpu().numpy(), want, (np.abs(x64) @ np.abs(w4).T) * (2 * P.U * (d / 16 + 24) + 2.0 ** -22), "student")
    s64, f64 = student.double().cpu().numpy(), full.double().cpu().numpy()
    best, probs = ids.cpu().numpy().view(np.uint32), top.cpu().numpy().astype(np.float64)
    t = targets.cpu().numpy()
    for r in range(rows):
        a = P.logprobs(f64[r], P.NONE, 1.0, k)
        assert np.array_equal(best[r], np.asarray(a["ids"], np.uint32))
        close(probs[r], a["top"], a["tol"] + P.U * 60, "teacher")
        b = P.distill(s64[r], best[r], probs[r], 1.0, 1.0, True, int(t[r]), float(g[r]), float(g[r]), "float32")
        close(float(kl[r]), b["kl"], b["tol"], "kl")
        close(float(ce[r]), b["ce"], b["tol_ce"], "ce")
        close(grad[r].double().cpu().numpy(), b["grad"], b["tol_g"], "gradient")
        c = P.logprobs(s64[r], int(t[r]), 1.0, 0)
        close(float(lp[r]), c["logprob"], c["tol"] + P.U * 6 * abs(c["logprob"]), "log probability")
        e, tol = P.logprob_grad(s64[r], int(t[r]), 1.0, stats[r].double().cpu().numpy(), float(h[r]), float(g[r]), float(g[r]), "float32")
        close(policy[r].double().cpu().numpy(), e, tol, "policy gradient")
    gpu.close()


@pytest.mark.parametrize("captured", [False, True])
def test_inputs_that_another_stream_or_a_copy_has_just_written(captured):
    """Each operator after a wait for another stream's kernel, and after a copy: the launch must wait for both. 30 rounds of inputs
    that change; the results are those of the same calls with the device idle before each."""
    import torch

    import pssa_b200
    side, other = torch.cuda.Stream(), torch.cuda.Stream()
    gpu = pssa_b200.B200Dispatch(0, side)
    rng = np.random.default_rng(5)
    rows, vocab, d, k, group = 64, 8192, 256, 6, 64
    rand = lambda *s: torch.from_numpy(rng.standard_normal(s).astype(np.float32)).cuda()  # noqa: E731
    a, b, w, x = rand(rows, vocab), rand(rows, vocab), rand(vocab, d), rand(2, d)
    targets = dev(rng.integers(0, vocab, rows).astype(np.uint32))
    logits, w2 = torch.zeros_like(a), torch.zeros_like(w)
    f = lambda *s: torch.zeros(*s, device="cuda")  # noqa: E731
    ids, top, lp, stats, grad = torch.zeros(rows, k, dtype=torch.int32, device="cuda"), f(rows, k), f(rows), f(rows, 2), f(rows, vocab)
    kl, dgrad, out = f(rows), f(rows, vocab), f(2, vocab)
    codes, scales = torch.zeros(vocab, d // 2, dtype=torch.uint8, device="cuda"), f(vocab, d // group)
    results = (ids, top, lp, stats, grad, kl, dgrad, codes, scales, out)
    g = torch.full((rows,), 1.0 / rows, device="cuda")
    torch.cuda.synchronize()

    def step(wait):
        def joined(write):
            other.wait_stream(side)
            with torch.cuda.stream(other):
                write()
            side.wait_stream(other)
            wait()
        joined(lambda: torch.mul(a, 0.5, out=logits))
        gpu.token_logprobs_dev(logits, rows, vocab, targets, logprob=lp, stats=stats, top_n=k, top_ids=ids, top_logprobs=top)
        wait()
        gpu.token_logprobs_grad_dev(logits, rows, vocab, targets, stats, grad, grad_logprob=g)
        wait()
        logits.copy_(b)  # on the operators' stream, behind the gradient that reads it
        wait()
        gpu.distill_topk_dev(logits, rows, vocab, ids, top, k, kl=kl, grad_kl=g, grad_logits=dgrad, rest=True)
        joined(lambda: torch.add(w, a[0, :d], out=w2))
        gpu.w4_quantize_dev(w2, vocab, d, group, codes, scales)
        wait()
        gpu.gemv_w4_dev(x, 2, codes, scales, None, vocab, d, group, out)
        wait()
        a.mul_(-0.9).add_(b, alpha=0.1)
        wait()

    start = a.clone()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        for _ in range(30):
            step(torch.cuda.synchronize)
        want = [t.clone() for t in results]
        a.copy_(start)
        torch.cuda.synchronize()
        if captured:
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=side, capture_error_mode="relaxed"):
                step(lambda: None)
            for _ in range(30):
                graph.replay()
        else:
            for _ in range(30):
                step(lambda: None)
    torch.cuda.synchronize()
    gpu.poll_status()
    for t, e in zip(results, want):
        assert torch.equal(t, e)
    gpu.close()
