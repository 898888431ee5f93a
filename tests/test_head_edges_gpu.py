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
