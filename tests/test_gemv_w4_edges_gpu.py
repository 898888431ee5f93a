"""Products with 4-bit weights whose inputs pass through shared memory in several turns, groups of an odd number of chunks, and fp32
inputs to their last bit."""
import numpy as np
import pytest

import head_plain as P
from test_gemv_w4_gpu import bound_of, gpu, product, weights_of  # noqa: F401
from test_token_logprobs_gpu import close

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,rows", [("bfloat16", 16), ("float16", 9), ("float32", 4), ("float32", 5), ("bfloat16", 1)])
@pytest.mark.parametrize("n,k,group,zeros", [(20000, 8192, 128, False), (33000, 8160, 64, True), (20000, 8192, 32, False)])
def test_inputs_that_take_several_turns(gpu, dtype, rows, n, k, group, zeros):  # noqa: F811
    """Enough weight rows that no cluster splits the columns: 64 chunks through shared memory 24 or 32 at a time, the codes of the next
    turn's first chunk on their way. Sums on the device in 64 bits."""
    import torch
    gen = torch.Generator(device="cuda").manual_seed(n + rows)
    groups = -(-k // group)
    codes = torch.randint(0, 256, (n, k // 2), device="cuda", generator=gen, dtype=torch.uint8)
    scales = torch.randn(n, groups, device="cuda", generator=gen) * 0.02
    z = torch.randint(0, 16, (n, groups), device="cuda", generator=gen, dtype=torch.uint8) if zeros else None
    x = torch.randn(rows, k, device="cuda", generator=gen).to(getattr(torch, dtype))
    out = torch.full((rows, n), 3.0, device="cuda").to(x.dtype)
    gpu.gemv_w4_dev(x, rows, codes, scales, z, n, k, group, out)
    at = torch.arange(k, device="cuda") // group
    for i in range(0, n, 4096):
        q = torch.stack([codes[i:i + 4096] & 15, codes[i:i + 4096] >> 4], 2).view(-1, k).double()
        w = (q - (8.0 if z is None else z[i:i + 4096].double()[:, at])) * scales[i:i + 4096].double()[:, at]
        want, size = x.double() @ w.T, x.double().abs() @ w.abs().T
        tol = size * (2 * P.U * (k / 16 + 24)) + P.HALF_STEP[dtype] * 1.01 * want.abs() + P.TINY[dtype]  # as in bound_of, the pieces of fp32 exact
        assert bool(((out[:, i:i + 4096].double() - want).abs() <= tol).all()), i


@pytest.mark.parametrize("dtype", ["float32", "bfloat16", "float16"])
@pytest.mark.parametrize("rows,n,k,group", [(1, 70, 1920, 384), (3, 70, 2080, 640), (20, 50, 1312, 384), (1, 40, 8192, 640), (2, 5000, 4000, 1152)])
@pytest.mark.parametrize("zeros", [False, True])
def test_groups_of_an_odd_number_of_chunks(gpu, dtype, rows, n, k, group, zeros):  # noqa: F811
    """384, 640 and 1152 columns, with a shorter last group."""
    import torch
    rng = np.random.default_rng(rows + n + k)
    codes, scales, z = weights_of(rng, n, k, group, zeros, "float32")
    x = torch.from_numpy(rng.standard_normal((rows, k))).to(getattr(torch, dtype)).cuda()
    x64, w = x.double().cpu().numpy(), P.dequantize(codes, scales, z, group)
    want = x64 @ w.T
    got = product(gpu, x, codes, scales, z, group).double().cpu().numpy()
    close(got, want, bound_of(x64, w, dtype) + P.HALF_STEP[dtype] * np.abs(want) * 1.01 + P.TINY[dtype], "product")


@pytest.mark.parametrize("rows", [1, 3, 11])
@pytest.mark.parametrize("power", [-100, -30, 0, 60])
def test_an_fp32_input_is_multiplied_to_its_last_bit(gpu, rows, power):  # noqa: F811
    """One input of a row that is not 0, a scale of 1: code times input is a number of 28 bits, and the result its fp32 rounding but for
    the order of its three pieces' sum, which rounds twice. The last of 24 bits of the input shows in codes of 1."""
    import torch
    rng = np.random.default_rng(power + 200)
    n, k = 64, 256
    codes = rng.integers(0, 16, (n, k)).astype(np.uint8)
    codes[:, ::3] = 9  # a weight of 1
    scales = torch.ones(n, k // 64)
    at = rng.integers(0, k // 3, rows) * 3
    bits = (rng.integers(0, 1 << 23, rows) | 1).astype(np.uint32) | np.uint32((127 + power) << 23)  # the last bit is set
    x = np.zeros((rows, k), np.float32)
    x[np.arange(rows), at] = bits.view(np.float32)
    got = product(gpu, torch.from_numpy(x).cuda(), codes, scales, None, 64).cpu().numpy()
    for r in range(rows):
        assert np.array_equal(got[r], np.full(n, x[r, at[r]]))  # to the bit: 1 times the pieces, whose sums are cut numbers of the input
    # other weights: three exact products of up to 12 bits each, summed with two roundings
    at = at + 1
    x = np.zeros((rows, k), np.float32)
    x[np.arange(rows), at] = bits.view(np.float32)
    got = product(gpu, torch.from_numpy(x).cuda(), codes, scales, None, 64).double().cpu().numpy()
    want = x.astype(np.float64) @ (codes.astype(np.float64) - 8).T
    assert (np.abs(got - want) <= 2 * 2 * P.U * np.abs(want)).all()
