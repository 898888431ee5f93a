"""Products with 4-bit weights and the quantisation of a matrix to them, against the plain forms in 64 bits."""
import numpy as np
import pytest

import head_plain as P
from test_token_logprobs_gpu import DTYPES, close

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def gpu():
    import torch

    import pssa_b200
    d = pssa_b200.B200Dispatch(0, torch.cuda.current_stream())
    yield d
    d.close()


def weights_of(rng, n, k, group, zeros, scale):
    """Random codes, scales of both signs and some zero, zeros."""
    import torch
    groups = -(-k // group)
    codes = rng.integers(0, 16, (n, k)).astype(np.uint8)
    s = rng.standard_normal((n, groups)) * 0.02
    s[rng.random(s.shape) < 0.05] = 0.0
    scales = torch.from_numpy(s).to(getattr(torch, scale))
    z = rng.integers(0, 16, (n, groups)).astype(np.uint8) if zeros else None
    return codes, scales, z


def product(gpu, x, codes, scales, zeros, group, epilogue=0, alpha=1.0, ldo=None, out=None):
    import torch
    n, k = codes.shape
    rows = x.shape[0]
    ldo = n if ldo is None else ldo
    if out is None:
        out = torch.full((rows, ldo), 3.0, dtype=x.dtype, device="cuda")
    gpu.gemv_w4_dev(x, rows, torch.from_numpy(P.pack(codes)).cuda(), scales.cuda(), None if zeros is None else torch.from_numpy(zeros).cuda(), n, k,
                    group, out, ldx=x.stride(0), ldo=out.stride(0), epilogue=epilogue, alpha=alpha)
    torch.cuda.synchronize()
    return out


def bound_of(x, w, dtype):
    """Sums of k products in fp32, in any order and with the matrix unit's truncation (a step, not half, for each addition); fp32 inputs
    come in pieces that leave 2^-22 of them; one rounding of the result."""
    k = x.shape[1]
    size = np.abs(x) @ np.abs(w).T
    return size * (2 * P.U * (k / 16 + 24) + (2.0 ** -22 if dtype == "float32" else 0.0))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,n,k,group", [(1, 1, 32, 32), (1, 17, 64, 32), (1, 5003, 384, 128), (2, 100, 192, 128), (3, 129, 768, 64), (4, 64, 4128, 32),
                                            (5, 33, 256, 256), (8, 200, 1024, 128), (9, 50, 96, 64), (16, 300, 640, 128), (17, 48, 2048, 64), (33, 95, 384, 32),
                                            (64, 160, 768, 128), (100, 40, 544, 64), (256, 70, 256, 128), (1, 40, 8192, 1024), (7, 16, 16384, 128)])
@pytest.mark.parametrize("zeros,scale", [(False, "float32"), (True, "float16"), (True, "bfloat16")])
def test_products_match_the_plain_form(gpu, dtype, rows, n, k, group, zeros, scale):
    import torch
    rng = np.random.default_rng(rows + n + k)
    codes, scales, z = weights_of(rng, n, k, group, zeros, scale)
    x = torch.from_numpy(rng.standard_normal((rows, k)) * np.exp(rng.uniform(-3, 3, (rows, 1)))).to(getattr(torch, dtype)).cuda()
    x64, w = x.double().cpu().numpy(), P.dequantize(codes, scales, z, group)
    want = x64 @ w.T
    got = product(gpu, x, codes, scales, z, group).double().cpu().numpy()
    close(got, want, bound_of(x64, w, dtype) + P.HALF_STEP[dtype] * np.abs(want) * 1.01 + P.TINY[dtype], "product")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("epilogue", range(6))
def test_epilogues(gpu, dtype, epilogue):
    import torch
    rng = np.random.default_rng(epilogue)
    codes, scales, z = weights_of(rng, 77, 256, 64, True, "float32")
    x = torch.from_numpy(rng.standard_normal((5, 256))).to(getattr(torch, dtype)).cuda()
    x64, w = x.double().cpu().numpy(), P.dequantize(codes, scales, z, 64)
    acc = x64 @ w.T
    f = {0: lambda a: a, 1: lambda a: np.log1p(np.exp(a)), 2: lambda a: 1 / (1 + np.exp(-a)), 3: lambda a: a / (1 + np.exp(-a)), 4: lambda a: 0.25 * a,
         5: lambda a: a + 3.0}[epilogue]
    want = f(acc)
    got = product(gpu, x, codes, scales, z, 64, epilogue, 0.25).double().cpu().numpy()
    # every epilogue's slope is at most 1.1; its own arithmetic costs a few roundings of its result
    close(got, want, 1.1 * bound_of(x64, w, dtype) + (P.HALF_STEP[dtype] * 1.01 + 8 * P.U) * np.abs(want) + P.TINY[dtype], "epilogue")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shift,ldx,ldo", [(1, 257, 50), (3, 260, 51), (0, 256, 64), (8, 264, 49)])
def test_rows_may_start_anywhere_and_what_lies_between_them_stays(gpu, dtype, shift, ldx, ldo):
    import torch
    rng = np.random.default_rng(ldx)
    n, k, rows = 49, 256, 6
    codes, scales, z = weights_of(rng, n, k, 128, False, "float32")
    t = getattr(torch, dtype)
    buf = torch.full((shift + rows * ldx + 16,), float("nan"), dtype=t, device="cuda")  # what lies between the rows is not read
    x = buf[shift:shift + rows * ldx].view(rows, ldx)[:, :k]
    x.copy_(torch.from_numpy(rng.standard_normal((rows, k))))
    obuf = torch.full((shift + rows * ldo + 16,), 5.0, dtype=t, device="cuda")
    out = obuf[shift:shift + rows * ldo].view(rows, ldo)[:, :n]
    product(gpu, x, codes, scales, z, 128, out=out)
    x64, w = x.double().cpu().numpy(), P.dequantize(codes, scales, z, 128)
    want = x64 @ w.T
    close(out.double().cpu().numpy(), want, bound_of(x64, w, dtype) + P.HALF_STEP[dtype] * np.abs(want) * 1.01 + P.TINY[dtype], "product")
    out.fill_(5.0)
    assert bool((obuf == 5.0).all())


def test_fp32_inputs_of_every_size_and_values_that_are_no_numbers(gpu):
    """Inputs from the smallest normal numbers to the largest go through whole; infinities and NaNs reach their own row only, as
    infinity or NaN."""
    import torch
    rng = np.random.default_rng(4)
    codes, scales, _ = weights_of(rng, 40, 128, 128, False, "float32")
    w = P.dequantize(codes, scales, None, 128)
    for dtype, powers in (("float32", (-80, -40, 0, 40, 100)), ("bfloat16", (-80, 0, 100)), ("float16", (-8, 0, 6))):
        x = torch.from_numpy(rng.standard_normal((len(powers), 128)) * 2.0 ** np.array(powers)[:, None]).to(getattr(torch, dtype)).cuda()
        x64 = x.double().cpu().numpy()
        want = x64 @ w.T
        got = product(gpu, x, codes, scales, None, 128).double().cpu().numpy()
        fine = np.abs(want) < float(torch.finfo(x.dtype).max) * 0.9
        tol = bound_of(x64, w, dtype) + P.HALF_STEP[dtype] * np.abs(want) * 1.01 + P.TINY[dtype]
        assert fine.any() and (np.abs(got - want)[fine] <= tol[fine]).all()
        x = torch.from_numpy(rng.standard_normal((12, 128))).to(x.dtype).cuda()
        clean = product(gpu, x, codes, scales, None, 128)
        x[3, 5], x[7, 100], x[11, 0] = float("nan"), float("inf"), -float("inf")
        dirty = product(gpu, x, codes, scales, None, 128)
        good = [r for r in range(12) if r not in (3, 7, 11)]
        assert torch.equal(clean[good], dirty[good]) and bool(torch.isnan(dirty[3]).all())
        live = torch.from_numpy((codes != 8).astype(np.uint8)).bool().cuda() & (scales.cuda() != 0)
        assert not bool(torch.isfinite(dirty[7][live[:, 100]]).any()) and not bool(torch.isfinite(dirty[11][live[:, 0]]).any())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,k,group", [(1, 32, 32), (7, 96, 64), (33, 192, 128), (20, 768, 64), (16, 1024, 256), (5, 544, 32), (3, 160, 256)])
@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("scale", DTYPES)
def test_quantisation_is_the_plain_one_bit_for_bit(gpu, dtype, n, k, group, zeros, scale):
    import torch
    rng = np.random.default_rng(n * k)
    w = rng.standard_normal((n, k)) * 0.05
    w[0, :group] = 0.0  # a group of nothing
    if n > 2:
        w[1] = np.abs(w[1])  # one sign only
        w[2, :32] *= 1e-9
    w = torch.from_numpy(w).to(getattr(torch, dtype))
    codes, scales, zs = P.quantize(w.float().numpy(), group, zeros, scale)
    groups = -(-k // group)
    c = torch.full((n, k // 2), 0xAA, dtype=torch.uint8, device="cuda")
    s = torch.full((n, groups), 9.0, dtype=getattr(torch, scale), device="cuda")
    z = torch.full((n, groups), 99, dtype=torch.uint8, device="cuda") if zeros else None
    gpu.w4_quantize_dev(w.cuda(), n, k, group, c, s, z)
    torch.cuda.synchronize()
    assert torch.equal(s.cpu(), scales) and np.array_equal(c.cpu().numpy(), P.pack(codes))
    assert z is None or np.array_equal(z.cpu().numpy(), zs)


@pytest.mark.parametrize("zeros", [False, True])
def test_quantisation_of_groups_that_are_no_numbers_or_too_large(gpu, zeros):
    import torch
    w = torch.randn(4, 128)
    w[0, 3], w[1, 70], w[2, 5] = float("nan"), float("inf"), 3e38
    w[2, 6] = -3e38
    for scale in DTYPES:
        codes, scales, zs = P.quantize(w.numpy(), 64, zeros, scale)
        c = torch.zeros(4, 64, dtype=torch.uint8, device="cuda")
        s = torch.zeros(4, 2, dtype=getattr(torch, scale), device="cuda")
        z = torch.zeros(4, 2, dtype=torch.uint8, device="cuda") if zeros else None
        gpu.w4_quantize_dev(w.cuda(), 4, 128, 64, c, s, z)
        torch.cuda.synchronize()
        s = s.cpu()
        assert torch.isnan(s[0, 0]) and torch.isnan(s[1, 1]) and torch.equal(s.nan_to_num(7.0), scales.nan_to_num(7.0))
        assert np.array_equal(c.cpu().numpy(), P.pack(codes)) and (z is None or np.array_equal(z.cpu().numpy(), zs))
        x = torch.ones(1, 128, device="cuda")
        out = product(gpu, x, codes, s, zs, 64)
        assert bool(torch.isnan(out[0, :2]).all())


def test_captured_and_replayed_and_on_two_streams(gpu):
    import torch

    import pssa_b200
    rng = np.random.default_rng(12)
    codes, scales, z = weights_of(rng, 600, 1024, 128, True, "float16")
    c, s, zz = torch.from_numpy(P.pack(codes)).cuda(), scales.cuda(), torch.from_numpy(z).cuda()
    x, y = torch.randn(3, 1024, device="cuda").half(), torch.randn(3, 1024, device="cuda").half()
    want = [product(gpu, a, codes, scales, z, 128) for a in (x, y)]
    out = torch.zeros(3, 600, device="cuda").half()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    gpu.set_stream(side)
    try:
        with torch.cuda.stream(side):
            gpu.gemv_w4_dev(x, 3, c, s, zz, 600, 1024, 128, out)
            side.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=side, capture_error_mode="relaxed"):
                gpu.gemv_w4_dev(x, 3, c, s, zz, 600, 1024, 128, out)
            graph.replay()
            side.synchronize()
            assert torch.equal(out, want[0])
            x.copy_(y)
            graph.replay()
            side.synchronize()
            assert torch.equal(out, want[1])
    finally:
        gpu.set_stream(torch.cuda.current_stream())
    streams = [torch.cuda.Stream() for _ in range(2)]
    ctx = [pssa_b200.B200Dispatch(0, q) for q in streams]
    try:
        outs = [[torch.zeros_like(out) for _ in range(6)] for _ in range(2)]
        torch.cuda.synchronize()
        for i in range(6):
            for j in range(2):
                ctx[j].gemv_w4_dev(y, 3, c, s, zz, 600, 1024, 128, outs[j][i])
        torch.cuda.synchronize()
        assert all(torch.equal(o, want[1]) for group in outs for o in group)
    finally:
        for g in ctx:
            g.close()


def test_offsets_beyond_32_bits(gpu):
    """More than 2^32 weights; the last rows are the ones that count."""
    import torch
    n, k, group = (1 << 19) + 5, 8192, 128
    rng = np.random.default_rng(2)
    codes, scales, _ = weights_of(rng, 37, k, group, False, "bfloat16")
    c = torch.zeros(n, k // 2, dtype=torch.uint8, device="cuda")
    s = torch.zeros(n, k // group, dtype=torch.bfloat16, device="cuda")
    c[-37:], s[-37:] = torch.from_numpy(P.pack(codes)).cuda(), scales.cuda()
    x = torch.randn(2, k, device="cuda").bfloat16()
    out = torch.full((2, n), 9.0, device="cuda").bfloat16()
    gpu.gemv_w4_dev(x, 2, c, s, None, n, k, group, out)
    torch.cuda.synchronize()
    want = product(gpu, x, codes, scales, None, group)
    x64, w = x.double().cpu().numpy(), P.dequantize(codes, scales, None, group)
    ref = x64 @ w.T
    close(out[:, -37:].double().cpu().numpy(), ref, bound_of(x64, w, "bfloat16") + P.HALF_STEP["bfloat16"] * np.abs(ref) * 1.01, "last rows")
    assert torch.equal(out[:, -37:].abs() > 0, want.abs() > 0) and not bool(out[:, :1000].any())
