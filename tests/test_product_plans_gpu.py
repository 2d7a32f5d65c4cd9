"""The product over weight planes on every kernel and plan that its rule chooses from: sums of small integers, which fp32 holds, so
that results are compared bit for bit; and the activations at values known to the bit."""
import ctypes
import math
import random

import pytest
import torch

import decoder_reference as ref
from test_decoder_gpu import BF, FF, HF, product

pytestmark = pytest.mark.gpu

# (blocks that share a tile, rows of X in it, blocks that share its K): sizes that take this plan, ragged ones among them
PLANS = {
    (0, 8, 1): [(1, 300, 500), (8, 129, 128)],
    (0, 8, 2): [(3, 70, 600), (8, 1000, 1001)],
    (0, 8, 4): [(5, 100, 1600)],
    (0, 8, 8): [(8, 333, 4100), (1, 17, 9000)],
    (1, 32, 1): [(20, 4096, 130), (300, 1000, 1000)],
    (1, 32, 2): [(394, 557, 2461)],
    (1, 32, 4): [(258, 133, 1475), (100, 900, 2048)],
    (1, 32, 8): [(9, 70, 1000), (48, 130, 4096)],
    (1, 64, 1): [(400, 2337, 500), (64, 32003, 260)],
    (1, 64, 2): [(627, 780, 4261)],
    (1, 64, 4): [(549, 140, 2189), (33, 4000, 8000)],
    (1, 64, 8): [(232, 131, 2775)],
    (1, 128, 1): [(513, 2300, 264), (700, 6000, 640)],
    (1, 128, 2): [(719, 784, 8668)],
    (1, 128, 4): [(363, 779, 3798)],
    (1, 128, 8): [(389, 287, 5917)],
    (2, 256, 1): [(400, 6000, 3000), (129, 30000, 1536), (1587, 1665, 3114)],
}


def plan(M, N, K):
    from apnn_tc_b200 import _cabi
    out = [ctypes.c_int() for _ in range(3)]
    assert _cabi.lib().apnn_linear_planes_plan(M, N, K, *(ctypes.addressof(o) for o in out)) == 0
    return tuple(o.value for o in out)


def test_every_plan_has_its_sizes(cuda_device):
    """The sizes below take the plans that they stand under, and no size takes a plan that none of them takes."""
    for want, sizes in PLANS.items():
        for s in sizes:
            assert plan(*s) == want, s
    rng = random.Random(0)
    for most in ((64, 4096, 16384), (4096, 32768, 16384), (65536, 262144, 65536)):
        for _ in range(20000):
            s = [int(2 ** rng.uniform(0, math.log2(m))) for m in most]
            assert plan(*s) in PLANS, s


def exact(M, N, K, wbits, dtype, zero, seed=0, keep=None):
    """x of integers up to 8 and levels less `zero` (a multiple of 1/2): sums below 2^23 halves; what lies behind a row of x is NaN."""
    assert 8 * 15 * 2 * (K if keep is None else keep) < 2 ** 24
    g = torch.Generator(device="cuda").manual_seed(seed + M + N + K)
    buf = torch.full((M, (K + 7) // 8 * 8 + 8 * (M % 2)), float("nan"), dtype=dtype, device="cuda")
    x = torch.randint(-8, 9, (M, K), generator=g, device="cuda")
    if keep is not None:
        x[:, torch.randperm(K, generator=g, device="cuda")[keep:]] = 0
    buf[:, :K] = x
    levels = torch.randint(0, 2 ** wbits, (N, K), generator=g, device="cuda")
    sums = x.double() @ (levels.double() - zero).t()
    return buf[:, :K], levels, sums


def planes_of(levels, wbits):
    import apnn_tc_b200 as ap
    return ap.Bit_compression(levels.to(torch.int32).contiguous(), wbits)


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("wbits", [1, 2, 3, 4])
@pytest.mark.parametrize("size", [s for sizes in PLANS.values() for s in sizes], ids=str)
def test_integer_sums(cuda_device, size, wbits, dtype):
    import apnn_tc_b200 as ap
    M, N, K = size
    zero = (2 ** wbits - 1) / 2
    x, levels, sums = exact(M, N, K, wbits, dtype, zero)
    planes = planes_of(levels, wbits)
    if M * N * K < 10 ** 8:
        assert torch.equal(planes.cpu(), ref.planes_of(levels, wbits))
    scale = torch.pow(2.0, -(torch.arange(N, device="cuda") % 5).float())
    got = ap.linear_planes(x, planes, scale, zero=zero, out_dtype=FF)
    assert torch.equal(got.double(), sums * scale.double())
    bias = (torch.arange(N, device="cuda") % 7).float()
    residual = torch.randint(-50, 50, (M, N), device="cuda").to(dtype)
    got = ap.linear_planes(x, planes, scale, zero=zero, bias=bias, activation="relu", residual=residual)
    want = ((sums * scale.double() + bias.double()).clamp(min=0).float() + residual.float()).to(dtype)      # exact before the one rounding
    assert torch.equal(got, want)


@pytest.mark.parametrize("act", ["none", "silu", "gelu", "gelu_tanh"])
@pytest.mark.parametrize("out", [None, FF])
def test_pair_epilogues(cuda_device, act, out):
    """What the pair of blocks does after its sums, rows and columns ragged, odd strides, the residual in place."""
    product(5, 1587, 1665, 3114, 2, BF, act, True, True, out, pad=8)
    product(6, 400, 6000, 3000, 3, HF, act, False, False, FF)


@pytest.mark.parametrize("M,N,K", [(400, 6000, 3000), (129, 30000, 1536)])
def test_pair_residual_in_place_and_repeated(cuda_device, M, N, K):
    import apnn_tc_b200 as ap
    x, levels, sums = exact(M, N, K, 4, BF, 7.5)
    planes, scale = planes_of(levels, 4), torch.full((N,), 0.125, device="cuda")
    for shift in (0, 1):      # pairs of columns stored together or not
        wide = torch.randint(-50, 50, (M, N + 5), device="cuda").to(BF)
        start = wide.clone()
        flag = torch.full((1,), 7, dtype=torch.int32, device="cuda")
        view = wide[:, shift:shift + N]
        ap.linear_planes(x, planes, scale, zero=7.5, residual=view, out=view, status_flag=flag)
        want = ((sums * 0.125).float() + start[:, shift:shift + N].float()).to(BF)
        assert torch.equal(view, want) and int(flag.item()) == 0
        assert torch.equal(wide[:, :shift], start[:, :shift]) and torch.equal(wide[:, shift + N:], start[:, shift + N:])


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("M,N,K", [(1, 200, 40), (8, 200, 40), (12, 200, 40), (40, 333, 64), (200, 300, 64), (400, 6000, 3000)])
def test_activations_apart(cuda_device, M, N, K, dtype):
    """fp32 results at values v known to the bit, each activation to its own roundings: v (|v| + 4) 2^-23 of the logistic function by one
    exponential (2 units of 2^-23, of an argument off by |v| 2^-23) and one reciprocal; for gelu_tanh of an argument u off by 7 half
    units of itself; |v| 2^-22 of erf (2 units of 2^-24 of itself and its argument's rounding).  The two gelus are hundreds of these apart."""
    import apnn_tc_b200 as ap
    x, levels, sums = exact(M, N, K, 4, dtype, 7.5, keep=40)
    scale = torch.full((N,), 2.0 ** -8, device="cuda")
    bias = (torch.arange(N, device="cuda") % 64 - 32).float() * 2.0 ** -4
    v = sums * 2.0 ** -8 + bias.double()
    assert torch.equal(v.float().double(), v) and float(v.abs().max()) > 3
    planes = planes_of(levels, 4)
    u = 2 * math.sqrt(2 / math.pi) * (v + 0.044715 * v ** 3)
    unit = 2.0 ** -23
    want = {"silu": (v * torch.sigmoid(v), (v.abs() + 4) * unit), "gelu_tanh": (v * torch.sigmoid(u), (4.5 * u.abs() + 4) * unit),
            "relu": (v.clamp(min=0), torch.zeros_like(v)), "none": (v, torch.zeros_like(v))}
    off = {k: y.abs() * r for k, (y, r) in want.items()}
    want = {k: y for k, (y, _) in want.items()}
    want["gelu"], off["gelu"] = 0.5 * v * torch.erfc(-v / math.sqrt(2.0)), v.abs() * 2 * unit
    for act, y in want.items():
        got = ap.linear_planes(x, planes, scale, zero=7.5, bias=bias, activation=act, out_dtype=FF).double()
        assert bool(((got - y).abs() <= off[act]).all()), (act, float(((got - y).abs() / (off[act] + 1e-300)).max()))
        for other in want:
            if other != act:
                assert bool(((got - want[other]).abs() > 10 * off[other] + 1e-7).any()), (act, other)
    assert float(((want["gelu"] - want["gelu_tanh"]).abs() / off["gelu"].clamp(min=1e-300)).max()) > 100
