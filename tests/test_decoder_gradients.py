"""The decoder-layer operators have no backward pass: outside ``no_grad`` they refuse tensors that require a gradient, in place of
returning results whose history ends there."""
import pytest
import torch

import apnn_tc_b200 as ap

BF = torch.bfloat16


def calls():
    """(name, argument, call): each floating-point argument in turn one that requires a gradient; CPU tensors and no cache, so that
    nothing else is looked at before."""
    g = lambda *shape, dtype=BF: torch.zeros(*shape, dtype=dtype, requires_grad=True)     # noqa: E731
    x, planes, scale = torch.zeros(2, 128, dtype=BF), torch.zeros(4, 8, 4, dtype=torch.int32), torch.ones(8)
    kw = dict(x=x, planes=planes, scale=scale)
    for name, t in (("x", g(2, 128)), ("scale", g(8, dtype=torch.float32)), ("bias", g(8, dtype=torch.float32)), ("residual", g(2, 8)), ("out", g(2, 8))):
        yield "linear_planes", name, lambda name=name, t=t: ap.linear_planes(**{**kw, name: t})
    k = torch.zeros(1, 2, 64, dtype=BF)
    kw2 = dict(k=k, v=k, q=k)
    for name, t in (("k", g(1, 2, 64)), ("v", g(1, 2, 64)), ("q", g(1, 2, 64)), ("q_out", g(1, 2, 64)), ("q_norm", g(64)), ("k_norm", g(64)),
                    ("rotary", g(4, 64, dtype=torch.float32))):
        yield "kv4_append", name, lambda name=name, t=t: ap.kv4_append(None, None, **{**kw2, name: t})
    for name, t in (("q", g(1, 2, 64)), ("out", g(1, 2, 64))):
        yield "kv4_attention", name, lambda name=name, t=t: ap.kv4_attention(None, None, **{"q": k, name: t})


@pytest.mark.parametrize("what,name,call", [pytest.param(*c, id=f"{c[0]}-{c[1]}") for c in calls()])
def test_gradients_are_refused(what, name, call):
    with pytest.raises(ValueError, match=what + ".*gradient"):
        call()
    with torch.no_grad(), pytest.raises(Exception) as other:      # the next check's: these are CPU tensors without a cache
        call()
    assert "gradient" not in str(other.value)


@pytest.mark.gpu
def test_parameters_under_no_grad(cuda_device):
    from test_decoder_gpu import Setup
    planes = torch.zeros(4, 8, 4, dtype=torch.int32, device="cuda")
    scale, bias = (torch.nn.Parameter(torch.ones(8, device="cuda")) for _ in range(2))
    x = torch.ones(2, 128, dtype=BF, device="cuda")
    with pytest.raises(ValueError, match="gradient"):
        ap.linear_planes(x, planes, scale, bias=bias)
    s = Setup(1, [1], [9], 1, 64, 16, BF)
    q = s.randn(1, 2, 64).cuda().requires_grad_()
    with torch.no_grad():
        assert bool((ap.linear_planes(x, planes, scale, bias=bias) == 1).all())
        want = ap.kv4_attention(s.cache, s.batch, q.detach())
        assert torch.equal(ap.kv4_attention(s.cache, s.batch, q), want)
    with torch.inference_mode():
        assert torch.equal(ap.kv4_attention(s.cache, s.batch, q), want)
