"""Decoder-layer operators on the GPU where finite inputs lie far apart: heads whose squares leave fp32's range."""
import pytest
import torch

import decoder_reference as ref
from test_decoder_gpu import BF, Setup, check_append

pytestmark = pytest.mark.gpu


# ------------------------------------------------------------------------------------------------------------ norm
def test_append_norm_of_squares_beyond_fp32(cuda_device):
    """bf16 heads with an element whose square is no fp32 number while the head's mean square is one, and heads of such elements."""
    s = Setup(1, [6], [20], 2, 128, 16, BF)
    k = s.randn(6, 2, 128)
    k[0, 0], k[0, 0, 3] = 1.0, 5e19
    k[1, 1, 100] = -2e19
    k[2] = k[2] * 1e18
    k[3, 0, :4] = 9e19
    check_append(s, 4, True, 0, False, k=k)
    check_append(s, 4, True, 128, True, k=k)


@pytest.mark.parametrize("D", [64, 128, 256])
def test_append_norm_over_the_whole_range(cuda_device, D):
    """Every power of two whose mean square fp32 holds, subnormal ones among them, without eps: queries to the bit."""
    top = list(range(-74, 67))
    s = Setup(2, [len(top)], [len(top)], 1, D, 16, BF)
    q = s.randn(len(top), 3, D) * torch.pow(2.0, torch.tensor(top, dtype=torch.float64))[:, None, None].float()
    q = q.clamp(-1.2e20, 1.2e20).to(BF)
    q[:, 1, 1:] *= 2.0 ** -9
    w = (s.randn(D).float() * 0.2 + 1).to(BF)
    got = s.ap.kv4_append(s.cache, s.batch, q[:, :1].cuda(), q[:, :1].cuda(), q=q.cuda(), q_norm=w.cuda(), eps=0.0)
    want = torch.from_numpy(ref.normed(q, w, 0.0)).to(BF)
    assert torch.equal(got.cpu().view(torch.int16), want.view(torch.int16))
