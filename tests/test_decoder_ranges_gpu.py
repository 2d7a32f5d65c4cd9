"""Decoder-layer operators on the GPU where finite inputs lie far apart: heads whose squares leave fp32's range, value rows whose
steps differ by many powers of two, in visible, negligible and masked places."""
import numpy as np
import pytest
import torch

import decoder_reference as ref
from test_decoder_gpu import BF, HF, Setup, check_append, check_attention

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


# ------------------------------------------------------------------------------------------------------------ attention
FORMS = [(64, 16, BF), (128, 16, HF), (128, 64, BF), (256, 8, BF), (64, 32, HF)]
LENGTHS = [1, 7, 40, 150]


def with_params(s, change):
    """The cache with its parameters changed in place: change(params [pages, heads, 2, page, 2])."""
    rows = s.plain()
    params = rows.params.copy()
    change(params)
    s.data.copy_(ref.words_of(rows.levels, params, s.dtype).cuda())


def at(s, b, j):
    """Page and slot of position j of sequence b."""
    return s.table[b, j // s.page], j % s.page


@pytest.mark.parametrize("D,page,dtype", FORMS)
@pytest.mark.parametrize("q", [4, 7, 40, 150])
@pytest.mark.parametrize("window", [0, 9])
def test_later_rows_do_not_reach_earlier_ones(cuda_device, D, page, dtype, q, window):
    """The last token's value step is 2^30 times the others' (bf16; fp16: the type's range): the rows before it do not see it."""
    s = Setup(D + q, [q, q], [q + 60, q + 5], 2, D, page, dtype)

    def change(params):
        if dtype == HF:
            params[:, :, 1] *= 2.0 ** -15
        for b in range(2):
            p, r = at(s, b, int(s.kv[b]) - 1)
            params[p, :, 1, r] = (2.0 ** 30, -7.5 * 2.0 ** 30) if dtype == BF else (2.0 ** 11, -7.5 * 2.0 ** 11)

    with_params(s, change)
    check_attention(s, 4, window=window)


@pytest.mark.parametrize("D,page,dtype", FORMS)
@pytest.mark.parametrize("q", LENGTHS)
@pytest.mark.parametrize("ratio", [22, 28, 31, 90])
def test_value_rows_without_weight(cuda_device, D, page, dtype, q, ratio):
    """Keys that every row sees with a weight of nothing, whose value steps lie `ratio` powers of two above the others'."""
    s = Setup(D + q + ratio, [q, q], [q + 300, q + 90], 1, D, page, dtype)
    small = -min(ratio, 28) + 12 if dtype == HF else 0

    def change(params):
        params[:, :, 1] *= 2.0 ** small
        for b in range(2):
            for j in (5, 40, 85):
                p, r = at(s, b, j)
                params[p, :, 0, r] = 0.1, -30.0 if ratio == 90 else -8.0
                step = 2.0 ** (small + (min(ratio, 28) if dtype == HF else ratio))
                params[p, :, 1, r] = step, -7.5 * step

    with_params(s, change)
    check_attention(s, 2, q=s.randn(s.T, 2, D).abs())


@pytest.mark.parametrize("D,page,dtype", FORMS)
@pytest.mark.parametrize("q", LENGTHS)
@pytest.mark.parametrize("order", ["mixed", "rising", "falling"])
def test_value_steps_far_apart(cuda_device, D, page, dtype, q, order):
    """Value steps over 80 powers of two (fp16: 24), of either sign, some 0; scores over some 40 of them, so that many keys of small
    steps and large weights meet few of large steps and small weights."""
    s = Setup(D + 3 * q, [q, q, 1], [q + 280, q + 40, 200], 1, D, page, dtype)
    low, high = (-14, 10) if dtype == HF else (-40, 40)

    def change(params):
        rng = np.random.default_rng(q)
        for b in range(3):
            e = rng.uniform(low, high, size=int(s.kv[b]))
            e = e if order == "mixed" else np.sort(e) if order == "rising" else -np.sort(-e)
            for j in range(int(s.kv[b])):
                p, r = at(s, b, j)
                step = 0.0 if j % 11 == 3 else 2.0 ** e[j] * (-1 if j % 5 == 0 else 1)
                params[p, :, 1, r, 0] = step
                params[p, :, 1, r, 1] = -step * rng.uniform(5, 10)

    with_params(s, change)
    x = s.randn(s.T, 3, D)
    x[:, 1] *= 4
    x[:, 2] = 0
    check_attention(s, 3, q=x)
    check_attention(s, 3, q=x, window=33)
    check_attention(s, 3, q=x, causal=False)


@pytest.mark.parametrize("q", [1, 4, 60, 300])
@pytest.mark.parametrize("least,most", [(-126, -100), (-126, 100), (80, 100)])
def test_value_steps_at_the_ends_of_the_range(cuda_device, q, least, most):
    """bf16 value steps from the smallest normal number on, and up to 2^100."""
    s = Setup(q, [q], [q + 200], 1, 64, 16, BF)

    def change(params):
        e = np.random.default_rng(q).integers(least, most + 1, size=int(s.kv[0]))
        for j in range(int(s.kv[0])):
            p, r = at(s, 0, j)
            params[p, :, 1, r] = 2.0 ** float(e[j]), -8.0 * 2.0 ** float(e[j])

    with_params(s, change)
    check_attention(s, 2)


@pytest.mark.parametrize("dtype", [BF, HF])
def test_value_steps_far_apart_over_split_sequences(cuda_device, dtype):
    """One step far above the others in one of the parts that a sequence's keys are shared out in."""
    for q, L, where in ((1, 3000, 100), (4, 3000, 2990), (40, 2500, 1700), (1, 3000, 1500)):
        s = Setup(q, [q], [L], 1, 64, 64, dtype)

        def change(params):
            if dtype == HF:
                params[:, :, 1] *= 2.0 ** -15
            p, r = at(s, 0, where)
            step = 2.0 ** 40 if dtype == BF else 2.0 ** 11
            params[p, :, 0, r] = 0.1, -8.0
            params[p, :, 1, r] = step, -7.5 * step

        with_params(s, change)
        check_attention(s, 2, q=s.randn(s.T, 2, 64).abs())
