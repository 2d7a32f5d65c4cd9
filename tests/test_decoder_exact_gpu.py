"""Attention whose result names the key it came from, at the borders of tiles, pages, warps and shares of the keys; key splits and long
blocks of prompts; and one decoder layer, operator by operator, beside the plain forms."""
import numpy as np
import pytest
import torch

import decoder_reference as ref
from test_decoder_gpu import BF, HF, Setup, check_attention, close, layer, layer_weights, rotary_table

pytestmark = pytest.mark.gpu


def borders(L, q):
    """Positions on both sides of the borders of 8 to 1024 keys, and those in between, spread over the length."""
    at = {0, 1, L - 1, L - 2, max(0, L - q), max(0, L - q - 1)}
    for size in (8, 16, 32, 64, 128, 256, 512, 1024):
        for k in (1, 2, 3, L // size):
            at |= {k * size - 1, k * size}
    at |= {int(v) for v in np.linspace(0, L - 1, 20)}
    return sorted(j for j in at if 0 <= j < L)


def one_key(D, page, dtype, q, L, heads, group, window=0, causal=True):
    """Every sequence has one key of score 40 (in log2 more than 50 above the others, whose scores are 0), each at another border: a row
    that sees it gets its value row, the others the mean of what they see."""
    at = borders(L, q)
    B = len(at)
    s = Setup(D + q + L, [q] * B, [L] * B, heads, D, page, dtype)
    rows = s.plain()
    params = rows.params.copy()
    params[:, :, 0] = 0
    params[:, :, 1] = 0.25, -2.0
    for b, j in enumerate(at):
        params[s.table[b, j // page], :, 0, j % page] = 0, 40.0 / D ** 0.5
    s.data.copy_(ref.words_of(rows.levels, params, dtype).cuda())
    x = torch.ones(s.T, heads * group, D, dtype=dtype, device="cuda")
    out, lse = s.ap.kv4_attention(s.cache, s.batch, x, causal=causal, window=window, lse=True)
    got = (out.float().cpu().numpy().reshape(B, q, heads, group, D) + 2.0) / 0.25
    lse = lse.cpu().numpy().reshape(B, q, heads * group)
    score = float(torch.tensor(40.0 / D ** 0.5).to(dtype)) * D ** 0.5      # of the key as it is held
    for b, j in enumerate(at):
        want = rows.levels[s.table[b, j // page], :, 1, j % page][None, :, None, :]      # [1, heads, 1, D]
        pos = L - q + np.arange(q)
        end = pos + 1 if causal else np.full(q, L)
        begin = np.maximum(0, end - window) if window else np.zeros(q, dtype=int)
        sees = (j < end) & (j >= begin)
        # off by a rounding of the weight (2^-11 of up to 8 steps), one of the result (2^-8 of up to 8 steps) and 2^-40 for the others
        assert np.abs(got[b, sees] - want).max(initial=0) < 8 * (2.0 ** -11 + 2.0 ** -8) + 1e-3, (b, j)
        full = np.where(sees, score, np.log(np.maximum(end - begin - sees, 1e-30)))       # exp(40) is 2e17: the others add below 2^-40
        assert np.abs(lse[b] - full[:, None]).max() < 40 * 2.0 ** -20, (b, j)


@pytest.mark.parametrize("D,page,dtype", [(64, 8, BF), (64, 64, HF), (128, 16, HF), (128, 256, BF), (256, 32, BF), (256, 8, HF)])
@pytest.mark.parametrize("q,L,heads,group", [(1, 3001, 1, 1), (1, 500, 2, 4), (3, 1500, 1, 4), (4, 257, 1, 4), (40, 1411, 1, 2), (150, 700, 2, 2)])
def test_one_key(cuda_device, D, page, dtype, q, L, heads, group):
    one_key(D, page, dtype, q, L, heads, group)
    one_key(D, page, dtype, q, L, heads, group, window=200)
    one_key(D, page, dtype, q, L, heads, group, causal=False)


@pytest.mark.parametrize("D,dtype", [(64, HF), (128, BF), (256, HF)])
@pytest.mark.parametrize("q", [1, 40])
def test_one_key_of_a_split_sequence(cuda_device, D, dtype, q):
    """A single sequence whose keys are shared out over the device, one border after the other."""
    L = 6000
    s = Setup(D, [q], [L], 1, D, 64, dtype)
    rows = s.plain()
    for j in borders(L, q)[::3]:
        params = rows.params.copy()
        params[:, :, 0] = 0
        params[:, :, 1] = 0.25, -2.0
        params[s.table[0, j // 64], :, 0, j % 64] = 0, 40.0 / D ** 0.5
        s.data.copy_(ref.words_of(rows.levels, params, dtype).cuda())
        out = s.ap.kv4_attention(s.cache, s.batch, torch.ones(q, 2, D, dtype=dtype, device="cuda"))
        sees = np.arange(L - q, L) >= j
        got = (out.float().cpu().numpy()[sees] + 2.0) / 0.25
        assert np.abs(got - rows.levels[s.table[0, j // 64], 0, 1, j % 64]).max() < 8 * (2.0 ** -11 + 2.0 ** -8) + 1e-3, j


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("q,L", [(40, 2500), (300, 1300), (40, 700)])
def test_prompt_key_splits(cuda_device, D, q, L):
    check_attention(Setup(D + q, [q], [L], 1, D, 64, BF), 2)
    check_attention(Setup(D + q, [q, 3], [L, 90], 1, D, 16, HF), 1, window=L // 2)


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("dtype", [BF, HF])
def test_prompt_blocks_of_many_tiles(cuda_device, D, dtype):
    """More blocks of rows than the device has room for at once: no split, every block walks up to 14 tiles of keys."""
    B = 76
    lens = np.random.default_rng(D).integers(1100, 1700, size=B)
    check_attention(Setup(D, [40] * B, list(lens), 2, D, 64, dtype), 2)


@pytest.mark.parametrize("q", [1, 3, 50])
def test_layer_operator_by_operator(cuda_device, q):
    """The run of a decoder layer: each operator's result against the plain form of its own inputs, and the run's as theirs."""
    import apnn_tc_b200 as ap
    E, Hq, H, D, F = 256, 4, 2, 64, 384
    w = layer_weights(E, Hq, H, D, F, seed=q)
    bits = dict(qkv=4, o=2, up=1, down=3)
    g = torch.Generator().manual_seed(q)
    levels = {}      # as layer_weights draws them
    gw = torch.Generator().manual_seed(q)
    for name, N, K in (("qkv", (Hq + 2 * H) * D, E), ("o", E, Hq * D), ("up", F, E), ("down", E, F)):
        levels[name] = torch.randint(0, 2 ** bits[name], (N, K), generator=gw)
        torch.rand(N, generator=gw)
        assert torch.equal(w[name].cpu(), ref.planes_of(levels[name], bits[name]))
    table = rotary_table(200, D)
    s = Setup(q, [q, 0, q], [q + 60, 9, q + 3], H, D, 16, BF)
    x = torch.randn(s.T, E, generator=g).to(BF)
    start = s.data.clone()
    ws = torch.empty(ap.kv4_attention_workspace_bytes(s.cache, s.batch, Hq), dtype=torch.uint8, device="cuda")
    whole = layer(ap, w, s.cache, s.batch, x.cuda(), table.cuda(), ws)
    held = s.data.clone()
    s.data.copy_(start)

    def product(name, t, zero, bias=None, act="none", residual=None):
        got = ap.linear_planes(t, w[name], w["s_" + name], zero=zero, bias=bias, activation=act, residual=residual)
        close(got, *ref.linear(t, levels[name], w["s_" + name], zero, bias, act, residual), BF)
        return got

    xd = x.cuda()
    qkv = product("qkv", xd, 7.5, bias=w["b_qkv"])
    qd, kd, vd = (part.unflatten(1, (-1, D)) for part in qkv.split((Hq * D, H * D, H * D), 1))
    before = s.plain()
    qr = ap.kv4_append(s.cache, s.batch, kd, vd, q=qd, q_norm=w["qn"], k_norm=w["kn"], rotary=table.cuda())
    pos, owner = s.positions()
    want = torch.from_numpy(ref.rotated(ref.normed(qd, w["qn"], 1e-6), table, pos, False)).to(BF)
    assert torch.equal(qr.cpu(), want)
    after, where = s.plain(), s.table[owner, pos // s.page]
    lv, par = before.levels.copy(), before.params.copy()
    for i, t in enumerate((ref.rotated(ref.normed(kd, w["kn"], 1e-6), table, pos, False), vd.float().cpu().numpy())):
        level, step, low = ref.quantise(t, BF)
        lv[where, :, i, pos % s.page], par[where, :, i, pos % s.page] = level, np.concatenate((step, low), -1)
    assert np.array_equal(after.levels, lv) and np.array_equal(after.params, par)
    o = ap.kv4_attention(s.cache, s.batch, qr, workspace=ws)
    wo, _, off, _ = ref.attention(qr, after, list(map(int, s.cu)), list(map(int, s.kv)), s.table, D ** -0.5, True, 0)
    close(o, torch.from_numpy(wo), torch.from_numpy(off), BF)
    y = product("o", o.view(s.T, Hq * D), 1.5, residual=xd)
    h = product("up", y, 0.5, act="silu")
    last = product("down", h, 3.5, residual=y)
    assert torch.equal(whole, last) and torch.equal(held, s.data)
