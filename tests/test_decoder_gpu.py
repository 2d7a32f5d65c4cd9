"""Decoder-layer operators on the GPU against plain 64-bit forms: product over weight planes with its epilogue, 4-bit cache
append and read, attention over the cache, and a run of them together."""
import numpy as np
import pytest
import torch

import decoder_reference as ref

pytestmark = pytest.mark.gpu
BF, HF, FF = torch.bfloat16, torch.float16, torch.float32


# ------------------------------------------------------------------------------------------------------------ product
def product(seed, M, N, K, wbits, dtype, act="none", bias=True, residual=False, out=None, zero=None, x=None, pad=0):
    import apnn_tc_b200 as ap
    g = torch.Generator().manual_seed(seed)
    zero = (2 ** wbits - 1) / 2 if zero is None else zero
    out = out or dtype
    wide = (K + 7) // 8 * 8 + pad
    buf = torch.full((M, wide), float("nan"), dtype=dtype)      # what lies behind a row is never used
    buf[:, :K] = torch.randn(M, K, generator=g).to(dtype) if x is None else x
    levels = torch.randint(0, 2 ** wbits, (N, K), generator=g)
    scale = (torch.rand(N, generator=g) + 0.5) / (2 ** wbits / 2 * K ** 0.5)
    b = torch.randn(N, generator=g) if bias else None
    r = torch.randn(M, N, generator=g).to(out) if residual else None
    dev = lambda t: None if t is None else t.cuda()     # noqa: E731
    xd = buf.cuda()[:, :K]
    got = ap.linear_planes(xd, ref.planes_of(levels, wbits).cuda(), dev(scale), zero=zero, bias=dev(b), activation=act,
                           residual=dev(r), out_dtype=out)
    want, off = ref.linear(buf[:, :K], levels, scale, zero, b, act, r)
    assert got.dtype == out and got.shape == (M, N)
    close(got, want, off, out)
    return got


def close(got, want, off, dtype):
    want = torch.as_tensor(want)
    tol = ref.STEP[dtype] * (want.abs() + off) + off + 2.0 ** -133      # one rounding of the result (bf16's and fp32's smallest steps)
    if dtype == HF:
        tol = tol + 2.0 ** -25                                            # fp16: half its smallest step
    err = (got.double().cpu() - want).abs()
    bad = ~(err <= tol)
    assert not bad.any(), (int(bad.sum()), err[bad].max().item(), (err / tol)[bad].max().item(), bad.nonzero()[0].tolist())


@pytest.mark.parametrize("wbits", [1, 2, 3, 4])
@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("M,N,K", [(1, 64, 128), (1, 1, 1), (3, 33, 200), (8, 256, 1024), (9, 40, 136), (17, 129, 392), (33, 65, 256),
                                   (64, 128, 2048), (65, 300, 520), (130, 257, 776), (257, 513, 129), (300, 1000, 1000), (40, 64, 8),
                                   (20, 4096, 1), (513, 2300, 264), (48, 130, 4096), (700, 6000, 640)])
def test_product(cuda_device, M, N, K, wbits, dtype):
    product(M + N + K, M, N, K, wbits, dtype)


@pytest.mark.parametrize("act", ["none", "relu", "silu", "gelu", "gelu_tanh"])
@pytest.mark.parametrize("M", [1, 12, 40, 200, 600])
@pytest.mark.parametrize("out", [None, FF])
def test_product_epilogues(cuda_device, act, M, out):
    for bias in (False, True):
        for residual in (False, True):
            product(M + 7, M, 200, 384, 3, BF if bias else HF, act, bias, residual, out, pad=8 * (M % 3))


@pytest.mark.parametrize("zero", [0.0, 0.5, 1.0, 7.5, 8.0, 14.5, 15.0])
@pytest.mark.parametrize("M", [2, 50, 280])
def test_product_zero_points(cuda_device, zero, M):
    for wbits in (1, 2, 4):
        product(M, M, 96, 300, wbits, BF, zero=zero)
        product(M, M, 96, 300, wbits, HF, zero=zero)


@pytest.mark.parametrize("M", [1, 8, 32, 100, 1000])
@pytest.mark.parametrize("dtype", [BF, HF])
def test_product_values_over_the_whole_range(cuda_device, M, dtype):
    """Rows of very large and of very small activations, zeros, and elements of one row far apart."""
    g = torch.Generator().manual_seed(5)
    x = torch.randn(M, 256, generator=g)
    top = 2.0 ** 60 if dtype == BF else 30000.0
    x[0] = x[0] * 1e-3 * top / 8
    x[0, 7] = top
    if M > 3:
        x[1] = 0
        x[2] = x[2] * (2.0 ** -100 if dtype == BF else 2.0 ** -14)
        x[3, ::2] *= 2.0 ** 12
    for out in (dtype, FF):
        if dtype == HF and out == HF:
            continue
        product(1, M, 70, 256, 4, dtype, bias=False, x=x, out=out)


@pytest.mark.parametrize("M", [1, 6, 24, 90, 400])
def test_product_not_finite(cuda_device, M):
    """An infinity or NaN stays in its row."""
    import apnn_tc_b200 as ap
    for dtype in (BF, HF):
        g = torch.Generator().manual_seed(1)
        x = torch.randn(M, 192, generator=g).to(dtype)
        levels = torch.randint(0, 16, (130, 192), generator=g)
        scale = torch.full((130,), 0.01)
        clean = ap.linear_planes(x.cuda(), ref.planes_of(levels, 4).cuda(), scale.cuda(), zero=7.5)
        x[0, 5] = float("inf")
        if M > 2:
            x[2, 100] = float("nan")
        got = ap.linear_planes(x.cuda(), ref.planes_of(levels, 4).cuda(), scale.cuda(), zero=7.5)
        hit = [0] + ([2] if M > 2 else [])
        assert not torch.isfinite(got[hit]).any()
        rest = [m for m in range(M) if m not in hit]
        assert torch.equal(got[rest], clean[rest])


@pytest.mark.parametrize("M", [1, 20, 70, 300])
def test_product_in_place_residual_strides_and_flag(cuda_device, M):
    import apnn_tc_b200 as ap
    g = torch.Generator().manual_seed(2)
    N, K = 136, 264
    x = torch.randn(M, K, generator=g).to(BF)
    levels = torch.randint(0, 4, (N, K), generator=g)
    scale, bias = torch.rand(N, generator=g) * 0.05, torch.randn(N, generator=g)
    stream = torch.randn(M, N + 11, generator=g).to(BF)     # the residual stream is a view of something wider, and is updated in place
    buf = stream.cuda()
    flag = torch.full((1,), 5, dtype=torch.int32, device="cuda")
    view = buf[:, 3:3 + N]
    got = ap.linear_planes(x.cuda(), ref.planes_of(levels, 2).cuda(), scale.cuda(), zero=1.5, bias=bias.cuda(), activation="gelu",
                           residual=view, out=view, status_flag=flag)
    assert got.data_ptr() == view.data_ptr() and int(flag.item()) == 0
    want, off = ref.linear(x, levels, scale, 1.5, bias, "gelu", stream[:, 3:3 + N])
    close(view, want, off, BF)
    assert torch.equal(buf[:, :3].cpu(), stream[:, :3]) and torch.equal(buf[:, 3 + N:].cpu(), stream[:, 3 + N:])


def test_product_empty_and_repeated(cuda_device):
    import apnn_tc_b200 as ap
    planes, scale = torch.zeros(4, 8, 4, dtype=torch.int32, device="cuda"), torch.ones(8, device="cuda")
    assert ap.linear_planes(torch.empty(0, 128, dtype=BF, device="cuda"), planes, scale).shape == (0, 8)
    for M in (1, 40, 513):
        a = product(3, M, 384, 640, 4, BF, residual=True)
        b = product(3, M, 384, 640, 4, BF, residual=True)
        assert torch.equal(a, b)


def test_product_refusals(cuda_device):
    import apnn_tc_b200 as ap
    x = torch.zeros(4, 128, dtype=BF, device="cuda")
    planes, scale = torch.zeros(4, 8, 4, dtype=torch.int32, device="cuda"), torch.ones(8, device="cuda")
    ok = dict(x=x, planes=planes, scale=scale)
    for kw, exc in [(dict(x=x.float()), ValueError), (dict(planes=planes[:, :, :3]), ValueError), (dict(scale=scale.half()), ValueError),
                    (dict(x=x.t()), ValueError), (dict(activation="swish"), ValueError), (dict(out_dtype=HF), ValueError),
                    (dict(residual=torch.zeros(4, 9, dtype=BF, device="cuda")), ValueError), (dict(bias=scale.cpu()), ValueError),
                    (dict(zero=0.3), ap.ApnnError), (dict(planes=torch.zeros(5, 8, 4, dtype=torch.int32, device="cuda")), ap.ApnnError),
                    (dict(x=x[:, :100][1:].as_strided((3, 100), (100, 1))), ap.ApnnError)]:
        with pytest.raises(exc):
            ap.linear_planes(**{**ok, **kw})


# ------------------------------------------------------------------------------------------------------------ cache
class Setup:
    """A cache of random rows and a batch over scattered pages."""

    def __init__(self, seed, lens_q, lens_kv, heads, D, page, dtype, spare_rows=0, wide=None, extra_pages=3, gap=0):
        import apnn_tc_b200 as ap
        rng = np.random.default_rng(seed)
        B = len(lens_kv)
        wide = wide or max(1, max((n + page - 1) // page for n in lens_kv))
        pages = B * wide + extra_pages
        order = rng.permutation(pages)[:B * wide].reshape(B, wide).astype(np.int32)
        self.levels = rng.integers(0, 16, size=(pages, heads, 2, page, D), dtype=np.uint8)
        self.params = np.empty((pages, heads, 2, page, 2), dtype=np.float32)
        self.params[..., 0] = rng.uniform(0.1, 0.4, size=self.params.shape[:-1])
        self.params[..., 1] = -self.params[..., 0] * 7.5 + rng.normal(size=self.params.shape[:-1]) * 0.2
        words = ref.words_of(self.levels, self.params, dtype)
        if gap:     # pages of one layer of a pool
            pool = torch.zeros(pages, words.shape[1] + gap, words.shape[2], dtype=torch.int32).cuda()
            pool[:, :heads] = words.cuda()
            self.data = pool[:, :heads]
        else:
            self.data = words.cuda()
        self.ap, self.dtype, self.page, self.D, self.heads = ap, dtype, page, D, heads
        self.cu = np.concatenate(([0], np.cumsum(lens_q))).astype(np.int32)
        self.kv, self.table = np.asarray(lens_kv, dtype=np.int32), order
        self.T = int(self.cu[-1]) + spare_rows
        self.rng = rng
        self.cache = ap.KVCache4(pages, heads, page, D, dtype, data=self.data)
        self.max_q = max(1, max(lens_q))
        self.refresh()

    def refresh(self):
        dev = lambda a: torch.from_numpy(np.ascontiguousarray(a)).cuda()     # noqa: E731
        self.batch = self.ap.KVBatch(dev(self.cu), dev(self.kv), dev(self.table), self.max_q)

    def plain(self):
        return ref.Cache(self.data, self.page, self.D, self.dtype)

    def randn(self, *shape):
        return torch.from_numpy(self.rng.normal(size=shape).astype(np.float32)).to(self.dtype)

    def positions(self):
        pos, owner = [], []
        for b in range(len(self.kv)):
            n = self.cu[b + 1] - self.cu[b]
            pos += list(range(self.kv[b] - n, self.kv[b]))
            owner += [b] * n
        return np.array(pos, dtype=np.int64), np.array(owner, dtype=np.int64)


def rotary_table(rows, rot):
    inverse = 10000.0 ** (-np.arange(0, rot, 2) / rot)
    angle = np.arange(rows)[:, None] * inverse
    return torch.from_numpy(np.concatenate((np.cos(angle), np.sin(angle)), 1).astype(np.float32))


def check_append(s, Hq, norm, rot, interleaved, k=None, v=None, rows=None):
    """Levels and parameters bit for bit, every other byte of the cache untouched, q to one rounding, and the read."""
    ap, T, D, H = s.ap, s.T, s.D, s.heads
    fused = torch.cat([t.reshape(T, -1) for t in (s.randn(T, Hq, D), s.randn(T, H, D) if k is None else k, s.randn(T, H, D) if v is None else v)], 1)
    q, k, v = (part.unflatten(1, (-1, D)) for part in fused.split((Hq * D, H * D, H * D), 1))
    qw, kw = ((s.randn(D).float() * 0.2 + 1).to(s.dtype), (s.randn(D).float() * 0.2 + 1).to(s.dtype)) if norm else (None, None)
    table = rotary_table(rows or int(max(1, s.kv.max())), rot) if rot else None
    pos, owner = s.positions()
    n = len(pos)
    dev = lambda t: None if t is None else t.cuda()     # noqa: E731
    fd = fused.cuda()
    qd, kd, vd = (part.unflatten(1, (-1, D)) for part in fd.split((Hq * D, H * D, H * D), 1))
    before = s.plain()
    q_out = torch.full((T, Hq, D), 3.0, dtype=s.dtype, device="cuda")
    got_q = ap.kv4_append(s.cache, s.batch, kd, vd, q=qd, q_out=q_out, q_norm=dev(qw), k_norm=dev(kw), eps=1e-5, rotary=dev(table),
                          interleaved=interleaved)
    after = s.plain()
    wk = ref.rotated(ref.normed(k[:n], kw, 1e-5), table, pos, interleaved)
    wq = ref.rotated(ref.normed(q[:n], qw, 1e-5), table, pos, interleaved)
    want_q = torch.from_numpy(wq).to(s.dtype)
    assert torch.equal(torch.nan_to_num(got_q[:n].cpu().float(), nan=9e9), torch.nan_to_num(want_q.float(), nan=9e9))
    assert (got_q[n:] == 3.0).all()
    levels, params = before.levels.copy(), before.params.copy()
    where = np.full(n, -1)
    inside = (pos >= 0) & (pos < s.table.shape[1] * s.page)
    where[inside] = s.table[owner[inside], pos[inside] // s.page]
    ok = (where >= 0) & (where < after.pages)
    for i, x in enumerate((wk, v[:n].float().numpy())):
        level, step, low = ref.quantise(x, s.dtype)
        levels[where[ok], :, i, pos[ok] % s.page] = level[ok]
        params[where[ok], :, i, pos[ok] % s.page] = np.concatenate((step, low), -1)[ok]
    assert np.array_equal(after.levels, levels)
    assert np.array_equal(after.params, params, equal_nan=True)
    gk, gv = ap.kv4_read(s.cache, s.batch, T)
    values = torch.from_numpy(after.values().astype(np.float32)).to(s.dtype)     # step * level + low: one rounding in fp32, one to the type
    for i, got in enumerate((gk, gv)):
        want = torch.full((n, H, D), float("nan"), dtype=s.dtype)
        want[torch.from_numpy(ok)] = values[where[ok], :, i, pos[ok] % s.page]
        assert torch.equal(torch.nan_to_num(got[:n].cpu().float(), nan=9e9), torch.nan_to_num(want.float(), nan=9e9))


@pytest.mark.parametrize("D,page,dtype", [(64, 16, BF), (128, 16, HF), (128, 64, BF), (256, 8, HF), (256, 32, BF), (64, 1024, HF)])
@pytest.mark.parametrize("norm,rot,interleaved", [(False, 0, False), (True, 0, False), (False, 1.0, False), (True, 1.0, True), (True, 0.5, False), (True, 0.25, True)])
def test_append(cuda_device, D, page, dtype, norm, rot, interleaved):
    s = Setup(D + page, [1, 0, 5, 37, 1], [1, 4, 5, 90, 33], 3, D, page, dtype, spare_rows=2)
    check_append(s, 6, norm, int(rot * D), interleaved)


@pytest.mark.parametrize("Hq,heads,B", [(1, 1, 1), (7, 7, 70), (40, 8, 300), (5, 1, 1100)])
def test_append_many_sequences(cuda_device, Hq, heads, B):
    rng = np.random.default_rng(B)
    lens_q = rng.integers(0, 3, size=B)
    lens_q[-1] = 1
    s = Setup(B, list(lens_q), list(lens_q + rng.integers(0, 20, size=B)), heads, 64, 8, BF, spare_rows=1, gap=1)
    check_append(s, Hq, True, 64, False)


@pytest.mark.parametrize("dtype", [BF, HF])
def test_append_odd_rows(cuda_device, dtype):
    """Constant rows, rows that are not finite, the largest and smallest values of the type, positions behind the rotary table."""
    s = Setup(1, [12], [20], 2, 128, 16, dtype)
    big, small = torch.finfo(dtype).max, torch.finfo(dtype).tiny
    k, v = s.randn(12, 2, 128), s.randn(12, 2, 128)
    for x in (k, v):
        x[0] = 0
        x[1] = 1.7
        x[2, 0, 5] = float("nan")
        x[3, 1, 7] = float("inf")
        x[4, 0, 9] = -float("inf")
        x[5, 0, 0], x[5, 0, 1] = big, -big
        x[6, 1] = small
        x[7] = x[7] * small * 4
        x[8] = -1e-3
        x[9, 0, :64] = 1.0
    check_append(s, 4, False, 0, False, k=k, v=v)
    check_append(Setup(1, [12], [20], 2, 128, 16, dtype), 4, False, 128, True, k=k, v=v, rows=18)
    check_append(Setup(1, [12], [20], 2, 128, 16, dtype), 4, True, 64, False, k=k, v=v, rows=18)


@pytest.mark.parametrize("Hq,heads,D,most,B,norm,rot", [(1, 1, 64, 5, 2500, True, 64), (3, 2, 128, 40, 260, False, 64), (1, 1, 64, 4, 30000, False, 0), (4, 3, 256, 900, 9, True, 256)])
def test_append_rows_that_share_a_block(cuda_device, Hq, heads, D, most, B, norm, rot):
    """So many rows that a block takes several, up to 32, across the borders of sequences and past the last one."""
    rng = np.random.default_rng(B)
    lens_q = rng.integers(0, most + 1, size=B)
    s = Setup(B, lens_q, lens_q + rng.integers(0, 12, size=B), heads, D, 16, BF, spare_rows=70)
    check_append(s, Hq, norm, rot, False, rows=most + 12)


@pytest.mark.parametrize("T,rows", [(20, 7), (9000, 7001), (9000, 8999), (60000, 59995)])
def test_append_and_read_no_further_than_their_tensors(cuda_device, T, rows):
    """Tensors of fewer rows than the batch's sequences: the cache and everything behind the tensors' rows stay as they were."""
    s = Setup(T, [T], [T], 1, 64, 1024, BF)
    k, v, q = (s.randn(rows + 40, n, 64).cuda() for n in (1, 1, 2))
    before = s.data.clone()
    q_out = torch.full_like(q, 3.0)
    s.ap.kv4_append(s.cache, s.batch, k[:rows], v[:rows], q=q[:rows], q_out=q_out[:rows])
    assert torch.equal(q_out[:rows], q[:rows]) and bool((q_out[rows:] == 3.0).all())
    outs = [torch.full((rows + 40, 1, 64), 3.0, dtype=BF, device="cuda") for _ in range(2)]
    s.ap.kv4_read(s.cache, s.batch, k_out=outs[0][:rows], v_out=outs[1][:rows])
    for out in outs:
        assert bool((out[rows:] == 3.0).all())
    held = s.plain()
    old = ref.Cache(before, s.page, s.D, s.dtype)
    where, at = s.table[0, np.arange(rows, T) // s.page], np.arange(rows, T) % s.page
    assert np.array_equal(held.levels[where, :, :, at], old.levels[where, :, :, at])
    assert np.array_equal(held.params[where, :, :, at], old.params[where, :, :, at])
    for i, out in enumerate(outs):
        want = torch.from_numpy(held.values()[s.table[0, np.arange(rows) // s.page], :, i, np.arange(rows) % s.page].astype(np.float32)).to(BF)
        assert torch.equal(out[:rows].cpu(), want)


def test_append_bad_pages_and_positions(cuda_device):
    """Page numbers outside the cache, lengths shorter than the rows, lengths behind the table: those rows are not written."""
    s = Setup(4, [6, 9, 4], [40, 5, 60], 2, 64, 16, BF, wide=3)
    s.table[0, 2], s.table[1, 0] = -1, s.cache.pages
    s.refresh()
    check_append(s, 2, False, 32, False, rows=64)


def test_append_in_place_and_alone(cuda_device):
    """q rotated into itself gives what a second tensor gives; without q only the cache is written; a second append of the same rows changes nothing."""
    s = Setup(2, [9], [9], 2, 128, 16, BF)
    q, k, v, table = s.randn(9, 4, 128).cuda(), s.randn(9, 2, 128).cuda(), s.randn(9, 2, 128).cuda(), rotary_table(9, 128).cuda()
    other = s.ap.kv4_append(s.cache, s.batch, k, v, q=q, rotary=table)
    held = s.data.clone()
    assert s.ap.kv4_append(s.cache, s.batch, k, v, rotary=table) is None
    assert s.ap.kv4_append(s.cache, s.batch, k, v, q=q, q_out=q, rotary=table) is q
    assert torch.equal(q, other) and torch.equal(s.data, held)
    assert s.ap.kv4_append(s.cache, s.batch, k[:0], v[:0]) is None


# ------------------------------------------------------------------------------------------------------------ attention
def check_attention(s, Hq, causal=True, window=0, scale=None, q=None, poison=False, max_q=None):
    ap, T, D = s.ap, s.T, s.D
    q = s.randn(T, Hq, D) if q is None else q
    scale = D ** -0.5 if scale is None else scale
    out = torch.full((T, Hq, D), 3.0, dtype=s.dtype, device="cuda")
    lse = torch.full((T, Hq), 3.0, device="cuda")
    plain = s.plain()
    ap.kv4_attention(s.cache, s.batch, q.cuda(), scale=scale, causal=causal, window=window, out=out, lse=lse)
    want, wlse, off, loff = ref.attention(q, plain, list(map(int, s.cu)), list(map(int, s.kv)), s.table, scale, causal, window, max_q)
    n = int(s.cu[-1])
    done = torch.from_numpy(~np.isnan(wlse[:n]))
    assert (out[n:] == 3.0).all() and (lse[n:] == 3.0).all()
    assert (out[:n].cpu()[~done] == 3.0).all()
    close(out[:n].cpu()[done], torch.from_numpy(want[:n])[done], torch.from_numpy(off[:n])[done], s.dtype)
    got, wl = lse[:n].cpu().double()[done], torch.from_numpy(wlse[:n])[done]
    empty = torch.isinf(wl)
    assert torch.equal(got[empty], wl[empty])
    assert ((got - wl).abs()[~empty] <= torch.from_numpy(loff[:n])[done][~empty]).all()
    return out, lse


FORMS = [(64, 16, BF), (128, 16, BF), (128, 64, HF), (256, 32, BF), (64, 8, HF), (128, 256, BF), (256, 8, HF)]


@pytest.mark.parametrize("D,page,dtype", FORMS)
@pytest.mark.parametrize("Hq,heads", [(1, 1), (4, 1), (8, 2), (14, 2), (3, 3), (24, 1)])
def test_attention_single_tokens(cuda_device, D, page, dtype, Hq, heads):
    check_attention(Setup(D + Hq, [1] * 7, [1, 2, 15, 16, 65, 130, 333], heads, D, page, dtype, spare_rows=1), Hq)


@pytest.mark.parametrize("D,page,dtype", FORMS)
@pytest.mark.parametrize("window", [0, 1, 20])
def test_attention_few_tokens(cuda_device, D, page, dtype, window):
    check_attention(Setup(D, [4, 0, 2, 4, 3], [4, 9, 77, 200, 3], 2, D, page, dtype, spare_rows=3, gap=1), 6, window=window)


@pytest.mark.parametrize("D,page,dtype", FORMS)
@pytest.mark.parametrize("window", [0, 50])
def test_attention_prompts(cuda_device, D, page, dtype, window):
    check_attention(Setup(D + 1, [70, 1, 131], [70, 100, 260], 2, D, page, dtype, spare_rows=1), 4, window=window)


@pytest.mark.parametrize("q", [2, 5, 40])
def test_attention_widest_window(cuda_device, q):
    """A window of 2^31 - 1 is none, also where rows stand before position 0."""
    check_attention(Setup(q, [q, 1, q], [q - 2, 70, 130], 2, 64, 16, BF), 4, window=2 ** 31 - 1)


@pytest.mark.parametrize("q", [1, 3, 40])
@pytest.mark.parametrize("dtype", [BF, HF])
def test_attention_all_keys(cuda_device, q, dtype):
    check_attention(Setup(q, [q, 1, q], [q + 3, 300, 129], 2, 128, 16, dtype), 4, causal=False)


@pytest.mark.parametrize("q", [1, 4, 50])
def test_attention_rows_that_see_nothing(cuda_device, q):
    """Lengths of zero, below zero, and shorter than the rows of the call."""
    s = Setup(9, [q, q, q, 1], [max(1, q - 2), q, q + 30, 40], 2, 64, 16, BF)
    s.kv[1], s.kv[3] = 0, -5
    s.refresh()
    check_attention(s, 4)
    check_attention(s, 4, causal=False)


@pytest.mark.parametrize("q", [1, 4, 60])
def test_attention_masked_places_hold_anything(cuda_device, q):
    """NaN and infinities in the rows behind each length and before the window, in unused pages; bad pages are masked."""
    s = Setup(6, [q, q], [q + 50, q + 5], 2, 128, 16, BF)
    _, _ = clean = check_attention(s, 8, window=32, q=s.randn(s.T, 8, 128))
    q0 = s.randn(s.T, 8, 128)
    clean = check_attention(s, 8, window=32, q=q0)
    rows = s.plain()
    params = rows.params.copy()
    bad = np.ones(params.shape[:1] + params.shape[3:4], dtype=bool)      # [pages, page]
    for b in range(2):
        for j in range(max(0, s.kv[b] - q - 31), s.kv[b]):
            bad[s.table[b, j // 16], j % 16] = False
    values = np.array([np.nan, np.inf, -np.inf, 3e38], dtype=np.float32)
    where = np.nonzero(bad)
    params[where[0], :, :, where[1]] = values[np.random.default_rng(0).integers(0, 4, size=(len(where[0]), 2, 2, 2))]
    s.data.copy_(ref.words_of(rows.levels, params, BF).cuda())
    again = s.ap.kv4_attention(s.cache, s.batch, q0.cuda(), window=32, lse=True)
    assert torch.equal(again[0], clean[0]) and torch.equal(again[1], clean[1])
    s.table[0, 1] = s.cache.pages + 7
    s.table[1, 0] = -3
    s.refresh()
    s.data.copy_(ref.words_of(rows.levels, rows.params, BF).cuda())
    check_attention(s, 8, q=q0)


@pytest.mark.parametrize("q", [1, 5, 40])
@pytest.mark.parametrize("dtype", [BF, HF])
def test_attention_scores_far_apart(cuda_device, q, dtype):
    """Scores of hundreds, value rows of very different steps, a constant value row, a zero query, a negative scale."""
    s = Setup(3, [q, q], [q + 200, q + 70], 2, 64, 16, dtype)
    rows = s.plain()
    params = rows.params.copy()
    params[:, :, 1, 0::3] *= 2.0 ** -9
    params[:, :, 1, 1::5, 0] = 0
    params[:, :, 1, 2::7] *= 64
    s.data.copy_(ref.words_of(rows.levels, params, dtype).cuda())
    x = s.randn(s.T, 4, 64)
    x[0, 0] = 0
    x[-1, 1] *= 30
    x[0, 2] *= 2.0 ** -12
    check_attention(s, 4, q=x)
    check_attention(s, 4, q=x, scale=-0.5)
    check_attention(s, 4, q=x, scale=0.0)


def test_attention_nan_row_is_seen(cuda_device):
    """A row held as NaN makes NaN of the rows that see it and of no others."""
    for q in (1, 4, 40):
        s = Setup(5, [q, q], [q + 60, q + 60], 1, 64, 16, BF)
        rows = s.plain()
        at = q + 60 - 1     # only the last row of each sequence sees it
        params = rows.params.copy()
        params[s.table[0, at // 16], 0, 0, at % 16] = np.nan
        params[s.table[1, at // 16], 0, 1, at % 16] = np.nan
        s.data.copy_(ref.words_of(rows.levels, params, BF).cuda())
        out = s.ap.kv4_attention(s.cache, s.batch, s.randn(s.T, 2, 64).cuda())
        assert torch.isnan(out[[q - 1, 2 * q - 1]]).all()
        rest = [t for t in range(2 * q) if t not in (q - 1, 2 * q - 1)]
        assert torch.isfinite(out[rest]).all()


@pytest.mark.parametrize("dtype", [BF, HF])
def test_attention_long_and_ragged(cuda_device, dtype):
    """Sequences split over the device: one long among short ones."""
    check_attention(Setup(8, [1, 1, 1, 1], [3000, 17, 1, 700], 1, 64, 32, dtype), 2)
    check_attention(Setup(8, [2, 2], [2100, 40], 2, 128, 64, dtype), 4, window=1500)
    check_attention(Setup(8, [40], [2500], 1, 64, 64, dtype), 2)


@pytest.mark.parametrize("B,window", [(128, 0), (129, 0), (300, 40), (1000, 0)])
def test_attention_many_sequences(cuda_device, B, window):
    """Work shared out over more sequences than a block looks at in one go, some without rows, a few long ones among them."""
    rng = np.random.default_rng(B)
    lens_q = rng.integers(0, 3, size=B)
    lens_kv = lens_q + rng.integers(0, 40, size=B)
    lens_kv[::37] = rng.integers(500, 900, size=len(lens_kv[::37]))
    lens_q[0], lens_q[-1] = 0, 2
    check_attention(Setup(B, lens_q, np.maximum(lens_kv, 1), 2, 64, 64, BF, spare_rows=2), 4, window=window)


def test_attention_more_rows_than_promised(cuda_device):
    """Rows of a sequence beyond max_q are left as they were."""
    for promised, q in ((1, 3), (2, 9), (40, 50)):
        s = Setup(2, [q, 1], [q + 9, 20], 1, 64, 16, BF)
        s.max_q = promised
        s.refresh()
        check_attention(s, 4, max_q=promised)


def test_attention_views_and_repeats(cuda_device):
    """q as a view of a fused projection, out as a view, a workspace that held something else, and twice the same bits."""
    for q in (1, 4, 70):
        s = Setup(7, [q, q], [q + 300, q + 20], 2, 128, 16, BF)
        fused = s.randn(s.T, 4 + 2 + 2, 128).cuda()
        x = fused[:, :4]
        ws = torch.full((s.ap.kv4_attention_workspace_bytes(s.cache, s.batch, 4),), 255, dtype=torch.uint8, device="cuda")
        plain = s.ap.kv4_attention(s.cache, s.batch, x.contiguous(), workspace=ws)
        wide = torch.zeros(s.T, 6, 128, dtype=BF, device="cuda")
        s.ap.kv4_attention(s.cache, s.batch, x, out=wide[:, :4], workspace=ws)
        assert torch.equal(wide[:, :4], plain) and not wide[:, 4:].any()
        assert torch.equal(s.ap.kv4_attention(s.cache, s.batch, x), plain)
        s.ap.kv4_attention_check(ws)


def test_attention_refusals(cuda_device):
    import apnn_tc_b200 as ap
    s = Setup(7, [1, 1], [9, 9], 2, 64, 16, BF)
    q = s.randn(2, 4, 64).cuda()
    for kw in (dict(q=q.half()), dict(q=q[:, :, :32]), dict(q=q.cpu()), dict(out=q[:1]), dict(lse=q), dict(causal=False, window=4)):
        with pytest.raises(ValueError):
            ap.kv4_attention(s.cache, s.batch, **{"q": q, **kw})
    for kw in (dict(q=q[:, :3]), dict(workspace=torch.empty(8, dtype=torch.uint8, device="cuda")), dict(scale=float("nan")), dict(window=-1)):
        with pytest.raises(ap.ApnnError):
            ap.kv4_attention(s.cache, s.batch, **{"q": q, **kw})
    assert ap.kv4_attention(s.cache, s.batch, q[:0]).shape == (0, 4, 64)


# ------------------------------------------------------------------------------------------------------------ together
def layer(ap, w, cache, batch, x, table, ws):
    """One decoder layer: fused projection with bias, append, attention, output projection onto the stream, two-layer block onto the stream."""
    T, D, Hq, H = x.shape[0], cache.head_dim, w["Hq"], cache.heads
    qkv = ap.linear_planes(x, w["qkv"], w["s_qkv"], zero=7.5, bias=w["b_qkv"])
    q, k, v = (part.unflatten(1, (-1, D)) for part in qkv.split((Hq * D, H * D, H * D), 1))
    q = ap.kv4_append(cache, batch, k, v, q=q, q_norm=w["qn"], k_norm=w["kn"], rotary=table)
    o = ap.kv4_attention(cache, batch, q, workspace=ws)
    x = ap.linear_planes(o.view(T, Hq * D), w["o"], w["s_o"], zero=1.5, residual=x)
    h = ap.linear_planes(x, w["up"], w["s_up"], zero=0.5, activation="silu")
    return ap.linear_planes(h, w["down"], w["s_down"], zero=3.5, residual=x)


def layer_weights(E, Hq, H, D, F, seed=0):
    g = torch.Generator().manual_seed(seed)
    w = dict(Hq=Hq)
    for name, N, K, bits in (("qkv", (Hq + 2 * H) * D, E, 4), ("o", E, Hq * D, 2), ("up", F, E, 1), ("down", E, F, 3)):
        w[name] = ref.planes_of(torch.randint(0, 2 ** bits, (N, K), generator=g), bits).cuda()
        w["s_" + name] = ((torch.rand(N, generator=g) + 0.5) / (2 ** bits / 2 * K ** 0.5)).cuda()
    w["b_qkv"] = (torch.randn((Hq + 2 * H) * D, generator=g) * 0.3).cuda()
    w["qn"], w["kn"] = ((torch.randn(D, generator=g) * 0.1 + 1).to(BF).cuda() for _ in range(2))
    return w


@pytest.mark.parametrize("q", [1, 4, 48])
def test_layer_captured_and_eager(cuda_device, q):
    """The run of operators, eagerly and as a captured graph whose lengths, table and inputs move on between replays; both on their own
    workspace and stream.  The cache after both is the same, and a step's outputs are."""
    import apnn_tc_b200 as ap
    E, Hq, H, D, F = 256, 4, 2, 64, 384
    w = layer_weights(E, Hq, H, D, F)
    table = rotary_table(400, D).cuda()
    runs = []
    for captured in (False, True):
        s = Setup(3, [q, q], [q + 30, q + 3], H, D, 16, BF, wide=12)
        x = torch.zeros(2 * q, E, dtype=BF, device="cuda")
        ws = torch.empty(ap.kv4_attention_workspace_bytes(s.cache, s.batch, Hq), dtype=torch.uint8, device="cuda")
        g = torch.Generator().manual_seed(11)
        outs = []
        if captured:
            side = torch.cuda.Stream()
            side.wait_stream(torch.cuda.current_stream())
            start = s.data.clone()
            with torch.cuda.stream(side):
                layer(ap, w, s.cache, s.batch, x, table, ws)
            torch.cuda.current_stream().wait_stream(side)
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                y = layer(ap, w, s.cache, s.batch, x, table, ws)
            s.data.copy_(start)
        for step in range(3):
            x.copy_(torch.randn(2 * q, E, generator=g).to(BF))
            if captured:
                graph.replay()
            else:
                y = layer(ap, w, s.cache, s.batch, x, table, ws)
            outs.append(y.clone())
            s.batch.kv_len += q
        runs.append((outs, s.data.clone()))
    for a, b in zip(*[r[0] for r in runs]):
        assert torch.equal(a, b) and torch.isfinite(a).all()
    assert torch.equal(runs[0][1], runs[1][1])


def test_two_streams_at_once(cuda_device):
    """Two calls of each operator at once on two streams, each with its own workspace."""
    import apnn_tc_b200 as ap
    w = layer_weights(256, 4, 2, 64, 384)
    table = rotary_table(700, 64).cuda()
    sets = [Setup(i, [q, q], [q + 500, q + 90], 2, 64, 16, BF) for i, q in enumerate((1, 40))]
    xs = [torch.randn(s.T, 256, generator=torch.Generator().manual_seed(4)).to(BF).cuda() for s in sets]
    want = []
    for s, x in zip(sets, xs):
        start = s.data.clone()
        ws = torch.empty(ap.kv4_attention_workspace_bytes(s.cache, s.batch, 4), dtype=torch.uint8, device="cuda")
        want.append(layer(ap, w, s.cache, s.batch, x, table, ws).clone())
        s.data.copy_(start)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    spaces = [torch.empty(ap.kv4_attention_workspace_bytes(s.cache, s.batch, 4), dtype=torch.uint8, device="cuda") for s in sets]
    for _ in range(5):
        got = []
        for s, x, st, ws in zip(sets, xs, streams, spaces):
            with torch.cuda.stream(st):
                got.append(layer(ap, w, s.cache, s.batch, x, table, ws))
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert torch.equal(a, b)
