"""The operators of a low-bit decoder layer, as measurable cases.

* ``linear`` -- ``linear_planes``: 16-bit activations times weights held as bit planes, with bias, activation and residual
  in the epilogue;
* ``append`` -- ``kv4_append`` (norm of each head, position rotation, 4-bit quantisation into the pages of a cache), then
  ``kv4_read`` of the rows it wrote: what a program does that hands a chunk's keys and values on as the cache holds them;
* ``attend`` -- ``kv4_attention`` over such a cache: single tokens, a few tokens to verify, prompts.

``own`` false computes the same from elementary torch operations in 32 bits.

A page of the cache holds, for each head, the key levels [page][D/2] (two per byte, even element in the low half), the value
levels, then (step, lowest) of every key row and of every value row in the cache's type.
"""
import math

import torch

own = False

TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
MOST_LINEAR = 2.0 * 4096 * 16384 * 4096            # operations of the largest product
MOST_ATTEND = 4.0 * 128 * 32 * 8192 * 8192 / 2     # and of the largest attention
MOST_APPEND = 8900 * 48 * 64                       # elements of the largest append
MOST_CACHE = 64 * 8192 * 8 * 136                   # bytes of cache that an append goes to


# ---------------------------------------------------------------------------------------------------------- cases
def linear(name, M, N, K, wbits, dtype, act="none", bias=True, residual=False, zero=None, out=None):
    return dict(name=name, kind="linear", M=M, N=N, K=K, wbits=wbits, dtype=dtype, act=act, bias=bias, residual=residual,
                zero=(2 ** wbits - 1) / 2 if zero is None else zero, out=out or dtype)


def append(name, B, most_q, Hq, Hkv, D, page, dtype, norm=True, rot=None, interleaved=False, before=1024):
    return dict(name=name, kind="append", B=B, most_q=most_q, Hq=Hq, Hkv=Hkv, D=D, page=page, dtype=dtype, norm=norm,
                rot=D if rot is None else rot, interleaved=interleaved, before=before)


def attend(name, B, most_q, least_kv, most_kv, Hq, Hkv, D, page, dtype, causal=True, window=0, lse=False):
    return dict(name=name, kind="attend", B=B, most_q=most_q, least_kv=least_kv, most_kv=most_kv, Hq=Hq, Hkv=Hkv, D=D, page=page,
                dtype=dtype, causal=causal, window=window, lse=lse)


def listed():
    return [
        # one token through a square projection: the call whose latency a user waits for
        linear("linear_m1_4096x4096_w4", 1, 4096, 4096, 4, "bf16"),
        # a small decoding batch through the widening half of a block, two-bit weights
        linear("linear_m16_16384x4096_w2", 16, 16384, 4096, 2, "fp16", act="gelu_tanh"),
        # +-1 weights onto float scores of a vocabulary that is no multiple of anything
        linear("linear_m64_32003x2048_w1_fp32", 64, 32003, 2048, 1, "bf16", bias=False, out="fp32"),
        # a ragged middle-sized product: odd rows and columns, K inside its padding, residual stream added
        linear("linear_m333_2337x2296_w3", 333, 2337, 2296, 3, "bf16", act="relu", residual=True),
        # a prompt through the widening half of a block
        linear("linear_m4096_16384x4096_w4", 4096, 16384, 4096, 4, "bf16", act="silu"),
        # one new token for each of 64 sequences: norms, rotation, 4-bit rows scattered over the pages
        append("append_b64_d128", 64, 1, 32, 8, 128, 16, "bf16", before=8192),
        # prompts of different lengths, adjacent pairs rotated, no norm
        append("append_b4_prompts_d64", 4, 4096, 16, 16, 64, 64, "fp16", norm=False, interleaved=True, before=100),
        # one short request: all latency
        attend("attend_b1_kv333_d128", 1, 1, 333, 333, 32, 8, 128, 16, "bf16"),
        # one long request: the cache's length is split over the device
        attend("attend_b1_kv65536_d128", 1, 1, 65536, 65536, 64, 8, 128, 64, "bf16"),
        # a decoding batch whose sequences are of very different lengths
        attend("attend_b64_kv16384_d128", 64, 1, 64, 16384, 32, 8, 128, 64, "bf16", lse=True),
        # four drafted tokens verified for each sequence, one query head per key head, a sliding window
        attend("attend_b24_q4_d64_window", 24, 4, 300, 6000, 16, 16, 64, 32, "fp16", window=2048),
        # a prompt
        attend("attend_prompt_8192_d128", 1, 8192, 8192, 8192, 32, 8, 128, 64, "bf16"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(("linear", "linear", "append", "attend", "attend"))
    dtype = rng.choice(("bf16", "bf16", "fp16"))
    Hkv, group = rng.choice((1, 2, 4, 8, 16)), rng.choice((1, 2, 4, 5, 7, 8))
    D, page = rng.choice((64, 128, 128, 256)), rng.choice((16, 16, 32, 64, 128))
    if Hkv * group > 64:
        group = 1
    if kind == "linear":
        M = rng.choice((1, _log(rng, 1, 16), _log(rng, 1, 4096), _log(rng, 64, 4096)))
        N, K = _log(rng, 64, 32768), _log(rng, 64, 16384)
        if rng.random() < 0.6:
            N = (N + 127) // 128 * 128
        K = (K + 127) // 128 * 128 if rng.random() < 0.7 else (K + 7) // 8 * 8
        while 2.0 * M * N * K > MOST_LINEAR:
            M = (M + 1) // 2
        wbits = rng.choice((1, 2, 3, 4, 4))
        c = linear("", M, N, K, wbits, dtype, rng.choice(("none", "none", "relu", "silu", "gelu", "gelu_tanh")),
                   rng.random() < 0.5, rng.random() < 0.4, rng.choice((None, 0.0, float(2 ** (wbits - 1)))),
                   rng.choice((dtype, dtype, "fp32")))
    elif kind == "append":
        B = _log(rng, 1, 256)
        most_q = 1 if rng.random() < 0.5 else _log(rng, 1, 8192)
        while B * most_q * Hkv * (group + 2) * D > MOST_APPEND:
            B, most_q = (B + 1) // 2, max(1, most_q // 2)
        before = _log(rng, 1, 8192)
        while B * (most_q + before) * Hkv * (D + 8) > MOST_CACHE:
            before //= 2
        c = append("", B, most_q, Hkv * group, Hkv, D, page, dtype, rng.random() < 0.6, rng.choice((0, D // 2, D, D)),
                   rng.random() < 0.4, before)
    else:
        form = rng.choice(("one", "one", "few", "prompt"))
        if form == "prompt":
            B, most_q = _log(rng, 1, 8), _log(rng, 16, 8192)
            most_kv = most_q + rng.choice((0, 0, _log(rng, 1, 8192)))
            least_kv = max(1, most_kv // 3)
            while 4.0 * D * Hkv * group * B * most_q * most_kv > MOST_ATTEND:
                if B > 1:
                    B -= 1
                else:
                    most_q, most_kv, least_kv = (most_q + 1) // 2, (most_kv + 1) // 2, (least_kv + 1) // 2
        else:
            most_q = 1 if form == "one" else rng.randint(2, 8)
            B, most_kv = _log(rng, 1, 128), _log(rng, most_q, 65536)
            while B * most_kv * Hkv * (D + 8) > 64 * 16384 * 8 * 136:
                B = (B + 1) // 2
                if B == 1:
                    break
            least_kv = rng.choice((most_kv, max(most_q, most_kv // 50)))
        causal = rng.random() < 0.85
        c = attend("", B, most_q, min(least_kv, most_kv), most_kv, Hkv * group, Hkv, D, page, dtype, causal,
                   _log(rng, 16, 8192) if causal and rng.random() < 0.25 else 0, rng.random() < 0.3)
    c.pop("name")
    return c


# ---------------------------------------------------------------------------------------------------------- the cache
def _quantise(x, dtype):
    """Float rows [..., D] -> levels (uint8 values 0..15), step and lowest value in ``dtype``; every operation rounds in 32 bits.

    A row that is not finite, or whose step or lowest value is not finite in ``dtype``, is held as NaN; a step below 2^-126 as 0."""
    lo, hi = x.amin(-1, keepdim=True), x.amax(-1, keepdim=True)
    step = (hi / 15 - lo / 15).to(dtype).float()
    low = lo.to(dtype).float()
    step = torch.where(step < 2.0 ** -126, torch.zeros_like(step), step)
    bad = ~(torch.isfinite(step) & torch.isfinite(low))
    inverse = torch.where(step > 0, 1 / torch.where(step > 0, step, torch.ones_like(step)), torch.zeros_like(step))
    level = torch.round((x - low) * inverse).clamp(0, 15)
    level = torch.where(bad, torch.zeros_like(level), level).to(torch.uint8)
    nan = torch.full_like(step, float("nan"))
    return level, torch.where(bad, nan, step).to(dtype), torch.where(bad, nan, low).to(dtype)


def _bytes_of(level, step, low):
    """Levels [..., page, D] with their (step, low) [..., page, 1] -> code bytes and parameter bytes, flat over the page."""
    codes = level[..., 0::2] | (level[..., 1::2] << 4)
    params = torch.cat((step, low), -1).contiguous().view(torch.uint8)
    return codes.flatten(-2), params.flatten(-2)


def _rows_of(data, D, page, dtype):
    """Cache words [..., heads, words] -> keys and values [..., heads, page, D] in 32 bits."""
    raw = data.contiguous().view(torch.uint8)
    n = page * D // 2
    out = []
    for at, par in ((0, 2 * n), (n, 2 * n + 4 * page)):
        code = raw[..., at:at + n].unflatten(-1, (page, D // 2))
        level = torch.stack((code & 15, code >> 4), -1).flatten(-2).float()
        p = raw[..., par:par + 4 * page].contiguous().view(dtype).unflatten(-1, (page, 2)).float()
        out.append(p[..., :1] * level + p[..., 1:])
    return out


def _fill_cache(pages, case, gen):
    """A cache of random rows: keys with channels of their own offset, as position-rotated keys have, and plain values."""
    D, page, H, dtype = case["D"], case["page"], case["Hkv"], TYPES[case["dtype"]]
    data = torch.empty((pages, H, page * (D + 8) // 4), dtype=torch.int32, device="cuda")
    raw = data.view(torch.uint8)
    n = page * D // 2
    offset = torch.randn((H, 1, D), device="cuda", generator=gen) * 0.5
    for i, at in enumerate((0, n)):
        x = torch.randn((pages, H, page, D), device="cuda", generator=gen)
        x = x + offset if i == 0 else x
        codes, params = _bytes_of(*_quantise(x, dtype))
        raw[..., at:at + n] = codes
        raw[..., 2 * n + 4 * page * i:2 * n + 4 * page * (i + 1)] = params
    return data


def _batch(case, gen, lengths_q, lengths_kv):
    """Offsets, lengths and a page table whose pages lie scattered over the cache."""
    B, page = len(lengths_kv), case["page"]
    wide = max(1, (max(lengths_kv) + page - 1) // page)
    pages = B * wide
    table = torch.randperm(pages, device="cuda", generator=gen).view(B, wide).to(torch.int32)
    cu = [0]
    for n in lengths_q:
        cu.append(cu[-1] + n)
    return dict(cu_q=torch.tensor(cu, dtype=torch.int32, device="cuda"), table=table, pages=pages, T=cu[-1], max_q=max(lengths_q),
                kv_len=torch.tensor(lengths_kv, dtype=torch.int32, device="cuda"))


def _spread(least, most, B):
    """B lengths over [least, most], evenly over their logarithm, the longest first: the same for every seed."""
    if B == 1:
        return [most]
    return [int(round(math.exp(math.log(most) + (math.log(max(least, 1)) - math.log(most)) * i / (B - 1)))) for i in range(B)]


def _lengths(case):
    B, most_q = case["B"], case["most_q"]
    if case["kind"] == "append":
        q = _spread(max(1, most_q // 4), most_q, B)
        return q, [n + (case["before"] * (i + 1)) // B for i, n in enumerate(q)]
    kv = _spread(case["least_kv"], case["most_kv"], B)
    return [min(most_q, n) for n in kv], kv


def _owners(cu_q, T):
    """For every query row its sequence and its place within it."""
    t = torch.arange(T, device=cu_q.device)
    b = torch.searchsorted(cu_q[1:].long(), t, right=True)
    return b, t - cu_q.long()[b]


# ---------------------------------------------------------------------------------------------------------- states
def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype = TYPES[case["dtype"]]

    def randn(*shape):
        return torch.randn(shape, device="cuda", generator=gen)

    if case["kind"] == "linear":
        M, N, K, wbits = case["M"], case["N"], case["K"], case["wbits"]
        level = torch.randint(0, 2 ** wbits, (N, K), device="cuda", generator=gen, dtype=torch.int32)
        s = dict(case=case, x=randn(M, K).to(dtype), planes=_planes(level, wbits),
                 scale=(torch.rand(N, device="cuda", generator=gen) + 0.5) / (2 ** wbits / 2 * math.sqrt(K)),
                 bias=randn(N) * 0.5 if case["bias"] else None,
                 residual=randn(M, N).to(TYPES[case["out"]]) if case["residual"] else None)
        if own:
            import apnn_tc_b200 as ap
            s["ap"] = ap
        return s
    s = dict(case=case, **_batch(case, gen, *_lengths(case)))
    s["cache"] = _fill_cache(s["pages"], case, gen)
    T, Hq, Hkv, D = s["T"], case["Hq"], case["Hkv"], case["D"]
    if case["kind"] == "append":
        qkv = randn(T, (Hq + 2 * Hkv) * D).to(dtype)     # the fused projection's rows: q, k and v are views of it
        s["q"], s["k"], s["v"] = (part.unflatten(1, (-1, D)) for part in qkv.split((Hq * D, Hkv * D, Hkv * D), 1))
        s["q_norm"] = (randn(D) * 0.2 + 1).to(dtype) if case["norm"] else None
        s["k_norm"] = (randn(D) * 0.2 + 1).to(dtype) if case["norm"] else None
        s["rotary"] = _rotary(int(s["kv_len"].max()), case["rot"]) if case["rot"] else None
    else:
        s["q"] = randn(T, Hq, D).to(dtype)
    if own:
        import apnn_tc_b200 as ap
        s["ap"] = ap
        s["kv"] = ap.KVCache4(s["pages"], Hkv, case["page"], D, dtype, data=s["cache"])
        s["batch"] = ap.KVBatch(s["cu_q"], s["kv_len"], s["table"], s["max_q"])
        if case["kind"] == "attend":
            s["workspace"] = torch.empty(ap.kv4_attention_workspace_bytes(s["kv"], s["batch"], Hq), dtype=torch.uint8, device="cuda")
    return s


def _planes(level, wbits):
    """Levels [N, K] -> bit planes [wbits, N, PAD128(K)/32]; element k is bit 31 - k % 32 of word k / 32."""
    N, K = level.shape
    full = torch.zeros((N, (K + 127) // 128 * 128), dtype=torch.int32, device=level.device)
    full[:, :K] = level
    shift = torch.arange(31, -1, -1, device=level.device, dtype=torch.int64)
    return torch.stack([((full >> p & 1).view(N, -1, 32).long() << shift).sum(-1).to(torch.int32) for p in range(wbits)])


def _rotary(positions, rot):
    """cos and sin [positions, rot/2 + rot/2] of the angles pos / 10000^(2i/rot), made in 64 bits."""
    inverse = 10000.0 ** (-torch.arange(0, rot, 2, dtype=torch.float64, device="cuda") / rot)
    angle = torch.arange(positions, dtype=torch.float64, device="cuda")[:, None] * inverse
    return torch.cat((angle.cos(), angle.sin()), 1).float()


# ---------------------------------------------------------------------------------------------------------- one pass
def run(state):
    case = state["case"]
    if own:
        ap = state["ap"]
        if case["kind"] == "linear":
            return ap.linear_planes(state["x"], state["planes"], state["scale"], zero=case["zero"], bias=state["bias"],
                                    activation=case["act"], residual=state["residual"], out_dtype=TYPES[case["out"]])
        if case["kind"] == "append":
            q = ap.kv4_append(state["kv"], state["batch"], state["k"], state["v"], q=state["q"], q_norm=state["q_norm"],
                              k_norm=state["k_norm"], eps=1e-6, rotary=state["rotary"], interleaved=case["interleaved"])
            return (q,) + ap.kv4_read(state["kv"], state["batch"], state["T"])
        return ap.kv4_attention(state["kv"], state["batch"], state["q"], causal=case["causal"], window=case["window"],
                                lse=case["lse"], workspace=state["workspace"])
    if case["kind"] == "linear":
        return _linear_plain(state)
    return _append_plain(state) if case["kind"] == "append" else _attend_plain(state)


def _levels(planes, K):
    shift = torch.arange(31, -1, -1, device=planes.device, dtype=torch.int32)
    wbits, N, words = planes.shape
    bits = (planes.unsqueeze(-1) >> shift & 1).view(wbits, N, words * 32)[:, :, :K]
    weight = (1 << torch.arange(wbits, device=planes.device, dtype=torch.int32)).view(-1, 1, 1)
    return (bits * weight).sum(0)


def _activate(y, act):
    if act == "relu":
        return y.clamp(min=0)
    if act == "silu":
        return y / (1 + torch.exp(-y))
    if act == "gelu":
        return 0.5 * y * (1 + torch.erf(y / math.sqrt(2.0)))
    if act == "gelu_tanh":
        return 0.5 * y * (1 + torch.tanh(math.sqrt(2.0 / math.pi) * (y + 0.044715 * y * y * y)))
    return y


def _linear_plain(s, real=torch.float32):
    case = s["case"]
    w = _levels(s["planes"], case["K"]).to(real) - case["zero"]
    y = (s["x"].to(real) @ w.t()) * s["scale"].to(real)
    if s["bias"] is not None:
        y = y + s["bias"].to(real)
    y = _activate(y, case["act"])
    if s["residual"] is not None:
        y = y + s["residual"].to(real)
    return y.to(TYPES[case["out"]])


def _normed(x, weight, real=torch.float32):
    """x / sqrt(mean(x^2) + 1e-6) * weight; the mean in 64 bits, every other operation rounded in 32."""
    y = x.to(real)
    if weight is None:
        return y
    mean = (y.double() * y.double()).mean(-1, keepdim=True) + 1e-6
    return y * (1 / torch.sqrt(mean.to(real))) * weight.to(real)


def _rotated(y, table, pos, interleaved):
    if table is None:
        return y
    half = table.shape[1] // 2
    row = table[pos].to(y.dtype).unsqueeze(1)
    c, s = row[..., :half], row[..., half:]
    turn, rest = y[..., :2 * half], y[..., 2 * half:]
    a, b = (turn[..., 0::2], turn[..., 1::2]) if interleaved else (turn[..., :half], turn[..., half:])
    first, second = a * c - b * s, b * c + a * s
    turn = torch.stack((first, second), -1).flatten(-2) if interleaved else torch.cat((first, second), -1)
    return torch.cat((turn, rest), -1)


def _positions(s):
    b, i = _owners(s["cu_q"], s["T"])
    n = (s["cu_q"][1:] - s["cu_q"][:-1]).long()
    return b, s["kv_len"].long()[b] - n[b] + i


def _append_plain(s):
    case = s["case"]
    D, page, dtype = case["D"], case["page"], TYPES[case["dtype"]]
    b, pos = _positions(s)
    q = _rotated(_normed(s["q"], s["q_norm"]), s["rotary"], pos, case["interleaved"])
    k = _rotated(_normed(s["k"], s["k_norm"]), s["rotary"], pos, case["interleaved"])
    where, slot = s["table"].long()[b, pos // page], pos % page
    raw, n = s["cache"].view(torch.uint8), page * D // 2
    row, quad = torch.arange(D // 2, device="cuda"), torch.arange(4, device="cuda")
    for i, x in enumerate((k, s["v"].float())):
        codes, params = _bytes_of(*(part.unsqueeze(-2) for part in _quantise(x, dtype)))     # [T, H, D/2] and [T, H, 4]
        raw[where[:, None], :, (n * i + slot * (D // 2))[:, None] + row] = codes.transpose(1, 2)
        raw[where[:, None], :, (2 * n + 4 * page * i + slot * 4)[:, None] + quad] = params.transpose(1, 2)
    k, v = _read_plain(s, b, pos)
    return q.to(dtype), k, v


def _read_plain(s, b, pos):
    """The values that the cache now holds for the batch's rows, gathered byte by byte."""
    case = s["case"]
    D, page, dtype = case["D"], case["page"], TYPES[case["dtype"]]
    where, slot = s["table"].long()[b, pos // page], pos % page
    raw, n = s["cache"].view(torch.uint8), page * D // 2
    row, quad = torch.arange(D // 2, device="cuda"), torch.arange(4, device="cuda")
    out = []
    for i in range(2):
        code = raw[where[:, None], :, (n * i + slot * (D // 2))[:, None] + row].transpose(1, 2)
        par = raw[where[:, None], :, (2 * n + 4 * page * i + slot * 4)[:, None] + quad].transpose(1, 2).contiguous()
        p = par.view(dtype).float()
        level = torch.stack((code & 15, code >> 4), -1).flatten(-2).float()
        out.append((p[..., :1] * level + p[..., 1:]).to(dtype))
    return out


def _visible(s, q_pos, keys):
    """Which keys [.., keys] a query at position q_pos [.., 1] of a sequence of s["kv_len"] sees."""
    case = s["case"]
    seen = keys < s["kv_len"].long().view(-1, 1, 1)
    if case["causal"]:
        seen = seen & (keys <= q_pos)
        if case["window"]:
            seen = seen & (keys > q_pos - case["window"])
    return seen


def _attend_plain(s):
    case = s["case"]
    Hq, Hkv, D, page, dtype = case["Hq"], case["Hkv"], case["D"], case["page"], TYPES[case["dtype"]]
    B, G, T, most = s["kv_len"].numel(), Hq // Hkv, s["T"], s["max_q"]
    b, i = _owners(s["cu_q"], T)
    k, v = (x.permute(0, 2, 1, 3, 4).flatten(2, 3) for x in _rows_of(s["cache"][s["table"].long()], D, page, dtype))   # [B, Hkv, L, D]
    q = torch.zeros((B, most, Hq, D), device="cuda")
    q[b, i] = s["q"].float()
    q = q.view(B, most, Hkv, G, D).permute(0, 2, 3, 1, 4).reshape(B, Hkv, G * most, D)
    scores = ((q @ k.transpose(2, 3)) / math.sqrt(D)).view(B, Hkv * G, most, -1)
    n = (s["cu_q"][1:] - s["cu_q"][:-1]).long()
    q_pos = (s["kv_len"].long() - n).view(-1, 1, 1) + torch.arange(most, device="cuda").view(1, -1, 1)
    seen = _visible(s, q_pos, torch.arange(scores.shape[-1], device="cuda").view(1, 1, -1)).unsqueeze(1)
    scores.masked_fill_(~seen, float("-inf"))
    top = scores.amax(-1, keepdim=True)
    top = torch.where(torch.isinf(top), torch.zeros_like(top), top)
    p = scores.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    o = (p.view(B, Hkv, G * most, -1) @ v).view(B, Hq, most, D) / torch.where(total > 0, total, torch.ones_like(total))
    out = o.permute(0, 2, 1, 3)[b, i].to(dtype)
    return (out, (top + torch.log(total)).squeeze(-1).transpose(1, 2)[b, i]) if case["lse"] else out


# ---------------------------------------------------------------------------------------------------------- what a pass needs
def work(case):
    size = {"bf16": 2, "fp16": 2, "fp32": 4}
    e = size[case["dtype"]]
    if case["kind"] == "linear":
        M, N, K = case["M"], case["N"], case["K"]
        o = size[case["out"]]
        return {"bytes": e * M * K + case["wbits"] * N * K / 8 + 4 * N * (2 if case["bias"] else 1) + o * M * N * (2 if case["residual"] else 1),
                "flops": 2.0 * M * N * K}
    lengths_q, lengths_kv = _lengths(case)
    T, Hq, Hkv, D = sum(lengths_q), case["Hq"], case["Hkv"], case["D"]
    if case["kind"] == "append":
        # rows in (q, k, v and the rotation of their positions); q, the cache's rows, and the keys and values read back out
        return {"bytes": T * (e * (Hq + 2 * Hkv) * D + 4 * case["rot"] + e * Hq * D + Hkv * (D + 8) + 2 * e * Hkv * D), "flops": 8.0 * T * (Hq + 2 * Hkv) * D}
    pairs, rows = 0, 0
    for nq, nk in zip(lengths_q, lengths_kv):
        first = nk - nq
        if not case["causal"]:
            pairs, rows = pairs + nq * nk, rows + nk
        else:
            w = case["window"] or nk
            pairs += sum(min(first + i + 1, w) for i in range(nq))
            rows += nk - max(0, first + 1 - w)
    return {"bytes": rows * Hkv * (D + 8) + 2 * e * T * Hq * D + (4 * T * Hq if case["lse"] else 0), "flops": 4.0 * D * Hq * pairs}


# ---------------------------------------------------------------------------------------------------------- in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "linear":
        return _linear_exact(s)
    if case["kind"] == "append":
        return _append_exact(s)
    return _attend_exact(s)


def _linear_exact(s):
    case = s["case"]
    planes, K = s["planes"], case["K"]
    w = torch.full((planes.shape[1], K), -float(case["zero"]), dtype=torch.float64, device="cuda")
    for p in range(planes.shape[0]):
        for r in range(32):
            n = len(range(r, K, 32))
            w[:, r::32] += ((planes[p, :, :n] >> (31 - r)) & 1).double() * 2 ** p
    y = torch.matmul(s["x"].double(), w.t())
    y *= s["scale"].double()
    if s["bias"] is not None:
        y += s["bias"].double()
    act = case["act"]
    if act == "relu":
        y = torch.where(y > 0, y, torch.zeros_like(y))
    elif act == "silu":
        y = y * torch.sigmoid(y)
    elif act == "gelu":
        y = y * 0.5 * torch.erfc(-y / 2 ** 0.5)
    elif act == "gelu_tanh":
        y = y * torch.sigmoid(2 * (2 / math.pi) ** 0.5 * (y + 0.044715 * y ** 3))
    if s["residual"] is not None:
        y += s["residual"].double()
    return y


def _append_exact(s):
    case = s["case"]
    D, dtype = case["D"], TYPES[case["dtype"]]
    b, pos = _positions(s)
    if case["rot"]:
        half = case["rot"] // 2
        c, sn = s["rotary"][pos, :half].double().unsqueeze(1), s["rotary"][pos, half:].double().unsqueeze(1)

    def turned(x, weight):
        x = x.double()
        if weight is not None:
            x = x * torch.rsqrt(x.pow(2).mean(-1, keepdim=True) + 1e-6) * weight.double()
        if not case["rot"]:
            return x
        out = x.clone()
        first = slice(0, 2 * half, 2) if case["interleaved"] else slice(0, half)
        second = slice(1, 2 * half, 2) if case["interleaved"] else slice(half, 2 * half)
        out[..., first] = x[..., first] * c - x[..., second] * sn
        out[..., second] = x[..., second] * c + x[..., first] * sn
        return out

    def held(x):
        lo = x.amin(-1, keepdim=True)
        step = ((x.amax(-1, keepdim=True) - lo) / 15).to(dtype).double()
        lo = lo.to(dtype).double()
        return lo + step * torch.nan_to_num(((x - lo) / step).round(), nan=0.0).clamp(0, 15)

    return turned(s["q"], s["q_norm"]), held(turned(s["k"], s["k_norm"])), held(s["v"].double())


def _attend_exact(s):
    case = s["case"]
    Hq, Hkv, D, page, dtype = case["Hq"], case["Hkv"], case["D"], case["page"], TYPES[case["dtype"]]
    G = Hq // Hkv
    out = torch.zeros((s["T"], Hq, D), dtype=torch.float64, device="cuda")
    lse = torch.full((s["T"], Hq), float("-inf"), dtype=torch.float64, device="cuda")
    cu, lengths, table = s["cu_q"].tolist(), s["kv_len"].tolist(), s["table"].long()
    n = page * D // 2
    for b, L in enumerate(lengths):
        nq = cu[b + 1] - cu[b]
        if nq == 0 or L == 0:
            continue
        raw = s["cache"][table[b, :(L + page - 1) // page]].view(torch.uint8)       # [pages, heads, bytes]
        code = raw[..., :2 * n].unflatten(-1, (2, page, D // 2))
        par = raw[..., 2 * n:].contiguous().view(dtype).unflatten(-1, (2, page, 2)).double()
        for h in range(Hkv):
            kv = []
            for i in range(2):
                x = code[:, h, i].reshape(-1, D // 2)[:L]
                level = torch.empty((L, D), dtype=torch.float64, device="cuda")
                level[:, 0::2], level[:, 1::2] = (x & 15).double(), (x >> 4).double()
                p = par[:, h, i].reshape(-1, 2)[:L]
                kv.append(torch.addcmul(p[:, 1:], level, p[:, :1]))
            for at in range(0, nq, 1024):
                i = torch.arange(at, min(nq, at + 1024), device="cuda")
                q = s["q"][cu[b] + i, h * G:(h + 1) * G].double()                    # [rows, G, D]
                x = torch.einsum("rgd,kd->rgk", q, kv[0]) * D ** -0.5
                place, key = (L - nq + i).view(-1, 1, 1), torch.arange(L, device="cuda").view(1, 1, -1)
                if case["causal"]:
                    hidden = (key > place) | ((key <= place - case["window"]) if case["window"] else torch.zeros_like(key, dtype=torch.bool))
                    x = x.masked_fill(hidden, float("-inf"))
                l = torch.logsumexp(x, -1, keepdim=True)
                p = torch.exp(x - l).nan_to_num(nan=0.0)
                out[cu[b] + i, h * G:(h + 1) * G] = torch.einsum("rgk,kd->rgd", p, kv[1])
                lse[cu[b] + i, h * G:(h + 1) * G] = l.squeeze(-1)
    return (out, lse) if case["lse"] else out
