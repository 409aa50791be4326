"""GPU parity of the long-context serving operators against plain 64-bit
restatements: packed prompt attention, the 4-bit KV cache (append, read,
single-token attention, eviction) and their refusals.

Bars, with A = sum_j p_j |v_j| (the result's magnitude before cancellation):
 - packed attention: the result is rounded to bf16 (8 significant bits: 2^-8
   of itself at most) and so are the probabilities (2^-8 of each at most, so
   2^-8 A), the scores' fp32 rounding adds less than 1e-4 A:
   |got - ref| <= 2^-8 |ref| + (2^-8 + 1e-4) A. lse: 1e-4 absolute (fp32
   sums of 128 products whose magnitudes add up to some tens).
 - 4-bit attention: probabilities as two bf16 pieces (2^-16 of each), fp32
   sums: 2^-14 A in fp32, and 2^-8 |ref| more in bf16. Weights: 2e-5 of the
   row's largest sum plus 2e-5 relative.
 - codes, positions, evictions: equal."""
import math

import pytest
import torch

import smoe_cuda as S

pytestmark = pytest.mark.gpu
BF16, F32, F64 = torch.bfloat16, torch.float32, torch.float64


def ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def starts(n):
    return ints([sum(n[:i]) for i in range(len(n) + 1)])


def gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


# ------------------------------------------------------- packed prompt attention
def packed_ref(q, k, v, lens, causal, window, scale):
    """(out, A, lse, has a key) per row in 64 bits; rows without a key: zeros and -inf."""
    out, mag = torch.zeros(q.shape, dtype=F64, device="cuda"), torch.zeros(q.shape, dtype=F64, device="cuda")
    lse = torch.full(q.shape[:2], -math.inf, dtype=F64, device="cuda")
    G = q.shape[1] // k.shape[1]
    q0 = k0 = 0
    for lq, lk in lens:
        i = torch.arange(lq, device="cuda")[:, None] + lk - lq
        j = torch.arange(lk, device="cuda")[None]
        shut = (j > i) if causal else torch.zeros(lq, lk, dtype=torch.bool, device="cuda")
        if window:
            shut = shut | (j <= i - window)
        for h in range(q.shape[1]):
            if lk == 0 or lq == 0:
                continue
            x = q[q0:q0 + lq, h].double() @ k[k0:k0 + lk, h // G].double().t() * scale
            x = x.masked_fill(shut, -math.inf)
            any_ = ~shut.all(-1)
            p = torch.softmax(x[any_], -1)
            vv = v[k0:k0 + lk, h // G].double()
            rows = torch.arange(q0, q0 + lq, device="cuda")[any_]
            out[rows, h], mag[rows, h] = p @ vv, p @ vv.abs()
            lse[rows, h] = torch.logsumexp(x[any_], -1)
        q0, k0 = q0 + lq, k0 + lk
    return out, mag, lse


def packed_inputs(lens, H, Hkv, hd, seed, strided=False, std=1.5):
    g = gen(seed)
    tq, tk = sum(a for a, _ in lens), sum(b for _, b in lens)

    def rows(n, heads, s):
        x = (torch.randn(n, heads, hd, generator=g, device="cuda") * s).to(BF16)
        if not strided:
            return x.contiguous()
        big = torch.full((heads, n, hd + 24), float("nan"), dtype=BF16, device="cuda")   # heads outermost, padded rows
        big[:, :, 8:8 + hd] = x.transpose(0, 1)
        return big.transpose(0, 1)[:, :, 8:8 + hd]
    return rows(tq, H, std), rows(tk, Hkv, 1.0), rows(tk, Hkv, 1.0)


def packed_run(ctx, q, k, v, lens, causal=True, window=0, scale=None):
    out = torch.full(q.shape, float("nan"), dtype=BF16, device="cuda")
    lse = torch.full(q.shape[:2], float("nan"), dtype=F32, device="cuda")
    args = S.packed_attn_args(q, k, v, out, starts([a for a, _ in lens]), starts([b for _, b in lens]), scale=scale,
                              causal=causal, window=window, lse=lse)
    ctx.attention_packed(args)
    ctx.synchronize()
    return out, lse


def packed_check(out, lse, ref):
    want, mag, wlse = ref
    assert torch.isfinite(out).all()
    assert ((out.double() - want).abs() <= 2 ** -8 * want.abs() + (2 ** -8 + 1e-4) * mag + 1e-30).all()
    none = wlse == -math.inf
    assert (lse[none] == -math.inf).all() and (out[none] == 0).all()
    assert ((lse.double() - wlse)[~none].abs() <= 1e-4).all()


PACKED = [
    # lens (q, k) of the sequences, heads, KV heads, head_dim, causal, window, strided
    ([(1, 1)], 32, 4, 128, True, 0, False),
    ([(45, 45)], 32, 4, 128, True, 0, False),
    ([(17, 17), (1, 1), (0, 0), (130, 130), (2, 2), (63, 63)], 32, 4, 128, True, 0, False),
    ([(300, 300), (5, 5), (257, 257)], 64, 4, 128, True, 0, True),
    ([(129, 129), (16, 16)], 8, 8, 128, True, 0, False),
    ([(33, 400), (1, 500), (128, 128), (100, 1001)], 16, 8, 64, True, 0, False),
    ([(33, 400), (1, 500), (200, 200), (100, 1001)], 16, 8, 64, True, 70, True),
    ([(300, 300), (40, 700)], 12, 4, 128, True, 1, False),
    ([(50, 20), (10, 0), (0, 7), (4, 3)], 32, 4, 128, True, 0, False),      # rows without a key
    ([(50, 20), (10, 0), (9, 300)], 6, 2, 64, False, 0, False),
    ([(70, 190), (3, 129)], 28, 4, 128, False, 0, True),
    ([(140, 140)], 5, 1, 96, True, 0, False),
    ([(37, 90), (64, 64)], 7, 7, 80, True, 33, False),
    ([(20, 20), (300, 310)], 4, 1, 8, True, 0, True),
    ([(40, 200)], 128, 1, 64, True, 0, False),
    ([(3, 640)], 100, 1, 128, True, 0, False),
    ([(1, 3000), (2, 5000), (1, 1)], 32, 4, 128, True, 0, False),
    ([(1100, 1100)], 32, 4, 128, True, 0, False),
    ([(7 * i % 23, 7 * i % 23 + i) for i in range(90)], 8, 2, 64, True, 0, False),
]


@pytest.mark.parametrize("case", range(len(PACKED)))
def test_packed_attention(ctx, case):
    lens, H, Hkv, hd, causal, window, strided = PACKED[case]
    q, k, v = packed_inputs(lens, H, Hkv, hd, 100 + case, strided)
    scale = 1 / math.sqrt(hd)
    out, lse = packed_run(ctx, q, k, v, lens, causal, window)
    packed_check(out, lse, packed_ref(q, k, v, lens, causal, window, scale))
    again, lse2 = packed_run(ctx, q, k, v, lens, causal, window)
    assert torch.equal(out, again) and torch.equal(lse, lse2)


@pytest.mark.parametrize("std", [0.0, 30.0])
def test_packed_attention_flat_and_peaked(ctx, std):
    """Equal scores (q = 0: plain means) and scores in the hundreds (one key decides, the maximum moves far)."""
    lens = [(400, 400), (3, 900)]
    q, k, v = packed_inputs(lens, 8, 2, 128, 7, std=std)
    out, lse = packed_run(ctx, q, k, v, lens)
    want, mag, wlse = packed_ref(q, k, v, lens, True, 0, 1 / math.sqrt(128))
    # at |score| in the hundreds fp32 scores are off by about 2^-24 * sum |q k| scale < 1e-3, and so are logs of probabilities
    slack = 1e-4 if std == 0 else 2e-3
    assert ((out.double() - want).abs() <= 2 ** -8 * want.abs() + (2 ** -8 + slack) * mag + 1e-30).all()
    assert ((lse.double() - wlse).abs() <= slack).all()


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf"), 3.38e38])
@pytest.mark.parametrize("causal", [True, False])
def test_packed_attention_masked_places(ctx, bad, causal):
    """Whatever later tokens, other sequences and rows outside the packing hold, earlier rows do not see it."""
    lens = [(150, 150), (40, 300), (77, 77)]
    q, k, v = packed_inputs(lens, 16, 2, 128, 11)
    clean, _ = packed_run(ctx, q, k, v, lens, causal)
    q2, k2, v2 = q.clone(), k.clone(), v.clone()
    q2[150:190] = bad                    # the middle sequence altogether
    k2[150:450], v2[150:450] = bad, bad
    if causal:                           # and the last token of the first
        k2[149], v2[149] = bad, bad
    out, lse = packed_run(ctx, q2, k2, v2, lens, causal)
    rows = list(range(149 if causal else 150)) + list(range(190, 267))
    assert torch.equal(out[rows], clean[rows])
    if bad != bad:
        assert out[150:190].isnan().all()
        if causal:
            assert out[149].isnan().all()


@pytest.mark.parametrize("kind", ["nan", "inf", "mixed"])
def test_packed_attention_nonfinite_values_seen(ctx, kind):
    """Infinities and NaN among the values reach just the rows that attend to them, column by column."""
    lens = [(300, 300)]
    q, k, v = packed_inputs(lens, 8, 2, 64, 12)
    v[40, 0, 3] = float("nan") if kind == "nan" else float("inf")
    v[200, 0, 5] = -float("inf")
    if kind == "mixed":
        v[250, 0, 3] = -float("inf")
    out, _ = packed_run(ctx, q, k, v, lens)
    assert torch.isfinite(out[:, 4:]).all() and torch.isfinite(out[:40]).all()
    got = out[:, :4].float()
    assert torch.isfinite(got[:, :, [0, 1, 2, 4] + list(range(6, 64))]).all()
    col = got[40:, :, 3]
    if kind == "nan":
        assert col.isnan().all()
    else:
        stop = 210 if kind == "mixed" else 260
        assert (col[:stop] == float("inf")).all()
        assert kind == "inf" or col[210:].isnan().all()
    assert torch.isfinite(got[:200, :, 5]).all() and (got[200:, :, 5] == -float("inf")).all()


def test_packed_attention_bad_rows_are_skipped(ctx):
    """Row ranges outside the buffers: an error at the next synchronize, the other sequences as they are."""
    lens = [(20, 20), (30, 30)]
    q, k, v = packed_inputs(lens, 8, 2, 64, 3)
    out = torch.zeros(q.shape, dtype=BF16, device="cuda")
    cu = ints([0, 20, 80])
    ctx.attention_packed(S.packed_attn_args(q, k, v, out, cu))
    with pytest.raises(S.SmoeCudaError, match="ERR_DEVICE"):
        ctx.synchronize()
    want, mag, _ = packed_ref(q[:20], k[:20], v[:20], lens[:1], True, 0, 1 / 8)
    assert ((out[:20].double() - want).abs() <= 2 ** -8 * want.abs() + (2 ** -8 + 1e-4) * mag).all()
    assert (out[20:] == 0).all()
    # nothing to do
    ctx.attention_packed(S.packed_attn_args(q[:0], k, v, out[:0], ints([0])))
    ctx.synchronize()


def test_packed_attention_refusals(ctx):
    lens = [(20, 20)]
    q, k, v = packed_inputs(lens, 8, 2, 64, 3)
    out = torch.zeros_like(q)

    def refused(what, **kw):
        a = S.packed_attn_args(q, k, v, out, starts([20]))
        for n, x in kw.items():
            setattr(a, n, x)
        with pytest.raises(S.SmoeCudaError, match=what):
            ctx.attention_packed(a)
    refused("ERR_ARG", q=None)
    refused("ERR_ARG", cu_q=None)
    refused("ERR_ARG", num_kv_heads=3)
    refused("ERR_ARG", q=q.data_ptr() + 2)
    refused("ERR_ARG", k_row=12)
    refused("ERR_ARG", causal=0, window=4)
    refused("ERR_UNSUPPORTED", head_dim=136)
    refused("ERR_UNSUPPORTED", head_dim=12)
    refused("ERR_UNSUPPORTED", num_heads=258)
    with pytest.raises(TypeError):
        S.packed_attn_args(q.float(), k, v, out, starts([20]))
    ctx.synchronize()
    assert (out == 0).all()


# ------------------------------------------------------------------ 4-bit cache
def quantised(x):
    """Codes [.., groups, 64], scale and bias of rows in fp32, as the header defines them."""
    g = x.float().unflatten(-1, (-1, 64))
    lo, hi = g.amin(-1, keepdim=True), g.amax(-1, keepdim=True)
    bias = lo.bfloat16().float()
    scale = ((hi - lo) * torch.tensor(1 / 15, dtype=F32, device=x.device)).bfloat16().float()
    code = torch.where(scale > 0, ((g - bias) / torch.where(scale > 0, scale, 1.0)).round(), 0.0).clamp(0, 15)
    return code, scale, bias


class Cache:
    """A cache over shuffled pages and the 64-bit values of its entries."""

    def __init__(self, Hkv, hd, lens, room, seed, garbage=True):
        self.g = gen(seed)
        self.Hkv, self.hd, self.B = Hkv, hd, len(lens)
        width = max((n + room + 63) // 64 for n in lens) + 1
        pages = self.B * width + 3
        self.blocks = torch.full((pages, Hkv, S.kv4_block_bytes(hd)), 255 if garbage else 0, dtype=torch.uint8,
                                 device="cuda")                    # scales of 0xffff: NaN where nothing was written
        self.table = torch.randperm(pages, generator=self.g, device="cuda")[: self.B * width].int().view(self.B, width)
        self.table = self.table.contiguous()
        self.len, self.seen = ints([0] * self.B), ints([0] * self.B)
        self.pos = torch.zeros(pages, Hkv, 64, dtype=torch.int32, device="cuda")
        self.score = torch.full((pages, Hkv, 64), float("nan"), device="cuda")
        self.lens = list(lens)
        self.n = [0] * self.B

    def desc(self):
        return S.kv4_cache(self.blocks, self.table, self.len, self.hd, seen=self.seen, pos=self.pos, score=self.score)

    def at(self, b, n, first=0):
        e = torch.arange(first, first + n, device="cuda")
        return self.table[b, e // 64].long(), e % 64

    def values(self, b, n):
        """K, V [n, Hkv, hd] in 64 bits from the bytes."""
        page, slot = self.at(b, n)
        ng = self.hd // 64
        raw = self.blocks[page]                                    # [n, Hkv, bytes]
        codes = raw[..., : ng * 4096].unflatten(-1, (2, ng, 64, 32))
        sb = raw[..., ng * 4096:].contiguous().view(BF16).unflatten(-1, (2, ng, 64, 2))
        i = torch.arange(n, device="cuda")
        c, s = codes[i, :, :, :, slot], sb[i, :, :, :, slot].double()
        c = torch.stack((c & 15, c >> 4), -1).flatten(-2).double()
        x = (c * s[..., 0:1] + s[..., 1:2]).flatten(-2)            # [n, Hkv, 2, hd]
        return x[:, :, 0], x[:, :, 1]

    def fill(self, ctx, dtype=BF16):
        rows = sum(self.lens)
        k = torch.randn(rows, self.Hkv, self.hd, generator=self.g, device="cuda").to(dtype)
        v = torch.randn(rows, self.Hkv, self.hd, generator=self.g, device="cuda").to(dtype)
        if rows:
            ctx.kv4_append(self.desc(), S.kv4_rows(k, v, starts(self.lens)))
        ctx.kv4_advance(self.len, self.seen, self.B, cu=starts(self.lens))
        ctx.synchronize()
        return k, v


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("Hkv,hd,lens,more", [(4, 128, [1], [1]), (2, 64, [63, 0, 64, 65], [2, 130, 1, 0]),
                                              (8, 128, [10, 200, 128], [54, 1, 300]), (1, 64, [5] * 70, [3] * 70),
                                              (3, 128, [700, 9], [0, 1])])
def test_kv4_append_and_read(ctx, dtype, Hkv, hd, lens, more):
    c = Cache(Hkv, hd, lens, max(more), 5)
    k0, v0 = c.fill(ctx, dtype)
    n = sum(more)
    big = torch.randn(n, 2, Hkv + 1, hd, generator=c.g, device="cuda").to(dtype)   # rows with gaps
    k1, v1 = big[:, 0, 1:], big[:, 1, :-1]
    if n:
        k1[0, 0] = 2.5                                             # a group of equal values
        v1[-1, -1] *= 1e30
    before = c.blocks.clone()
    ctx.kv4_append(c.desc(), S.kv4_rows(k1, v1, starts(more)))
    ctx.synchronize()
    assert c.len.tolist() == lens and c.seen.tolist() == lens
    total = [a + b for a, b in zip(lens, more)]
    back = [torch.full((sum(total), Hkv, hd), float("nan"), dtype=dtype, device="cuda") for _ in range(2)]
    ctx.kv4_read(c.desc(), None, S.kv4_rows(*back, starts(total)))
    part = [torch.zeros(n, Hkv, hd, dtype=dtype, device="cuda") for _ in range(2)]
    ctx.kv4_read(c.desc(), c.len, S.kv4_rows(*part, starts(more)))
    ctx.synchronize()
    row = old = new = 0
    written = torch.zeros(c.blocks.shape[:2] + (64,), dtype=torch.bool, device="cuda")
    for b in range(len(lens)):
        for side, (x0, x1) in enumerate(((k0, k1), (v0, v1))):
            want = torch.cat((x0[old: old + lens[b]], x1[new: new + more[b]]))
            code, scale, bias = quantised(want)
            value = (code * scale + bias).flatten(-2)
            assert torch.equal(back[side][row: row + total[b]], value.to(dtype))
            assert torch.equal(part[side][new: new + more[b]], value[lens[b]:].to(dtype))
            if total[b]:
                assert ((c.values(b, total[b])[side] - value.double()).abs() <= 1e-6 * value.double().abs() + 1e-6).all()
        page, slot = c.at(b, total[b])
        assert (c.pos[page, :, slot] == torch.arange(total[b], device="cuda")[:, None]).all()
        page, slot = c.at(b, more[b], lens[b])
        assert (c.score[page, :, slot] == 0).all()
        written[page, :, slot] = True
        row, old, new = row + total[b], old + lens[b], new + more[b]
    codes = lambda t: t[..., : hd * 64].unflatten(-1, (-1, 64, 32)).transpose(2, 3)
    assert torch.equal(codes(c.blocks)[~written], codes(before)[~written])          # nothing else was touched


def test_kv4_append_nonfinite(ctx):
    """A group with an infinity or NaN stays in its group and entry."""
    c = Cache(2, 128, [3], 1, 9)
    k, v = (torch.randn(3, 2, 128, generator=c.g, device="cuda") for _ in range(2))
    k[1, 0, 70] = float("nan")
    v[2, 1, 5] = float("inf")
    ctx.kv4_append(c.desc(), S.kv4_rows(k, v, starts([3])))
    ko, vo = torch.zeros_like(k), torch.zeros_like(v)
    ctx.kv4_read(c.desc(), None, S.kv4_rows(ko, vo, starts([3])))
    ctx.synchronize()
    bad_k, bad_v = torch.zeros_like(k, dtype=torch.bool), torch.zeros_like(k, dtype=torch.bool)
    bad_v[2, 1, :64] = True
    bad_k[1, 0, 64:] = True
    for x, o, bad in ((k, ko, bad_k), (v, vo, bad_v)):
        code, scale, bias = quantised(x)
        assert torch.equal(o[~bad], (code * scale + bias).flatten(-2)[~bad])
    assert not torch.isfinite(vo[bad_v]).any()


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_kv4_append_magnitudes(ctx, dtype):
    """Groups from subnormal to 1e37, groups far from zero, constant ones, whole numbers that end half-way between two codes."""
    n = 200
    c = Cache(2, 128, [n], 1, 10)
    k = torch.randn(n, 2, 128, generator=c.g, device="cuda")
    v = k * 10.0 ** torch.linspace(-44, 37, n, device="cuda")[:, None, None]
    k[:40] = 1000 + k[:40] * 1e-3
    k[40:80] = -7e5 + k[40:80] * 2
    k[80:120] = torch.arange(128, device="cuda") % 31 - 4.0         # (scale 2: every other value is half-way)
    k[120:130] = 3.25
    k, v = k.to(dtype), v.to(dtype)
    ctx.kv4_append(c.desc(), S.kv4_rows(k, v, starts([n])))
    ko, vo = torch.zeros(n, 2, 128, device="cuda"), torch.zeros(n, 2, 128, device="cuda")
    c.len += n
    ctx.kv4_read(c.desc(), None, S.kv4_rows(ko, vo, starts([n])))
    ctx.synchronize()
    for x, o in ((k, ko), (v, vo)):
        code, scale, bias = quantised(x)
        assert torch.equal(o, (code * scale + bias).flatten(-2))


def test_kv4_bad_pages_are_skipped(ctx):
    c = Cache(2, 64, [64, 64], 70, 9)
    c.fill(ctx)
    good = c.table.clone()
    c.table[0, 1] = c.blocks.shape[0]
    k = torch.randn(4, 2, 64, device="cuda")
    ctx.kv4_append(c.desc(), S.kv4_rows(k, k, starts([2, 2])))
    with pytest.raises(S.SmoeCudaError, match="ERR_DEVICE"):
        ctx.synchronize()
    c.len[1] = c.table.shape[1] * 64 - 1                           # one entry of room
    ctx.kv4_append(c.desc(), S.kv4_rows(k, k, starts([0, 2])))
    with pytest.raises(S.SmoeCudaError, match="ERR_DEVICE"):
        ctx.synchronize()
    c.table = good
    out = torch.zeros(2, 2, 64, device="cuda")
    ctx.kv4_read(c.desc(), ints([0, 64]), S.kv4_rows(out, out, starts([0, 2])))
    ctx.synchronize()
    code, scale, bias = quantised(k[2:])
    assert torch.equal(out, (code * scale + bias).flatten(-2))


def attn_run(ctx, c, q, max_len, extra=0, score=False, decay=1.0, in_place=False):
    out = torch.full(q.shape, float("nan"), dtype=q.dtype, device="cuda")
    so = None if not score else c.score if in_place else torch.full_like(c.score, -1.0)
    args = S.kv4_attn_args(q, out, max_len, extra=extra, score_out=so, decay=decay)
    ws = torch.full((max(1, S.kv4_attention_workspace(c.desc(), args)),), 255, dtype=torch.uint8, device="cuda")
    ctx.kv4_attention(c.desc(), S.kv4_attn_set_workspace(args, ws))
    ctx.synchronize()
    return out, so


def attn_check(c, q, lens, out, so=None, old=None, decay=1.0):
    scale = 1 / math.sqrt(c.hd)
    for b, n in enumerate(lens):
        if n == 0:
            assert (out[b] == 0).all()
            continue
        k, v = c.values(b, n)
        x = torch.einsum("kgd,nkd->kgn", q[b].double().view(c.Hkv, -1, c.hd), k) * scale
        p = torch.softmax(x, -1)
        want = torch.einsum("kgn,nkd->kgd", p, v).reshape(q.shape[1:])
        mag = torch.einsum("kgn,nkd->kgd", p, v.abs()).reshape(q.shape[1:])
        tol = 2 ** -14 * mag + (2 ** -8 * want.abs() if q.dtype == BF16 else 0)
        assert ((out[b].double() - want).abs() <= tol).all(), (b, n, float(((out[b].double() - want).abs() / mag).max()))
        if so is not None:
            page, slot = c.at(b, n)
            w = p.sum(1).t()
            if decay:
                w = w + decay * old[page, :, slot].double()
            assert ((so[page, :, slot].double() - w).abs() <= 2e-5 * (w.abs() + p.sum(1).max())).all()


ATTN = [
    # heads, KV heads, head_dim, lengths, extra
    (32, 4, 128, [1], 0),
    (32, 4, 128, [300], 0),
    (32, 4, 128, [64, 65, 0, 127, 1, 640], 0),
    (64, 4, 128, [45, 1000, 333], 0),
    (8, 8, 64, [17, 900], 1),
    (12, 4, 128, [5, 70, 2049], 0),
    (5, 1, 64, [129, 64], 1),
    (28, 4, 64, [500, 1], 0),
    (40, 2, 128, [77, 1300], 0),
    (33, 1, 128, [90], 0),
    (32, 4, 128, [5000, 12345], 0),
    (16, 8, 64, [6000], 1),
    (4, 2, 128, [20 + 3 * i for i in range(70)], 0),
]


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("case", range(len(ATTN)))
def test_kv4_attention(ctx, dtype, case):
    """Entries after the last hold NaN scales, and the last page ends inside a tile."""
    H, Hkv, hd, lens, extra = ATTN[case]
    c = Cache(Hkv, hd, lens, 1, 20 + case)
    c.fill(ctx)
    if extra:
        c.len -= extra
    q = (torch.randn(len(lens), H, hd, generator=c.g, device="cuda") * 2).to(dtype)
    c.score.copy_(torch.rand(c.score.shape, generator=c.g, device="cuda"))
    old = c.score.clone()
    out, _ = attn_run(ctx, c, q, max(lens) + 5, extra)
    attn_check(c, q, lens, out)
    for decay in (1.0, 0.0, 0.5):
        out2, so = attn_run(ctx, c, q, max(lens), extra, score=True, decay=decay)
        attn_check(c, q, lens, out2, so, old, decay)
    rest = torch.ones(so.shape, dtype=torch.bool, device="cuda")
    for b, n in enumerate(lens):
        page, slot = c.at(b, n)
        rest[page, :, slot] = False
    assert (so[rest] == -1).all()                                  # entries that were not attended to stay
    again, so2 = attn_run(ctx, c, q, max(lens), extra, score=True, decay=0.5)
    assert torch.equal(out2, again) and torch.equal(so, so2)
    attn_run(ctx, c, q, max(lens), extra, score=True, decay=0.5, in_place=True)
    assert torch.equal(c.score[~rest], so[~rest]) and torch.equal(c.score[rest], old[rest])


@pytest.mark.parametrize("lens", [[14300, 0, 14250, 3], [56900], [28500, 28400]])
def test_kv4_attention_long_stretches(ctx, lens):
    """Enough pages that every warp has eight or more: stretches of two lengths, which cut pairs at any page."""
    Hkv = 32 if sum(lens) < 40000 else 16
    c = Cache(Hkv, 64, lens, 1, 55)
    c.fill(ctx)
    assert sum((n + 63) // 64 for n in lens) * Hkv > 8 * 1776
    q = torch.randn(len(lens), Hkv, 64, generator=c.g, device="cuda") * 2
    c.score.copy_(torch.rand(c.score.shape, generator=c.g, device="cuda"))
    old = c.score.clone()
    out, so = attn_run(ctx, c, q, max(lens), score=True, decay=0.5)
    attn_check(c, q, lens, out, so, old, 0.5)
    again, so2 = attn_run(ctx, c, q, max(lens), score=True, decay=0.5)
    assert torch.equal(out, again) and torch.equal(so, so2)


@pytest.mark.parametrize("std", [0.0, 40.0])
def test_kv4_attention_flat_and_peaked(ctx, std):
    """Equal scores, and scores in the hundreds (fp32 scores are then off by 2^-24 of some hundreds: 1e-4 of a probability)."""
    c = Cache(2, 128, [3000, 700], 1, 77)
    c.fill(ctx)
    q = torch.randn(2, 16, 128, generator=c.g, device="cuda") * std
    out, _ = attn_run(ctx, c, q, 3000)
    for b, n in enumerate([3000, 700]):
        k, v = c.values(b, n)
        p = torch.softmax(torch.einsum("kgd,nkd->kgn", q[b].double().view(2, -1, 128), k) / math.sqrt(128), -1)
        want, mag = (torch.einsum("kgn,nkd->kgd", p, x).reshape(16, 128) for x in (v, v.abs()))
        assert ((out[b].double() - want).abs() <= (2 ** -14 + (3e-4 if std else 0)) * mag).all()


def test_kv4_attention_too_long_and_refusals(ctx):
    c = Cache(2, 64, [100, 30], 1, 3)
    c.fill(ctx)
    q = torch.randn(2, 4, 64, generator=c.g, device="cuda")
    out = torch.zeros_like(q)
    args = S.kv4_attn_args(q, out, 64)
    ws = torch.zeros(max(16, S.kv4_attention_workspace(c.desc(), args)), dtype=torch.uint8, device="cuda")
    S.kv4_attn_set_workspace(args, ws)
    ctx.kv4_attention(c.desc(), args)
    with pytest.raises(S.SmoeCudaError, match="ERR_DEVICE"):
        ctx.synchronize()
    attn_check(c, q, [64, 30], out)

    def refused(what, cache=None, **kw):
        a = S.kv4_attn_set_workspace(S.kv4_attn_args(q, out, 100, score_out=c.score), ws)
        for n, x in kw.items():
            setattr(a, n, x)
        with pytest.raises(S.SmoeCudaError, match=what):
            ctx.kv4_attention(cache or c.desc(), a)
    refused("ERR_ARG", q=None)
    refused("ERR_ARG", num_heads=3)
    refused("ERR_ARG", dtype=2)
    refused("ERR_ARG", workspace_bytes=0)
    refused("ERR_ARG", q=q.data_ptr() + 4)
    bad = c.desc()
    bad.head_dim = 96
    refused("ERR_UNSUPPORTED", bad)
    bad = c.desc()
    bad.table = None
    refused("ERR_ARG", bad)
    with pytest.raises(S.SmoeCudaError):
        S.kv4_block_bytes(80)
    ctx.synchronize()


def evict_ref(scores, pos, seen, n, keep, recent):
    """entries that end up in the slots [0, min(n, keep)), by the rule of the header."""
    if n <= keep:
        return list(range(n))
    late = [p + recent >= seen for p in pos]
    key = [(math.inf, 1) if l else (-math.inf, -1) if s != s else (s, 0) for l, s in zip(late, scores)]
    best = set(sorted(range(n), key=lambda i: ((-key[i][0], -key[i][1]), i))[:keep])
    into = list(range(keep))
    free = [i for i in range(keep) if i not in best]
    for i, j in zip(free, sorted(i for i in best if i >= keep)):
        into[i] = j
    return into


EVICT = [
    # KV heads, head_dim, lengths, keep, recent, scores
    (2, 128, [100, 64, 65, 1, 0], 64, 8, "random"),
    (4, 128, [1100, 1024, 1500], 1024, 100, "random"),
    (1, 64, [3000], 70, 64, "random"),
    (3, 64, [500, 333], 100, 1, "ties"),
    (2, 128, [500, 333], 100, 30, "equal"),
    (2, 64, [400], 33, 200, "random"),       # more recent ones than stay
    (2, 64, [400, 90], 40, 3, "special"),
    (1, 128, [5000], 4900, 0, "random"),
    (1, 64, [7], 1, 0, "random"),
]


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("case", range(len(EVICT)))
def test_kv4_evict(ctx, case, in_place):
    Hkv, hd, lens, keep, recent, kind = EVICT[case]
    c = Cache(Hkv, hd, lens, 1, 50 + case)
    c.fill(ctx)
    shape = c.score.shape
    s = torch.rand(shape, generator=c.g, device="cuda")
    if kind == "ties":
        s = (s * 5).floor()
    elif kind == "equal":
        s = torch.full(shape, 0.25, device="cuda")
    elif kind == "special":
        pick = torch.randint(0, 8, shape, generator=c.g, device="cuda")
        for i, x in enumerate((float("nan"), float("inf"), -float("inf"), 0.0, -0.0, -1.0)):
            s[pick == i] = x
    c.score.copy_(s)
    # positions of the entries as they were left by an earlier eviction: out of order past the first 20
    for b, n in enumerate(lens):
        page, slot = c.at(b, n)
        perm = torch.stack([torch.randperm(n, generator=c.g, device="cuda") for _ in range(Hkv)], 1)
        c.pos[page, :, slot] = perm.int()
    old_blocks, old_pos, old_score = c.blocks.clone(), c.pos.clone(), c.score.clone()
    pos_out = None if in_place else torch.full_like(c.pos, -7)
    score_out = None if in_place else torch.full_like(c.score, -7.0)
    ws = torch.full((S.kv4_evict_workspace(c.desc(), max(lens) + 3),), 255, dtype=torch.uint8, device="cuda")
    for _ in range(1 if in_place else 2):    # with separate outputs a second call does the same again
        ctx.kv4_evict(c.desc(), keep, recent, max(lens) + 3, ws, pos_out, score_out)
    ctx.synchronize()
    new_pos, new_score = (c.pos, c.score) if in_place else (pos_out, score_out)
    same = torch.ones(shape, dtype=torch.bool, device="cuda")
    eq = lambda a, b: ((a == b) | (a.isnan() & b.isnan())).all()
    ng = hd // 64
    codes = lambda t: t[..., : ng * 4096].unflatten(-1, (2 * ng, 64, 32))
    sb = lambda t: t[..., ng * 4096:].unflatten(-1, (2 * ng, 64, 4))
    for b, n in enumerate(lens):
        page, slot = c.at(b, n)
        for h in range(Hkv):
            into = evict_ref(old_score[page, h, slot].tolist(), old_pos[page, h, slot].tolist(), n, n, keep, recent)
            src = torch.tensor(into, dtype=torch.long, device="cuda")
            tp, ts, fp, fs = page[: len(into)], slot[: len(into)], page[src], slot[src]
            assert (new_pos[tp, h, ts] == old_pos[fp, h, fs]).all()
            assert eq(new_score[tp, h, ts], old_score[fp, h, fs])
            assert torch.equal(codes(c.blocks)[tp, h, :, ts], codes(old_blocks)[fp, h, :, fs])
            assert torch.equal(sb(c.blocks)[tp, h, :, ts], sb(old_blocks)[fp, h, :, fs])
            same[tp, h, ts] = False
    assert torch.equal(codes(c.blocks).transpose(2, 3)[same], codes(old_blocks).transpose(2, 3)[same])
    if in_place:
        assert (c.pos[same] == old_pos[same]).all() and eq(c.score[same], old_score[same])
    else:
        assert (pos_out[same] == -7).all() and (score_out[same] == -7).all()
        assert torch.equal(c.pos, old_pos) and eq(c.score, old_score)
    ctx.kv4_advance(c.len, c.seen, c.B, n_each=0, keep=keep)
    ctx.synchronize()
    assert c.len.tolist() == [min(n, keep) for n in lens] and c.seen.tolist() == lens


def test_kv4_evict_refusals(ctx):
    c = Cache(2, 64, [100], 1, 3)
    c.fill(ctx)
    c.score.fill_(1.0)
    ws = torch.zeros(S.kv4_evict_workspace(c.desc(), 100), dtype=torch.uint8, device="cuda")
    with pytest.raises(S.SmoeCudaError, match="ERR_ARG"):
        ctx.kv4_evict(c.desc(), 0, 1, 100, ws)
    with pytest.raises(S.SmoeCudaError, match="ERR_ARG"):
        ctx.kv4_evict(c.desc(), 10, 1, 200, ws)                    # workspace too small
    with pytest.raises(S.SmoeCudaError, match="ERR_ARG"):
        ctx.kv4_evict(c.desc(), 10, 1, 100, ws, pos_out=torch.zeros_like(c.pos))
    with pytest.raises(S.SmoeCudaError, match="ERR_ARG"):
        ctx.kv4_evict(c.desc(), 10, 1, 100, ws, pos_out=c.pos, score_out=c.score)
    bare = S.kv4_cache(c.blocks, c.table, c.len, 64)
    with pytest.raises(S.SmoeCudaError, match="ERR_ARG"):
        ctx.kv4_evict(bare, 10, 1, 100, ws)
    with pytest.raises(S.SmoeCudaError, match="ERR_ARG"):
        ctx.kv4_append(c.desc(), S.Kv4Rows())
    ctx.synchronize()


def test_serving_step_in_a_graph_on_another_stream(ctx):
    """append, attention with weights, eviction and advance captured once and replayed, against the same calls one by one."""
    lens, keep = [90, 130], 96

    def make():
        c = Cache(2, 128, lens, 20, 41)
        c.fill(ctx)
        c.score.fill_(0.0)
        c.k = torch.randn(2, 2, 128, generator=c.g, device="cuda")
        c.q = torch.randn(2, 16, 128, generator=c.g, device="cuda")
        c.out = torch.zeros_like(c.q)
        c.args = S.kv4_attn_args(c.q, c.out, 160, extra=1, score_out=c.score)
        c.ws = torch.zeros(max(S.kv4_attention_workspace(c.desc(), c.args), S.kv4_evict_workspace(c.desc(), 160)),
                           dtype=torch.uint8, device="cuda")
        S.kv4_attn_set_workspace(c.args, c.ws)
        c.cu = starts([1, 1])
        return c

    def step(x, c):
        x.kv4_append(c.desc(), S.kv4_rows(c.k, c.k, c.cu))
        x.kv4_attention(c.desc(), c.args)
        x.kv4_advance(c.len, c.seen, 2, n_each=1)
        x.kv4_evict(c.desc(), keep, 16, 160, c.ws)
        x.kv4_advance(c.len, c.seen, 2, n_each=0, keep=keep)
    one, two = make(), make()
    other = S.Context(0, max_batch=4)
    s = torch.cuda.Stream()
    other.set_stream(s.cuda_stream)
    torch.cuda.synchronize()
    for _ in range(9):
        step(ctx, one)
    ctx.synchronize()
    with torch.cuda.stream(s):
        step(other, two)
        other.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            step(other, two)
        for _ in range(8):
            graph.replay()
    other.synchronize()
    assert torch.equal(one.out, two.out) and one.len.tolist() == two.len.tolist() == [96, 96]
    assert torch.equal(one.pos, two.pos) and one.seen.tolist() == [99, 139]
    assert torch.equal(one.score.nan_to_num(-1), two.score.nan_to_num(-1)) and torch.equal(one.blocks, two.blocks)
    del graph
    other.close()
