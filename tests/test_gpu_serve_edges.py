"""GPU tests of the long-context serving operators at their edges: strides,
NaN in cache rows, scales of 0, row ranges outside their buffers, outliers
among the cache's groups. Bars as in test_gpu_serve.py unless derived here."""
import math

import pytest
import torch

import smoe_cuda as S
import test_gpu_serve as T
from test_gpu_serve import BF16, F32, attn_run, ints, quantised, starts

pytestmark = pytest.mark.gpu


# ---------------------------------------------------------------------- strides
@pytest.mark.parametrize("lens,H,Hkv,hd", [([(45, 45), (3, 200)], 32, 4, 128),                # a CTA per pair
                                           ([(150, 900), (40, 1300), (77, 777)], 16, 2, 64),   # equal shares
                                           ([(940, 1300), (1500, 1500), (333, 333)], 32, 8, 128)])     # the list
@pytest.mark.parametrize("which", ["k", "v", "kv"])
def test_packed_attention_shared_kv_heads(ctx, lens, H, Hkv, hd, which):
    """K and V expanded over their heads (stride 0) give the bits of copies."""
    q, k, v = T.packed_inputs(lens, H, Hkv, hd, 600)
    a, b = (x[:, :1].contiguous().expand(-1, Hkv, -1) if n in which else x for n, x in (("k", k), ("v", v)))
    assert (a.stride(1) == 0) == ("k" in which)
    out, lse = T.packed_run(ctx, q, a, b, lens)
    want, want_lse = T.packed_run(ctx, q, a.contiguous(), b.contiguous(), lens)
    assert torch.equal(out, want) and torch.equal(lse, want_lse)
    T.packed_check(out, lse, T.packed_ref(q, a, b, lens, True, 0, 1 / math.sqrt(hd)))


def test_packed_attention_stride_refusals(ctx):
    """Strides of 0 and outputs that overlap are refused; a dimension of one element may have any stride."""
    lens = [(20, 20)]
    q, k, v = T.packed_inputs(lens, 8, 2, 64, 601)
    out = torch.zeros_like(q)

    def refused(q=q, k=k, v=v, out=out, **kw):
        a = S.packed_attn_args(q, k, v, out, starts([20]))
        for n, x in kw.items():
            setattr(a, n, x)
        with pytest.raises(S.SmoeCudaError, match="ERR_ARG"):
            ctx.attention_packed(a)
    refused(q=q[:, :1].expand(-1, 8, -1))
    refused(q=q[:1].expand(20, -1, -1))
    refused(k=k[:1].expand(20, -1, -1))
    refused(v=v[:1].expand(20, -1, -1))
    refused(out=out[:, :1].expand(-1, 8, -1))
    refused(out=out[:1].expand(20, -1, -1))
    refused(out_row=64 * 7)              # rows that end in the next one
    refused(out_head=56)
    refused(out_row=8 * 64 * 10, out_head=8 * 64 * 10)
    ctx.synchronize()
    assert (out == 0).all()
    # one row, one query head per call: their strides are nobody's
    want, want_lse = T.packed_run(ctx, q[:1], k[:1], v[:1], [(1, 1)])
    a = S.packed_attn_args(q[:1], k[:1], v[:1], out[:1], starts([1]))
    a.q_row, a.k_row, a.v_row, a.out_row = 0, 3, 5, 0
    ctx.attention_packed(a)
    q1, k1, v1 = q[:, :1].contiguous(), k[:, :1].contiguous(), v[:, :1].contiguous()
    one = torch.zeros_like(q1)
    b = S.packed_attn_args(q1, k1, v1, one, starts([20]))
    b.q_head, b.k_head, b.v_head, b.out_head = 1, 0, 7, 0
    ctx.attention_packed(b)
    ctx.synchronize()
    assert torch.equal(out[:1], want)
    want, _ = T.packed_run(ctx, q1, k1, v1, lens)
    assert torch.equal(one, want)


def test_kv4_outputs_that_overlap_are_refused(ctx):
    c = T.Cache(2, 64, [20, 30], 1, 610)
    k, v = c.fill(ctx)
    x = torch.zeros(50, 2, 64, device="cuda")
    cu = starts([20, 30])

    def refused(k, v, **kw):
        r = S.kv4_rows(k, v, cu)
        for n, y in kw.items():
            setattr(r, n, y)
        with pytest.raises(S.SmoeCudaError, match="ERR_ARG"):
            ctx.kv4_read(c.desc(), None, r)
    refused(x[:, :1].expand(-1, 2, -1), x)
    refused(x, x[:1].expand(50, -1, -1))
    refused(x, x.clone(), k_row=64)
    refused(x, x.clone(), v_head=60)
    q = torch.randn(2, 4, 64, device="cuda")
    out = torch.zeros_like(q)
    args = S.kv4_attn_args(q, out, 40)
    ws = torch.zeros(S.kv4_attention_workspace(c.desc(), args), dtype=torch.uint8, device="cuda")
    S.kv4_attn_set_workspace(args, ws)
    for row in (0, 64, 4 * 64 - 4):
        args.out_row = row
        with pytest.raises(S.SmoeCudaError, match="ERR_ARG"):
            ctx.kv4_attention(c.desc(), args)
    ctx.synchronize()
    assert (x == 0).all() and (out == 0).all()
    # rows that are read may be expanded, and the outputs' heads lie outside their rows
    ctx.kv4_append(c.desc(), S.kv4_rows(k[:1, :1].expand(3, 2, -1), v[:1].expand(3, -1, -1), starts([0, 3])))
    ko, vo = (torch.zeros(2, 3, 64, dtype=BF16, device="cuda").transpose(0, 1) for _ in range(2))
    ctx.kv4_read(c.desc(), ints([0, 30]), S.kv4_rows(ko, vo, starts([0, 3])))
    ctx.synchronize()
    for got, x in ((ko, k[:1, :1].expand(3, 2, -1)), (vo, v[:1].expand(3, -1, -1))):
        code, scale, bias = quantised(x)
        assert torch.equal(got, (code * scale + bias).flatten(-2).to(BF16))


def odd(n, heads, hd, dtype, g):
    """Rows [n, heads, hd] whose strides are multiples of 4 elements and not of 8, heads outermost."""
    x = torch.randn(heads, n, hd + 4, generator=g, device="cuda").to(dtype)
    return x[:, :, :hd].transpose(0, 1)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("Hkv,hd", [(3, 128), (2, 64)])
def test_kv4_strides_of_four(ctx, dtype, Hkv, hd):
    """bf16 rows that start on 8 bytes and not on 16: append, read, and attention's q and out."""
    lens = [130, 1, 70]
    c = T.Cache(Hkv, hd, lens, 1, 611)
    n = sum(lens)
    k, v = odd(n, Hkv, hd, dtype, c.g), odd(n, Hkv, hd, dtype, c.g)
    assert k.stride(0) % 8 == 4
    ctx.kv4_append(c.desc(), S.kv4_rows(k, v, starts(lens)))
    ctx.kv4_advance(c.len, c.seen, 3, cu=starts(lens))
    ko, vo = odd(n, Hkv, hd, dtype, c.g), odd(n, Hkv, hd, dtype, c.g)
    ctx.kv4_read(c.desc(), None, S.kv4_rows(ko, vo, starts(lens)))
    ctx.synchronize()
    for x, o in ((k, ko), (v, vo)):
        code, scale, bias = quantised(x)
        assert torch.equal(o, (code * scale + bias).flatten(-2).to(dtype))
    H = 4 * Hkv
    wide = torch.randn(3, H * hd + 12, generator=c.g, device="cuda").to(dtype)
    q = wide[:, : H * hd].view(3, H, hd)
    res = torch.full((3, H * hd + 4), -5.0, dtype=dtype, device="cuda")
    out = res[:, : H * hd].view(3, H, hd)
    args = S.kv4_attn_args(q, out, 130)
    ws = torch.zeros(S.kv4_attention_workspace(c.desc(), args), dtype=torch.uint8, device="cuda")
    ctx.kv4_attention(c.desc(), S.kv4_attn_set_workspace(args, ws))
    ctx.synchronize()
    T.attn_check(c, q, lens, out)
    assert (res[:, H * hd:] == -5).all()


# -------------------------------------------------------------- nothing to do
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_kv4_no_rows(ctx, dtype):
    """A step in which no sequence has a row: tensors without elements have no address, and nothing changes."""
    c = T.Cache(2, 64, [20, 30], 1, 620)
    c.fill(ctx)
    before, pos = c.blocks.clone(), c.pos.clone()
    none = torch.zeros(0, 2, 64, dtype=dtype, device="cuda")
    cu = ints([0, 0, 0])
    ctx.kv4_append(c.desc(), S.kv4_rows(none, none, cu))
    ctx.kv4_read(c.desc(), None, S.kv4_rows(none, none.clone(), cu))
    ctx.kv4_advance(c.len, c.seen, 2, cu=cu)
    ctx.synchronize()
    assert torch.equal(c.blocks, before) and torch.equal(c.pos, pos) and c.len.tolist() == [20, 30]


def test_packed_attention_no_keys_at_all(ctx):
    """Rows, but not one key in the call: zeros and -inf."""
    q = torch.randn(40, 8, 64, device="cuda").to(BF16)
    none = torch.zeros(0, 2, 64, dtype=BF16, device="cuda")
    for causal in (True, False):
        out, lse = T.packed_run(ctx, q, none, none.clone(), [(30, 0), (10, 0)], causal)
        assert (out == 0).all() and (lse == -math.inf).all()


@pytest.mark.parametrize("rows,H,Hkv", [(100, 8, 2), (700, 16, 2), (6000, 32, 4)])     # each of the call's paths
def test_packed_attention_sequences_without_rows(ctx, rows, H, Hkv):
    """Rows and keys that belong to no sequence: nothing is written."""
    q, k, v = T.packed_inputs([(rows, rows + 1000)], H, Hkv, 64, 640)
    out = torch.full_like(q, 7.0)
    lse = torch.full(q.shape[:2], 7.0, device="cuda")
    ctx.attention_packed(S.packed_attn_args(q, k, v, out, ints([0, 0, 0]), lse=lse))
    ctx.attention_packed(S.packed_attn_args(q, k, v, out, ints([rows] * 4), ints([0, 9, 9, rows]), lse=lse))
    ctx.synchronize()
    assert (out == 7).all() and (lse == 7).all()


@pytest.mark.parametrize("score", [False, True])
def test_kv4_attention_empty_sequences(ctx, score):
    """No sequence has an entry: zeros, and no weight is written."""
    c = T.Cache(2, 128, [0, 0, 0], 1, 641)
    q = torch.randn(3, 8, 128, device="cuda")
    for max_len in (0, 5000):
        out, so = attn_run(ctx, c, q, max_len, score=score)
        assert (out == 0).all() and (so is None or (so == -1).all())


# --------------------------------------------------------------------- limits
def test_limits(ctx):
    """Shapes past what a launch takes are refused before anything runs; 6,144 query heads on one KV head are served."""
    c = T.Cache(1, 64, [70], 1, 630)
    c.fill(ctx)
    for heads in (6144, 6145):
        q = torch.randn(1, heads, 64, generator=c.g, device="cuda")
        out, so = torch.zeros_like(q), torch.zeros_like(c.score)
        args = S.kv4_attn_args(q, out, 70, score_out=so, decay=0.0)
        ws = torch.zeros(S.kv4_attention_workspace(c.desc(), args), dtype=torch.uint8, device="cuda")
        S.kv4_attn_set_workspace(args, ws)
        if heads == 6144:
            ctx.kv4_attention(c.desc(), args)
            ctx.synchronize()
            T.attn_check(c, q, [70], out, so, decay=0.0)
        else:
            before = ctx.dispatches()
            with pytest.raises(S.SmoeCudaError, match="ERR_UNSUPPORTED"):
                ctx.kv4_attention(c.desc(), args)
            assert ctx.dispatches() == before
    q, k, v = T.packed_inputs([(20, 20)], 8, 2, 64, 631)
    a = S.packed_attn_args(q, k, v, torch.zeros_like(q), starts([20]))
    a.n_seqs = a.total_q = 0xffffffff
    before = ctx.dispatches()
    with pytest.raises(S.SmoeCudaError, match="ERR_UNSUPPORTED"):
        ctx.attention_packed(a)
    assert ctx.dispatches() == before


# ------------------------------------------------------------- NaN in cache rows
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("other", [0.0, math.inf, -math.inf])
def test_kv4_append_carries_nan(ctx, dtype, other):
    """One NaN makes its whole group NaN (bias = min of the group), wherever it is and whatever else is there, and no other group."""
    n = 64
    c = T.Cache(2, 128, [n], 1, 500)
    k, v = ((torch.randn(n, 2, 128, generator=c.g, device="cuda")).to(dtype) for _ in range(2))
    for i in range(n):                   # each place of a group, both groups, heads and sides
        k[i, i % 2, 64 + i] = math.nan
        v[i, 1 - i % 2, i] = -math.nan
        if other:
            k[i, i % 2, 64 + (i + 17) % 64] = other
    ctx.kv4_append(c.desc(), S.kv4_rows(k, v, starts([n])))
    ko, vo = torch.zeros_like(k), torch.zeros_like(v)
    ctx.kv4_read(c.desc(), None, S.kv4_rows(ko, vo, starts([n])))
    ctx.synchronize()
    for x, o in ((k, ko), (v, vo)):
        bad = x.isnan().unflatten(-1, (2, 64)).any(-1, keepdim=True).expand(-1, -1, -1, 64).flatten(-2)
        assert bad.sum() == 64 * n and o[bad].isnan().all()
        code, scale, bias = quantised(x)
        assert torch.equal(o[~bad], (code * scale + bias).flatten(-2).to(dtype)[~bad])


def test_kv4_attention_over_a_nan(ctx):
    """A NaN among the keys makes its KV head's results NaN, among the values those of its group; nothing else."""
    c = T.Cache(2, 128, [300], 1, 501)
    k, v = (torch.randn(300, 2, 128, generator=c.g, device="cuda") for _ in range(2))
    k[200, 0, 5] = math.nan
    v[100, 1, 70] = math.nan
    ctx.kv4_append(c.desc(), S.kv4_rows(k, v, starts([300])))
    c.len += 300
    q = torch.randn(1, 8, 128, generator=c.g, device="cuda")
    out, _ = attn_run(ctx, c, q, 300)
    assert out[0, :4].isnan().all() and out[0, 4:, 64:].isnan().all() and torch.isfinite(out[0, 4:, :64]).all()


# ------------------------------------------------------------------ scales of 0
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("scale", [0.0, 1e-37, 1e-20, 0.05])
def test_kv4_attention_small_scales(ctx, dtype, scale):
    """Equal probabilities at a scale of 0, for zero, tiny and ordinary queries, with lengths that end inside a page, and their weights."""
    lens = [1, 63, 65, 200, 1000]
    c = T.Cache(2, 64, lens, 1, 510)
    c.fill(ctx)
    q = torch.randn(len(lens), 16, 64, generator=c.g, device="cuda")
    q[:, 0] = 0
    q[:, 1] *= 1e-12
    q[:, 2] *= 1e-30
    q[:, 3] *= 1e-42
    q = q.to(dtype)
    out, so = torch.full_like(q, math.nan), torch.full_like(c.score, -1.0)
    args = S.kv4_attn_args(q, out, max(lens), scale=scale, score_out=so, decay=0.0)
    ws = torch.full((S.kv4_attention_workspace(c.desc(), args),), 255, dtype=torch.uint8, device="cuda")
    ctx.kv4_attention(c.desc(), S.kv4_attn_set_workspace(args, ws))
    ctx.synchronize()
    assert torch.isfinite(out).all()
    for b, n in enumerate(lens):
        k, v = c.values(b, n)
        p = torch.softmax(torch.einsum("kgd,nkd->kgn", q[b].double().view(2, -1, 64), k) * scale, -1)
        want, mag = (torch.einsum("kgn,nkd->kgd", p, x).reshape(16, 64) for x in (v, v.abs()))
        assert ((out[b].double() - want).abs() <= 2 ** -14 * mag + (2 ** -8 * want.abs() if dtype == BF16 else 0)).all()
        page, slot = c.at(b, n)
        w = p.sum(1).t()
        assert ((so[page, :, slot].double() - w).abs() <= 2e-5 * (w + p.sum(1).max())).all()


# ------------------------------------------------------------------- row ranges
RANGES = [
    # starts, rows, sequences that must be skipped
    ([0, 5, 9, 9], 7, [1]),              # the second one ends past the rows
    ([0, 7, 12, 12], 7, [1]),            # .. and starts there
    ([0, 4, 4, 200], 9, [2]),
    ([0, 3, 6, 2 ** 31 + 5], 9, [2]),
    ([0, 6, 2, 2], 8, [1]),              # one that ends before it starts
]


@pytest.mark.parametrize("case", range(len(RANGES)))
@pytest.mark.parametrize("what", ["append", "read"])
def test_kv4_rows_outside_their_buffer(ctx, case, what):
    """A sequence whose rows are not all there is skipped as a whole and reported; the others are served."""
    cu, total, bad = RANGES[case]
    c = T.Cache(2, 64, [70, 10, 64], 300, 520)
    c.fill(ctx)
    before = c.blocks.clone()
    k, v = (torch.randn(total, 2, 64, generator=c.g, device="cuda") for _ in range(2))
    cu_t = torch.tensor([x - (x >> 31 << 32) for x in cu], dtype=torch.int32, device="cuda")
    ko, vo = torch.full_like(k, -9), torch.full_like(v, -9)
    if what == "append":
        ctx.kv4_append(c.desc(), S.kv4_rows(k, v, cu_t))
    else:
        ctx.kv4_read(c.desc(), None, S.kv4_rows(ko, vo, cu_t))
    with pytest.raises(S.SmoeCudaError, match="ERR_DEVICE"):
        ctx.synchronize()
    ctx.synchronize()                    # reported once
    lens = [70, 10, 64]
    for s in range(3):
        n = cu[s + 1] - cu[s]
        if s in bad or n == 0 or any(cu[b + 1] < cu[b] for b in bad) and s > 0:
            continue
        if what == "append":
            page, slot = c.at(s, n, lens[s])
            assert (c.pos[page, :, slot] == torch.arange(lens[s], lens[s] + n, device="cuda")[:, None]).all()
            got = T.Cache.values(c, s, lens[s] + n)[0][lens[s]:]
            code, scale, bias = quantised(k[cu[s]: cu[s + 1]])
            assert ((got - (code * scale + bias).flatten(-2).double()).abs() <= 1e-5).all()
        else:
            want = c.values(s, n)[0]
            assert ((ko[cu[s]: cu[s + 1]].double() - want).abs() <= 1e-5).all()
    for s in bad:
        if what == "append":             # nothing was written for it
            page, slot = c.at(s, 64, lens[s])
            assert torch.equal(c.blocks[page], before[page]) and (c.pos[page, :, slot] == 0).all()
        elif cu[s] < min(cu[s + 1], total):
            assert (ko[cu[s]: cu[s + 1]] == -9).all() and (vo[cu[s]: cu[s + 1]] == -9).all()


def test_kv4_advance_reports_a_range_that_runs_backwards(ctx):
    lens, seen = ints([10, 20, 30]), ints([11, 21, 31])
    ctx.kv4_advance(lens, seen, 3, cu=ints([0, 4, 1, 8]))
    with pytest.raises(S.SmoeCudaError, match="ERR_DEVICE"):
        ctx.synchronize()
    assert lens.tolist() == [14, 20, 37] and seen.tolist() == [15, 21, 38]


# ----------------------------------------------------------- accuracy of decode
def test_kv4_attention_accuracy(ctx):
    """fp32 results over ordinary rows: norm of the error within 2^-19 of the result's. (Scores of magnitude up to 8 in
    units of log2 take some six roundings of 2^-24 of that: 7e-7 rms of a probability, likewise of the result; products
    of codes that are not centred would be at 2.8e-6.)"""
    lens = [1000, 300, 64, 777]
    c = T.Cache(4, 128, lens, 1, 530)
    c.fill(ctx)
    q = torch.randn(4, 32, 128, generator=c.g, device="cuda") * 2
    out, _ = attn_run(ctx, c, q, 1000)
    want = torch.zeros(q.shape, dtype=torch.float64, device="cuda")
    for b, n in enumerate(lens):
        k, v = c.values(b, n)
        p = torch.softmax(torch.einsum("kgd,nkd->kgn", q[b].double().view(4, -1, 128), k) / math.sqrt(128), -1)
        want[b] = torch.einsum("kgn,nkd->kgd", p, v).reshape(32, 128)
    assert float((out.double() - want).norm() / want.norm()) <= 2 ** -19


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("hd,n", [(128, 700), (64, 30000), (128, 30000)])      # a page a warp; three
@pytest.mark.parametrize("kind", ["no weight", "some weight", "own head", "later maximum"])
@pytest.mark.parametrize("size", [2.0 ** 14, 2.0 ** 30, 2.0 ** 100])
def test_kv4_attention_outliers(ctx, dtype, hd, n, kind, size):
    """Values that are much larger than all others but have (almost) no weight leave the result as exact as without them.
    A score in fp32 is off by some 4 x 2^-24 of its products' magnitudes, and a probability by that in units of log2. They
    add up to 16 where outliers have no weight (2^-18 of the magnitude); to 100 where outliers of some weight decide the
    result (2^-15); to 900 where a score of 212 or 300 does (2^-12)."""
    Hkv, H = 8, 24
    c = T.Cache(Hkv, hd, [n], 1, 540)
    g = c.g
    k, v = (torch.randn(n, Hkv, hd, generator=g, device="cuda") for _ in range(2))
    q = torch.randn(1, H, hd, generator=g, device="cuda")
    q[..., 0] = 6.0                      # dimension 0 sets the scores: 6 k[0] / sqrt(hd)
    page = torch.arange(0, n - 63, 64, device="cuda")
    slot = torch.randint(0, 64, page.shape, generator=g, device="cuda")
    at = (page + slot)[::5]              # every fifth page has an outlier
    unit = math.sqrt(hd) / 6
    if kind == "later maximum":          # every third page has a key that is 300 above, the outliers' pages come before it
        at = (page + slot)[::3]
        k[(page + slot)[2::3], :, 0] = 300 * unit
    else:
        k[at, :, 0] = (-14 if kind == "some weight" else -212) * unit
    if kind == "own head":
        at = at[len(at) // 2:][:1]
        q[0, 5, 0] = q[0, 13, 0] = -6.0  # this one decides
    v[at] *= size
    ctx.kv4_append(c.desc(), S.kv4_rows(k, v, starts([n])))
    c.len += n
    q = q.to(dtype)
    out, _ = attn_run(ctx, c, q, n)
    kk, vv = c.values(0, n)
    p = torch.softmax(torch.einsum("kgd,nkd->kgn", q[0].double().view(Hkv, -1, hd), kk) / math.sqrt(hd), -1)
    want, mag = (torch.einsum("kgn,nkd->kgd", p, x).reshape(H, hd) for x in (vv, vv.abs()))
    assert torch.isfinite(out).all()
    bar = 2 ** (-18 if kind == "no weight" else -15 if kind == "some weight" else -12)
    assert ((out[0].double() - want).abs() <= bar * mag + (2 ** -8 * want.abs() if dtype == BF16 else 0)).all()
