"""GPU parity of the long-context serving operators on the paths that large
calls take: packed attention from the sorted list of tile pairs and with a
CTA per pair past the list's size, infinities and bad row ranges on each of
its paths, its calls in a captured graph, and evictions by clusters of CTAs
(several words a lane, keys that shared memory does not hold). Bars as in
test_gpu_serve.py."""
import math

import pytest
import torch

import smoe_cuda as S
import test_gpu_serve as T
from test_gpu_serve import BF16, F32, ints, packed_check, packed_inputs, packed_ref, packed_run, starts

pytestmark = pytest.mark.gpu


def plan_of(lens, H, Hkv):
    """How the entry runs a call: 'direct', 'shares' or 'list' (its rule, restated)."""
    tokens = 128 // (H // Hkv)
    tq, tk = sum(a for a, _ in lens), sum(b for _, b in lens)
    pairs = tq // (2 * tokens) + min(len(lens), tq)
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    if (pairs * Hkv <= sms and tk <= 1024) or pairs > 65536:
        return "direct"
    return "list" if pairs * Hkv >= 4 * sms else "shares"


RAGGED = [(n, n) for n in (17, 0, 900, 1, 33, 0, 1300, 64, 250, 31, 32, 700, 5, 411, 0, 1024)]
LISTED = [
    # lens (q, k) of the sequences, heads, KV heads, head_dim, causal, window, strided
    (RAGGED, 32, 4, 128, True, 0, False),
    ([(a, a + 7 * i) for i, (a, _) in enumerate(RAGGED)], 32, 4, 128, True, 300, True),
    ([(1 + i * 37 % 61, 1 + i * 37 % 61 + i * 53 % 400) for i in range(90)], 8, 8, 64, True, 45, False),
    ([(1 + i * 11 % 40, i * 29 % 50) for i in range(160)], 16, 4, 96, True, 0, False),        # rows without a key among them
    ([(60, 300), (1, 5), (45, 45)] * 50, 8, 4, 128, False, 0, True),
    ([(3000, 3000)], 64, 4, 64, True, 0, False),
]


@pytest.mark.parametrize("case", range(len(LISTED)))
def test_packed_attention_from_the_list(ctx, case):
    lens, H, Hkv, hd, causal, window, strided = LISTED[case]
    assert plan_of(lens, H, Hkv) == "list"
    q, k, v = packed_inputs(lens, H, Hkv, hd, 300 + case, strided)
    out, lse = packed_run(ctx, q, k, v, lens, causal, window)
    packed_check(out, lse, packed_ref(q, k, v, lens, causal, window, 1 / math.sqrt(hd)))
    again, lse2 = packed_run(ctx, q, k, v, lens, causal, window)
    assert torch.equal(out, again) and torch.equal(lse, lse2)


def test_packed_attention_more_pairs_than_the_list_holds(ctx):
    """70,000 tile pairs: a CTA each."""
    lens = [(70, 70)] * 2000
    assert plan_of(lens, 128, 1) == "direct"
    q, k, v = packed_inputs(lens, 128, 1, 8, 310)
    out, lse = packed_run(ctx, q, k, v, lens)
    for s in (0, 1, 777, 1998, 1999):
        r = slice(70 * s, 70 * s + 70)
        packed_check(out[r], lse[r], packed_ref(q[r], k[r], v[r], [(70, 70)], True, 0, 1 / math.sqrt(8)))
    assert torch.isfinite(out).all() and torch.isfinite(lse).all()


PATHS = {
    "direct": ([(150, 150), (40, 300), (77, 77)], 16, 2, 128),
    "shares": ([(150, 900), (40, 1300), (77, 777)], 16, 2, 128),       # pairs are cut, and joined
    "list": ([(150, 250), (940, 1300), (77, 77), (1500, 1500)] * 2, 32, 4, 128),
}


@pytest.mark.parametrize("path", list(PATHS))
@pytest.mark.parametrize("window", [0, 200])
def test_packed_attention_nonfinite_values(ctx, path, window):
    """Infinities and NaN among the values reach the rows that attend to them, in their column, and no others."""
    lens, H, Hkv, hd = PATHS[path]
    assert plan_of(lens, H, Hkv) == path
    q, k, v = packed_inputs(lens, H, Hkv, hd, 320)
    want, mag, wlse = packed_ref(q, k, v, lens, True, window, 1 / math.sqrt(hd))
    q0 = k0 = 0
    G = H // Hkv
    for lq, lk in lens:                  # per sequence: a key near the end, one that is older, in two columns of KV head 1
        for at, col, x in ((lk - 30, 3, math.inf), (lk - min(lk, 130), 70, -math.inf), (lk - 12, 3, -math.inf), (lk - 60, 90, math.nan)):
            v[k0 + at, 1, col] = x
            i = torch.arange(lq, device="cuda") + lk - lq
            sees = (i >= at) & ((i < at + window) if window else (i >= 0))
            w = want[q0: q0 + lq, G: 2 * G, col]
            w[sees] = w[sees] + x        # (0 * inf has no place here: every probability is above 0)
        q0, k0 = q0 + lq, k0 + lk
    out, lse = packed_run(ctx, q, k, v, lens, True, window)
    fine = torch.isfinite(want)
    assert torch.isfinite(out[fine]).all()
    assert torch.equal(out[~fine].double().nan_to_num(3, 1, 2), want[~fine].nan_to_num(3, 1, 2))
    assert ((out.double() - want).abs() <= 2 ** -8 * want.abs() + (2 ** -8 + 1e-4) * mag + 1e-30)[fine].all()
    assert ((lse.double() - wlse).abs() <= 1e-4).all()


@pytest.mark.parametrize("path", list(PATHS))
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_packed_attention_masked_places_on_each_path(ctx, path, bad):
    """What later tokens and another sequence hold does not change a bit of the other rows."""
    lens, H, Hkv, hd = PATHS[path]
    q, k, v = packed_inputs(lens, H, Hkv, hd, 330)
    clean, clean_lse = packed_run(ctx, q, k, v, lens)
    (a, ka), (b, kb) = lens[:2]
    q[a: a + b] = bad                    # the second sequence altogether
    k[ka: ka + kb], v[ka: ka + kb] = bad, bad
    k[ka - 1], v[ka - 1] = bad, bad      # and the last token of the first
    out, lse = packed_run(ctx, q, k, v, lens)
    rows = torch.ones(len(out), dtype=torch.bool, device="cuda")
    rows[a - 1: a + b] = False
    assert torch.equal(out[rows], clean[rows]) and torch.equal(lse[rows], clean_lse[rows])
    if bad != bad:
        assert out[~rows].isnan().all()


@pytest.mark.parametrize("path", list(PATHS))
@pytest.mark.parametrize("side", ["q", "k"])
def test_packed_attention_bad_rows_on_each_path(ctx, path, side):
    """A row range outside its buffer: an error at the next synchronize, the other sequences as they are."""
    lens, H, Hkv, hd = PATHS[path]
    q, k, v = packed_inputs(lens, H, Hkv, hd, 340)
    out = torch.full(q.shape, -3.0, dtype=BF16, device="cuda")
    cu, cu_k = starts([a for a, _ in lens]), starts([b for _, b in lens])
    (cu if side == "q" else cu_k)[-1] += 5                             # the last sequence's
    ctx.attention_packed(S.packed_attn_args(q, k, v, out, cu, cu_k))
    with pytest.raises(S.SmoeCudaError, match="ERR_DEVICE"):
        ctx.synchronize()
    n, nk = q.shape[0] - lens[-1][0], k.shape[0] - lens[-1][1]
    want, mag, _ = packed_ref(q[:n], k[:nk], v[:nk], lens[:-1], True, 0, 1 / math.sqrt(hd))
    assert ((out[:n].double() - want).abs() <= 2 ** -8 * want.abs() + (2 ** -8 + 1e-4) * mag + 1e-30).all()
    assert (out[n:] == -3).all()


def test_packed_attention_in_a_graph(ctx):
    """Calls of all paths captured together and replayed over new inputs, against the same calls one by one."""
    states = []
    for path, (lens, H, Hkv, hd) in PATHS.items():
        q, k, v = packed_inputs(lens, H, Hkv, hd, 350)
        out, lse = torch.zeros_like(q), torch.zeros(q.shape[:2], device="cuda")
        cu, cu_k = starts([a for a, _ in lens]), starts([b for _, b in lens])
        states.append((S.packed_attn_args(q, k, v, out, cu, cu_k, lse=lse), q, k, v, out, lse, cu, cu_k))
    other = S.Context(0, max_batch=4)
    s = torch.cuda.Stream()
    other.set_stream(s.cuda_stream)
    torch.cuda.synchronize()

    def calls(x):
        for st in states:
            x.attention_packed(st[0])
    with torch.cuda.stream(s):
        calls(other)
        other.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            calls(other)
            calls(other)
        for i in range(3):
            for st in states:
                for x in st[1:4]:
                    x.copy_(x.roll(i + 1, 0))
            graph.replay()
            other.synchronize()
            got = [(st[4].clone(), st[5].clone()) for st in states]
            for st in states:
                st[4].zero_()
                st[5].zero_()
            calls(other)
            other.synchronize()
            for st, (out, lse) in zip(states, got):
                assert torch.equal(st[4], out) and torch.equal(st[5], lse) and out.any()
    del graph
    other.close()


# ------------------------------------------------------------------- eviction
def evict_into(score, pos, seen, n, keep, recent):
    """The entries that end up in the slots [0, min(n, keep)), by stable sorts of whole columns."""
    if n <= keep:
        return torch.arange(n, device="cuda")
    rank = torch.where(pos.long() + recent >= seen, 2, torch.where(score.isnan(), 0, 1))
    key = torch.where(rank == 1, score.nan_to_num(0.0, math.inf, -math.inf), 0.0) + 0.0
    order = key.argsort(descending=True, stable=True)
    order = order[rank[order].argsort(descending=True, stable=True)]
    best = torch.zeros(n, dtype=torch.bool, device="cuda")
    best[order[:keep]] = True
    into = torch.arange(keep, device="cuda")
    into[~best[:keep]] = best[keep:].nonzero()[:, 0] + keep
    return into


CLUSTERS = [
    # KV heads, head_dim, lengths, max_len, keep, recent, scores
    (2, 64, [8193, 8200, 64, 0, 1001], 8200, 1000, 50, "random"),              # two CTAs a pair
    (2, 128, [20000, 20000, 100], 20000, 4096, 512, "ties"),                   # four; ties across them
    (1, 64, [20000, 16385], 20000, 19990, 3, "random"),                        # few moves
    (1, 64, [9000, 300, 40, 257], 60000, 256, 64, "random"),                   # short ones under a large max_len: CTAs without entries
    (1, 128, [70000, 33000], 70000, 4096, 0, "special"),                       # eight
    (1, 64, [40000], 40000, 20000, 20000, "equal"),                            # the oldest go up to the recent ones
    (2, 64, [30000], 30000, 500, 2000, "random"),                              # more recent ones than stay
    (1, 64, [140000, 9], 140000, 60000, 1000, "ties"),                         # several words a lane
    (1, 64, [400003], 400003, 30000, 100, "random"),                           # keys that shared memory does not hold
    (1, 64, [399000], 400003, 398000, 0, "ties"),
]


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("case", range(len(CLUSTERS)))
def test_kv4_evict_clusters(ctx, case, in_place):
    Hkv, hd, lens, max_len, keep, recent, kind = CLUSTERS[case]
    c = T.Cache(Hkv, hd, lens, 1, 400 + case)
    c.blocks.copy_(torch.randint(0, 256, c.blocks.shape, generator=c.g, device="cuda", dtype=torch.uint8))
    c.len, c.seen = ints(lens), ints([n + 5 for n in lens])
    s = torch.rand(c.score.shape, generator=c.g, device="cuda")
    if kind == "ties":
        s = (s * 7).floor()
    elif kind == "equal":
        s = torch.full_like(s, 0.25)
    elif kind == "special":
        pick = torch.randint(0, 9, s.shape, generator=c.g, device="cuda")
        for i, x in enumerate((math.nan, math.inf, -math.inf, 0.0, -0.0, -1.0)):
            s[pick == i] = x
    c.score.copy_(s)
    for b, n in enumerate(lens):         # positions out of order, as earlier evictions leave them
        page, slot = c.at(b, n)
        c.pos[page, :, slot] = torch.stack([torch.randperm(n, generator=c.g, device="cuda") for _ in range(Hkv)], 1).int() + 5
    old_blocks, old_pos, old_score = c.blocks.clone(), c.pos.clone(), c.score.clone()
    pos_out = None if in_place else torch.full_like(c.pos, -7)
    score_out = None if in_place else torch.full_like(c.score, -7.0)
    ws = torch.full((S.kv4_evict_workspace(c.desc(), max_len),), 255, dtype=torch.uint8, device="cuda")
    ctx.kv4_evict(c.desc(), keep, recent, max_len, ws, pos_out, score_out)
    ctx.synchronize()
    want_blocks = old_blocks.clone()
    want_pos, want_score = (old_pos.clone(), old_score.clone()) if in_place else (torch.full_like(c.pos, -7), torch.full_like(c.score, -7.0))
    ng = hd // 64

    def parts(t):                        # codes and pairs [pages, heads, side and group, slot, bytes]
        return t[..., : ng * 4096].unflatten(-1, (2 * ng, 64, 32)), t[..., ng * 4096:].unflatten(-1, (2 * ng, 64, 4))
    for b, n in enumerate(lens):
        page, slot = c.at(b, n)
        for h in range(Hkv):
            src = evict_into(old_score[page, h, slot], old_pos[page, h, slot], n + 5, n, keep, recent)
            m = len(src)
            for to, frm in zip(parts(want_blocks), parts(old_blocks)):
                to[page[:m], h, :, slot[:m]] = frm[page[src], h, :, slot[src]]
            want_pos[page[:m], h, slot[:m]] = old_pos[page[src], h, slot[src]]
            want_score[page[:m], h, slot[:m]] = old_score[page[src], h, slot[src]]
    assert torch.equal(c.blocks, want_blocks)
    new_pos, new_score = (c.pos, c.score) if in_place else (pos_out, score_out)
    assert torch.equal(new_pos, want_pos)
    assert torch.equal(new_score.view(torch.int32), want_score.view(torch.int32))
    if not in_place:
        assert torch.equal(c.pos, old_pos) and torch.equal(c.score.view(torch.int32), old_score.view(torch.int32))
