"""The long-context serving operators as a user's program calls them: packed
prompt attention, writes to and reads from the 4-bit KV cache, single-token
attention over that cache, and eviction from it. listed() names the cases,
prepare() makes one's inputs, run() is one pass: with `own` false in a plain
form (elementary torch operations in 32 bits), with `own` true through the
framework's entry points."""
import functools
import math
import os
import random
import sys

import torch

own = False

PAGE = 64            # entries of one page of the 4-bit cache
GROUP = 64           # values that share a scale and a bias
BLOCK = 4608         # bytes of one page of one KV head, per 64 values of head_dim
F32 = torch.float32
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}


def listed():
    return [
        # one chat prompt of the framework's bench length: latency of a single small call
        _prompt("prompt_45", 32, 4, 128, 1, 45, 45, split=1),
        # a packed batch of prompts of very different lengths, as a server collects them
        _prompt("prompt_ragged", 32, 4, 128, 24, 17, 2048, split=2),
        # chunked prefill: new tokens of four conversations over what they hold already, smaller heads, a window
        _prompt("prompt_chunk", 16, 8, 64, 4, 200, 512, prefix=6001, window=4096, split=3),
        # one long document
        _prompt("prompt_16k", 32, 4, 128, 1, 16384, 16384, split=4),
        # a packed chunk of eight prompts goes to the cache, and their whole contexts come back for its attention
        _write("write_chunk", 4, 128, 8, 100, 1200, held=4000, back="all", dtype="bf16", split=5),
        # one decode step of 256 sequences: their new token's K and V, in the trunk's type
        _write("write_step", 4, 128, 256, 1, 1, held=600, back="new", dtype="f32", split=6),
        # one sequence, a short context: latency of a decode step
        _decode("decode_one", 32, 4, 128, 1, 300, 300, dtype="f32", score=False, split=7),
        # a batch of ragged contexts whose attention weights are kept for eviction
        _decode("decode_batch", 32, 4, 128, 32, 512, 8192, dtype="bf16", score=True, split=8),
        # many short sequences of the wide shape (16 query heads to a KV head)
        _decode("decode_wide", 64, 4, 128, 128, 45, 1000, dtype="f32", score=False, split=9),
        # two very long contexts
        _decode("decode_long", 32, 4, 128, 2, 120000, 131072, dtype="bf16", score=True, split=10),
        # between decode steps: a few sequences a little over what they may hold
        _evict("evict_step", 4, 128, 8, 1088, 1150, keep=1024, recent=128, split=11),
        # after long prompts: most of what they wrote goes
        _evict("evict_prompt", 4, 128, 16, 6000, 32768, keep=4096, recent=512, split=12),
    ]


def _prompt(name, heads, kv_heads, head_dim, seqs, lo, hi, prefix=0, window=0, split=0):
    return {"name": name, "op": "prompt", "heads": heads, "kv_heads": kv_heads, "head_dim": head_dim, "seqs": seqs,
            "lo": lo, "hi": hi, "prefix": prefix, "window": window, "split": split}


def _write(name, kv_heads, head_dim, seqs, lo, hi, held=0, back="all", dtype="bf16", split=0):
    return {"name": name, "op": "write", "kv_heads": kv_heads, "head_dim": head_dim, "seqs": seqs, "lo": lo, "hi": hi,
            "held": held, "back": back, "dtype": dtype, "split": split}


def _decode(name, heads, kv_heads, head_dim, seqs, lo, hi, dtype="bf16", score=False, split=0):
    return {"name": name, "op": "decode", "heads": heads, "kv_heads": kv_heads, "head_dim": head_dim, "seqs": seqs,
            "lo": lo, "hi": hi, "dtype": dtype, "score": score, "split": split}


def _evict(name, kv_heads, head_dim, seqs, lo, hi, keep, recent, split=0):
    return {"name": name, "op": "evict", "kv_heads": kv_heads, "head_dim": head_dim, "seqs": seqs, "lo": lo, "hi": hi,
            "keep": keep, "recent": recent, "split": split}


def _log(rng, lo, hi):
    """A whole number between lo and hi, spread over the logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(("prompt", "write", "decode", "evict"))
    split = rng.randrange(1 << 20)
    heads, kv_heads = rng.choice(((32, 4), (64, 4), (16, 8), (8, 8), (28, 4), (12, 4), (5, 1), (32, 8)))
    head_dim = rng.choice((64, 128, 128))
    if op == "prompt":
        head_dim = rng.choice((64, 128, 128, 96))
        seqs, hi = _log(rng, 1, 32), _log(rng, 1, 16384)
        prefix = rng.choice((0, 0, _log(rng, 1, 8192)))
        room = 16384 * 16384 * 32
        while seqs > 1 and seqs * hi * (hi + prefix) * heads > room:
            seqs = seqs // 2
        while seqs * hi * (hi + prefix) * heads > room:
            hi = hi * 2 // 3
        window = rng.choice((0, 0, 0, _log(rng, 16, 4096)))
        c = _prompt("", heads, kv_heads, head_dim, seqs, _log(rng, 1, hi), hi, prefix, window, split)
    elif op == "write":
        seqs, hi = _log(rng, 1, 256), _log(rng, 1, 4096)
        held = rng.choice((0, _log(rng, 1, 8192)))
        while seqs > 1 and seqs * (hi + held) * kv_heads * head_dim > (1 << 25):
            seqs = seqs * 2 // 3
        while hi > 1 and seqs * (hi + held) * kv_heads * head_dim > (1 << 25):
            hi, held = hi * 2 // 3, held * 2 // 3
        c = _write("", kv_heads, head_dim, seqs, _log(rng, 1, hi), hi, held, rng.choice(("all", "new")),
                   rng.choice(("bf16", "f32")), split)
    elif op == "decode":
        seqs, hi = _log(rng, 1, 256), _log(rng, 1, 131072)
        while seqs * hi * kv_heads * head_dim > 2 * 131072 * 4 * 128:
            seqs, hi = max(1, seqs * 2 // 3), hi if seqs > 1 else hi * 2 // 3
        c = _decode("", heads, kv_heads, head_dim, seqs, _log(rng, 1, hi), hi, rng.choice(("bf16", "f32")),
                    rng.random() < 0.5, split)
    else:
        seqs, hi = _log(rng, 1, 64), _log(rng, 65, 65536)
        while seqs * hi * kv_heads * head_dim > 16 * 32768 * 4 * 128:
            seqs, hi = max(1, seqs * 2 // 3), hi if seqs > 1 else hi * 2 // 3
        keep = _log(rng, 32, hi - 1)
        c = _evict("", kv_heads, head_dim, seqs, max(1, int(hi * rng.uniform(0.3, 1.0))), hi, keep,
                   _log(rng, 1, keep), split)
    del c["name"]
    return c


# ------------------------------------------------------------ lengths and work
def _lengths(case):
    """Per sequence: (new tokens, entries held before). The first sequence has the most of both."""
    r = random.Random(case["split"])
    n = [case["hi"]] + [_log(r, case["lo"], case["hi"]) for _ in range(case["seqs"] - 1)]
    most = case.get("prefix", case.get("held", 0))
    held = [most] + [_log(r, 1, most) if most else 0 for _ in range(case["seqs"] - 1)]
    return n, held


def work(case):
    n, held = _lengths(case)
    hd, hkv, ng = case["head_dim"], case["kv_heads"], case["head_dim"] // GROUP
    if case["op"] == "prompt":
        pairs = 0
        for q, p in zip(n, held):
            w = case["window"] or q + p
            first = max(0, min(q, w - p))            # tokens whose window reaches the first key
            pairs += first * p + first * (first + 1) // 2 + (q - first) * w
        rows = 2 * sum(n) * case["heads"] * (hd + 2) + 2 * 2 * (sum(n) + sum(held)) * hkv * hd
        return {"bytes": rows, "flops": 4 * pairs * case["heads"] * hd}
    entry = hkv * ng * 72                            # one entry's codes, scales and biases, K and V
    if case["op"] == "write":
        size = 4 if case["dtype"] == "f32" else 2
        back = sum(n) + (sum(held) if case["back"] == "all" else 0)
        return {"bytes": sum(n) * (2 * hkv * hd * size + entry + 8 * hkv) + back * (entry + 2 * hkv * hd * size),
                "flops": 0}
    if case["op"] == "decode":
        size = 4 if case["dtype"] == "f32" else 2
        score = 8 * hkv * sum(n) if case["score"] else 0
        return {"bytes": sum(n) * entry + 2 * case["seqs"] * case["heads"] * hd * size + score,
                "flops": 4 * sum(n) * case["heads"] * hd}
    bytes_ = 0.0
    for k in n:
        keep = min(k, case["keep"])
        late = min(case["recent"], k - keep)
        moved = late + (k - keep - late) * (keep - late) / max(1, k - late)
        bytes_ += hkv * (8 * k + 8 * keep) + 2 * entry * moved
    return {"bytes": bytes_, "flops": 0}


# ------------------------------------------------------------------- inputs
def _quantise(x):
    """4-bit codes and (scale, bias) of groups of 64: x [..., head_dim] in f32."""
    g = x.unflatten(-1, (-1, GROUP))
    low, high = g.amin(-1, keepdim=True), g.amax(-1, keepdim=True)
    bias = low.bfloat16().float()
    scale = ((high - low) * torch.tensor(1 / 15, dtype=F32, device=x.device)).bfloat16().float()
    code = torch.where(scale > 0, (g - bias) / torch.where(scale > 0, scale, 1.0), 0.0).round().clamp(0, 15)
    return code.to(torch.uint8), torch.cat((scale, bias), -1).bfloat16()


def _views(blocks, head_dim):
    """Codes [pages, heads, K/V, group, slot, 32] and (scale, bias) [pages, heads, K/V, group, slot, 2] of the blocks."""
    ng = head_dim // GROUP
    codes = blocks[..., : ng * 4096].unflatten(-1, (2, ng, PAGE, 32))
    sb = blocks.view(torch.bfloat16)[..., ng * 2048:].unflatten(-1, (2, ng, PAGE, 2))
    return codes, sb


def _store(blocks, head_dim, page, slot, k, v):
    """Quantised rows k, v [n, heads, head_dim] into the entries (page, slot)."""
    codes, sb = _views(blocks, head_dim)
    c, s = _quantise(torch.stack((k, v), 2))                       # [n, heads, 2, groups, 64]
    codes[page, :, :, :, slot] = c[..., 0::2] | (c[..., 1::2] << 4)
    sb[page, :, :, :, slot] = s


def _load(blocks, head_dim, page, slot):
    """Values [n, heads, 2, head_dim] that the entries (page, slot) stand for, in f32."""
    codes, sb = _views(blocks, head_dim)
    c = codes[page, :, :, :, slot]                                 # [n, heads, 2, groups, 32]
    c = torch.stack((c & 15, c >> 4), -1).flatten(-2).float()
    s = sb[page, :, :, :, slot].float()
    return (c * s[..., 0:1] + s[..., 1:2]).flatten(-2)


def _cache(g, case, lens, scored):
    """A cache of entries made from Gaussian rows, its pages in a random order; room for `lens` entries of each sequence."""
    hd, hkv = case["head_dim"], case["kv_heads"]
    width = (max(lens) + PAGE - 1) // PAGE
    need = [(n + PAGE - 1) // PAGE for n in lens]
    table = torch.zeros(len(lens), width, dtype=torch.int32, device="cuda")
    order = torch.randperm(sum(need) + 1, generator=g, device="cuda").int()
    held = torch.arange(width, device="cuda")[None] < torch.tensor(need, device="cuda")[:, None]
    table[held] = order[: sum(need)]
    pages = sum(need) + 1
    blocks = torch.empty(pages, hkv, hd // GROUP * BLOCK, dtype=torch.uint8, device="cuda")
    codes, sb = _views(blocks, hd)
    step = max(1, (1 << 26) // (hkv * PAGE * hd * 2))
    for p in range(0, pages, step):
        m = min(step, pages - p)
        x = torch.randn(m, hkv, 2, PAGE, hd, generator=g, device="cuda")
        c, s = _quantise(x)
        codes[p: p + m] = (c[..., 0::2] | (c[..., 1::2] << 4)).transpose(3, 4)
        sb[p: p + m] = s.transpose(3, 4)
    st = {"blocks": blocks, "table": table}
    if scored:  # accumulated weights have a long tail
        st["score"] = torch.randn(pages, hkv, PAGE, generator=g, device="cuda").mul_(2).exp_().mul_(0.05)
    return st


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    n, held = _lengths(case)
    hd, hkv = case["head_dim"], case["kv_heads"]

    def ints(v):
        return torch.tensor(v, dtype=torch.int32, device="cuda")

    def starts(v):
        return ints([sum(v[:i]) for i in range(len(v) + 1)])

    def randn(*shape, std=1.0, dtype=torch.bfloat16):
        return torch.randn(*shape, generator=g, device="cuda").mul_(std).to(dtype)

    st = {"case": case, "n": n, "held": held, "cu": starts(n)}
    if case["op"] == "prompt":
        total = [a + b for a, b in zip(n, held)]
        st["q"] = randn(sum(n), case["heads"], hd, std=2.0)        # peaked, as after per-head norms
        st["k"], st["v"] = randn(sum(total), hkv, hd), randn(sum(total), hkv, hd)
        st["cu_k"], st["total"] = starts(total), total
        st["out"] = torch.zeros_like(st["q"])
        st["lse"] = torch.zeros(sum(n), case["heads"], device="cuda")
    elif case["op"] == "write":
        dtype = TYPES[case["dtype"]]
        st.update(_cache(g, case, [a + b for a, b in zip(n, held)], scored=True))
        st["k"], st["v"] = randn(sum(n), hkv, hd, dtype=dtype), randn(sum(n), hkv, hd, dtype=dtype)
        st["pos"] = torch.zeros(st["score"].shape, dtype=torch.int32, device="cuda")
        st["len"], st["seen"] = ints(held), ints([h + 7 * (i % 3) for i, h in enumerate(held)])
        back = [a + b for a, b in zip(n, held)] if case["back"] == "all" else n
        st["first"] = ints([0] * len(n)) if case["back"] == "all" else ints(held)
        st["back"], st["cu_back"] = back, starts(back)
        st["k_back"] = torch.zeros(sum(back), hkv, hd, dtype=dtype, device="cuda")
        st["v_back"] = torch.zeros_like(st["k_back"])
    elif case["op"] == "decode":
        dtype = TYPES[case["dtype"]]
        st.update(_cache(g, case, n, scored=case["score"]))
        st["q"] = randn(len(n), case["heads"], hd, std=2.0, dtype=dtype)
        st["out"] = torch.zeros_like(st["q"])
        st["len"] = ints([k - 1 for k in n])                       # this step's entry is in the cache already
        if case["score"]:
            st["score_out"] = torch.zeros_like(st["score"])
    else:
        st.update(_cache(g, case, n, scored=True))
        hp, width = st["table"].shape[1] * PAGE, st["table"].shape[1]
        st["len"], st["seen"] = ints(n), ints([2 * k for k in n])
        # entries still in the order of their positions, with gaps that earlier evictions left
        gap = torch.randint(0, 2, (len(n), hkv, hp), generator=g, device="cuda")
        back = torch.arange(hp, device="cuda")[None, None] - st["len"][:, None, None]
        pos = st["seen"][:, None, None] + back - torch.where(back < -case["recent"], gap, 0)
        st["pos"] = torch.zeros(st["score"].shape, dtype=torch.int32, device="cuda")
        inside = torch.arange(width, device="cuda")[None] * PAGE < st["len"][:, None]
        st["pos"][st["table"][inside].long()] = pos.clamp(min=0).int().unflatten(-1, (width, PAGE)).transpose(1, 2)[inside]
        st["score_out"], st["pos_out"] = torch.zeros_like(st["score"]), torch.zeros_like(st["pos"])
    if own:
        st["call"] = _call(st)
    return st


# --------------------------------------------------------- the framework's calls
@functools.lru_cache(None)
def _framework():
    sys.path.insert(0, os.path.join(os.getcwd(), "s-moe_b200"))
    import smoe_cuda
    ctx = smoe_cuda.Context(0, max_batch=4)
    ctx.set_stream(torch.cuda.current_stream().cuda_stream or 1)   # 1: the handle of torch's default stream
    return smoe_cuda, ctx


def _call(st):
    """The argument structures and the workspace that a program makes once for its buffers."""
    S, ctx = _framework()
    case = st["case"]
    if case["op"] == "prompt":
        return S.packed_attn_args(st["q"], st["k"], st["v"], st["out"], st["cu"], st["cu_k"], causal=True,
                                  window=case["window"], lse=st["lse"])
    cache = S.kv4_cache(st["blocks"], st["table"], st["len"], case["head_dim"], pos=st.get("pos"),
                        score=st.get("score"), seen=st.get("seen"))
    if case["op"] == "write":
        return cache, S.kv4_rows(st["k"], st["v"], st["cu"]), S.kv4_rows(st["k_back"], st["v_back"], st["cu_back"])
    if case["op"] == "decode":
        args = S.kv4_attn_args(st["q"], st["out"], max_len=case["hi"], extra=1, score_out=st.get("score_out"))
        size = S.kv4_attention_workspace(cache, args)
        st["workspace"] = torch.empty(size, dtype=torch.uint8, device="cuda")
        return cache, S.kv4_attn_set_workspace(args, st["workspace"])
    size = S.kv4_evict_workspace(cache, case["hi"])
    st["workspace"] = torch.empty(size, dtype=torch.uint8, device="cuda")
    return cache


def _run_own(st):
    _, ctx = _framework()
    case, call = st["case"], st["call"]
    if case["op"] == "prompt":
        ctx.attention_packed(call)
        return {"out": st["out"], "lse": st["lse"]}
    if case["op"] == "write":
        cache, rows, back = call
        ctx.kv4_append(cache, rows)
        ctx.kv4_read(cache, st["first"], back)
        return {"k": st["k_back"], "v": st["v_back"], "pos": st["pos"], "score": st["score"]}
    if case["op"] == "decode":
        ctx.kv4_attention(*call)
        return {"out": st["out"], "score": st["score_out"]} if case["score"] else {"out": st["out"]}
    ctx.kv4_evict(call, case["keep"], case["recent"], case["hi"], st["workspace"], pos_out=st["pos_out"],
                  score_out=st["score_out"])
    return {"blocks": st["blocks"], "pos": st["pos_out"], "score": st["score_out"]}


# -------------------------------------------------------------- the plain form
def _spread(cu, width):
    """For starts cu [n + 1]: packed row numbers [n, width], and which of them are in their sequence."""
    at = cu[:-1, None].long() + torch.arange(width, device="cuda")[None]
    inside = at < cu[1:, None]
    return torch.where(inside, at, 0), inside


def _plain_prompt(st):
    case = st["case"]
    b, h, hkv, hd = len(st["n"]), case["heads"], case["kv_heads"], case["head_dim"]
    mq, mk, g = max(st["n"]), max(st["total"]), h // hkv
    rq, in_q = _spread(st["cu"], mq)
    rk, in_k = _spread(st["cu_k"], mk)
    q = st["q"][rq].float().unflatten(2, (hkv, g)).permute(0, 2, 3, 1, 4).reshape(b, hkv, g * mq, hd)
    k, v = (st[x][rk].float().transpose(1, 2) for x in "kv")       # [b, hkv, mk, hd]
    lq, lk = st["cu"].diff(), st["cu_k"].diff()
    i = torch.arange(mq, device="cuda")[None, :, None] + (lk - lq)[:, None, None]
    j = torch.arange(mk, device="cuda")[None, None]
    shut = (j > i) | ~in_k[:, None, :]
    if case["window"]:
        shut |= j <= i - case["window"]
    s = torch.matmul(q.mul_(1 / math.sqrt(hd)), k.transpose(2, 3)).view(b, hkv, g, mq, mk)
    s.masked_fill_(shut[:, None, None], -math.inf)
    top = s.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, 0.0, top)
    s.sub_(top).exp_()
    total = s.sum(-1, keepdim=True)
    o = torch.matmul(s.view(b, hkv, g * mq, mk), v).view(b, hkv, g, mq, hd)
    o = torch.where(total > 0, o / total, 0.0)
    lse = (top + total.log()).squeeze(-1)
    o = o.permute(0, 3, 1, 2, 4).reshape(b, mq, h, hd)[in_q]
    return {"out": o.to(st["q"].dtype), "lse": lse.permute(0, 3, 1, 2).reshape(b, mq, h)[in_q]}


def _entries(st, first, counts, cu):
    """Sequence, page and slot of each packed row, where sequence b's rows are its entries first[b], first[b] + 1, ..."""
    seq = torch.repeat_interleave(torch.arange(len(counts), device="cuda"), cu.diff().long(), output_size=sum(counts))
    at = torch.arange(sum(counts), device="cuda") - cu[seq].long() + first[seq].long()
    return seq, st["table"][seq, at // PAGE].long(), at % PAGE


def _plain_write(st):
    hd = st["case"]["head_dim"]
    seq, page, slot = _entries(st, st["len"], st["n"], st["cu"])
    _store(st["blocks"], hd, page, slot, st["k"].float(), st["v"].float())
    ahead = torch.arange(len(seq), device="cuda") - st["cu"][seq].long()
    st["pos"][page, :, slot] = (st["seen"][seq] + ahead).int()[:, None]
    st["score"][page, :, slot] = 0.0
    _, page, slot = _entries(st, st["first"], st["back"], st["cu_back"])
    x = _load(st["blocks"], hd, page, slot).to(st["k"].dtype)
    return {"k": x[:, :, 0], "v": x[:, :, 1], "pos": st["pos"], "score": st["score"]}


def _plain_decode(st):
    case = st["case"]
    hd, hkv = case["head_dim"], case["kv_heads"]
    codes, sb = _views(st["blocks"], hd)
    table = st["table"].long()
    c = codes[table]                                               # [b, pages, hkv, 2, groups, slot, 32]
    c = torch.stack((c & 15, c >> 4), -1).flatten(-2).float()
    s = sb[table].float()
    kv = c.mul_(s[..., 0:1]).add_(s[..., 1:2])                     # [b, pages, hkv, 2, groups, slot, 64]
    kv = kv.permute(3, 0, 2, 1, 5, 4, 6).flatten(5).flatten(3, 4)  # [2, b, hkv, entries, hd]
    valid = st["len"] + 1
    q = st["q"].float().unflatten(1, (hkv, -1)) * (1 / math.sqrt(hd))
    p = torch.matmul(q, kv[0].transpose(2, 3))                     # [b, hkv, g, entries]
    shut = torch.arange(p.shape[-1], device="cuda")[None] >= valid[:, None]
    p.masked_fill_(shut[:, None, None], -math.inf)
    p = (p - p.amax(-1, keepdim=True)).exp()
    p = p / p.sum(-1, keepdim=True)
    out = {"out": torch.matmul(p, kv[1]).flatten(1, 2).to(st["q"].dtype)}
    if case["score"]:
        w = p.sum(2).unflatten(-1, (-1, PAGE)).transpose(1, 2)     # [b, pages, hkv, slot]
        some = ~shut.unflatten(-1, (-1, PAGE))
        used = some.any(-1)
        page = table[used]
        st["score_out"][page] = torch.where(some[used][:, None], st["score"][page] + w[used], st["score_out"][page])
        out["score"] = st["score_out"]
    return out


def _plain_evict(st):
    case = st["case"]
    keep, hd, hkv = case["keep"], case["head_dim"], case["kv_heads"]
    table = st["table"].long()
    b, width = table.shape
    n = width * PAGE
    score = st["score"][table].transpose(1, 2).reshape(b, hkv, n)
    pos = st["pos"][table].transpose(1, 2).reshape(b, hkv, n)
    at = torch.arange(n, device="cuda")[None, None]
    length = st["len"][:, None, None]
    late = pos + case["recent"] >= st["seen"][:, None, None]
    rank = torch.where(late, math.inf, score)
    rank = torch.where(at < length, rank, -math.inf)
    order = rank.argsort(dim=-1, descending=True, stable=True)
    kept = torch.zeros(b, hkv, n, dtype=torch.bool, device="cuda")
    kept.scatter_(-1, order[..., :keep], True)
    kept = (kept | (length <= keep)) & (at < length)
    # the j-th kept entry past `keep` goes to the j-th free one before it
    free = ~kept & (at < keep) & (at < length)
    far = (kept & (at >= keep)).int().argsort(dim=-1, descending=True, stable=True)
    source = torch.where(free, far.gather(-1, (free.cumsum(-1) - 1).clamp(min=0)), at.expand(b, hkv, n))
    seq, head, to = (at.expand(b, hkv, n) < length.clamp(max=keep)).nonzero(as_tuple=True)
    src = source[seq, head, to]
    sp, ss, dp, ds = table[seq, src // PAGE], src % PAGE, table[seq, to // PAGE], to % PAGE
    codes, sb = _views(st["blocks"], hd)
    new_codes, new_sb = codes[sp, head, :, :, ss], sb[sp, head, :, :, ss]
    codes[dp, head, :, :, ds], sb[dp, head, :, :, ds] = new_codes, new_sb
    st["pos_out"][dp, head, ds], st["score_out"][dp, head, ds] = st["pos"][sp, head, ss], st["score"][sp, head, ss]
    return {"blocks": st["blocks"], "pos": st["pos_out"], "score": st["score_out"]}


def run(state):
    if own:
        return _run_own(state)
    return {"prompt": _plain_prompt, "write": _plain_write, "decode": _plain_decode,
            "evict": _plain_evict}[state["case"]["op"]](state)


# ------------------------------------------------------------------- in 64 bits
def _dequantised(st, b, first, count):
    """K and V [heads, count, head_dim] of sequence b's entries in 64 bits, byte by byte from the block layout."""
    hd = st["case"]["head_dim"]
    ng = hd // GROUP
    e = torch.arange(first, first + count, device="cuda")
    raw = st["blocks"][st["table"][b].long()][e // PAGE]           # [count, heads, bytes]
    slot = e % PAGE
    d = torch.arange(hd, device="cuda")
    both = []
    for kv in range(2):
        byte = (kv * ng + d[None] // GROUP) * PAGE * 32 + slot[:, None] * 32 + d[None] % GROUP // 2
        pair = ((kv * ng + d[None] // GROUP) * PAGE + slot[:, None]) * 4 + ng * 4096
        code = raw.gather(2, byte[:, None].expand(-1, raw.shape[1], -1)).int() >> (4 * (d % 2)).int() & 15
        half = [raw.gather(2, (pair + i)[:, None].expand(-1, raw.shape[1], -1)).int() for i in range(4)]
        scale, bias = ((lo | hi << 8) << 16 for lo, hi in (half[:2], half[2:]))
        both.append((code.double() * scale.view(F32).double() + bias.view(F32).double()).transpose(0, 1))
    return both


def exact(case, seed):
    global own
    before, own = own, False
    st = prepare(case, seed)
    own = before
    hd, hkv = case["head_dim"], case["kv_heads"]
    scale = 1 / math.sqrt(hd)
    if case["op"] == "prompt":
        g = case["heads"] // hkv
        out = torch.zeros(st["q"].shape, dtype=torch.float64, device="cuda")
        lse = torch.zeros(st["lse"].shape, dtype=torch.float64, device="cuda")
        q0 = k0 = 0
        for q, k in zip(st["n"], st["total"]):
            i = torch.arange(q, device="cuda")[:, None] + (k - q)
            j = torch.arange(k, device="cuda")[None]
            open_ = (j <= i) & ((j > i - case["window"]) if case["window"] else (j >= 0))
            for head in range(case["heads"]):
                x = st["q"][q0: q0 + q, head].double() @ st["k"][k0: k0 + k, head // g].double().t() * scale
                x = x.masked_fill(~open_, -math.inf)
                lse[q0: q0 + q, head] = torch.logsumexp(x, -1)
                out[q0: q0 + q, head] = torch.softmax(x, -1) @ st["v"][k0: k0 + k, head // g].double()
            q0, k0 = q0 + q, k0 + k
        return {"out": out, "lse": lse}
    if case["op"] == "write":
        new = []
        for x in (st["k"], st["v"]):
            x = x.double().unflatten(-1, (-1, GROUP))
            low = x.amin(-1, keepdim=True)
            bias, s = low.bfloat16().double(), ((x.amax(-1, keepdim=True) - low) / 15).bfloat16().double()
            new.append((((x - bias) / s).round().clamp(0, 15) * s + bias).flatten(-2))
        ks, vs, row = [], [], 0
        for b, (n, h) in enumerate(zip(st["n"], st["held"])):
            if case["back"] == "all":
                k, v = _dequantised(st, b, 0, h)
                ks.append(k.transpose(0, 1))
                vs.append(v.transpose(0, 1))
            ks.append(new[0][row: row + n])
            vs.append(new[1][row: row + n])
            row += n
        return {"k": torch.cat(ks), "v": torch.cat(vs), "pos": None, "score": None}
    if case["op"] == "decode":
        out = torch.zeros(st["q"].shape, dtype=torch.float64, device="cuda")
        score = torch.zeros(st["score"].shape, dtype=torch.float64, device="cuda") if case["score"] else None
        for b, n in enumerate(st["n"]):
            k, v = _dequantised(st, b, 0, n)
            x = st["q"][b].double().view(hkv, -1, hd) @ k.transpose(1, 2) * scale
            p = torch.softmax(x, -1)
            out[b] = (p @ v).flatten(0, 1)
            if case["score"]:
                e = torch.arange(n, device="cuda")
                page, slot = st["table"][b, e // PAGE].long(), e % PAGE
                score[page, :, slot] = st["score"][page, :, slot].double() + p.sum(1).t()
        return {"out": out, "score": score} if case["score"] else {"out": out}
    score = torch.zeros(st["score"].shape, dtype=torch.float64, device="cuda")
    for b, n in enumerate(st["n"]):
        e = torch.arange(n, device="cuda")
        page, slot = st["table"][b, e // PAGE].long(), e % PAGE
        values, pos = st["score"][page, :, slot].double(), st["pos"][page, :, slot]
        for head in range(hkv):
            s = [math.inf if p + case["recent"] >= int(st["seen"][b]) else v
                 for p, v in zip(pos[:, head].tolist(), values[:, head].tolist())]
            best = sorted(sorted(range(n), key=lambda i: (-s[i], i))[: case["keep"]])
            into = [i for i in range(min(n, case["keep"]))]
            free = sorted(set(into) - set(best))
            for i, j in zip(free, (i for i in best if i >= case["keep"])):
                into[i] = j
            to = torch.arange(len(into), device="cuda")
            score[page[to], head, slot[to]] = values[torch.tensor(into, device="cuda"), head]
    return {"blocks": None, "pos": None, "score": score}           # the others are whole numbers
