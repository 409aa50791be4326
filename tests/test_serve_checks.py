"""CPU: what the long-context serving calls check of their tensors against one
another before anything is launched (the library behind them is a recorder
here). A mismatch that came through would be a read or write out of range."""
import pytest
import torch

import smoe_cuda as S


class Recorder:
    def __init__(self):
        self.called = []

    def __getattr__(self, name):
        return lambda *a: self.called.append(name) or S.SMOE_OK


@pytest.fixture
def ctx(monkeypatch):
    """A context whose library only records, and for which host tensors pass as the GPU's."""
    c = S.Context.__new__(S.Context)
    c.L, c.h = Recorder(), None
    monkeypatch.setattr(S, "_host", lambda **t: None)
    monkeypatch.setattr(S, "_need_gpu", lambda t, name: None)
    return c


def ints(*v):
    return torch.tensor(v, dtype=torch.int32)


def cache(n_seqs=3, heads=2, hd=128, pages=5):
    return S.kv4_cache(torch.zeros(pages, heads, S.kv4_block_bytes(hd), dtype=torch.uint8),
                       torch.zeros(n_seqs, 2, dtype=torch.int32), torch.zeros(n_seqs, dtype=torch.int32), hd,
                       pos=torch.zeros(pages, heads, 64, dtype=torch.int32), score=torch.zeros(pages, heads, 64))


def rows(n=7, heads=2, hd=128, cu=(0, 2, 4, 7), dtype=torch.float32):
    return S.kv4_rows(torch.zeros(n, heads, hd, dtype=dtype), torch.zeros(n, heads, hd, dtype=dtype), ints(*cu))


def refused(ctx, match, call):
    with pytest.raises(ValueError, match=match):
        call()
    assert ctx.L.called == []


def test_rows_against_the_cache(ctx):
    for call in (lambda r: ctx.kv4_append(cache(), r), lambda r: ctx.kv4_read(cache(), None, r)):
        refused(ctx, "KV heads", lambda: call(rows(heads=1)))
        refused(ctx, "KV heads", lambda: call(rows(heads=4)))
        refused(ctx, "KV heads", lambda: call(rows(hd=64)))
        refused(ctx, "cu", lambda: call(rows(cu=(0, 2, 7))))
    with pytest.raises(ValueError, match="cu"):
        S.kv4_rows(torch.zeros(1, 2, 64), torch.zeros(1, 2, 64), ints())
    ctx.kv4_append(cache(), rows())
    ctx.kv4_read(cache(), ints(0, 0, 0), rows(dtype=torch.bfloat16))
    assert ctx.L.called == ["smoe_cuda_kv4_append", "smoe_cuda_kv4_read"]


def test_first_entries(ctx):
    refused(ctx, "first", lambda: ctx.kv4_read(cache(), torch.zeros(3, dtype=torch.int64), rows()))
    refused(ctx, "first", lambda: ctx.kv4_read(cache(), ints(0, 0), rows()))
    refused(ctx, "first", lambda: ctx.kv4_read(cache(), ints(0, 0, 0, 0, 0, 0)[::2], rows()))


def test_attention_against_the_cache(ctx):
    def args(n=3, hd=128, **kw):
        return S.kv4_attn_args(torch.zeros(n, 8, hd), torch.zeros(n, 8, hd), 100, **kw)
    refused(ctx, "q and out", lambda: ctx.kv4_attention(cache(), args(n=2)))
    refused(ctx, "q and out", lambda: ctx.kv4_attention(cache(), args(hd=64)))
    refused(ctx, "score_out", lambda: ctx.kv4_attention(cache(), args(score_out=torch.zeros(4, 2, 64))))
    for bad in (torch.zeros(5, 2, 64, dtype=torch.bfloat16), torch.zeros(5, 2, 128)[:, :, ::2], torch.zeros(1, 1, 1).expand(5, 2, 64)):
        with pytest.raises(ValueError, match="score_out"):
            args(score_out=bad)
    for kw in ({"extra": -1}, {"extra": 1 << 32}):
        with pytest.raises(ValueError, match="extra"):
            args(**kw)
    with pytest.raises(ValueError, match="max_len"):
        S.kv4_attn_args(torch.zeros(3, 8, 64), torch.zeros(3, 8, 64), -1)
    with pytest.raises(ValueError, match="workspace"):
        S.kv4_attn_set_workspace(args(), torch.zeros(1, dtype=torch.uint8).expand(1 << 20))
    ctx.kv4_attention(cache(), args(score_out=torch.zeros(5, 2, 64)))
    assert ctx.L.called == ["smoe_cuda_kv4_attention"]


def test_eviction_against_the_cache(ctx):
    ws, pos, score = torch.zeros(10000, dtype=torch.uint8), torch.zeros(5, 2, 64, dtype=torch.int32), torch.zeros(5, 2, 64)
    ev = lambda **kw: ctx.kv4_evict(cache(), 10, 2, 100, **{"workspace": ws, "pos_out": pos, "score_out": score, **kw})
    refused(ctx, "pos_out", lambda: ev(pos_out=pos.long()))
    refused(ctx, "pos_out", lambda: ev(pos_out=pos[:4]))
    refused(ctx, "score_out", lambda: ev(score_out=score.bfloat16()))
    refused(ctx, "score_out", lambda: ev(score_out=score[:, :1]))
    refused(ctx, "workspace", lambda: ev(workspace=ws[::2]))
    refused(ctx, "keep", lambda: ctx.kv4_evict(cache(), -1, 2, 100, ws))
    refused(ctx, "recent", lambda: ctx.kv4_evict(cache(), 1, -2, 100, ws))
    ev()
    ev(pos_out=None, score_out=None)
    assert ctx.L.called == ["smoe_cuda_kv4_evict"] * 2


def test_advance(ctx):
    lens = ints(1, 2, 3)
    refused(ctx, "lens", lambda: ctx.kv4_advance(lens.long(), None, 3))
    refused(ctx, "lens", lambda: ctx.kv4_advance(lens, None, 4))
    refused(ctx, "seen", lambda: ctx.kv4_advance(lens, lens[:2], 3))
    refused(ctx, "cu", lambda: ctx.kv4_advance(lens, None, 3, cu=ints(0, 1, 2)))
    refused(ctx, "keep", lambda: ctx.kv4_advance(lens, None, 3, keep=-1))
    ctx.kv4_advance(lens, ints(1, 2, 3), 3, cu=ints(0, 1, 2, 3))
    assert ctx.L.called == ["smoe_cuda_kv4_advance"]


def test_packed_arguments(ctx):
    q, k = torch.zeros(4, 8, 64, dtype=torch.bfloat16), torch.zeros(6, 2, 64, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="cu_q"):                  # no starts at all: n_seqs would be 2^32 - 1
        S.packed_attn_args(q, k, k, q.clone(), ints())
    with pytest.raises(ValueError, match="window"):
        S.packed_attn_args(q, k, k, q.clone(), ints(0, 4), window=-1)
    ctx.attention_packed(S.packed_attn_args(q, k, k, q.clone(), ints(0, 4), ints(0, 6)))
    assert ctx.L.called == ["smoe_cuda_attention_packed"]


def test_host_tensors_are_refused():
    """Host memory in the place of a GPU tensor."""
    ctx = S.Context.__new__(S.Context)
    ctx.L, ctx.h = Recorder(), None
    q, k = torch.zeros(3, 8, 128, dtype=torch.bfloat16), torch.zeros(3, 2, 128, dtype=torch.bfloat16)
    refused(ctx, "on the GPU", lambda: ctx.attention_packed(S.packed_attn_args(q, k, k, q.clone(), ints(0, 3))))
    refused(ctx, "on the GPU", lambda: ctx.kv4_append(cache(), rows()))
    refused(ctx, "on the GPU", lambda: ctx.kv4_read(cache(), None, rows()))
    refused(ctx, "on the GPU", lambda: ctx.kv4_attention(cache(), S.kv4_attn_args(q, q.clone(), 10)))
    refused(ctx, "on the GPU", lambda: ctx.kv4_evict(cache(), 10, 2, 100, torch.zeros(100)))
    refused(ctx, "on the GPU", lambda: ctx.kv4_advance(ints(1), None, 1))


def test_structures_filled_in_by_hand_pass(ctx):
    """Without a builder there is nothing to compare: the library checks what it can."""
    ctx.kv4_append(S.Kv4Cache(), S.Kv4Rows())
    ctx.kv4_attention(S.Kv4Cache(), S.Kv4AttnArgs())
    ctx.attention_packed(S.PackedAttnArgs())
    ctx.kv4_advance(1 << 20, None, 3)
    assert len(ctx.L.called) == 4
