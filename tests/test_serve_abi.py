"""CPU: the long-context serving entries' structures, their builders' checks,
and the host-side queries that need no GPU."""
import ctypes

import pytest
import torch

import smoe_cuda as S


def test_struct_layouts():
    assert ctypes.sizeof(S.PackedAttnArgs) == 7 * 8 + 8 * 8 + 8 * 4 + 4 + 4      # padded to 8
    assert ctypes.sizeof(S.Kv4Cache) == 6 * 8 + 5 * 4 + 4
    assert ctypes.sizeof(S.Kv4Rows) == 3 * 8 + 4 * 8 + 2 * 4
    assert ctypes.sizeof(S.Kv4AttnArgs) == 4 * 8 + 3 * 8 + 3 * 4 + 3 * 4
    assert S.kv4_block_bytes(64) == 4608 and S.kv4_block_bytes(128) == 9216
    for hd in (0, 32, 80, 96, 256):
        with pytest.raises(S.SmoeCudaError):
            S.kv4_block_bytes(hd)


def rows(n, h, d, dtype=torch.bfloat16):
    return torch.zeros(n, h, d, dtype=dtype)


def test_packed_attn_args():
    q, k = rows(10, 8, 64), rows(12, 2, 64)
    cu = torch.tensor([0, 4, 10], dtype=torch.int32)
    a = S.packed_attn_args(q, k, k.clone(), rows(10, 8, 64), cu, torch.tensor([0, 6, 12], dtype=torch.int32), window=5)
    assert (a.n_seqs, a.total_q, a.total_k, a.num_heads, a.num_kv_heads, a.head_dim) == (2, 10, 12, 8, 2, 64)
    assert (a.q_row, a.q_head, a.k_row, a.k_head, a.causal, a.window) == (512, 64, 128, 64, 1, 5) and abs(a.scale - 0.125) < 1e-7
    heads_first = rows(8, 10, 64).transpose(0, 1)
    b = S.packed_attn_args(heads_first, k, k, rows(10, 8, 64), cu)
    assert (b.q_row, b.q_head, b.cu_k) == (64, 640, None)
    with pytest.raises(TypeError):
        S.packed_attn_args(q.float(), k, k, q, cu)
    with pytest.raises(ValueError):
        S.packed_attn_args(q, k, k, rows(9, 8, 64), cu)
    with pytest.raises(ValueError):
        S.packed_attn_args(q.transpose(1, 2), k, k, q, cu)
    with pytest.raises(ValueError):
        S.packed_attn_args(q, k, k, q, cu.long())
    with pytest.raises(ValueError):
        S.packed_attn_args(q, k, k, q, cu, lse=torch.zeros(10, 7))


def test_kv4_builders():
    blocks, table = torch.zeros(5, 2, 9216, dtype=torch.uint8), torch.zeros(3, 2, dtype=torch.int32)
    lens = torch.zeros(3, dtype=torch.int32)
    c = S.kv4_cache(blocks, table, lens, 128)
    assert (c.n_pages, c.n_seqs, c.table_stride, c.num_kv_heads, c.head_dim) == (5, 3, 2, 2, 128)
    assert (c.seen, c.pos, c.score) == (None, None, None)
    with pytest.raises(ValueError):
        S.kv4_cache(blocks, table, lens, 64)
    with pytest.raises(ValueError):
        S.kv4_cache(blocks, table, lens[:2], 128)
    with pytest.raises(ValueError):
        S.kv4_cache(blocks, table, lens, 128, score=torch.zeros(4, 2, 64))
    r = S.kv4_rows(rows(7, 2, 128, torch.float32), rows(7, 2, 128, torch.float32), lens)
    assert (r.total, r.dtype, r.k_row, r.v_head) == (7, S.DTYPE_F32, 256, 128)
    with pytest.raises(TypeError):
        S.kv4_rows(rows(7, 2, 128, torch.float16), rows(7, 2, 128, torch.float16), lens)
    with pytest.raises(ValueError):
        S.kv4_rows(rows(7, 2, 128), rows(6, 2, 128), lens)
    q = rows(3, 16, 128)
    a = S.kv4_attn_args(q, rows(3, 16, 128), max_len=100)
    plain = S.kv4_attention_workspace(c, a)
    scored = S.kv4_attention_workspace(c, S.kv4_attn_args(q, rows(3, 16, 128), max_len=100, score_out=torch.zeros(5, 2, 64)))
    assert 0 < plain and scored >= plain + 3 * 16 * 128 * 4       # a row of scores per head, whole pages
    assert S.kv4_evict_workspace(c, 100) >= 3 * 2 * 100 * 4
    with pytest.raises(ValueError):
        S.kv4_attn_args(q.transpose(0, 1), q, max_len=1)


def test_refusals_without_a_context():
    L = S.lib()
    assert L.smoe_cuda_attention_packed(None, None) == S.SMOE_ERR_ARG
    assert L.smoe_cuda_kv4_append(None, None, None) == S.SMOE_ERR_ARG
    assert L.smoe_cuda_kv4_read(None, None, None, None) == S.SMOE_ERR_ARG
    assert L.smoe_cuda_kv4_attention(None, None, None) == S.SMOE_ERR_ARG
    assert L.smoe_cuda_kv4_evict(None, None, 1, 1, 1, None, None, None, 0) == S.SMOE_ERR_ARG
    assert L.smoe_cuda_kv4_advance(None, None, None, 1, None, 1, 0) == S.SMOE_ERR_ARG
    assert S.last_error() != ""
