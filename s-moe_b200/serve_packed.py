"""Long-context serving of one attention layer: several conversations over a
4-bit KV cache, with the operators as a server calls them.

 1. prompt   the prompts of all conversations, packed: Q/K/V projections, one
             attention_packed over all of them, kv4_append of their K and V;
 2. chunk    (--chunk N) N further tokens of each, as a chunked prefill does:
             append, kv4_read of the whole contexts, attention_packed of the
             new rows over them (cu_k beside cu_q);
 3. decode   one token per conversation and step: append, kv4_attention over
             the cache (keeping each entry's accumulated weight), and one
             kv4_advance a step for all layers;
 4. evict    when the longest conversation passes --limit entries: kv4_evict
             down to --keep, the last --recent positions always kept.

The projections are smoe_cuda_gemm_bf16, per-head norms and RoPE plain torch
on the same stream (keys enter the cache after RoPE, so entries may move).
Weights and inputs are random; what is printed is the time of each part and
how far the 4-bit steps are from attention over unquantised keys and values.

    python s-moe_b200/serve_packed.py --seqs 16 --prompt 2000 --steps 64
"""
from __future__ import annotations

import argparse
import json
import os
import sys

import torch

HERE = os.path.dirname(os.path.abspath(__file__))
sys.path.insert(0, HERE)
import smoe_cuda as S  # noqa: E402
from decode import Shape, rope_inv_freq  # noqa: E402


def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _starts(n):
    return _ints([sum(n[:i]) for i in range(len(n) + 1)])


class Layer:
    """One layer's projections and 4-bit cache for `lens` conversations with
    room for `room` entries each."""

    def __init__(self, ctx, shape: Shape, n_seqs: int, room: int, seed: int = 1):
        self.ctx, self.sh, self.n_seqs = ctx, shape, n_seqs
        g = torch.Generator(device="cuda")
        g.manual_seed(seed)
        rows = {"w_q": shape.q_dim, "w_k": shape.kv_dim, "w_v": shape.kv_dim, "w_o": shape.d_model}
        cols = {"w_o": shape.q_dim}
        self.w = {n: (torch.randn(r, cols.get(n, shape.d_model), generator=g, device="cuda") * 0.02).to(torch.bfloat16)
                  for n, r in rows.items()}
        self.inv_freq = torch.from_numpy(rope_inv_freq(shape)).cuda()
        width = (room + S.KV4_PAGE - 1) // S.KV4_PAGE
        pages = n_seqs * width
        hkv, hd = shape.num_kv_heads, shape.head_dim
        self.blocks = torch.zeros(pages, hkv, S.kv4_block_bytes(hd), dtype=torch.uint8, device="cuda")
        self.table = torch.randperm(pages, generator=g, device="cuda").int().view(n_seqs, width).contiguous()
        self.len, self.seen = _ints([0] * n_seqs), _ints([0] * n_seqs)
        self.pos = torch.zeros(pages, hkv, S.KV4_PAGE, dtype=torch.int32, device="cuda")
        self.score = torch.zeros(pages, hkv, S.KV4_PAGE, device="cuda")
        self.cache = S.kv4_cache(self.blocks, self.table, self.len, hd, seen=self.seen, pos=self.pos, score=self.score)
        self.room = width * S.KV4_PAGE
        self.out = torch.zeros(n_seqs, shape.num_heads, hd, device="cuda")
        self.attn = None                       # kv4_attention's arguments, made at the first step
        self.evict_ws = torch.empty(S.kv4_evict_workspace(self.cache, self.room), dtype=torch.uint8, device="cuda")

    def project(self, name, x):
        y = torch.empty(x.shape[0], self.w[name].shape[0], device="cuda")
        self.ctx.gemm_bf16(self.w[name], x, y, self.w[name].shape[0], x.shape[1], x.shape[0])
        return y

    def qkv(self, x, pos):
        """Q and K (normed per head, with RoPE) and V of rows x [n, d_model] at positions pos [n], fp32."""
        sh = self.sh
        q, k, v = (self.project(n, x).view(len(x), -1, sh.head_dim) for n in ("w_q", "w_k", "w_v"))
        ang = pos.float()[:, None] * self.inv_freq
        cos, sin = ang.cos()[:, None], ang.sin()[:, None]

        def norm_rope(y):
            y = y * torch.rsqrt(y.square().mean(-1, keepdim=True) + 1e-6)
            a, b = y.chunk(2, -1)
            return torch.cat((a * cos - b * sin, b * cos + a * sin), -1).contiguous()
        return norm_rope(q), norm_rope(k), v.contiguous()

    def prompt(self, x, new, held):
        """Rows x of sequences with `new` tokens each after `held` ones: attention output [n, heads, head_dim] bf16."""
        total = [a + b for a, b in zip(new, held)]
        pos = torch.cat([torch.arange(h, t, device="cuda") for h, t in zip(held, total)])
        q, k, v = self.qkv(x, pos)
        qb, kb, vb = (t.to(torch.bfloat16) for t in (q, k, v))
        cu = _starts(new)
        self.ctx.kv4_append(self.cache, S.kv4_rows(kb, vb, cu))
        cu_k = None
        if any(held):                          # the earlier tokens come back from the cache, with the new ones
            cu_k = _starts(total)
            kb, vb = (torch.empty(sum(total), *kb.shape[1:], dtype=kb.dtype, device="cuda") for _ in range(2))
            self.ctx.kv4_read(self.cache, None, S.kv4_rows(kb, vb, cu_k))
        out = torch.empty_like(qb)
        self.ctx.attention_packed(S.packed_attn_args(qb, kb, vb, out, cu, cu_k))
        self.ctx.kv4_advance(self.len, self.seen, self.n_seqs, cu=cu)
        return out, (qb, k, v)

    def step(self, x, pos):
        """One token per sequence: attention output [n_seqs, heads, head_dim] fp32."""
        q, k, v = self.qkv(x, pos)
        self.ctx.kv4_append(self.cache, S.kv4_rows(k, v, self.one))
        if self.attn is None:
            self.q = torch.empty_like(q)
            self.attn = S.kv4_attn_args(self.q, self.out, self.room, extra=1, score_out=self.score)
            self.attn_ws = torch.empty(S.kv4_attention_workspace(self.cache, self.attn), dtype=torch.uint8, device="cuda")
            S.kv4_attn_set_workspace(self.attn, self.attn_ws)
        self.q.copy_(q)
        self.ctx.kv4_attention(self.cache, self.attn)
        self.ctx.kv4_advance(self.len, self.seen, self.n_seqs, n_each=1)
        return self.out, (q, k, v)

    @property
    def one(self):
        if not hasattr(self, "_one"):
            self._one = _starts([1] * self.n_seqs)
        return self._one

    def evict(self, keep, recent):
        self.ctx.kv4_evict(self.cache, keep, recent, self.room, self.evict_ws)
        self.ctx.kv4_advance(self.len, self.seen, self.n_seqs, n_each=0, keep=keep)


def serve(shape: Shape, seqs: int, prompt: int, chunk: int, steps: int, limit: int, keep: int, recent: int, seed: int = 3):
    """Runs the parts above; returns a dict of times (ms) and, for the decode
    steps before the first eviction, the relative distance of the 4-bit
    outputs from attention over the unquantised keys and values."""
    lens = [max(1, prompt - (i * prompt) // (2 * seqs)) for i in range(seqs)]
    more = [chunk] * seqs
    ctx = S.Context(0, max_batch=max(sum(lens), chunk * seqs, 4), max_d_model=max(shape.d_model, shape.q_dim), max_d_ff=64,
                    max_experts=16)
    stream = torch.cuda.Stream()
    ctx.set_stream(stream.cuda_stream)
    report = {"lens": lens}
    with torch.cuda.stream(stream):
        room = min(limit + 1, max(lens) + chunk + steps) if limit else max(lens) + chunk + steps
        layer = Layer(ctx, shape, seqs, max(room, max(lens) + chunk + 1), seed)
        g = torch.Generator(device="cuda")
        g.manual_seed(seed + 1)
        marks = [(torch.cuda.Event(enable_timing=True), "start")]
        marks[0][0].record()

        def mark(name):
            marks.append((torch.cuda.Event(enable_timing=True), name))
            marks[-1][0].record()
        x = torch.randn(sum(lens), shape.d_model, generator=g, device="cuda")
        layer.prompt(x, lens, [0] * seqs)      # warm-up of the libraries; forgotten again
        layer.len.zero_()
        layer.seen.zero_()
        mark("warm")
        out, (_, k, v) = layer.prompt(x, lens, [0] * seqs)
        mark("prompt")
        exact_k, exact_v = (list(t.split(lens)) for t in (k, v))
        total = lens
        if chunk:
            y = torch.randn(chunk * seqs, shape.d_model, generator=g, device="cuda")
            mark("idle")
            out, (_, k, v) = layer.prompt(y, more, lens)
            mark("chunk")
            exact_k = [torch.cat(p) for p in zip(exact_k, k.split(more))]
            exact_v = [torch.cat(p) for p in zip(exact_v, v.split(more))]
            total = [a + b for a, b in zip(lens, more)]
        held, evictions, worst, G = list(total), 0, 0.0, shape.num_heads // shape.num_kv_heads
        for i in range(steps):
            if limit and max(held) >= limit:
                mark("idle")
                layer.evict(keep, recent)
                mark("evict")
                held, evictions = [min(h, keep) for h in held], evictions + 1
            z = torch.randn(seqs, shape.d_model, generator=g, device="cuda")
            pos = _ints([t + i for t in total])
            mark("idle")
            out, (q, k, v) = layer.step(z, pos)
            mark("decode")
            held = [h + 1 for h in held]
            if evictions == 0 and i < 2:
                for b in range(seqs):
                    exact_k[b], exact_v[b] = torch.cat((exact_k[b], k[b: b + 1])), torch.cat((exact_v[b], v[b: b + 1]))
                    s = torch.einsum("kgd,nkd->kgn", q[b].view(-1, G, shape.head_dim), exact_k[b]) / shape.head_dim ** 0.5
                    want = torch.einsum("kgn,nkd->kgd", s.softmax(-1), exact_v[b]).reshape(out[b].shape)
                    worst = max(worst, float((out[b] - want).norm() / want.norm()))
        layer.project("w_o", out.reshape(seqs, -1).float().contiguous())
        mark("end")
        ctx.synchronize()
        for (a, _), (b, name) in zip(marks, marks[1:]):
            report.setdefault(name, []).append(a.elapsed_time(b))
        report["lengths"], report["seen"] = layer.len.tolist(), layer.seen.tolist()
        assert report["lengths"] == held and report["seen"] == [t + steps for t in total]
    report = {n: (round(sum(v) / len(v), 4) if n in ("prompt", "chunk", "decode", "evict") else v) for n, v in report.items()
              if n not in ("warm", "idle", "end")}
    report.update(evictions=evictions, rel_distance=round(worst, 5), cache_bytes=layer.blocks.numel(), finite=bool(out.isfinite().all()))
    ctx.close()
    return report


def main():
    ap = argparse.ArgumentParser(description=__doc__.split("\n\n")[0])
    ap.add_argument("--seqs", type=int, default=16)
    ap.add_argument("--prompt", type=int, default=2000, help="tokens of the longest prompt")
    ap.add_argument("--chunk", type=int, default=256)
    ap.add_argument("--steps", type=int, default=64)
    ap.add_argument("--limit", type=int, default=2280)
    ap.add_argument("--keep", type=int, default=2048)
    ap.add_argument("--recent", type=int, default=256)
    a = ap.parse_args()
    print(json.dumps(serve(Shape(layers=1), a.seqs, a.prompt, a.chunk, a.steps, a.limit, a.keep, a.recent)))


if __name__ == "__main__":
    main()
