// prompt_attn.cuh - attention over packed prompts: causal, grouped heads,
// sequences of different lengths in one launch, on the tcgen05 tensor cores.
#pragma once
#include <cuda.h>

#include "serve.cuh"
#include "tc05.cuh"

namespace smoe {

// Tile rows are (token, head of the group) pairs, token-major: a KV head's
// keys and values then serve all its query heads from one shared-memory copy,
// and a short prompt fills a tile with G times fewer tokens. A CTA works on
// two tiles of 128 rows at a time (the tensor cores work for one while the
// other's softmax runs) and walks the keys 64 at a time. Each tile has room for
// the scores of two blocks: the next block's are there when the softmax has
// done one (with 128 keys and one place it waited for two products every
// time; 24 prompts of 17 to 2,048 tokens took 1.13 times as long).
//
// Small calls run a CTA per tile pair. Otherwise there is one CTA an SM, which
// goes from pair to pair with the next one's loads in flight:
//  - many pairs: each CTA takes the next one from a list, the longest first
//    (k_packed_plan sorts it). CTAs that run side by side then walk the same
//    keys at the same time, which the L2 serves them together - with shares
//    of neighbouring pairs instead, 16,384 tokens took 1.18 times as long;
//  - few pairs: each CTA takes an equal share of the line of all pairs' key
//    blocks, and the parts of a pair that is cut are joined by k_packed_join.
//
// Softmax by the running maximum and sum; probabilities go back to tensor
// memory as bf16 (over the scores) and are the left operand of the second
// product, which takes both operands of one type, the values'. Their sum and
// the lse are taken before that rounding. (Results are 1.8e-3 to 2.2e-3 from
// 64 bits, with fp32 probabilities 1.6e-3 to 1.7e-3.) A block of 64 keys
// takes a tile pair 1,800 cycles, of which the exponentials' unit needs 1,024
// (its two tiles take it by turns, 900 each) and the tensor cores 1,060.
// 16,384 causal tokens of 32 / 4 heads of 128: 1.75 ms, 1,260 TFLOP/s in
// short runs, 1.97 ms, 1,117 for seconds on end (the power limit); 24 prompts
// of 17 to 2,048: 180 us, 826 TFLOP/s, and 190, 782; 4 x 200..512 tokens over
// 6,000 keys, heads of 64: 36 us; 45 tokens: 8.4 us.
// (Without turns 1.05 times as long; part of the exponentials by polynomial,
// chunks of 16 were no faster.)
constexpr uint32_t kPaRows = 128, kPaKeys = 64;
constexpr int kPaThreads = 384;                  // 2 x 4 softmax warps; TMA, MMA of each tile and items, a warp each
constexpr int kPaItems = 2;                       // items that a CTA has at hand: the one in work and the next
constexpr uint32_t kPaMaxPairs = 65536;          // tile pairs of a planned call (per KV head)

// A place in the line: KV head, sequence, first token of the pair, and the
// block of its keys (counted from the pair's first).
struct PaPlace {
    uint32_t kvh, seq, tok, blk;
};

struct PackedArgs {
    SmoeCudaPackedAttnArgs a;
    uint32_t group, tokens;                      // query heads per KV head, tokens per tile (128 / group)
    uint32_t k_step, v_step;                     // 1, or 0 where all KV heads have the same keys / values
    float scale_log2;                            // scale * log2(e), positive
    uint32_t* err;
    const PaPlace* plan;                         // [CTAs + 1] where each CTA's share starts, or null
    const uint2* list;                           // [*pairs] (sequence, token) of the pairs, longest first, or null
    uint32_t* taken;                             // pairs (times KV heads) taken from it so far, and the number of pairs
                                                 // (both null: a CTA per pair)
    float* part;                                 // [2 per CTA][256 rows][head_dim 64 or 128] sums of the cut pairs' parts
    float2* stat;                                // [2 per CTA][256 rows] maximum (of the unscaled scores), sum
};

template <int HP>                                // head_dim rounded up to 64 or 128
struct PackedSmem {
    static constexpr uint32_t TILE = HP / 64 * 16384;            // 128 rows, 64-column halves of 128-byte rows
    static constexpr uint32_t BLOCK = TILE * kPaKeys / kPaRows;  // 64 rows of keys or values, likewise
    static constexpr int STAGES = 8;                             // even: keys in the even ones, values in the odd
    static constexpr uint32_t Q = 0, KV = 2 * TILE, OUT = KV + STAGES * BLOCK;        // OUT: 4 KB a softmax warp, rows on their way out
    static constexpr uint32_t BAR = OUT + 8 * 4096, ITEMS = BAR + 512, END = ITEMS + kPaItems * 64;
    static constexpr uint32_t bytes() { return END + 1024; }     // the base is rounded up to 1024
};

// Keys [lo, hi) of a token at index i of its sequence.
struct PackedSeq {
    uint32_t q0, k0, len_q, len_k;
    uint16_t causal, bad;                        // bad: its rows are not in the buffers (len_q 0 then)
    uint32_t window;
    SMOE_DEVINL uint32_t hi(uint32_t i) const {
        if (!causal) return len_k;
        const int64_t h = int64_t(i) + 1 + int64_t(len_k) - int64_t(len_q);
        return h < 0 ? 0u : uint32_t(h);                         // (h <= len_k)
    }
    SMOE_DEVINL uint32_t lo(uint32_t i) const {
        const uint32_t h = hi(i);
        return window && h > window ? h - window : 0u;
    }
    // first block of the pair at `tok`, and the blocks that its tile t takes from there
    SMOE_DEVINL uint32_t first_block(uint32_t tok) const { return lo(tok) / kPaKeys; }
    SMOE_DEVINL uint32_t blocks(uint32_t tok, uint32_t tokens, uint32_t t) const {
        const uint32_t first = tok + t * tokens;
        if (first >= len_q) return 0u;
        const uint32_t end = (hi(min(first + tokens, len_q) - 1) + kPaKeys - 1) / kPaKeys, b0 = first_block(tok);
        return end > b0 ? end - b0 : 0u;
    }
};

// Sequence s; len_q 0 for one whose rows are not in the buffers.
SMOE_DEVINL PackedSeq packed_seq(const SmoeCudaPackedAttnArgs& a, uint32_t s) {
    const uint32_t* ck = a.cu_k ? a.cu_k : a.cu_q;
    const uint32_t q0 = ld_plain(a.cu_q + s), q1 = ld_plain(a.cu_q + s + 1), k0 = ld_plain(ck + s), k1 = ld_plain(ck + s + 1);
    const bool ok = q0 <= q1 && q1 <= a.total_q && k0 <= k1 && k1 <= a.total_k;
    return {q0, k0, ok ? q1 - q0 : 0u, ok ? k1 - k0 : 0u, uint16_t(a.causal != 0), uint16_t(!ok), a.window};
}

// What a CTA does next: some blocks of a tile pair. Worked out by a warp of
// its own, some items ahead, and passed to the others in shared memory.
struct alignas(16) PaItem {
    PackedSeq S;
    uint32_t kvh, tok;
    uint32_t key0;                               // first key of the first block
    uint32_t cnt[2];                             // blocks of each tile
    uint32_t inner_hi, inner_lo;                 // some row may not see some key of a block that ends past / starts before these
    uint16_t whole, starts;                      // all of the pair's blocks; its first block among them
    uint16_t more, pad;                          // 0: there was no further item
};
static_assert(sizeof(PaItem) == 64, "an item's place in shared memory");
struct PaWalk {
    PaPlace at, end;
    bool single;                                 // just the pair at `at`
    // the next item, false when there is none; afterwards `at` is behind it
    SMOE_DEVINL bool next(const PackedArgs& p, PaItem& it) {
#pragma unroll 1
        for (;;) {
            if (at.kvh > end.kvh || (at.kvh == end.kvh && (at.seq > end.seq || (at.seq == end.seq && at.tok > end.tok)))) return false;
            const bool last = at.kvh == end.kvh && at.seq == end.seq && at.tok == end.tok;
            if (last && at.blk >= end.blk && !single) return false;
            if (at.seq >= p.a.n_seqs) {
                at = {at.kvh + 1, 0u, 0u, 0u};
                if (at.kvh >= p.a.num_kv_heads) return false;
                continue;
            }
            it.S = packed_seq(p.a, at.seq);
            if (at.tok >= it.S.len_q) {
                at = {at.kvh, at.seq + 1, 0u, 0u};
                continue;
            }
            it.kvh = at.kvh;
            it.tok = at.tok;
            const uint32_t n0 = it.S.blocks(at.tok, p.tokens, 0), n1 = it.S.blocks(at.tok, p.tokens, 1), all = max(n0, n1);
            const uint32_t ba = at.blk, bb = last && !single ? min(end.blk, all) : all;
            it.key0 = (it.S.first_block(at.tok) + ba) * kPaKeys;
            it.cnt[0] = min(bb, n0) > ba ? min(bb, n0) - ba : 0u;
            it.cnt[1] = min(bb, n1) > ba ? min(bb, n1) - ba : 0u;
            it.inner_hi = it.S.hi(at.tok);
            it.inner_lo = it.S.lo(min(at.tok + 2 * p.tokens, it.S.len_q) - 1);
            it.whole = ba == 0 && bb == all;
            it.starts = ba == 0;
            at = {at.kvh, at.seq, at.tok + 2 * p.tokens, 0u};
            if (single) at.kvh = end.kvh + 1;
            return true;
        }
    }
};

// One CTA: the places where `ctas` equal shares of the work start. A pair
// costs its blocks and two more.
constexpr int kPlThreads = 1024;
SMOE_DEVINL uint32_t pl_scan(uint32_t v, uint32_t* sums, uint32_t& all) {      // exclusive sum over the CTA
    const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    uint32_t incl = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const uint32_t x = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= uint32_t(o)) incl += x;
    }
    __syncthreads();
    if (lane == 31) sums[warp] = incl;
    __syncthreads();
    const uint32_t w = sums[lane];
    uint32_t wi = w;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const uint32_t x = __shfl_up_sync(0xffffffffu, wi, o);
        if (lane >= uint32_t(o)) wi += x;
    }
    all = __shfl_sync(0xffffffffu, wi, 31);
    return __shfl_sync(0xffffffffu, wi - w, warp) + incl - v;
}
// cost: [kPaMaxPairs] scratch, the exclusive sums of the pairs' costs; place:
// [kPaMaxPairs] (sequence, token) of each pair. (The host has checked that
// the call cannot have more pairs.) With `list` instead of `plan`: the places
// sorted by their costs, longest first (by 128 keys; those past 1023 such, and
// equal ones, in any order).
__global__ void __launch_bounds__(kPlThreads) k_packed_plan(const PackedArgs p, PaPlace* plan, uint32_t ctas, uint32_t* cost, uint2* place,
                                                            uint2* list) {
    __shared__ uint32_t sums[32], bins[kPlThreads];
    pdl_release();
    pdl_acquire();
    const uint32_t tid = threadIdx.x, span = 2 * p.tokens;
    uint32_t pairs = 0, all;
#pragma unroll 1
    for (uint32_t b = 0; b < p.a.n_seqs; b += kPlThreads) {      // the pairs' places, a thread a sequence
        const uint32_t s = b + tid;
        uint32_t n = 0;
        PackedSeq S{};
        if (s < p.a.n_seqs) {
            S = packed_seq(p.a, s);
            if (S.bad) serve_err(p.err, SMOE_DEVERR_BAD_RANGE);
            n = (S.len_q + span - 1) / span;
        }
        const uint32_t first = pairs + pl_scan(n, sums, all);
        // (one long sequence: its places are written by all threads below)
#pragma unroll 1
        for (uint32_t i = 0; i < min(n, 8u); ++i)
            if (first + i < kPaMaxPairs) place[first + i] = make_uint2(s, i * span);
        uint32_t more = __ballot_sync(0xffffffffu, n > 8);
#pragma unroll 1
        while (more) {
            const int l = __ffs(more) - 1;
            more &= more - 1;
            const uint32_t nn = __shfl_sync(0xffffffffu, n, l), ff = __shfl_sync(0xffffffffu, first, l), ss = __shfl_sync(0xffffffffu, s, l);
#pragma unroll 1
            for (uint32_t i = 8 + (tid & 31); i < nn; i += 32)
                if (ff + i < kPaMaxPairs) place[ff + i] = make_uint2(ss, i * span);
        }
        pairs += all;
    }
    pairs = min(pairs, kPaMaxPairs);
    __syncthreads();
    if (list) {
        bins[tid] = 0;
        __syncthreads();
#pragma unroll 1
        for (uint32_t i = tid; i < pairs; i += kPlThreads) {
            const uint2 at = place[i];
            const PackedSeq S = packed_seq(p.a, at.x);
            const uint32_t n = min(uint32_t(kPlThreads - 1), max(S.blocks(at.y, p.tokens, 0), S.blocks(at.y, p.tokens, 1)) / 2);
            cost[i] = n;
            atomicAdd(&bins[kPlThreads - 1 - n], 1u);
        }
        __syncthreads();
        const uint32_t before = pl_scan(bins[tid], sums, all);
        bins[tid] = before;
        __syncthreads();
#pragma unroll 1
        for (uint32_t i = tid; i < pairs; i += kPlThreads) list[atomicAdd(&bins[kPlThreads - 1 - cost[i]], 1u)] = place[i];
        if (tid == 0) {
            p.taken[0] = 0;
            p.taken[1] = pairs;
        }
        return;
    }
    uint32_t total = 0;                          // (below 2^31: the host bounds it)
#pragma unroll 1
    for (uint32_t b = 0; b < pairs; b += kPlThreads) {
        const uint32_t i = b + tid;
        uint32_t n = 0;
        if (i < pairs) {
            const uint2 at = place[i];
            const PackedSeq S = packed_seq(p.a, at.x);
            n = max(S.blocks(at.y, p.tokens, 0), S.blocks(at.y, p.tokens, 1)) + 2;
        }
        const uint32_t before = total + pl_scan(n, sums, all);
        if (i < pairs) cost[i] = before;
        total += all;
    }
    __syncthreads();
#pragma unroll 1
    for (uint32_t c = tid; c <= ctas; c += kPlThreads) {
        PaPlace at{p.a.num_kv_heads, 0u, 0u, 0u};
        const uint64_t x = uint64_t(total) * p.a.num_kv_heads * c / ctas;
        if (c < ctas && pairs) {
            uint32_t kvh = uint32_t(x / total), y = uint32_t(x % total), lo = 0, hi = pairs - 1;
#pragma unroll 1
            while (lo < hi) {                    // the last pair whose cost starts at or before y
                const uint32_t mid = (lo + hi + 1) / 2;
                if (cost[mid] <= y) lo = mid;
                else hi = mid - 1;
            }
            const uint32_t n = (lo + 1 < pairs ? cost[lo + 1] : total) - cost[lo] - 2, off = y - cost[lo];
            uint32_t blk = off > 1 ? off - 2 : 0u;
            if (blk < 4) blk = 0;                // (no part of few blocks)
            if (n < blk + 4 && blk) {
                blk = 0;
                if (++lo == pairs) lo = 0, ++kvh;
            }
            const uint2 q = place[lo];
            at = {kvh, q.x, q.y, blk};
            if (kvh == p.a.num_kv_heads) at = {kvh, 0u, 0u, 0u};
        }
        plan[c] = at;
    }
}

// Shared-memory descriptors, 128-byte swizzle (rows of 128 bytes, groups of 8
// rows 1024 bytes apart). K-major operands step through K by moving the
// start; for an MN-major one (the values: keys are K, head_dim is N) the
// leading offset is the distance between 64-column halves.
SMOE_DEVINL uint64_t tc_desc_sw128(uint32_t saddr, uint32_t lbo) {
    return uint64_t((saddr >> 4) & 0x3FFFu) | (uint64_t((lbo >> 4) & 0x3FFFu) << 16) | (uint64_t(1024 >> 4) << 32) |
           (uint64_t(1) << 46) | (uint64_t(2) << 61);
}
// kind::f16 with bf16 operands and an fp32 accumulator; bmn: B is MN-major.
__host__ __device__ constexpr uint32_t tc_idesc_bf16(uint32_t m, uint32_t n, uint32_t bmn) {
    return (1u << 4) | (1u << 7) | (1u << 10) | (bmn << 16) | ((n >> 3) << 17) | ((m >> 4) << 24);
}
// D[tmem] (+)= A[tmem] * B[smem]
SMOE_DEVINL void tc_mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
        " tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}\n"
        :: "r"(d), "r"(a), "l"(b), "r"(idesc), "r"(accumulate) : "memory");
}
SMOE_DEVINL void tmem_ld32(uint32_t taddr, float* v) {
    uint32_t r[32];
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
        "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
        "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
          "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
          "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
          "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(taddr));
#pragma unroll
    for (int i = 0; i < 32; ++i) v[i] = __uint_as_float(r[i]);
}
SMOE_DEVINL void tmem_st16(uint32_t taddr, const uint32_t* r) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
        "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};"
        :: "r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
           "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
        : "memory");
}
SMOE_DEVINL float tmem_ld1(uint32_t taddr) {
    uint32_t r;
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x1.b32 {%0}, [%1];\n tcgen05.wait::ld.sync.aligned;"
                 : "=r"(r) : "r"(taddr) : "memory");
    return __uint_as_float(r);
}
SMOE_DEVINL void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
SMOE_DEVINL float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
SMOE_DEVINL uint32_t cvt_bf16x2(float lo, float hi) {
    uint32_t d;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(d) : "f"(hi), "f"(lo));
    return d;
}
// Barriers and words in shared memory by their 32-bit addresses: the softmax
// warps have no register to spare for generic pointers.
struct Bar {
    uint32_t a;
    SMOE_DEVINL Bar operator+(uint32_t i) const { return {a + 8 * i}; }
    SMOE_DEVINL void init(uint32_t count) const { asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" :: "r"(a), "r"(count)); }
    SMOE_DEVINL void arrive() const { asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" :: "r"(a) : "memory"); }
    SMOE_DEVINL void expect(uint32_t bytes) const {
        asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" :: "r"(a), "r"(bytes) : "memory");
    }
    SMOE_DEVINL void commit() const {            // arrives when all products issued so far are done
        asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" :: "r"(a) : "memory");
    }
    SMOE_DEVINL bool try_wait(uint32_t parity) const {
        uint32_t ok;
        asm volatile("{ .reg .pred p; mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2; selp.u32 %0, 1, 0, p; }"
                     : "=r"(ok) : "r"(a), "r"(parity) : "memory");
        return ok != 0;
    }
};
struct Word {
    uint32_t a;
    SMOE_DEVINL Word operator+(uint32_t i) const { return {a + 4 * i}; }
    SMOE_DEVINL uint32_t get() const {
        uint32_t v;
        asm volatile("ld.volatile.shared.u32 %0, [%1];" : "=r"(v) : "r"(a) : "memory");
        return v;
    }
    SMOE_DEVINL void set(uint32_t v) const { asm volatile("st.volatile.shared.u32 [%0], %1;" :: "r"(a), "r"(v) : "memory"); }
};
// A bounded wait, small enough to be inlined at each place (a call would
// bring the calling convention's registers into the softmax warps' budget):
// some tenths of a second of polls. After one ran out, all others of the CTA
// give up within 256; the roles then finish on whatever the buffers hold
// (every address stays in the CTA's own memory) and the error word is set.
constexpr uint32_t kPaPolls = 1u << 24;
SMOE_DEVINL void pa_wait(Bar bar, uint32_t parity, Word fail, uint32_t* err) {
#pragma unroll 1
    for (uint32_t i = 0; !bar.try_wait(parity); ++i)
        if ((i & 255) == 255 && (fail.get() || i >= kPaPolls)) {
            fail.set(1u);
            atomicCAS(err, 0u, uint32_t(SMOE_DEVERR_MBAR_TIMEOUT));
            break;
        }
}
// The same regardless of earlier failures: for copies and products in flight.
SMOE_DEVINL void pa_drain(Bar bar, uint32_t parity) {
#pragma unroll 1
    for (uint32_t i = 0; i < kPaPolls && !bar.try_wait(parity); ++i) {}
}
// No multicast; x (element coordinate) a multiple of 64.
SMOE_DEVINL void tma_load3(uint32_t dst, const CUtensorMap* map, uint32_t x, uint32_t y, uint32_t z, Bar bar) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cta.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];"
        :: "r"(dst), "l"(map), "r"(x), "r"(y), "r"(z), "r"(bar.a) : "memory");
}

template <int HP>
__global__ void __launch_bounds__(kPaThreads, 1)
k_attention_packed(const __grid_constant__ CUtensorMap mq, const __grid_constant__ CUtensorMap mk,
                   const __grid_constant__ CUtensorMap mv, const PackedArgs p) {
    using SM = PackedSmem<HP>;
    constexpr int ST = SM::STAGES, NH = HP / 64;
    constexpr uint32_t TMEM_O = 256;             // columns: S of tile 0, S of tile 1, O of tile 0, O of tile 1
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
    const uint32_t base = smem_u32(smem);
    const Bar qf{base + SM::BAR}, qe = qf + 2, sf = qf + 4, pr = qf + 8, of = qf + 12, itf = qf + 16, ite = itf + kPaItems,
              xb = ite + kPaItems, turn = xb + 3, kvf = turn + 8, kve = kvf + ST;
    const Word fail{(kve + ST).a}, begun = fail + 1, odds = fail + 4;          // begun[t]: the accumulator holds something before block 0's P V; odds: a word of each softmax warp, by turns in two
    uint32_t* const tslot = reinterpret_cast<uint32_t*>(smem + SM::BAR + ((kve + ST).a - qf.a)) + 3;
    PaItem* const items = reinterpret_cast<PaItem*>(smem + SM::ITEMS);
    const uint32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const SmoeCudaPackedAttnArgs& a = p.a;

    pdl_release();
    if (warp == 8 && lane == 0) {
        for (int i = 0; i < 2; ++i) {
            (qf + i).init(1);
            (qe + i).init(1);
        }
        for (int i = 0; i < 4; ++i) {            // sf, pr, of: of tile i / 2, for its even and odd blocks
            (sf + i).init(1);
            (pr + i).init(4);
            (of + i).init(1);
        }
        for (int i = 0; i < kPaItems; ++i) {
            (itf + i).init(1);
            (ite + i).init(11);              // the TMA lane, the MMA lanes, eight softmax warps
        }
        for (int i = 0; i < 3; ++i) (xb + i).init(i < 2 ? 4 : 8);
        for (int i = 0; i < 8; ++i) (turn + i).init(1);
        for (int i = 0; i < ST; ++i) {
            (kvf + i).init(1);
            (kve + i).init(2);               // the MMA lanes
        }
        fail.set(0u);
        begun.set(0u);
        (begun + 1).set(0u);
        fence_mbar_init();
    }
    if (warp == 9) tmem_alloc(tslot, 512);
    pdl_acquire();

    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tslot;
    auto wait = [&](Bar b, uint32_t ph) { pa_wait(b, ph & 1, fail, p.err); };
    // item k, of a role; and done with it
    auto item = [&](uint32_t k) -> const PaItem& {
        wait(itf + k % kPaItems, k / kPaItems);
        return items[k % kPaItems];
    };
    auto item_done = [&](uint32_t k) { (ite + k % kPaItems).arrive(); };
    if (warp == 8) {
        // ---------------------------------------------------- loads (one lane)
        if (elect_one()) {
            uint32_t j = 0, nq[2] = {0u, 0u};    // units sent for, Q tiles sent for
#pragma unroll 1
            for (uint32_t k = 0; !fail.get(); ++k) {
                const PaItem& it = item(k);
                if (!it.more) break;
                const uint32_t m = max(it.cnt[0], it.cnt[1]), kvh = it.kvh, row_q = it.S.q0 + it.tok, row_k = it.S.k0 + it.key0;
                const uint32_t cnt[2] = {it.cnt[0], it.cnt[1]}, head_k = kvh * p.k_step, head_v = kvh * p.v_step;
                item_done(k);
#pragma unroll 1
                for (uint32_t i = 0; i < 2 * m; ++i, ++j) {      // K0 V0 K1 V1 .., the Q tiles around K0
                    if (i < 2 && (i ? cnt[1] : cnt[0])) {
                        const uint32_t q = i ? nq[1]++ : nq[0]++;
                        if (q) wait(qe + i, q - 1);
                        (qf + i).expect(p.group * p.tokens * 128 * NH);
                        for (int h = 0; h < NH; ++h)
                            tma_load3(base + SM::Q + i * SM::TILE + h * 16384, &mq, h * 64, kvh * p.group, row_q + i * p.tokens, qf + i);
                    }
                    const uint32_t st = j % ST, round = j / ST;
                    if (round) wait(kve + st, round - 1);
                    (kvf + st).expect(SM::BLOCK);
                    for (int h = 0; h < NH; ++h)
                        tma_load3(base + SM::KV + st * SM::BLOCK + h * 8192, i & 1 ? &mv : &mk, h * 64, i & 1 ? head_v : head_k, row_k + i / 2 * kPaKeys, kvf + st);
                }
            }
            // nothing may be in flight when the CTA ends (the MMA lanes have
            // waited for all of it unless a wait ran out)
#pragma unroll 1
            for (uint32_t k = j > ST ? j - ST : 0; k < j; ++k) pa_drain(kvf + k % ST, (k / ST) & 1);
            for (int t = 0; t < 2; ++t)
                if (nq[t]) pa_drain(qf + t, (nq[t] - 1) & 1);
        }
    } else if (warp == 9 || warp == 10) {
        // ------------------------------------- MMA (one lane each for the two
        // tiles: a wait or a commit costs a lane some 90 cycles, and with one
        // lane for both the tensor cores stood still for a third of the time)
        if (elect_one()) {
            constexpr uint32_t IQK = tc_idesc_bf16(128, kPaKeys, 0), IPV = tc_idesc_bf16(128, HP, 1);
            const uint32_t t = warp - 9, ts = tmem + t * 128, to = tmem + TMEM_O + t * 128, skv = base + SM::KV;
            const uint64_t qd = tc_desc_sw128(base + SM::Q + t * SM::TILE, 16);
            uint32_t j0 = 0, nq = 0, nb = 0;     // units, Q tiles, blocks of the tile so far
            auto qk = [&](uint32_t st, uint32_t n, bool last) {  // scores of the tile's block n
                const uint64_t kd = tc_desc_sw128(skv + st * SM::BLOCK, 16);
#pragma unroll
                for (int s = 0; s < HP / 16; ++s)
                    tc_mma_f16(ts + n % 2 * 64, qd + ((s / 4 * 16384 + s % 4 * 32) >> 4), kd + ((s / 4 * 8192 + s % 4 * 32) >> 4), IQK, s > 0);
                (sf + t * 2 + n % 2).commit();
                if (last) (qe + t).commit();     // the tile's Q has been read
            };
            auto pv = [&](uint32_t st, uint32_t n, bool more) {
                const uint64_t vd = tc_desc_sw128(skv + st * SM::BLOCK, 8192);
#pragma unroll
                for (int s = 0; s < int(kPaKeys) / 16; ++s)
                    tc_mma_ts(to, ts + n % 2 * 64 + s * 8, vd + ((s * 2048) >> 4), IPV, more || s > 0);
                (of + t * 2 + n % 2).commit();
            };
#pragma unroll 1
            for (uint32_t k = 0; !fail.get(); ++k) {
                const PaItem& it = item(k);
                if (!it.more) break;
                const uint32_t nt = it.cnt[t], m = max(it.cnt[0], it.cnt[1]);
                item_done(k);
#pragma unroll 1
                for (uint32_t i = 0; i < min(m, 2u); ++i) {      // the first two blocks' scores
                    const uint32_t jk = j0 + 2 * i;
                    wait(kvf + jk % ST, jk / ST);    // (all of them in turn: a phase skipped could be taken for another)
                    if (i < nt) {
                        if (i == 0) wait(qf + t, nq++);
                        tc_fence_after();
                        qk(jk % ST, nb + i, i + 1 == nt);
                    }
                    (kve + jk % ST).commit();
                }
#pragma unroll 1
                for (uint32_t i = 0; i < m; ++i) {
                    const uint32_t jv = j0 + 2 * i + 1, jk = jv + 3, sv = jv % ST, sk = jk % ST;
                    wait(kvf + sv, jv / ST);
                    if (i < nt) {
                        // (of an item's first block this also says that the
                        // softmax warps have read the last item's sums)
                        wait(pr + t * 2 + nb % 2, nb / 2);
                        tc_fence_after();
                        pv(sv, nb, i > 0 || (begun + t).get());
                    }
                    (kve + sv).commit();
                    if (i + 2 < m) wait(kvf + sk, jk / ST);
                    if (i + 2 < nt) {
                        tc_fence_after();
                        qk(sk, nb, i + 3 == nt); // (where the block's probabilities were)
                    }
                    if (i + 2 < m) (kve + sk).commit();
                    nb += i < nt;
                }
                j0 += 2 * m;
            }
            if (j0) pa_drain(kve + (j0 - 1) % ST, ((j0 - 1) / ST) & 1);                // all MMAs done: the last commit
        }
    } else if (warp == 11) {
        // ------------------------------------------------------------- items
        PaWalk walk;
        walk.single = !p.plan;
        uint32_t pairs = 0;
        if (p.list) {
            pairs = ld_plain(p.taken + 1);
        } else if (p.plan) {
            walk.at = p.plan[blockIdx.x];
            walk.end = p.plan[blockIdx.x + 1];
        } else {
            // The CTA's tile pair, counted from the last one backwards: later
            // tokens have more keys, so long tiles start first. One lane a sequence.
            const uint32_t kvh = blockIdx.x % a.num_kv_heads, me = blockIdx.x / a.num_kv_heads, span = 2 * p.tokens;
            auto count = [&](uint32_t s) -> uint32_t {
                if (s >= a.n_seqs) return 0u;
                const PackedSeq S = packed_seq(a, s);
                if (S.bad && blockIdx.x == 0) serve_err(p.err, SMOE_DEVERR_BAD_RANGE);
                return (S.len_q + span - 1) / span;
            };
            uint32_t total = 0, seq = a.n_seqs, tok = 0, n = 0, before = 0;
#pragma unroll 1
            for (uint32_t b = 0; b < a.n_seqs; b += 32) total += __reduce_add_sync(0xffffffffu, n = count(b + lane));
            const uint32_t want = total - 1 - me;
#pragma unroll 1
            for (uint32_t b = 0; b < a.n_seqs && me < total && before <= want; b += 32) {
                if (a.n_seqs > 32) n = count(b + lane);          // (else they are still at hand)
                uint32_t incl = n;
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) {
                    const uint32_t v = __shfl_up_sync(0xffffffffu, incl, o);
                    if (lane >= uint32_t(o)) incl += v;
                }
                const uint32_t first = before + incl - n, hit = __ballot_sync(0xffffffffu, want >= first && want < first + n);
                if (hit) {
                    seq = b + __ffs(hit) - 1;
                    tok = __shfl_sync(0xffffffffu, (want - first) * span, __ffs(hit) - 1);
                }
                before += __shfl_sync(0xffffffffu, incl, 31);
            }
            walk.at = {kvh, seq, tok, 0u};
            walk.end = walk.at;
            if (seq >= a.n_seqs) walk.at.kvh = kvh + 1;          // past the last pair
        }
        if (elect_one()) {
            bool more = true;
#pragma unroll 1
            for (uint32_t k = 0; more && !fail.get(); ++k) {
                PaItem it{};
                if (k >= kPaItems) wait(ite + k % kPaItems, k / kPaItems - 1);
                if (p.list) {
                    const uint32_t i = atomicAdd(p.taken, 1u), pair = i / a.num_kv_heads;
                    const uint2 q = pair < pairs ? ld_plain(p.list + pair) : make_uint2(0u, 0u);
                    walk.at = {i % a.num_kv_heads, q.x, q.y, 0u};
                    walk.end = walk.at;
                    if (pair >= pairs) walk.at.kvh = walk.end.kvh + 1;
                }
                more = walk.next(p, it);
                it.more = more;
                items[k % kPaItems] = it;
                (itf + k % kPaItems).arrive();
            }
        }
    } else {
        // ----------------------------------------------------------- softmax
        // One thread a row. The reference maximum is only moved when the
        // running one is more than 8 (in log2) above it, so the
        // accumulator is rarely rescaled; probabilities stay below 2^8.
        const uint32_t t = warp >> 2, r = tid & 127;
        const uint32_t ts = tmem + t * 128 + ((warp & 3) << 21), to = tmem + TMEM_O + t * 128 + ((warp & 3) << 21);
        const float sl = p.scale_log2;
        const uint32_t tk = r / p.group, hd = r % p.group;       // the row's token of the tile and head of the group
        uint32_t j0 = 0, nb = 0;                 // units and this tile's blocks so far
        // A meeting of this tile's four warps, or of both tiles' eight. (An
        // mbarrier and not a named one, so that the wait is bounded.)
        uint32_t met[2] = {0u, 0u};
        auto meet = [&](bool all) {
            const uint32_t x = all ? 2u : t, turn = all ? met[1]++ : met[0]++;
            __syncwarp();
            if (lane == 0) (xb + x).arrive();
            wait(xb + x, turn);
            __syncwarp();
        };
        // The exponentials by turns with the warp of the other tile that has the
        // same scheduler, tile 0 first.
        const Bar mine_b = turn + warp, yours_b = turn + (warp ^ 4);
        auto await = [&](uint32_t u) {
            if (t) wait(mine_b, u);
            else if (u) wait(mine_b, u - 1);
        };
        auto pass = [&] {
            if (lane == 0) yours_b.arrive();
        };
#pragma unroll 1
        for (uint32_t k = 0;; ++k) {
            const PaItem& im = item(k);
            if (__any_sync(0xffffffffu, fail.get() || !im.more)) break;
            const uint32_t nt = im.cnt[t];
            const bool live = r < p.group * p.tokens && im.tok + t * p.tokens + tk < im.S.len_q;
            float m = -INFINITY, l = 0.0f;
            if (nt) {
                const uint32_t last = min(im.tok + (t + 1) * p.tokens, im.S.len_q) - 1, mine = min(im.tok + t * p.tokens + tk, last);
                const uint32_t lo = im.S.lo(mine), hi = im.S.hi(mine), first_key = im.key0, cnt_o = im.cnt[t ^ 1];
                const uint32_t inner_hi = im.inner_hi, inner_lo = im.inner_lo;
#pragma unroll 1
                for (uint32_t i = 0; i < nt; ++i) {
                    const uint32_t key0 = first_key + i * kPaKeys, jv = j0 + 2 * i + 1;
                    const bool masked = key0 + kPaKeys > inner_hi || key0 < inner_lo, both = i < cnt_o;   // some row of the pair may not see some key of the block
                    const uint32_t ja = lo > key0 ? lo - key0 : 0u, jb = hi > key0 ? hi - key0 : 0u;       // columns [ja, jb)
                    uint4* const vt = reinterpret_cast<uint4*>(smem + SM::KV + jv % ST * SM::BLOCK);
                    const uint32_t n = nb + i, tp = ts + n % 2 * 64;             // the block's scores, and then its probabilities
                    float x[kPaKeys];
                    wait(sf + t * 2 + n % 2, n / 2);
                    tc_fence_after();
                    tmem_ld32(tp, x);
                    tmem_ld32(tp + 32, x + 32);
                    tmem_ld_wait();
                    if (masked) {
#pragma unroll
                        for (int c = 0; c < 2; ++c) {            // bits of the 32 columns in [ja, jb)
                            auto below = [](uint32_t n) { return n >= 32 ? 0xffffffffu : (1u << n) - 1u; };
                            const uint32_t from = ja > c * 32u ? ja - c * 32u : 0u, to_ = jb > c * 32u ? jb - c * 32u : 0u, open = below(to_) & ~below(from);
#pragma unroll
                            for (int j = 0; j < 32; ++j)
                                if (!(open >> j & 1u)) x[c * 32 + j] = -INFINITY;
                        }
                    }
                    float mq[8];                 // eight chains: the maximum's latency is the softmax warps' to wait for
#pragma unroll
                    for (int j = 0; j < 8; ++j) mq[j] = fmaxf(x[2 * j], x[2 * j + 1]);
#pragma unroll
                    for (int j = 16; j < int(kPaKeys); j += 2) mq[j / 2 % 8] = fmaxf(fmaxf(mq[j / 2 % 8], x[j]), x[j + 1]);
#pragma unroll
                    for (int w = 4; w; w >>= 1)
#pragma unroll
                        for (int j = 0; j < w; ++j) mq[j] = fmaxf(mq[j], mq[j + w]);
                    const float mx = fmaxf(m, mq[0]);
                    // (each row for itself - a factor of 1 leaves the others of the
                    // warp as they are - so a row's bits do not depend on its neighbours)
                    const bool move = live && ((mx - m) * sl > 8.0f || (mx > m && m == -INFINITY));
                    if (__any_sync(0xffffffffu, move)) {
                        const float f = !move ? 1.0f : m == -INFINITY ? 0.0f : ex2((m - mx) * sl);
                        if (i) {
                            wait(of + t * 2 + (n - 1) % 2, (n - 1) / 2);
                            tc_fence_after();
#pragma unroll 1
                            for (int c = 0; c < HP; c += 16) {
                                float o[16];
                                uint32_t w[16];
                                tmem_ld16(to + c, o);
                                tmem_ld_wait();
#pragma unroll
                                for (int k = 0; k < 16; ++k) w[k] = __float_as_uint(o[k] * f);
                                tmem_st16(to + c, w);
                            }
                        }
                        l *= f;
                        if (move) m = mx;
                    }
                    // A zero probability does not silence an infinity or NaN
                    // among the values in the matrix product, and a masked block
                    // has keys that not every row may see: was there one?
                    bool odd = false;
                    if (masked) {
                        wait(kvf + jv % ST, jv / ST);            // (its scores are there: the stage's earlier loads are long done)
                        const __nv_bfloat162 zero = __float2bfloat162_rn(0.0f);
                        __nv_bfloat162 acc[4] = {zero, zero, zero, zero};
#pragma unroll 4
                        for (uint32_t q = r; q < SM::BLOCK / 16; q += 128) {     // 0 times one of those is a NaN
                            const uint4 v = vt[q];
                            acc[0] = __hfma2(*reinterpret_cast<const __nv_bfloat162*>(&v.x), zero, acc[0]);
                            acc[1] = __hfma2(*reinterpret_cast<const __nv_bfloat162*>(&v.y), zero, acc[1]);
                            acc[2] = __hfma2(*reinterpret_cast<const __nv_bfloat162*>(&v.z), zero, acc[2]);
                            acc[3] = __hfma2(*reinterpret_cast<const __nv_bfloat162*>(&v.w), zero, acc[3]);
                        }
                        const __nv_bfloat162 all = __hadd2(__hadd2(acc[0], acc[1]), __hadd2(acc[2], acc[3]));
                        const bool mine = __any_sync(0xffffffffu, __hisnan(all.x) || __hisnan(all.y));
                        const Word w = odds + (met[0] & 1) * 8 + t * 4;
                        if (lane == 0) (w + (warp & 3)).set(mine);
                        meet(false);
                        odd = (w + 0).get() | (w + 1).get() | (w + 2).get() | (w + 3).get();
                    }
                    const float ml = m == -INFINITY ? 0.0f : m * sl;
                    const uint64_t sl2 = pack2(sl, sl), ml2 = pack2(-ml, -ml);
                    uint64_t sums[2] = {0ull, 0ull};
                    await(j0 / 2 + i);
                    if (i == 0 && r == 0) (begun + t).set(odd);        // the product then adds to what the rows put there
#pragma unroll
                    for (int c = 0; c < 2; ++c) {
                        uint32_t w[16];
#pragma unroll
                        for (int k = 0; k < 16; ++k) {
                            float u, v;
                            unpack2(fma2(pack2(x[c * 32 + 2 * k], x[c * 32 + 2 * k + 1]), sl2, ml2), u, v);
                            u = ex2(u);
                            v = ex2(v);
                            sums[k % 2] = add2(sums[k % 2], pack2(u, v));
                            w[k] = cvt_bf16x2(u, v);
                        }
                        if (c == 1) pass();
                        tmem_st16(tp + c * 16, w);               // (over scores that have been read)
                    }
                    if (odd) {
                        // Rare. Each row adds its own share of the infinities and
                        // NaN to its accumulator; then they are zeroed in the
                        // shared tile, for both tiles' products.
                        tmem_st_wait();
                        if (i) {
                            wait(of + t * 2 + (n - 1) % 2, (n - 1) / 2);
                            tc_fence_after();
                        }
#pragma unroll 1
                        for (int c = 0; c < HP; c += 16) {
                            float o[16];
                            if (i) {
                                tmem_ld16(to + c, o);
                                tmem_ld_wait();
                            } else {
#pragma unroll
                                for (int k = 0; k < 16; ++k) o[k] = 0.0f;
                            }
#pragma unroll 1
                            for (uint32_t j = 0; j < kPaKeys; ++j) {
                                const uint32_t pp = __float_as_uint(tmem_ld1(tp + j / 2));
                                const float x = __uint_as_float(j & 1 ? pp & 0xffff0000u : pp << 16);
                                if (j < ja || j >= jb) continue;
#pragma unroll
                                for (int h = 0; h < 2; ++h) {    // 8 columns: one swizzled 16-byte piece of key j's row
                                    const uint4 v = vt[c / 64 * 512 + j * 8 + (((c % 64) / 8 + h) ^ (j & 7))];
                                    const uint32_t vs[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
                                    for (int k = 0; k < 4; ++k) {
                                        const float va = __uint_as_float(vs[k] << 16), vb = __uint_as_float(vs[k] & 0xffff0000u);
                                        if (!isfinite(va)) o[h * 8 + 2 * k] = fmaf(x, va, o[h * 8 + 2 * k]);
                                        if (!isfinite(vb)) o[h * 8 + 2 * k + 1] = fmaf(x, vb, o[h * 8 + 2 * k + 1]);
                                    }
                                }
                            }
                            uint32_t w[16];
#pragma unroll
                            for (int k = 0; k < 16; ++k) w[k] = __float_as_uint(o[k]);
                            tmem_st16(to + c, w);
                        }
                        meet(both);  // all rows of both tiles have read them
#pragma unroll 1
                        for (uint32_t k = both ? tid : r; k < SM::BLOCK / 16; k += both ? 256 : 128) {
                            uint4 x = vt[k];
                            uint32_t xs[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
                            for (int q = 0; q < 4; ++q) {
                                if ((xs[q] & 0x7f80u) == 0x7f80u) xs[q] &= 0xffff0000u;
                                if ((xs[q] & 0x7f800000u) == 0x7f800000u) xs[q] &= 0x0000ffffu;
                            }
                            vt[k] = make_uint4(xs[0], xs[1], xs[2], xs[3]);
                        }
                        fence_proxy_async();     // the tensor core reads what these threads wrote
                        meet(both);
                    }
                    float sum_x, sum_y;
                    unpack2(add2(sums[0], sums[1]), sum_x, sum_y);
                    l += sum_x + sum_y;
                    tmem_st_wait();
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) (pr + t * 2 + n % 2).arrive();
                }
                nb += nt;
            }
            for (uint32_t i = nt; i < im.cnt[t ^ 1]; ++i) {
                await(j0 / 2 + i);
                pass();
            }
            j0 += 2 * max(im.cnt[0], im.cnt[1]);
            // Rows go out through shared memory, 128 bytes of each at a time:
            // eight lanes a row, four whole lines an instruction (a thread
            // storing its own row touches 32 lines with each).
            const uint32_t token = im.tok + t * p.tokens + tk, head = im.kvh * p.group + hd;
            const bool whole = im.whole, keys = live && im.S.hi(token) > im.S.lo(token);
            uint4* const out = reinterpret_cast<uint4*>(smem + SM::OUT) + warp * 256;
            const uint32_t row = lane / 8, piece = lane % 8;
            uint8_t* dst;
            if (whole) {
                const float inv = keys ? 1.0f / l : 0.0f;
                dst = live ? reinterpret_cast<uint8_t*>(a.out + uint64_t(im.S.q0 + token) * a.out_row + uint64_t(head) * a.out_head) : nullptr;
                if (a.lse && live)
                    a.lse[uint64_t(im.S.q0 + token) * a.num_heads + head] = keys ? m * a.scale + logf(l) : -INFINITY;
                l = inv;
            } else {
                // a part: 2 * CTA when it continues a pair (or is the CTA's only one), 2 * CTA + 1 when it starts one
                const uint64_t at = (uint64_t(2 * blockIdx.x + im.starts) * 2 + t) * 128 + r;
                dst = nt ? reinterpret_cast<uint8_t*>(p.part + at * HP) : nullptr;
                p.stat[at] = make_float2(m, nt ? l : 0.0f);
            }
            if (nt) {
                wait(of + t * 2 + (nb - 1) % 2, (nb - 1) / 2);
                tc_fence_after();
            }
            const uint32_t row_bytes = whole ? a.head_dim * 2 : HP * 4;
#pragma unroll 1
            for (uint32_t c = 0; c * 128 < row_bytes; ++c) {     // 64 columns of the result, or 32 of a part
                __syncwarp();                    // (the last round's have been read)
#pragma unroll 1
                for (uint32_t h = 0; h < (whole ? 2u : 1u); ++h) {
                    float o[32];
                    if (nt) {
                        tmem_ld32(to + (whole ? c * 64 + h * 32 : c * 32), o);
                        tmem_ld_wait();
                    }
                    if (whole) {
#pragma unroll
                        for (uint32_t k = 0; k < 4; ++k)
                            out[lane * 8 + ((h * 4 + k) ^ (lane & 7))] =
                                keys ? make_uint4(cvt_bf16x2(o[8 * k] * l, o[8 * k + 1] * l), cvt_bf16x2(o[8 * k + 2] * l, o[8 * k + 3] * l),
                                                  cvt_bf16x2(o[8 * k + 4] * l, o[8 * k + 5] * l), cvt_bf16x2(o[8 * k + 6] * l, o[8 * k + 7] * l))
                                     : make_uint4(0u, 0u, 0u, 0u);
                    } else if (nt) {
#pragma unroll
                        for (uint32_t k = 0; k < 8; ++k)
                            out[lane * 8 + (k ^ (lane & 7))] =
                                make_uint4(__float_as_uint(o[4 * k]), __float_as_uint(o[4 * k + 1]), __float_as_uint(o[4 * k + 2]), __float_as_uint(o[4 * k + 3]));
                    }
                }
                __syncwarp();
                const uint32_t byte = c * 128 + piece * 16;
#pragma unroll
                for (uint32_t g = 0; g < 8; ++g) {
                    const uint32_t from = g * 4 + row;
                    uint8_t* const at = reinterpret_cast<uint8_t*>(__shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(dst), from));
                    const uint4 w = out[from * 8 + (piece ^ (from & 7))];
                    if (at && byte < row_bytes) *reinterpret_cast<uint4*>(at + byte) = w;
                }
            }
            tc_fence_before();                   // (the sums have been read: the next pr says so)
            __syncwarp();
            if (lane == 0) item_done(k);
        }
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (warp == 9) tmem_dealloc(tmem, 512);
}

// The parts of the cut pairs. grid (CTAs of the attention, 8): block (c, y)
// does 32 of the 256 rows of the pair that CTA c is the first to continue:
// CTA c - 1 has its first part, c, c + 1, .. the others. A warp does four rows
// side by side, eight lanes a row.
template <int HP>
__global__ void __launch_bounds__(256) k_packed_join(const PackedArgs p) {
    __shared__ uint32_t list[1024];              // the parts' numbers (more CTAs than that no GPU has SMs for)
    __shared__ uint32_t parts;
    pdl_release();
    pdl_acquire();
    const SmoeCudaPackedAttnArgs& a = p.a;
    const uint32_t c = blockIdx.x, tid = threadIdx.x;
    const PaPlace at = p.plan[c], before = p.plan[c ? c - 1 : 0];
    auto same = [&](const PaPlace& x) { return x.kvh == at.kvh && x.seq == at.seq && x.tok == at.tok; };
    if (c == 0 || at.blk == 0 || (same(before) && before.blk)) return;         // (an earlier CTA continues it, too)
    if (tid == 0) {
        uint32_t n = 0;
        list[n++] = 2 * (c - 1) + 1;
        PaPlace x = at;
#pragma unroll 1
        for (uint32_t e = c; e < gridDim.x && same(x) && n < 1024; ++e) {
            const PaPlace y = p.plan[e + 1];
            if (!(same(y) && y.blk == x.blk)) list[n++] = 2 * e;               // (a CTA whose share is empty has written nothing)
            x = y;
        }
        parts = n;
    }
    __syncthreads();
    const PackedSeq S = packed_seq(a, at.seq);
    const uint32_t row = blockIdx.y * 32 + tid / 8, t = row / 128, r = row % 128, q = tid % 8, n = parts;
    const uint32_t token = at.tok + t * p.tokens + r / p.group, head = at.kvh * p.group + r % p.group;
    if (r >= p.group * p.tokens || token >= S.len_q) return;
    constexpr int V = HP / 32;                   // four columns a lane, V times
    float mx = -INFINITY, l = 0.0f;
    float4 o[V];
#pragma unroll
    for (int v = 0; v < V; ++v) o[v] = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
    for (uint32_t i = 0; i < n; ++i) mx = fmaxf(mx, p.stat[(uint64_t(list[i]) * 2 + t) * 128 + r].x);
#pragma unroll 2
    for (uint32_t i = 0; i < n; ++i) {
        const uint64_t src = (uint64_t(list[i]) * 2 + t) * 128 + r;
        const float2 st = p.stat[src];
        const bool none = st.x == -INFINITY && st.y == 0.0f;     // no key in this part (its sums may not be written)
        const float f = none ? 0.0f : st.x == -INFINITY ? 1.0f : ex2((st.x - mx) * p.scale_log2);     // (-inf scores alone: NaN stays)
        l = fmaf(st.y, f, l);
#pragma unroll
        for (int v = 0; v < V; ++v) {
            if (none) continue;
            const float4 x = *reinterpret_cast<const float4*>(p.part + src * HP + v * 32 + q * 4);
            o[v].x = fmaf(x.x, f, o[v].x);
            o[v].y = fmaf(x.y, f, o[v].y);
            o[v].z = fmaf(x.z, f, o[v].z);
            o[v].w = fmaf(x.w, f, o[v].w);
        }
    }
    const bool keys = S.hi(token) > S.lo(token);
    const float inv = keys ? 1.0f / l : 0.0f;
    uint16_t* dst = a.out + uint64_t(S.q0 + token) * a.out_row + uint64_t(head) * a.out_head;
#pragma unroll
    for (int v = 0; v < V; ++v)
        if (v * 32 + q * 4 < a.head_dim)         // (head_dim is a multiple of 8)
            *reinterpret_cast<uint2*>(dst + v * 32 + q * 4) = keys ? make_uint2(cvt_bf16x2(o[v].x * inv, o[v].y * inv), cvt_bf16x2(o[v].z * inv, o[v].w * inv))
                                                                   : make_uint2(0u, 0u);
    if (a.lse && q == 0) a.lse[uint64_t(S.q0 + token) * a.num_heads + head] = keys ? mx * a.scale + logf(l) : -INFINITY;
}

}  // namespace smoe
