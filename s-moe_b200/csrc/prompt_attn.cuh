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
// other's softmax runs) and walks the keys 128 at a time.
//
// Small calls run a CTA per tile pair. Otherwise there is one CTA an SM, which
// goes from pair to pair with the next one's loads in flight:
//  - many pairs: each CTA takes the next one from a list, the longest first
//    (k_packed_plan sorts it). CTAs that run side by side then walk the same
//    keys at the same time, which the L2 serves them together - with shares
//    of neighbouring pairs instead, 16,384 tokens took 1.18 times as long;
//  - few pairs: each CTA takes an equal share of the line of all pairs' key
//    blocks, and the parts of a pair that is cut are joined by k_packed_join.
constexpr uint32_t kPaRows = 128, kPaKeys = 128;
constexpr int kPaThreads = 384;                  // 2 x 4 softmax warps; TMA warp, MMA warp, the items' warp and an idle one (a register split goes by four)
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
    static constexpr int STAGES = HP == 128 ? 5 : 8;
    static constexpr uint32_t Q = 0, KV = 2 * TILE, BAR = KV + STAGES * TILE, ITEMS = BAR + 384, END = ITEMS + kPaItems * 64;
    static constexpr uint32_t bytes() { return END + 1024; }     // the base is rounded up to 1024
};

// Keys [lo, hi) of a token at index i of its sequence.
struct PackedSeq {
    uint32_t q0, k0, len_q, len_k, causal, window;
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
    return {q0, k0, ok ? q1 - q0 : 0u, ok ? k1 - k0 : 0u, a.causal, a.window};
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
// costs its blocks and one more.
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
// sorted by their costs, longest first (those past 1023 blocks, and equal
// ones, in any order).
__global__ void __launch_bounds__(kPlThreads) k_packed_plan(const PackedArgs p, PaPlace* plan, uint32_t ctas, uint32_t* cost, uint2* place,
                                                            uint2* list) {
    __shared__ uint32_t sums[32], bins[kPlThreads];
    pdl_release();
    pdl_acquire();
    const uint32_t tid = threadIdx.x, span = 2 * p.tokens;
    uint32_t pairs = 0, all;
    for (uint32_t b = 0; b < p.a.n_seqs; b += kPlThreads) {      // the pairs' places, a thread a sequence
        const uint32_t s = b + tid;
        uint32_t n = 0;
        PackedSeq S{};
        if (s < p.a.n_seqs) {
            S = packed_seq(p.a, s);
            const uint32_t* ck = p.a.cu_k ? p.a.cu_k : p.a.cu_q;
            if (S.len_q != ld_plain(p.a.cu_q + s + 1) - S.q0 || S.len_k != ld_plain(ck + s + 1) - S.k0) serve_err(p.err, SMOE_DEVERR_BAD_RANGE);
            n = (S.len_q + span - 1) / span;
        }
        const uint32_t first = pairs + pl_scan(n, sums, all);
        // (one long sequence: its places are written by all threads below)
        for (uint32_t i = 0; i < min(n, 8u); ++i)
            if (first + i < kPaMaxPairs) place[first + i] = make_uint2(s, i * span);
        uint32_t more = __ballot_sync(0xffffffffu, n > 8);
        while (more) {
            const int l = __ffs(more) - 1;
            more &= more - 1;
            const uint32_t nn = __shfl_sync(0xffffffffu, n, l), ff = __shfl_sync(0xffffffffu, first, l), ss = __shfl_sync(0xffffffffu, s, l);
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
        for (uint32_t i = tid; i < pairs; i += kPlThreads) {
            const uint2 at = place[i];
            const PackedSeq S = packed_seq(p.a, at.x);
            const uint32_t n = min(uint32_t(kPlThreads - 1), max(S.blocks(at.y, p.tokens, 0), S.blocks(at.y, p.tokens, 1)));
            cost[i] = n;
            atomicAdd(&bins[kPlThreads - 1 - n], 1u);
        }
        __syncthreads();
        const uint32_t before = pl_scan(bins[tid], sums, all);
        bins[tid] = before;
        __syncthreads();
        for (uint32_t i = tid; i < pairs; i += kPlThreads) list[atomicAdd(&bins[kPlThreads - 1 - cost[i]], 1u)] = place[i];
        if (tid == 0) {
            p.taken[0] = 0;
            p.taken[1] = pairs;
        }
        return;
    }
    uint32_t total = 0;                          // (below 2^31: the host bounds it)
    for (uint32_t b = 0; b < pairs; b += kPlThreads) {
        const uint32_t i = b + tid;
        uint32_t n = 0;
        if (i < pairs) {
            const uint2 at = place[i];
            const PackedSeq S = packed_seq(p.a, at.x);
            n = max(S.blocks(at.y, p.tokens, 0), S.blocks(at.y, p.tokens, 1)) + 1;
        }
        const uint32_t before = total + pl_scan(n, sums, all);
        if (i < pairs) cost[i] = before;
        total += all;
    }
    __syncthreads();
    for (uint32_t c = tid; c <= ctas; c += kPlThreads) {
        PaPlace at{p.a.num_kv_heads, 0u, 0u, 0u};
        const uint64_t x = uint64_t(total) * p.a.num_kv_heads * c / ctas;
        if (c < ctas && pairs) {
            uint32_t kvh = uint32_t(x / total), y = uint32_t(x % total), lo = 0, hi = pairs - 1;
            while (lo < hi) {                    // the last pair whose cost starts at or before y
                const uint32_t mid = (lo + hi + 1) / 2;
                if (cost[mid] <= y) lo = mid;
                else hi = mid - 1;
            }
            const uint32_t n = (lo + 1 < pairs ? cost[lo + 1] : total) - cost[lo] - 1, off = y - cost[lo];
            uint32_t blk = off > 0 ? off - 1 : 0u;
            if (blk < 2) blk = 0;                // (no part of a single block)
            if (n < blk + 2 && blk) {
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
// No multicast; x (element coordinate) a multiple of 64.
SMOE_DEVINL void tma_load3(void* dst, const CUtensorMap* map, uint32_t x, uint32_t y, uint32_t z, uint64_t* bar) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cta.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];"
        :: "r"(smem_u32(dst)), "l"(map), "r"(x), "r"(y), "r"(z), "r"(smem_u32(bar)) : "memory");
}
SMOE_DEVINL float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// Two fp32 operations in one instruction.
SMOE_DEVINL uint64_t pack2(float a, float b) {
    uint64_t d;
    asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "f"(a), "f"(b));
    return d;
}
SMOE_DEVINL void unpack2(uint64_t x, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(x)); }
SMOE_DEVINL uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
    return d;
}
SMOE_DEVINL uint64_t add2(uint64_t a, uint64_t b) {
    uint64_t d;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}
SMOE_DEVINL uint32_t cvt_bf16x2(float lo, float hi) {
    uint32_t d;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(d) : "f"(hi), "f"(lo));
    return d;
}
// (Inlined: a call would bring the calling convention's registers into the
// softmax warps' budget.) A bounded wait: after one ran out, all others of the CTA return at once.
// The roles then finish their loops on whatever the buffers hold (every
// address stays in the CTA's own memory) and the error word is set.
SMOE_DEVINL void pa_wait_slow(uint64_t* bar, uint32_t parity, volatile uint32_t* fail, uint32_t* err) {
    const uint64_t end = gtimer() + SMOE_WAIT_NS_DEFAULT;
#pragma unroll 1
    for (uint32_t i = 0; i < SMOE_SPIN_LIMIT; ++i) {
        if (mbar_try_wait(bar, parity)) return;
        if ((i & 15) == 15 && (*fail || gtimer() > end)) break;
    }
    *fail = 1u;
    atomicCAS(err, 0u, uint32_t(SMOE_DEVERR_MBAR_TIMEOUT));
}

// The same regardless of earlier failures: for copies and products in flight.
SMOE_DEVINL void pa_drain(uint64_t* bar, uint32_t parity) {
    const uint64_t end = gtimer() + SMOE_WAIT_NS_DEFAULT;
#pragma unroll 1
    for (uint32_t i = 0; i < SMOE_SPIN_LIMIT; ++i)
        if (mbar_try_wait(bar, parity) || ((i & 15) == 15 && gtimer() > end)) return;
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
    uint64_t* bars = reinterpret_cast<uint64_t*>(smem + SM::BAR);
    uint64_t *qf = bars, *qe = bars + 2, *sf = bars + 4, *pr = bars + 6, *of = bars + 8, *itf = bars + 10, *ite = itf + kPaItems, *xb = ite + kPaItems, *kvf = xb + 3, *kve = kvf + ST;
    uint32_t* words = reinterpret_cast<uint32_t*>(kve + ST);
    PaItem* items = reinterpret_cast<PaItem*>(smem + SM::ITEMS);
    volatile uint32_t *fail = words, *begun = words + 1;         // begun[t]: the accumulator holds something before block 0's P V
    uint32_t* tslot = words + 3;
    volatile uint32_t* xflag = words + 6;                        // [3 meetings of softmax warps][3 turns] somebody said yes
    uint32_t* where = words + 4;                                 // without a plan: the CTA's sequence and first token
    const uint32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const SmoeCudaPackedAttnArgs& a = p.a;

    pdl_release();
    if (warp == 8 && lane == 0) {
        for (int i = 0; i < 2; ++i) {
            mbar_init(qf + i, 1);
            mbar_init(qe + i, 1);
            mbar_init(sf + i, 1);
            mbar_init(pr + i, 4);
            mbar_init(of + i, 1);
        }
        for (int i = 0; i < kPaItems; ++i) {
            mbar_init(itf + i, 1);
            mbar_init(ite + i, 10);              // the TMA lane, the MMA lane, eight softmax warps
        }
        for (int i = 0; i < 3; ++i) mbar_init(xb + i, i < 2 ? 4 : 8);
        for (int i = 0; i < 9; ++i) xflag[i] = 0u;
        for (int i = 0; i < ST; ++i) {
            mbar_init(kvf + i, 1);
            mbar_init(kve + i, 1);
        }
        *fail = begun[0] = begun[1] = 0u;
        fence_mbar_init();
    }
    if (warp == 9) tmem_alloc(tslot, 512);
    pdl_acquire();

    PaWalk walk;
    walk.single = !p.plan;
    if (p.list) {
    } else if (p.plan) {
        walk.at = p.plan[blockIdx.x];
        walk.end = p.plan[blockIdx.x + 1];
    } else {
        // The CTA's tile pair, counted from the last one backwards: later
        // tokens have more keys, so long tiles start first. One lane per sequence.
        const uint32_t kvh = blockIdx.x % a.num_kv_heads, span = 2 * p.tokens;
        if (warp == 0) {
            uint32_t total = 0;
            auto pairs = [&](uint32_t s) -> uint32_t {
                if (s >= a.n_seqs) return 0u;
                const PackedSeq S = packed_seq(a, s);
                const uint32_t* ck = a.cu_k ? a.cu_k : a.cu_q;
                if (blockIdx.x == 0 && (S.len_q != ld_plain(a.cu_q + s + 1) - S.q0 || S.len_k != ld_plain(ck + s + 1) - S.k0))
                    serve_err(p.err, SMOE_DEVERR_BAD_RANGE);
                return (S.len_q + span - 1) / span;
            };
            for (uint32_t b = 0; b < a.n_seqs; b += 32) total += __reduce_add_sync(0xffffffffu, pairs(b + lane));
            const uint32_t me = blockIdx.x / a.num_kv_heads;
            if (lane == 0) where[0] = a.n_seqs;
            __syncwarp();
            if (me < total) {
                uint32_t want = total - 1 - me, before = 0;
                for (uint32_t b = 0; b < a.n_seqs; b += 32) {
                    const uint32_t n = pairs(b + lane);
                    uint32_t incl = n;
#pragma unroll
                    for (int o = 1; o < 32; o <<= 1) {
                        const uint32_t v = __shfl_up_sync(0xffffffffu, incl, o);
                        if (lane >= uint32_t(o)) incl += v;
                    }
                    const uint32_t first = before + incl - n;
                    if (want >= first && want < first + n) {
                        where[0] = b + lane;
                        where[1] = (want - first) * span;
                    }
                    before += __shfl_sync(0xffffffffu, incl, 31);
                    if (before > want) break;
                }
            }
        }
        __syncthreads();
        walk.at = {kvh, where[0], where[1], 0u};
        walk.end = walk.at;
        if (where[0] >= a.n_seqs) walk.at.kvh = walk.end.kvh + 1;              // past the last pair
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tslot;
    auto wait = [&](uint64_t* b, uint32_t ph) { if (!*fail && !mbar_try_wait(b, ph & 1)) pa_wait_slow(b, ph & 1, fail, p.err); };
    // item k, of a role; and done with it
    auto item = [&](uint32_t k) -> const PaItem& {
        wait(itf + k % kPaItems, k / kPaItems);
        return items[k % kPaItems];
    };
    auto item_done = [&](uint32_t k) { mbar_arrive(ite + k % kPaItems); };
    // 384 threads start with 168 registers: 256 x 208 + 128 x 80 of them
    if (warp >= 8) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 80;");
    if (warp == 8) {
        // ---------------------------------------------------- loads (one lane)
        if (elect_one()) {
            uint32_t j = 0, nq[2] = {0u, 0u};    // units sent for, Q tiles sent for
            for (uint32_t k = 0; !*fail; ++k) {
                const PaItem& it = item(k);
                if (!it.more) break;
                const uint32_t m = max(it.cnt[0], it.cnt[1]), kvh = it.kvh, row_q = it.S.q0 + it.tok, row_k = it.S.k0 + it.key0;
                const uint32_t cnt[2] = {it.cnt[0], it.cnt[1]};
                item_done(k);
                for (uint32_t i = 0; i < 2 * m; ++i, ++j) {      // K0 V0 K1 V1 .., the Q tiles around K0
                    if (i < 2 && (i ? cnt[1] : cnt[0])) {
                        const uint32_t q = i ? nq[1]++ : nq[0]++;
                        if (q) wait(qe + i, q - 1);
                        mbar_arrive_expect_tx(qf + i, p.group * p.tokens * 128 * NH);
                        for (int h = 0; h < NH; ++h)
                            tma_load3(smem + SM::Q + i * SM::TILE + h * 16384, &mq, h * 64, kvh * p.group, row_q + i * p.tokens, qf + i);
                    }
                    const uint32_t st = j % ST, round = j / ST;
                    if (round) wait(kve + st, round - 1);
                    mbar_arrive_expect_tx(kvf + st, SM::TILE);
                    for (int h = 0; h < NH; ++h)
                        tma_load3(smem + SM::KV + st * SM::TILE + h * 16384, i & 1 ? &mv : &mk, h * 64, kvh, row_k + i / 2 * kPaKeys, kvf + st);
                }
            }
            // nothing may be in flight when the CTA ends (the MMA warp has
            // waited for all of it unless a wait ran out)
            for (uint32_t k = j > ST ? j - ST : 0; k < j; ++k) pa_drain(kvf + k % ST, (k / ST) & 1);
            for (int t = 0; t < 2; ++t)
                if (nq[t]) pa_drain(qf + t, (nq[t] - 1) & 1);
        }
    } else if (warp == 9) {
        // ------------------------------------------------------ MMA (one lane)
        if (elect_one()) {
            constexpr uint32_t IQK = tc_idesc_bf16(128, 128, 0), IPV = tc_idesc_bf16(128, HP, 1);
            const uint32_t sq = smem_u32(smem + SM::Q), skv = smem_u32(smem + SM::KV);
            uint32_t j0 = 0, nq[2] = {0u, 0u}, nb[2] = {0u, 0u}; // units, Q tiles, blocks of each tile so far
            auto qk = [&](uint32_t t, uint32_t st, bool last) {
                const uint64_t qd = tc_desc_sw128(sq + t * SM::TILE, 16), kd = tc_desc_sw128(skv + st * SM::TILE, 16);
#pragma unroll
                for (int s = 0; s < HP / 16; ++s) {
                    const uint32_t o = (s / 4 * 16384 + s % 4 * 32) >> 4;
                    tc_mma_f16(tmem + t * 128, qd + o, kd + o, IQK, s > 0);
                }
                tc_commit(sf + t);
                if (last) tc_commit(qe + t);     // the tile's Q has been read
            };
            auto pv = [&](uint32_t t, uint32_t st, bool more) {
                const uint64_t vd = tc_desc_sw128(skv + st * SM::TILE, 16384);
#pragma unroll
                for (int s = 0; s < kPaKeys / 16; ++s)
                    tc_mma_ts(tmem + TMEM_O + t * 128, tmem + t * 128 + s * 8, vd + ((s * 2048) >> 4), IPV, more || s > 0);
                tc_commit(of + t);
            };
            for (uint32_t k = 0; !*fail; ++k) {
                const PaItem& it = item(k);
                if (!it.more) break;
                const uint32_t c0 = it.cnt[0], c1 = it.cnt[1], m = max(c0, c1);
                item_done(k);
                if (m) {
                    wait(kvf + j0 % ST, j0 / ST);
#pragma unroll
                    for (uint32_t t = 0; t < 2; ++t)
                        if (t ? c1 : c0) {
                            wait(qf + t, nq[t]++);
                            tc_fence_after();
                            qk(t, j0 % ST, (t ? c1 : c0) == 1);
                        }
                    tc_commit(kve + j0 % ST);
                }
                for (uint32_t i = 0; i < m; ++i) {
                    const uint32_t jv = j0 + 2 * i + 1, jk = jv + 1, sv = jv % ST, sk = jk % ST;
                    wait(kvf + sv, jv / ST);
                    if (i + 1 < m) wait(kvf + sk, jk / ST);
#pragma unroll
                    for (uint32_t t = 0; t < 2; ++t) {
                        const uint32_t nt = t ? c1 : c0;
                        if (i < nt) {
                            // (of an item's first block this also says that the
                            // softmax warps have read the last item's sums)
                            wait(pr + t, nb[t]++);
                            tc_fence_after();
                            pv(t, sv, i > 0 || begun[t]);
                        }
                        if (i + 1 < nt) qk(t, sk, i + 2 == nt);
                    }
                    tc_commit(kve + sv);
                    if (i + 1 < m) tc_commit(kve + sk);
                }
                j0 += 2 * m;
            }
            if (j0) pa_drain(kve + (j0 - 1) % ST, ((j0 - 1) / ST) & 1);                // all MMAs done: the last commit
        }
    } else if (warp == 10) {
        // ------------------------------------------------------------- items
        if (elect_one()) {
            bool more = true;
            const uint32_t pairs = p.list ? ld_plain(p.taken + 1) : 0u;
            for (uint32_t k = 0; more && !*fail; ++k) {
                PaItem it{};
                if (k >= kPaItems) wait(ite + k % kPaItems, k / kPaItems - 1);
                if (p.list) {
                    const uint32_t i = atomicAdd(p.taken, 1u), pair = i / a.num_kv_heads;
                    more = pair < pairs;
                    if (more) {
                        const uint2 q = ld_plain(p.list + pair);
                        walk.at = {i % a.num_kv_heads, q.x, q.y, 0u};
                        walk.end = walk.at;
                        walk.next(p, it);
                    }
                } else {
                    more = walk.next(p, it);
                }
                it.more = more;
                items[k % kPaItems] = it;
                mbar_arrive(itf + k % kPaItems);
            }
        }
    }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 208;");
        // ----------------------------------------------------------- softmax
        // One thread a row: the scores of a block come from tensor memory
        // as 128 registers. The reference maximum is only moved when the
        // running one is more than 8 (in log2) above it, so the
        // accumulator is rarely rescaled; probabilities stay below 2^8.
        const uint32_t t = warp >> 2, r = tid & 127;
        const uint32_t ts = tmem + t * 128 + ((warp & 3) << 21), to = tmem + TMEM_O + t * 128 + ((warp & 3) << 21);
        const float sl = p.scale_log2;
        const uint32_t tk = r / p.group, hd = r % p.group;       // the row's token of the tile and head of the group
        uint32_t j0 = 0, nb = 0;                 // units and this tile's blocks so far
        // A meeting of this tile's four warps, or of both tiles' eight: whether
        // any thread came with yes. (An mbarrier and not a named one, so that
        // the wait is bounded. A turn's flag is cleared a turn ahead: by then all have read its last use.)
        uint32_t met[2] = {0u, 0u};
        auto any = [&](bool all, bool yes) -> bool {
            const uint32_t x = all ? 2u : t, turn = all ? met[1]++ : met[0]++;
            const bool mine = __any_sync(0xffffffffu, yes);
            __syncwarp();
            if (lane == 0) {
                xflag[x * 3 + (turn + 1) % 3] = 0u;
                if (mine) xflag[x * 3 + turn % 3] = 1u;
                mbar_arrive(xb + x);
            }
            wait(xb + x, turn);
            return __any_sync(0xffffffffu, xflag[x * 3 + turn % 3] != 0u);
        };
        for (uint32_t k = 0;; ++k) {
            const PaItem& im = item(k);
            if (__any_sync(0xffffffffu, *fail || !im.more)) break;
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
                    const bool masked = key0 + kPaKeys > inner_hi || key0 < inner_lo, both = i < cnt_o;
                    float s[128];
                    wait(sf + t, nb + i);
                    tc_fence_after();
#pragma unroll
                    for (int c = 0; c < 4; ++c) tmem_ld32(ts + c * 32, s + c * 32);
                    tmem_ld_wait();
                    bool odd = false;            // this block's values hold an infinity or NaN
                    const uint32_t ja = lo > key0 ? lo - key0 : 0u, jb = hi > key0 ? hi - key0 : 0u;       // columns [ja, jb)
                    uint4* const vt = reinterpret_cast<uint4*>(smem + SM::KV + jv % ST * SM::TILE);
                    if (masked) {
#pragma unroll
                        for (int j = 0; j < 128; ++j)
                            if (uint32_t(j) < ja || uint32_t(j) >= jb) s[j] = -INFINITY;
                        // A zero probability does not silence an infinity or NaN
                        // in the matrix product, and this block has keys that
                        // not every row may see: look for one.
                        wait(kvf + jv % ST, jv / ST);
                        __nv_bfloat162 acc = __float2bfloat162_rn(0.0f);
                        const __nv_bfloat162 zero = acc;
#pragma unroll 4
                        for (uint32_t k = r; k < SM::TILE / 16; k += 128) {
                            const uint4 x = vt[k];
                            const uint32_t xs[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
                            for (int q = 0; q < 4; ++q)
                                acc = __hfma2(*reinterpret_cast<const __nv_bfloat162*>(&xs[q]), zero, acc);
                        }
                        odd = any(both, __hisnan(acc.x) || __hisnan(acc.y));
                    }
                    float mq[8];                 // eight chains: the maximum's latency is the softmax warps' to wait for
#pragma unroll
                    for (int j = 0; j < 8; ++j) mq[j] = fmaxf(s[2 * j], s[2 * j + 1]);
#pragma unroll
                    for (int j = 16; j < 128; j += 2) mq[j / 2 % 8] = fmaxf(fmaxf(mq[j / 2 % 8], s[j]), s[j + 1]);
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
                            wait(of + t, nb + i - 1);
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
                    const float ml = m == -INFINITY ? 0.0f : m * sl;
                    const uint64_t sl2 = pack2(sl, sl), ml2 = pack2(-ml, -ml);
                    uint64_t sums[2] = {0ull, 0ull};
#pragma unroll
                    for (int c = 0; c < 4; ++c) {
                        uint32_t w[16];
#pragma unroll
                        for (int k = 0; k < 16; ++k) {
                            float x, y;
                            unpack2(fma2(pack2(s[c * 32 + 2 * k], s[c * 32 + 2 * k + 1]), sl2, ml2), x, y);
                            x = ex2(x);
                            y = ex2(y);
                            sums[k % 2] = add2(sums[k % 2], pack2(x, y));
                            w[k] = cvt_bf16x2(x, y);
                        }
                        tmem_st16(ts + c * 16, w);
                    }
                    if (i == 0 && r == 0) begun[t] = odd;        // the product then adds to what the rows put there
                    if (odd) {
                        // Rare. Each row adds its own share of the infinities and
                        // NaN to its accumulator; then they are zeroed in the
                        // shared tile, for both tiles' products.
                        tmem_st_wait();
                        if (i) {
                            wait(of + t, nb + i - 1);
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
                            for (uint32_t j = 0; j < 128; ++j) {
                                const uint32_t pp = __float_as_uint(tmem_ld1(ts + j / 2));
                                const float x = __uint_as_float(j & 1 ? pp & 0xffff0000u : pp << 16);
                                if (j < ja || j >= jb) continue;
#pragma unroll
                                for (int h = 0; h < 2; ++h) {    // 8 columns: one swizzled 16-byte piece of key j's row
                                    const uint4 v = vt[c / 64 * 1024 + j * 8 + (((c % 64) / 8 + h) ^ (j & 7))];
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
                        any(both, false);  // all rows of both tiles have read them
#pragma unroll 1
                        for (uint32_t k = both ? tid : r; k < SM::TILE / 16; k += both ? 256 : 128) {
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
                        any(both, false);
                    }
                    float sum_x, sum_y;
                    unpack2(add2(sums[0], sums[1]), sum_x, sum_y);
                    l += sum_x + sum_y;
                    tmem_st_wait();
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(pr + t);
                }
                nb += nt;
                wait(of + t, nb - 1);
                tc_fence_after();
            }
            j0 += 2 * max(im.cnt[0], im.cnt[1]);
            const uint32_t token = im.tok + t * p.tokens + tk, head = im.kvh * p.group + hd;
            if (im.whole) {
                const bool keys = live && im.S.hi(token) > im.S.lo(token);
                const float inv = keys ? 1.0f / l : 0.0f;
                uint16_t* dst = a.out + uint64_t(im.S.q0 + token) * a.out_row + uint64_t(head) * a.out_head;
#pragma unroll 1
                for (uint32_t c = 0; c < HP; c += 32) {
                    float o[32];
                    if (nt) {
                        tmem_ld32(to + c, o);
                        tmem_ld_wait();
                    }
#pragma unroll
                    for (int h = 0; h < 4; ++h)
                        if (live && c + h * 8 < a.head_dim) {
                            uint4 w = make_uint4(0u, 0u, 0u, 0u);
                            if (keys) {
                                w.x = cvt_bf16x2(o[h * 8] * inv, o[h * 8 + 1] * inv);
                                w.y = cvt_bf16x2(o[h * 8 + 2] * inv, o[h * 8 + 3] * inv);
                                w.z = cvt_bf16x2(o[h * 8 + 4] * inv, o[h * 8 + 5] * inv);
                                w.w = cvt_bf16x2(o[h * 8 + 6] * inv, o[h * 8 + 7] * inv);
                            }
                            *reinterpret_cast<uint4*>(dst + c + h * 8) = w;
                        }
                }
                if (a.lse && live)
                    a.lse[uint64_t(im.S.q0 + token) * a.num_heads + head] = keys ? m * a.scale + logf(l) : -INFINITY;
            } else {
                // a part: 2 * CTA when it continues a pair (or is the CTA's only one), 2 * CTA + 1 when it starts one
                const uint64_t row = (uint64_t(2 * blockIdx.x + im.starts) * 2 + t) * 128 + r;
                if (nt) {
                    float4* dst = reinterpret_cast<float4*>(p.part + row * HP);
#pragma unroll 1
                    for (uint32_t c = 0; c < HP; c += 32) {
                        float o[32];
                        tmem_ld32(to + c, o);
                        tmem_ld_wait();
#pragma unroll
                        for (int k = 0; k < 8; ++k) dst[c / 4 + k] = make_float4(o[4 * k], o[4 * k + 1], o[4 * k + 2], o[4 * k + 3]);
                    }
                }
                p.stat[row] = make_float2(m, nt ? l : 0.0f);
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
// does 32 of the 256 rows of the pair that CTA c is the first to continue,
// a warp four rows: CTA c - 1 has its first part, c, c + 1, .. the others.
template <int HP>
__global__ void __launch_bounds__(256) k_packed_join(const PackedArgs p) {
    pdl_release();
    pdl_acquire();
    const SmoeCudaPackedAttnArgs& a = p.a;
    const uint32_t c = blockIdx.x, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const PaPlace at = p.plan[c];
    if (c == 0 || at.blk == 0) return;
    auto same = [&](const PaPlace& x) { return x.kvh == at.kvh && x.seq == at.seq && x.tok == at.tok; };
    const PaPlace before = p.plan[c - 1];
    if (same(before) && before.blk) return;      // an earlier CTA continues this pair, too
    uint32_t end = c + 1;                        // parts of CTAs c - 1 (its start) and c .. end - 1
    while (end < gridDim.x) {
        const PaPlace x = p.plan[end];
        if (!same(x)) break;
        ++end;
    }
    const PackedSeq S = packed_seq(a, at.seq);
    constexpr int V = HP / 32;                   // columns of a lane
    for (uint32_t k = 0; k < 4; ++k) {
        const uint32_t row = blockIdx.y * 32 + warp * 4 + k, t = row / 128, r = row % 128;
        const uint32_t token = at.tok + t * p.tokens + r / p.group, head = at.kvh * p.group + r % p.group;
        if (r >= p.group * p.tokens || token >= S.len_q) continue;
        const uint64_t row0 = (uint64_t(2 * (c - 1) + 1) * 2 + t) * 128 + r;   // of CTA c - 1; those after: 2 (c + i)
        auto part = [&](uint32_t i) { return i == 0 ? row0 : (uint64_t(2 * (c + i - 1)) * 2 + t) * 128 + r; };
        const uint32_t parts = end - c + 1;
        // (a CTA whose share is empty has written nothing)
        auto idle = [&](uint32_t i) { return i && same(p.plan[c + i]) && p.plan[c + i].blk == p.plan[c + i - 1].blk; };
        float mx = -INFINITY, l = 0.0f, o[V];
#pragma unroll
        for (int v = 0; v < V; ++v) o[v] = 0.0f;
        for (uint32_t i = 0; i < parts; ++i)
            if (!idle(i)) mx = fmaxf(mx, p.stat[part(i)].x);
        for (uint32_t i = 0; i < parts; ++i) {
            if (idle(i)) continue;
            const float2 st = p.stat[part(i)];
            if (st.x == -INFINITY && st.y == 0.0f) continue;     // no key in this part (its sums may not be written)
            const float f = st.x == -INFINITY ? 1.0f : ex2((st.x - mx) * p.scale_log2);         // (-inf scores alone: NaN stays)
            l = fmaf(st.y, f, l);
#pragma unroll
            for (int v = 0; v < V; ++v) o[v] = fmaf(p.part[part(i) * HP + v * 32 + lane], f, o[v]);
        }
        const bool keys = S.hi(token) > S.lo(token);
        const float inv = keys ? 1.0f / l : 0.0f;
        uint16_t* dst = a.out + uint64_t(S.q0 + token) * a.out_row + uint64_t(head) * a.out_head;
#pragma unroll
        for (int v = 0; v < V; ++v)
            if (v * 32 + lane < a.head_dim) dst[v * 32 + lane] = __bfloat16_as_ushort(__float2bfloat16_rn(keys ? o[v] * inv : 0.0f));
        if (a.lse && lane == 0) a.lse[uint64_t(S.q0 + token) * a.num_heads + head] = keys ? mx * a.scale + logf(l) : -INFINITY;
    }
}

}  // namespace smoe
