// prompt_attn.cuh - attention over packed prompts: causal, grouped heads,
// sequences of different lengths in one launch, on the tcgen05 tensor cores.
#pragma once
#include <cuda.h>

#include "serve.cuh"
#include "tc05.cuh"

namespace smoe {

// Tile rows are (token, head of the group) pairs, token-major: a KV head's
// keys and values then serve all its query heads from one shared-memory copy,
// and a short prompt fills a tile with G times fewer tokens. A CTA owns two
// tiles of 128 rows (the tensor cores work for one while the other's softmax
// runs) and walks the keys 128 at a time.
constexpr uint32_t kPaRows = 128, kPaKeys = 128;
constexpr int kPaThreads = 320;                  // 2 x 4 softmax warps, TMA warp, MMA warp

struct PackedArgs {
    SmoeCudaPackedAttnArgs a;
    uint32_t group, tokens;                      // query heads per KV head, tokens per tile (128 / group)
    float scale_log2;                            // scale * log2(e)
    uint32_t* err;
};

template <int HP>                                // head_dim rounded up to 64 or 128
struct PackedSmem {
    static constexpr uint32_t TILE = HP / 64 * 16384;            // 128 rows, 64-column halves of 128-byte rows
    static constexpr int STAGES = HP == 128 ? 5 : 8;
    static constexpr uint32_t Q = 0, KV = 2 * TILE, BAR = KV + STAGES * TILE, END = BAR + 256;
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
};

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
SMOE_DEVINL uint32_t cvt_bf16x2(float lo, float hi) {
    uint32_t d;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(d) : "f"(hi), "f"(lo));
    return d;
}
// Named barriers of the softmax warps (1, 2: those of one tile; 3: both):
// arrive, wait, and learn whether any thread came with p.
template <int BARRIER, int THREADS>
SMOE_DEVINL bool bar_any(bool p) {
    uint32_t r;
    asm volatile(
        "{\n .reg .pred p, q;\n setp.ne.u32 p, %3, 0;\n barrier.cta.red.or.pred q, %1, %2, p;\n selp.u32 %0, 1, 0, q;\n}\n"
        : "=r"(r) : "n"(BARRIER), "n"(THREADS), "r"(uint32_t(p)) : "memory");
    return r != 0;
}
SMOE_DEVINL bool pa_any(bool both, uint32_t t, bool p) {
    return both ? bar_any<3, 256>(p) : t ? bar_any<2, 128>(p) : bar_any<1, 128>(p);
}

// A bounded wait: after one ran out, all others of the CTA return at once.
// The roles then finish their loops on whatever the buffers hold (every
// address stays in the CTA's own memory) and the error word is set.
static __device__ __noinline__ void pa_wait_slow(uint64_t* bar, uint32_t parity, volatile uint32_t* fail, uint32_t* err) {
    const uint64_t end = gtimer() + SMOE_WAIT_NS_DEFAULT;
#pragma unroll 1
    for (uint32_t i = 0; i < SMOE_SPIN_LIMIT; ++i) {
        if (mbar_try_wait(bar, parity)) return;
        if ((i & 15) == 15 && (*fail || gtimer() > end)) break;
    }
    *fail = 1u;
    atomicCAS(err, 0u, uint32_t(SMOE_DEVERR_MBAR_TIMEOUT));
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
    uint64_t *qf = bars, *sf = bars + 2, *pr = bars + 4, *of = bars + 6, *kvf = bars + 8, *kve = bars + 8 + ST;
    uint32_t* words = reinterpret_cast<uint32_t*>(bars + 8 + 2 * ST);
    volatile uint32_t *fail = words, *begun = words + 1;         // begun[t]: the accumulator holds something before block 0's P V
    uint32_t* tslot = words + 3;
    uint32_t* where = words + 4;                                 // the CTA's sequence and first token
    const uint32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const SmoeCudaPackedAttnArgs& a = p.a;

    pdl_release();
    if (warp == 8 && lane == 0) {
        for (int i = 0; i < 2; ++i) {
            mbar_init(qf + i, 1);
            mbar_init(sf + i, 1);
            mbar_init(pr + i, 4);
            mbar_init(of + i, 1);
        }
        for (int i = 0; i < ST; ++i) {
            mbar_init(kvf + i, 1);
            mbar_init(kve + i, 1);
        }
        *fail = begun[0] = begun[1] = 0u;
        fence_mbar_init();
    }
    if (warp == 9) tmem_alloc(tslot, 512);
    pdl_acquire();

    // The CTA's tile pair, counted from the last one backwards: later tokens
    // have more keys, so long tiles start first. One lane per sequence.
    const uint32_t kvh = blockIdx.x % a.num_kv_heads, span = 2 * p.tokens;
    const uint32_t* ck = a.cu_k ? a.cu_k : a.cu_q;
    if (warp == 0) {
        uint32_t total = 0;
        auto pairs = [&](uint32_t s) -> uint32_t {
            if (s >= a.n_seqs) return 0u;
            const uint32_t q0 = ld_plain(a.cu_q + s), q1 = ld_plain(a.cu_q + s + 1), k0 = ld_plain(ck + s), k1 = ld_plain(ck + s + 1);
            if (q1 < q0 || q1 > a.total_q || k1 < k0 || k1 > a.total_k) {
                if (blockIdx.x == 0) serve_err(p.err, SMOE_DEVERR_BAD_RANGE);
                return 0u;
            }
            return (q1 - q0 + span - 1) / span;
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
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tslot, seq = where[0];
    if (seq < a.n_seqs) {                        // (else: a CTA past the last tile pair)
        const uint32_t tok0 = where[1];
        const PackedSeq S{ld_plain(a.cu_q + seq), ld_plain(ck + seq), ld_plain(a.cu_q + seq + 1) - ld_plain(a.cu_q + seq),
                          ld_plain(ck + seq + 1) - ld_plain(ck + seq), a.causal, a.window};
        // blocks of 128 keys: the pair's first one, and how many each tile takes from there
        const uint32_t b0 = S.lo(tok0) / kPaKeys;
        auto blocks = [&](uint32_t t) -> uint32_t {
            const uint32_t first = tok0 + t * p.tokens;
            if (first >= S.len_q) return 0u;
            const uint32_t end = (S.hi(min(first + p.tokens, S.len_q) - 1) + kPaKeys - 1) / kPaKeys;
            return end > b0 ? end - b0 : 0u;
        };
        const uint32_t n0 = blocks(0), n1 = blocks(1), n = max(n0, n1);

        if (warp == 8) {
            // ------------------------------------------------ loads (one lane)
            if (lane == 0) {
                auto wait = [&](uint64_t* b, uint32_t ph) { if (!*fail && !mbar_try_wait(b, ph)) pa_wait_slow(b, ph, fail, p.err); };
                auto load_q = [&](uint32_t t) {
                    mbar_arrive_expect_tx(qf + t, p.group * p.tokens * 128 * NH);
                    for (int h = 0; h < NH; ++h)
                        tma_load3(smem + SM::Q + t * SM::TILE + h * 16384, &mq, h * 64, kvh * p.group,
                                  S.q0 + tok0 + t * p.tokens, qf + t);
                };
                if (n0) load_q(0);
                if (n1) load_q(1);
                for (uint32_t j = 0; j < 2 * n; ++j) {           // K0 V0 K1 V1 ..
                    const uint32_t st = j % ST, round = j / ST;
                    if (round) wait(kve + st, (round - 1) & 1);
                    mbar_arrive_expect_tx(kvf + st, SM::TILE);
                    for (int h = 0; h < NH; ++h)
                        tma_load3(smem + SM::KV + st * SM::TILE + h * 16384, j & 1 ? &mv : &mk, h * 64, kvh,
                                  S.k0 + (b0 + j / 2) * kPaKeys, kvf + st);
                }
                // nothing may be in flight when the CTA ends (the MMA warp has
                // waited for all of it unless a wait ran out)
                for (uint32_t j = 2 * n > ST ? 2 * n - ST : 0; j < 2 * n; ++j) mbar_wait_bounded(kvf + j % ST, (j / ST) & 1);
                if (n0) mbar_wait_bounded(qf, 0);
                if (n1) mbar_wait_bounded(qf + 1, 0);
            }
        } else if (warp == 9) {
            // -------------------------------------------------- MMA (one lane)
            if (lane == 0) {
                auto wait = [&](uint64_t* b, uint32_t ph) { if (!*fail && !mbar_try_wait(b, ph)) pa_wait_slow(b, ph, fail, p.err); };
                constexpr uint32_t IQK = tc_idesc_bf16(128, 128, 0), IPV = tc_idesc_bf16(128, HP, 1);
                const uint32_t sq = smem_u32(smem + SM::Q), skv = smem_u32(smem + SM::KV);
                auto qk = [&](uint32_t t, uint32_t st) {
                    const uint64_t qd = tc_desc_sw128(sq + t * SM::TILE, 16), kd = tc_desc_sw128(skv + st * SM::TILE, 16);
#pragma unroll
                    for (int s = 0; s < HP / 16; ++s) {
                        const uint32_t o = (s / 4 * 16384 + s % 4 * 32) >> 4;
                        tc_mma_f16(tmem + t * 128, qd + o, kd + o, IQK, s > 0);
                    }
                    tc_commit(sf + t);
                };
                auto pv = [&](uint32_t t, uint32_t st, bool more) {
                    const uint64_t vd = tc_desc_sw128(skv + st * SM::TILE, 16384);
#pragma unroll
                    for (int s = 0; s < kPaKeys / 16; ++s)
                        tc_mma_ts(tmem + TMEM_O + t * 128, tmem + t * 128 + s * 8, vd + ((s * 2048) >> 4), IPV, more || s > 0);
                };
                if (n) {
                    wait(kvf, 0);
                    for (uint32_t t = 0; t < 2; ++t)
                        if (t ? n1 : n0) {
                            wait(qf + t, 0);
                            tc_fence_after();
                            qk(t, 0);
                        }
                    tc_commit(kve);
                }
                for (uint32_t i = 0; i < n; ++i) {
                    const uint32_t jv = 2 * i + 1, jk = jv + 1, sv = jv % ST, sk = jk % ST;
                    wait(kvf + sv, (jv / ST) & 1);
                    if (i + 1 < n) wait(kvf + sk, (jk / ST) & 1);
#pragma unroll
                    for (uint32_t t = 0; t < 2; ++t) {
                        const uint32_t nt = t ? n1 : n0;
                        if (i < nt) {
                            wait(pr + t, i & 1);
                            tc_fence_after();
                            pv(t, sv, i > 0 || begun[t]);
                            tc_commit(of + t);
                        }
                        if (i + 1 < nt) qk(t, sk);
                    }
                    tc_commit(kve + sv);
                    if (i + 1 < n) tc_commit(kve + sk);
                }
                if (n) {                         // all MMAs done: this slot's last commit was the loop's last one
                    const uint32_t j = 2 * n - 1;
                    mbar_wait_bounded(kve + j % ST, (j / ST) & 1);
                }
            }
        } else {
            // ------------------------------------------------------- softmax
            // One thread a row: the scores of a block come from tensor memory
            // as 128 registers. The reference maximum is only moved when the
            // running one is more than 8 (in log2) above it, so the
            // accumulator is rarely rescaled; probabilities stay below 2^8.
            const uint32_t t = warp >> 2, r = tid & 127, nt = t ? n1 : n0;
            const uint32_t first = tok0 + t * p.tokens;
            const uint32_t token = first + r / p.group, head = kvh * p.group + r % p.group;
            const bool live = r < p.group * p.tokens && token < S.len_q;
            const uint32_t ts = tmem + t * 128 + ((warp & 3) << 21), to = tmem + TMEM_O + t * 128 + ((warp & 3) << 21);
            auto wait = [&](uint64_t* b, uint32_t ph) { if (!*fail && !mbar_try_wait(b, ph)) pa_wait_slow(b, ph, fail, p.err); };
            float m = -INFINITY, l = 0.0f;
            if (nt) {
                const uint32_t last = min(first + p.tokens, S.len_q) - 1;
                const uint32_t lo = S.lo(min(token, last)), hi = S.hi(min(token, last));
                // some row of the pair may not see some key of a block that
                // ends past `inner_hi` or starts before `inner_lo`
                const uint32_t inner_hi = S.hi(tok0), inner_lo = S.lo(min(tok0 + span, S.len_q) - 1);
                const float sl = p.scale_log2;
                for (uint32_t i = 0; i < nt; ++i) {
                    const uint32_t key0 = (b0 + i) * kPaKeys;
                    const bool masked = key0 + kPaKeys > inner_hi || key0 < inner_lo, both = i < n0 && i < n1;
                    float s[128];
                    wait(sf + t, i & 1);
                    tc_fence_after();
#pragma unroll
                    for (int c = 0; c < 4; ++c) tmem_ld32(ts + c * 32, s + c * 32);
                    tmem_ld_wait();
                    bool odd = false;            // this block's values hold an infinity or NaN
                    const uint32_t ja = lo > key0 ? lo - key0 : 0u, jb = hi > key0 ? hi - key0 : 0u;       // columns [ja, jb)
                    uint4* const vt = reinterpret_cast<uint4*>(smem + SM::KV + (2 * i + 1) % ST * SM::TILE);
                    if (masked) {
#pragma unroll
                        for (int j = 0; j < 128; ++j)
                            if (uint32_t(j) < ja || uint32_t(j) >= jb) s[j] = -INFINITY;
                        // A zero probability does not silence an infinity or NaN
                        // in the matrix product, and this block has keys that
                        // not every row may see: look for one.
                        wait(kvf + (2 * i + 1) % ST, ((2 * i + 1) / ST) & 1);
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
                        odd = pa_any(both, t, __hisnan(acc.x) || __hisnan(acc.y));
                    }
                    float mx = m;
#pragma unroll
                    for (int j = 0; j < 128; ++j) mx = fmaxf(mx, s[j]);
                    // (each row for itself - a factor of 1 leaves the others of the
                    // warp as they are - so a row's bits do not depend on its neighbours)
                    const bool move = live && ((mx - m) * sl > 8.0f || (mx > m && m == -INFINITY));
                    if (__any_sync(0xffffffffu, move)) {
                        const float f = !move ? 1.0f : m == -INFINITY ? 0.0f : ex2((m - mx) * sl);
                        if (i) {
                            wait(of + t, (i - 1) & 1);
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
                    float sum = 0.0f;
#pragma unroll
                    for (int c = 0; c < 4; ++c) {
                        uint32_t w[16];
#pragma unroll
                        for (int k = 0; k < 16; ++k) {
                            const float x = ex2(fmaf(s[c * 32 + 2 * k], sl, -ml)), y = ex2(fmaf(s[c * 32 + 2 * k + 1], sl, -ml));
                            sum += x + y;
                            w[k] = cvt_bf16x2(x, y);
                        }
                        tmem_st16(ts + c * 16, w);
                    }
                    if (odd) {
                        // Rare. Each row adds its own share of the infinities and
                        // NaN to its accumulator; then they are zeroed in the
                        // shared tile, for both tiles' products.
                        tmem_st_wait();
                        if (i) {
                            wait(of + t, (i - 1) & 1);
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
                        if (r == 0 && i == 0) begun[t] = 1u;
                        pa_any(both, t, false);  // all rows of both tiles have read them
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
                        pa_any(both, t, false);
                    }
                    l += sum;
                    tmem_st_wait();
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(pr + t);
                }
                wait(of + t, (nt - 1) & 1);
                tc_fence_after();
            }
            const bool keys = live && S.hi(token) > S.lo(token);
            const float inv = keys ? 1.0f / l : 0.0f;
            uint16_t* dst = a.out + uint64_t(S.q0 + token) * a.out_row + uint64_t(head) * a.out_head;
#pragma unroll 1
            for (uint32_t c = 0; c < HP; c += 16) {
                float o[16];
                if (nt) {
                    tmem_ld16(to + c, o);
                    tmem_ld_wait();
                }
#pragma unroll
                for (int h = 0; h < 2; ++h)
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
                a.lse[uint64_t(S.q0 + token) * a.num_heads + head] = keys ? m * a.scale + logf(l) : -INFINITY;
        }
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (warp == 9) tmem_dealloc(tmem, 512);
}

}  // namespace smoe
