// kv4.cuh - the paged 4-bit KV cache: quantised append, read-back, attention
// of one query token per sequence, eviction by accumulated attention weight.
#pragma once
#include "serve.cuh"

namespace smoe {

constexpr uint32_t kKvPage = SMOE_KV4_PAGE;      // entries of a page
constexpr uint32_t kKvPlane = kKvPage * 32;      // bytes of one group's codes in a block (32 a entry)

// Block of one page and KV head, ng = head_dim / 64 groups.
struct Kv4Geom {
    uint32_t ng, block;                          // bytes of a block
    __host__ __device__ explicit Kv4Geom(uint32_t head_dim) : ng(head_dim / 64), block(head_dim / 64 * 4608) {}
    __host__ __device__ uint32_t codes(uint32_t kv, uint32_t g) const { return (kv * ng + g) * kKvPlane; }
    __host__ __device__ uint32_t sb(uint32_t kv, uint32_t g) const { return ng * 2 * kKvPlane + (kv * ng + g) * kKvPage * 4; }
};

struct Kv4Args {
    SmoeKv4Cache c;
    uint32_t* err;
};

// Page of entry e of sequence s; ~0u (and the error word set) when the entry
// is past the table or the page past the cache.
SMOE_DEVINL uint32_t kv4_page(const SmoeKv4Cache& c, uint32_t s, uint64_t e, uint32_t* err) {
    if (e >= uint64_t(c.table_stride) * kKvPage) {
        serve_err(err, SMOE_DEVERR_BAD_PAGE);
        return ~0u;
    }
    const uint32_t p = ld_plain(c.table + size_t(s) * c.table_stride + e / kKvPage);
    if (p >= c.n_pages) {
        serve_err(err, SMOE_DEVERR_BAD_PAGE);
        return ~0u;
    }
    return p;
}

// ------------------------------------------------------------ append and read
// One half-warp per (row, KV head, K or V, group of 64): 4 values a lane, the
// group's minimum and maximum by four shuffles, 4 codes (2 bytes) a lane, so a
// group's loads (128 or 256 bytes) and stores (32) are whole sectors. A warp
// takes two units of one row; the rows of a CTA are consecutive.
SMOE_DEVINL float4 kv4_load4(const void* p, size_t at, int dtype) {
    if (dtype == SMOE_DTYPE_F32) return *(reinterpret_cast<const float4*>(static_cast<const float*>(p) + at));
    const uint2 u = *(reinterpret_cast<const uint2*>(static_cast<const uint16_t*>(p) + at));
    return make_float4(__uint_as_float(u.x << 16), __uint_as_float(u.x & 0xffff0000u), __uint_as_float(u.y << 16),
                       __uint_as_float(u.y & 0xffff0000u));
}

__global__ void __launch_bounds__(256) k_kv4_append(Kv4Args a, SmoeKv4Rows r) {
    pdl_release();
    pdl_acquire();
    const Kv4Geom G(a.c.head_dim);
    const uint32_t lane = threadIdx.x & 31, hl = lane & 15;
    const uint32_t row = blockIdx.x * 8 + (threadIdx.x >> 5);
    if (row >= r.total) return;
    const uint32_t s = seq_of_row(r.cu, a.c.n_seqs, row, lane);
    if (s >= a.c.n_seqs) return;                 // rows past the last sequence
    const uint32_t t = row - ld_plain(r.cu + s);
    const uint64_t e = uint64_t(ld_plain(a.c.len + s)) + t;
    const uint32_t page = kv4_page(a.c, s, e, a.err);
    if (page == ~0u) return;
    const uint32_t slot = uint32_t(e % kKvPage), units = a.c.num_kv_heads * 2 * G.ng;
    for (uint32_t u = lane >> 4; u < units; u += 2) {
        const uint32_t g = u % G.ng, kv = u / G.ng & 1, h = u / (2 * G.ng);
        const size_t at = kv ? row * r.v_row + h * r.v_head : row * r.k_row + h * r.k_head;
        const float4 x = kv4_load4(kv ? r.v : r.k, at + g * 64 + hl * 4, r.dtype);
        float lo = fminf(fminf(x.x, x.y), fminf(x.z, x.w)), hi = fmaxf(fmaxf(x.x, x.y), fmaxf(x.z, x.w));
        const uint32_t m = lane < 16 ? 0x0000ffffu : 0xffff0000u;
#pragma unroll
        for (int o = 8; o; o >>= 1) {
            lo = fminf(lo, __shfl_xor_sync(m, lo, o));
            hi = fmaxf(hi, __shfl_xor_sync(m, hi, o));
        }
        const __nv_bfloat16 bb = __float2bfloat16_rn(lo);
        const __nv_bfloat16 sb = __float2bfloat16_rn(__fmul_rn(__fsub_rn(hi, lo), 1.0f / 15.0f));
        const float bias = __bfloat162float(bb), scale = __bfloat162float(sb);
        const float xs[4] = {x.x, x.y, x.z, x.w};
        uint32_t code = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float q = scale > 0.0f ? rintf(__fdiv_rn(__fsub_rn(xs[i], bias), scale)) : 0.0f;
            code |= uint32_t(fminf(fmaxf(q, 0.0f), 15.0f)) << (4 * i);
        }
        uint8_t* blk = a.c.blocks + (size_t(page) * a.c.num_kv_heads + h) * G.block;
        *reinterpret_cast<uint16_t*>(blk + G.codes(kv, g) + slot * 32 + hl * 2) = uint16_t(code);
        if (hl == 0) {
            *reinterpret_cast<uint32_t*>(blk + G.sb(kv, g) + slot * 4) =
                uint32_t(__bfloat16_as_ushort(sb)) | uint32_t(__bfloat16_as_ushort(bb)) << 16;
            if (kv == 0 && g == 0) {
                const size_t i = (size_t(page) * a.c.num_kv_heads + h) * kKvPage + slot;
                if (a.c.pos) a.c.pos[i] = ld_plain((a.c.seen ? a.c.seen : a.c.len) + s) + t;
                if (a.c.score) a.c.score[i] = 0.0f;
            }
        }
    }
}

__global__ void __launch_bounds__(256) k_kv4_read(Kv4Args a, const uint32_t* first, SmoeKv4Rows r) {
    pdl_release();
    pdl_acquire();
    const Kv4Geom G(a.c.head_dim);
    const uint32_t lane = threadIdx.x & 31, hl = lane & 15;
    const uint32_t row = blockIdx.x * 8 + (threadIdx.x >> 5);
    if (row >= r.total) return;
    const uint32_t s = seq_of_row(r.cu, a.c.n_seqs, row, lane);
    if (s >= a.c.n_seqs) return;
    const uint64_t e = uint64_t(first ? ld_plain(first + s) : 0u) + (row - ld_plain(r.cu + s));
    const uint32_t page = kv4_page(a.c, s, e, a.err);
    if (page == ~0u) return;
    const uint32_t slot = uint32_t(e % kKvPage), units = a.c.num_kv_heads * 2 * G.ng;
    for (uint32_t u = lane >> 4; u < units; u += 2) {
        const uint32_t g = u % G.ng, kv = u / G.ng & 1, h = u / (2 * G.ng);
        const uint8_t* blk = a.c.blocks + (size_t(page) * a.c.num_kv_heads + h) * G.block;
        const uint32_t code = *reinterpret_cast<const uint16_t*>(blk + G.codes(kv, g) + slot * 32 + hl * 2);
        const uint32_t sb = *reinterpret_cast<const uint32_t*>(blk + G.sb(kv, g) + slot * 4);
        const float scale = __uint_as_float(sb << 16), bias = __uint_as_float(sb & 0xffff0000u);
        float v[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = __fadd_rn(__fmul_rn(float(code >> (4 * i) & 15u), scale), bias);
        const size_t at = (kv ? row * r.v_row + h * r.v_head : row * r.k_row + h * r.k_head) + g * 64 + hl * 4;
        void* dst = kv ? r.v : r.k;
        if (r.dtype == SMOE_DTYPE_F32)
            *reinterpret_cast<float4*>(static_cast<float*>(dst) + at) = make_float4(v[0], v[1], v[2], v[3]);
        else
            *reinterpret_cast<uint2*>(static_cast<uint16_t*>(dst) + at) =
                make_uint2(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]));
    }
}

// ---------------------------------------------------------------- attention
// One query token per sequence. With a group's codes c (0..15), scales s and
// biases b:
//   q . k = sum_g s_g (q_g . c_g) + b_g sum(q_g)
//   sum_j p_j v_j = sum_j (p_j s_j) c_j + sum_j p_j b_j          (per group)
// so the raw codes are the tensor cores' operands (exact in fp16) and scales
// and biases stay in fp32. q goes in as one (bf16 q) or two fp16 pieces, each
// head scaled by a power of two so that its largest value is near 2^14; p s
// as two fp16 pieces (22 bits), times a power of two per group that follows
// the largest scale seen. (bf16 pieces need no such power, but three more
// instructions for every 16 codes.)
// The entries are the M rows of both products and a KV head's query heads
// the N columns (8 or 16), so a page is dequantised once for all of them.
//
// A CTA of 4 warps takes a stretch of pages of one (sequence, KV head), a
// warp every fourth page: each warp copies its pages - one block, one bulk
// copy - into a ring of its own, keeps its own running maximum and sums, and
// the four are joined at the end.
constexpr int kKaWarps = 4, kKaStages = 2;

struct Kv4Attn {
    Kv4Args a;
    SmoeKv4AttnArgs t;
    uint32_t group, chunks;                      // query heads per KV head; CTAs of a KV head's query heads
    uint32_t split_pages, splits;                // pages of a CTA, CTAs along a sequence of max_len
    float* part;                                 // [n_seqs][num_heads][splits][head_dim] weighted sums, splits > 1 or weights
    float2* stat;                                // [n_seqs][num_heads][splits] maximum, sum
    float* logits;                               // [n_seqs][num_kv_heads][row][gs] log2-scaled scores, with weights
    uint32_t rows, gs;
    float scale_log2;
};

// Entries of sequence s that the token attends to.
SMOE_DEVINL uint32_t kv4_valid(const Kv4Attn& p, uint32_t s) {
    const uint64_t n = uint64_t(ld_plain(p.a.c.len + s)) + p.t.extra;
    if (n > p.t.max_len) {
        if (threadIdx.x == 0) serve_err(p.a.err, SMOE_DEVERR_BAD_RANGE);
        return p.t.max_len;
    }
    return uint32_t(n);
}

// 8 codes as fp16 pairs (code n, code n + 4): 1024 + c and 1024 + 16 c are
// exact, and so is what the subtraction or the multiply-add makes of them.
SMOE_DEVINL void kv4_half_codes(uint32_t w, uint32_t* r) {
    constexpr uint32_t M0 = 0x000F000Fu, M1 = 0x00F000F0u, ONE = 0x64006400u;
    const uint32_t w8 = w >> 8;
    r[0] = hsub_1024(lop3_and_or(w, M0, ONE));
    asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(r[1]) : "r"(lop3_and_or(w, M1, ONE)), "r"(0x2C002C00u), "r"(0xD400D400u));
    r[2] = hsub_1024(lop3_and_or(w8, M0, ONE));
    asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(r[3]) : "r"(lop3_and_or(w8, M1, ONE)), "r"(0x2C002C00u), "r"(0xD400D400u));
}
SMOE_DEVINL void mma_f16f32_16816(float* d, const uint32_t* a, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
SMOE_DEVINL uint32_t movm_trans(uint32_t x) {
    uint32_t y;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}
SMOE_DEVINL float kv4_ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
SMOE_DEVINL uint32_t cvt_f16x2(float lo, float hi) {
    uint32_t d;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(d) : "f"(hi), "f"(lo));
    return d;
}
SMOE_DEVINL float half_lo(uint32_t x) { return __half2float(__ushort_as_half(uint16_t(x))); }
SMOE_DEVINL float half_hi(uint32_t x) { return __half2float(__ushort_as_half(uint16_t(x >> 16))); }
SMOE_DEVINL float lo_f(uint32_t x) { return __uint_as_float(x << 16); }
SMOE_DEVINL float hi_f(uint32_t x) { return __uint_as_float(x & 0xffff0000u); }

template <int NG, int NT>
struct Kv4AttnSmem {
    static constexpr uint32_t BLOCK = NG * 4608, HD = NG * 64, HEADS = NT * 8;
    static constexpr uint32_t RING = 0, RING_BYTES = kKaWarps * kKaStages * BLOCK;
    // float [HEADS][HD + 4], in the last warp's last stage until the fragments are made: three CTAs then fit an SM
    static constexpr uint32_t QROW = HD + 4, Q = RING + RING_BYTES - (HEADS * QROW * 4 + 127) / 128 * 128;
    static_assert(HEADS * QROW * 4 <= (NT == 1 ? 1 : 2) * BLOCK, "q's place");
    static constexpr uint32_t QSUM = RING + RING_BYTES;          // float [NG][HEADS]
    static constexpr uint32_t QINV = QSUM + NG * HEADS * 4;      // float [HEADS]: scale_log2 over the head's power of two
    static constexpr uint32_t ML = QINV + HEADS * 4;             // float [warps][HEADS][2]
    static constexpr uint32_t BAR = ML + kKaWarps * HEADS * 8;
    static constexpr uint32_t BYTES = BAR + kKaWarps * kKaStages * 8;
    static_assert(kKaWarps * HEADS * HD * 4 <= RING_BYTES, "the joined accumulators take the ring's place");
};

// NG groups of 64 (head_dim / 64), NT tiles of 8 query heads, QP pieces of q.
template <int NG, int NT, int QP>
__global__ void __launch_bounds__(kKaWarps * 32, NT == 1 && QP == 1 ? 3 : 2) k_kv4_attention(const Kv4Attn p) {
    using SM = Kv4AttnSmem<NG, NT>;
    constexpr uint32_t HD = SM::HD, HEADS = SM::HEADS;
    extern __shared__ __align__(128) uint8_t kv4_smem[];
    uint8_t* smem = kv4_smem;
    const SmoeKv4Cache& c = p.a.c;
    const Kv4Geom G(HD);
    const uint32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, gr = lane >> 2, cl = lane & 3;
    const uint32_t split = blockIdx.x, kvh = blockIdx.y / p.chunks, chunk = blockIdx.y % p.chunks, s = blockIdx.z;
    uint64_t* bars = reinterpret_cast<uint64_t*>(smem + SM::BAR) + warp * kKaStages;
    pdl_release();
    if (lane == 0) {
        for (int i = 0; i < kKaStages; ++i) mbar_init(bars + i, 1);
        fence_mbar_init();
    }
    __syncwarp();
    pdl_acquire();
    const uint32_t n = kv4_valid(p, s), pages = (n + kKvPage - 1) / kKvPage;
    const uint32_t p0 = split * p.split_pages, p1 = min(pages, p0 + p.split_pages);
    const uint32_t h0 = chunk * HEADS, heads = min(HEADS, p.group - h0);        // of this CTA, in the KV head's group
    if (p0 >= p1 && !(n == 0 && p.splits == 1)) return;

    // this warp's pages: p0 + warp, + 4, ..; their numbers are fetched 32 at a time
    const uint32_t mine = p1 > p0 + warp ? (p1 - p0 - warp + kKaWarps - 1) / kKaWarps : 0u;
    uint32_t ids = ~0u, ids_base = 0;
    auto fetch_ids = [&](uint32_t base) {
        ids_base = base;
        ids = base + lane < mine ? kv4_page(c, s, uint64_t(p0 + warp + (base + lane) * kKaWarps) * kKvPage, p.a.err) : ~0u;
    };
    if (mine) fetch_ids(0);
    uint8_t* ring = smem + SM::RING + warp * kKaStages * SM::BLOCK;
    auto issue = [&](uint32_t i) -> uint32_t {                   // whole warp; the page's number
        if (i >= ids_base + 32) fetch_ids(i);
        const uint32_t page = __shfl_sync(0xffffffffu, ids, i - ids_base);
        if (lane == 0) {
            if (page != ~0u) {
                mbar_arrive_expect_tx(bars + i % kKaStages, SM::BLOCK);
                bulk_g2s(ring + i % kKaStages * SM::BLOCK, c.blocks + (size_t(page) * c.num_kv_heads + kvh) * SM::BLOCK,
                         SM::BLOCK, bars + i % kKaStages);
            } else {
                mbar_arrive(bars + i % kKaStages);               // nothing to wait for; its entries are masked
            }
        }
        return page;
    };
    uint32_t good = 0;                                           // bit st: the page in stage st can be read
    const uint32_t early = warp + 1 < kKaWarps ? kKaStages : NT == 1 ? kKaStages - 1 : 0;   // stages that q is not in
    for (uint32_t i = 0; i < early && i < mine; ++i) good |= uint32_t(issue(i) != ~0u) << i;

    // q: fp32 in shared memory, each head times a power of two, its group sums
    float* qs = reinterpret_cast<float*>(smem + SM::Q);
    float* qsum = reinterpret_cast<float*>(smem + SM::QSUM);
    float* qinv = reinterpret_cast<float*>(smem + SM::QINV);
    for (uint32_t h = warp; h < HEADS; h += kKaWarps) {
        float x[HD / 32], mx = 0.0f;
#pragma unroll
        for (uint32_t i = 0; i < HD / 32; ++i) {
            const size_t at = s * p.t.q_row + (kvh * p.group + h0 + h) * HD + i * 32 + lane;
            x[i] = h >= heads ? 0.0f : p.t.dtype == SMOE_DTYPE_F32 ? ld_plain(static_cast<const float*>(p.t.q) + at)
                                                                    : bf16_bits_to_f32(ld_plain(static_cast<const uint16_t*>(p.t.q) + at));
            mx = fmaxf(mx, fabsf(x[i]));
        }
#pragma unroll
        for (int o = 16; o; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
        // 2^e with mx 2^e in [2^14, 2^15), kept within what fp32 can invert (an infinity or NaN in q stays one)
        const int e = max(-100, min(100, 14 - (int(__float_as_uint(mx) >> 23) - 127)));
        const float up = __uint_as_float(uint32_t(127 + e) << 23);
#pragma unroll
        for (uint32_t i = 0; i < HD / 32; ++i) {
            // the pieces that go to the tensor cores, and their sum
            const float y = x[i] * up, hi = __half2float(__float2half_rn(y));
            const float lo = QP == 2 ? __half2float(__float2half_rn(y - hi)) : 0.0f;
            qs[h * SM::QROW + i * 32 + lane] = y;
            x[i] = hi + lo;
        }
#pragma unroll
        for (int g = 0; g < NG; ++g) {
            float t = x[2 * g] + x[2 * g + 1];
#pragma unroll
            for (int o = 16; o; o >>= 1) t += __shfl_xor_sync(0xffffffffu, t, o);
            if (lane == 0) qsum[g * HEADS + h] = t;
        }
        if (lane == 0) qinv[h] = p.scale_log2 * __uint_as_float(uint32_t(127 - e) << 23);
    }
    __syncthreads();
    // this lane's fragments of q: head gr (+ 8), dimensions in the order kv4_half_codes gives the codes
    uint32_t qf[NT][NG][4][QP][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int g = 0; g < NG; ++g)
#pragma unroll
            for (int st = 0; st < 4; ++st)
#pragma unroll
                for (int b = 0; b < 2; ++b) {
                    const float* y = qs + (nt * 8 + gr) * SM::QROW + g * 64 + cl * 16 + st / 2 * 8 + st % 2 * 2 + b;
                    const __half y0 = __float2half_rn(y[0]), y1 = __float2half_rn(y[4]);
                    qf[nt][g][st][0][b] = pack_half2(y0, y1);
                    if (QP == 2)
                        qf[nt][g][st][QP - 1][b] = pack_half2(__float2half_rn(y[0] - __half2float(y0)), __float2half_rn(y[4] - __half2float(y1)));
                }
    if (early < uint32_t(kKaStages)) fence_proxy_async();        // q's place goes to the bulk copies
    __syncthreads();
    for (uint32_t i = early; i < uint32_t(kKaStages) && i < mine; ++i) good |= uint32_t(issue(i) != ~0u) << i;
    float qsm[NT][NG][2], sc[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            sc[nt][k] = qinv[nt * 8 + 2 * cl + k];
#pragma unroll
            for (int g = 0; g < NG; ++g) qsm[nt][g][k] = qsum[g * HEADS + nt * 8 + 2 * cl + k];
        }

    float m[NT][2], l[NT][2], bacc[NT][NG][2], o[NT][NG][4][4], up[NG];      // up: the group's power of two in o
#pragma unroll
    for (int g = 0; g < NG; ++g) up[g] = 0.0f;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            m[nt][k] = -INFINITY;
            l[nt][k] = 0.0f;
#pragma unroll
            for (int g = 0; g < NG; ++g) {
                bacc[nt][g][k] = 0.0f;
#pragma unroll
                for (int i = 0; i < 4; ++i) o[nt][g][i][k] = o[nt][g][i][2 + k] = 0.0f;
            }
        }
    bool failed = false;
    float* lrow = p.logits ? p.logits + ((size_t(s) * c.num_kv_heads + kvh) * p.rows) * p.gs : nullptr;
#pragma unroll 1
    for (uint32_t i = 0; i < mine; ++i) {
        const uint8_t* blk = ring + i % kKaStages * SM::BLOCK;
        if (!failed && !mbar_wait_bounded(bars + i % kKaStages, (i / kKaStages) & 1)) {
            failed = true;                       // (the results are void, the error word says so)
            atomicCAS(p.a.err, 0u, uint32_t(SMOE_DEVERR_MBAR_TIMEOUT));
        }
        const uint32_t e0 = (p0 + warp + i * kKaWarps) * kKvPage;
        const uint32_t have = good >> (i % kKaStages) & 1u ? min(kKvPage, n - e0) : 0u;        // entries of this page
        float x[4][NT][4];                       // scores: entry 16 mt + gr (0, 1) and + 8 (2, 3), heads 2 cl, 2 cl + 1
#pragma unroll
        for (int mt = 0; mt < 4; ++mt) {
            const uint32_t ka = mt * 16 + gr, kb = ka + 8;
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int k = 0; k < 4; ++k) x[mt][nt][k] = 0.0f;
#pragma unroll
            for (int g = 0; g < NG; ++g) {
                const uint2 wa = *reinterpret_cast<const uint2*>(blk + G.codes(0, g) + ka * 32 + cl * 8);
                const uint2 wb = *reinterpret_cast<const uint2*>(blk + G.codes(0, g) + kb * 32 + cl * 8);
                const uint32_t sa = *reinterpret_cast<const uint32_t*>(blk + G.sb(0, g) + ka * 4);
                const uint32_t sb = *reinterpret_cast<const uint32_t*>(blk + G.sb(0, g) + kb * 4);
                float d[NT][4];
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) d[nt][0] = d[nt][1] = d[nt][2] = d[nt][3] = 0.0f;
#pragma unroll
                for (int w = 0; w < 2; ++w) {
                    uint32_t ra[4], rb[4];
                    kv4_half_codes(w ? wa.y : wa.x, ra);
                    kv4_half_codes(w ? wb.y : wb.x, rb);
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const uint32_t af[4] = {ra[2 * h], rb[2 * h], ra[2 * h + 1], rb[2 * h + 1]};
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                            for (int q = 0; q < QP; ++q)
                                mma_f16f32_16816(d[nt], af, qf[nt][g][w * 2 + h][q][0], qf[nt][g][w * 2 + h][q][1]);
                    }
                }
                const float s0 = lo_f(sa), b0 = hi_f(sa), s1 = lo_f(sb), b1 = hi_f(sb);
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int k = 0; k < 2; ++k) {
                        x[mt][nt][k] = fmaf(s0, d[nt][k], fmaf(b0, qsm[nt][g][k], x[mt][nt][k]));
                        x[mt][nt][2 + k] = fmaf(s1, d[nt][2 + k], fmaf(b1, qsm[nt][g][k], x[mt][nt][2 + k]));
                    }
            }
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int k = 0; k < 4; ++k) x[mt][nt][k] *= sc[nt][k & 1];
        }
        if (have < kKvPage)
#pragma unroll
            for (int mt = 0; mt < 4; ++mt)
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int k = 0; k < 4; ++k)
                        if (mt * 16 + gr + (k < 2 ? 0 : 8) >= have) x[mt][nt][k] = -INFINITY;
        if (lrow) {
            float* at = lrow + size_t(e0 + gr) * p.gs + h0 + 2 * cl;
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int mt = 0; mt < 4; ++mt)
#pragma unroll
                    for (int k = 0; k < 2; ++k)
                        if (nt * 8 + 2 * cl < heads && e0 + mt * 16 + k * 8 + gr < n)
                            *reinterpret_cast<float2*>(at + (mt * 16 + k * 8) * p.gs + nt * 8) = make_float2(x[mt][nt][2 * k], x[mt][nt][2 * k + 1]);
        }
        // running maximum; moved only when it is 2^8 too low
        float f[NT][2];
        bool move = false;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                float mx = x[0][nt][k];
#pragma unroll
                for (int mt = 0; mt < 4; ++mt) mx = fmaxf(fmaxf(mx, x[mt][nt][k]), x[mt][nt][2 + k]);
#pragma unroll
                for (int d = 4; d < 32; d <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, d));
                f[nt][k] = 1.0f;
                if (mx > m[nt][k] + 8.0f || (mx > m[nt][k] && m[nt][k] == -INFINITY)) {
                    f[nt][k] = m[nt][k] == -INFINITY ? 0.0f : kv4_ex2(m[nt][k] - mx);
                    m[nt][k] = mx;
                    move = true;
                }
            }
        if (__any_sync(0xffffffffu, move)) {
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    l[nt][k] *= f[nt][k];
#pragma unroll
                    for (int g = 0; g < NG; ++g) {
                        bacc[nt][g][k] *= f[nt][k];
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            o[nt][g][j][k] *= f[nt][k];
                            o[nt][g][j][2 + k] *= f[nt][k];
                        }
                    }
                }
        }
        // the power of two of a group's p s: its largest scale near 2^3, and below
        // 2^7 as pages follow, so that with p <= 2^8 nothing passes fp16's range
#pragma unroll
        for (int g = 0; g < NG; ++g) {
            const uint2 w = *reinterpret_cast<const uint2*>(blk + G.sb(1, g) + lane * 8);
            const uint32_t big = __reduce_max_sync(0xffffffffu, max(2 * lane < have ? w.x & 0x7fffu : 0u, 2 * lane + 1 < have ? w.y & 0x7fffu : 0u));
            if (__uint_as_float(big << 16) * up[g] > 128.0f || up[g] == 0.0f) {
                const float now = __uint_as_float(uint32_t(max(27, min(227, 257 - int(big >> 7)))) << 23);
                const float r = up[g] == 0.0f ? 0.0f : now / up[g];
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int j = 0; j < 4; ++j)
#pragma unroll
                        for (int k = 0; k < 4; ++k) o[nt][g][j][k] *= r;
                up[g] = now;
            }
        }
#pragma unroll
        for (int mt = 0; mt < 4; ++mt) {
            const uint32_t ka = mt * 16 + gr, kb = ka + 8;
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const float mm = m[nt][k & 1] == -INFINITY ? 0.0f : m[nt][k & 1];
                    x[mt][nt][k] = kv4_ex2(x[mt][nt][k] - mm);
                    l[nt][k & 1] += x[mt][nt][k];
                }
#pragma unroll
            for (int g = 0; g < NG; ++g) {
                // entries past the last one may hold anything: their scales count as 0
                uint32_t sa = *reinterpret_cast<const uint32_t*>(blk + G.sb(1, g) + ka * 4);
                uint32_t sb = *reinterpret_cast<const uint32_t*>(blk + G.sb(1, g) + kb * 4);
                if (have < kKvPage) {
                    if (ka >= have) sa = 0u;
                    if (kb >= have) sb = 0u;
                }
                const float s0 = lo_f(sa) * up[g], b0 = hi_f(sa), s1 = lo_f(sb) * up[g], b1 = hi_f(sb);
                // codes of this lane's 8 dimensions (8 gr ..) of the entries 2 cl, 2 cl + 1, 2 cl + 8, 2 cl + 9 of the tile;
                // lanes cl >= 2 load the pair the other way round (the four entries of a load then lie in different banks)
                uint32_t w[4];
#pragma unroll
                for (int k = 0; k < 4; ++k)
                    w[k] = *reinterpret_cast<const uint32_t*>(blk + G.codes(1, g) + (mt * 16 + 2 * cl + ((k & 1) ^ (cl >> 1)) + (k >> 1) * 8) * 32 + gr * 4);
                // even and odd bytes of the pair side by side, so that a register's halves are the two entries' codes of one dimension
                const uint32_t p_lo = cl < 2 ? 0x5410u : 0x1054u, p_hi = cl < 2 ? 0x7632u : 0x3276u;
                uint32_t c0[8], c1[8];           // dimension n: entries (2 cl, 2 cl + 1), and + 8
                kv4_half_codes(__byte_perm(w[0], w[1], p_lo), c0);
                kv4_half_codes(__byte_perm(w[0], w[1], p_hi), c0 + 4);
                kv4_half_codes(__byte_perm(w[2], w[3], p_lo), c1);
                kv4_half_codes(__byte_perm(w[2], w[3], p_hi), c1 + 4);
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                    bacc[nt][g][0] = fmaf(x[mt][nt][0], b0, fmaf(x[mt][nt][2], b1, bacc[nt][g][0]));
                    bacc[nt][g][1] = fmaf(x[mt][nt][1], b0, fmaf(x[mt][nt][3], b1, bacc[nt][g][1]));
                    const float y0 = x[mt][nt][0] * s0, y1 = x[mt][nt][1] * s0, y2 = x[mt][nt][2] * s1, y3 = x[mt][nt][3] * s1;
                    const uint32_t u0 = cvt_f16x2(y0, y1), u1 = cvt_f16x2(y2, y3);
                    const uint32_t t0 = movm_trans(u0), t1 = movm_trans(u1);
                    const uint32_t v0 = movm_trans(cvt_f16x2(y0 - half_lo(u0), y1 - half_hi(u0)));
                    const uint32_t v1 = movm_trans(cvt_f16x2(y2 - half_lo(u1), y3 - half_hi(u1)));
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const uint32_t af[4] = {c0[2 * j], c0[2 * j + 1], c1[2 * j], c1[2 * j + 1]};
                        mma_f16f32_16816(o[nt][g][j], af, t0, t1);
                        mma_f16f32_16816(o[nt][g][j], af, v0, v1);
                    }
                }
            }
        }
        __syncwarp();                            // the stage has been read
        if (i + kKaStages < mine) {
            const uint32_t bit = i % kKaStages;
            good = (good & ~(1u << bit)) | uint32_t(issue(i + kKaStages) != ~0u) << bit;
        }
    }
    if (failed)                                  // no copy may be in flight when the CTA ends
        for (uint32_t i = mine > uint32_t(kKaStages) ? mine - kKaStages : 0u; i < mine; ++i)
            mbar_wait_bounded(bars + i % kKaStages, (i / kKaStages) & 1);

    // join the lanes' sums, then the warps
#pragma unroll
    for (int d = 4; d < 32; d <<= 1)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                l[nt][k] += __shfl_xor_sync(0xffffffffu, l[nt][k], d);
#pragma unroll
                for (int g = 0; g < NG; ++g) bacc[nt][g][k] += __shfl_xor_sync(0xffffffffu, bacc[nt][g][k], d);
            }
    float* ml = reinterpret_cast<float*>(smem + SM::ML);
    if (gr == 0)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                float* at = ml + (warp * HEADS + nt * 8 + 2 * cl + k) * 2;
                at[0] = m[nt][k];
                at[1] = l[nt][k];
            }
    __syncthreads();                             // (every warp is done with its ring, too)
    float* acc = reinterpret_cast<float*>(smem + SM::RING) + warp * HEADS * HD;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int k = 0; k < 2; ++k)
#pragma unroll
            for (int g = 0; g < NG; ++g)
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    float* at = acc + (nt * 8 + 2 * cl + k) * HD + g * 64 + gr * 8 + 2 * j;
                    const float down = up[g] == 0.0f ? 0.0f : 1.0f / up[g];          // (exact: a power of two)
                    *reinterpret_cast<float2*>(at) = make_float2(fmaf(o[nt][g][j][k], down, bacc[nt][g][k]), fmaf(o[nt][g][j][2 + k], down, bacc[nt][g][k]));
                }
    __syncthreads();
    acc = reinterpret_cast<float*>(smem + SM::RING);
    for (uint32_t h = warp; h < heads; h += kKaWarps) {
        float top = -INFINITY, sum = 0.0f, f[kKaWarps];
#pragma unroll
        for (int w = 0; w < kKaWarps; ++w) top = fmaxf(top, ml[(w * HEADS + h) * 2]);
#pragma unroll
        for (int w = 0; w < kKaWarps; ++w) {
            const float mw = ml[(w * HEADS + h) * 2];
            f[w] = mw == -INFINITY ? 0.0f : kv4_ex2(mw - top);
            // (a warp without entries has zeros; one whose statistics are NaN passes them on)
            sum = fmaf(ml[(w * HEADS + h) * 2 + 1], mw == -INFINITY ? 1.0f : f[w], sum);
        }
        const uint32_t head = kvh * p.group + h0 + h;
        if (p.part) {
            const size_t at = (size_t(s) * p.t.num_heads + head) * p.splits + split;
            float* dst = p.part + at * HD;
#pragma unroll
            for (uint32_t i = 0; i < HD / 32; ++i) {
                float v = 0.0f;
#pragma unroll
                for (int w = 0; w < kKaWarps; ++w) v = fmaf(acc[(w * HEADS + h) * HD + i * 32 + lane], f[w], v);
                dst[i * 32 + lane] = v;
            }
            if (lane == 0) p.stat[at] = make_float2(top, sum);
        } else {
            const float inv = n ? 1.0f / sum : 0.0f;
#pragma unroll
            for (uint32_t i = 0; i < HD / 32; ++i) {
                float v = 0.0f;
#pragma unroll
                for (int w = 0; w < kKaWarps; ++w) v = fmaf(acc[(w * HEADS + h) * HD + i * 32 + lane], f[w], v);
                const size_t at = s * p.t.out_row + head * HD + i * 32 + lane;
                if (p.t.dtype == SMOE_DTYPE_F32) static_cast<float*>(p.t.out)[at] = v * inv;
                else static_cast<__nv_bfloat16*>(p.t.out)[at] = __float2bfloat16_rn(v * inv);
            }
        }
    }
}

// The parts of a (sequence, KV head): its query heads' results from the
// splits in their order, and - with weights - each entry's new weight from
// the stored scores and the heads' joined maximum and sum. grid (x, KV head,
// sequence): every CTA forms the statistics it needs again; the first
// `outs` take kKjOuts outputs each (four threads an output, a quarter of
// the splits each, so that the chain of loads is short), the others 1024
// entries each.
constexpr int kKjThreads = 256, kKjOuts = 64, kKjEntries = 4 * kKjThreads;
__global__ void __launch_bounds__(kKjThreads) k_kv4_join(const Kv4Attn p, uint32_t outs) {
    extern __shared__ float kv4_join_smem[];     // [group] log2 of the sum of exponentials; weights of the splits
    __shared__ float part_sum[kKjThreads];
    pdl_release();
    pdl_acquire();
    const SmoeKv4Cache& c = p.a.c;
    const uint32_t kvh = blockIdx.y, s = blockIdx.z, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, HD = c.head_dim;
    const uint32_t n = kv4_valid(p, s), pages = (n + kKvPage - 1) / kKvPage;
    const uint32_t splits = (pages + p.split_pages - 1) / p.split_pages;       // those that have entries
    const bool is_out = blockIdx.x < outs;
    const uint32_t e0 = (blockIdx.x - outs) * kKjEntries;
    if (!is_out && e0 >= n) return;
    const size_t first = (size_t(s) * p.t.num_heads + kvh * p.group) * p.splits;
    // an output CTA's 64 outputs belong to one head (head_dim is 64 or 128)
    const uint32_t h_lo = is_out ? blockIdx.x * kKjOuts / HD : 0u, h_hi = is_out ? h_lo + 1 : p.group;
    float* lse = kv4_join_smem;
    float* wgt = kv4_join_smem + p.group;        // [splits] of the output CTA's head: its share of the whole
    for (uint32_t h = h_lo + warp; h < h_hi; h += kKjThreads / 32) {
        const float2* st = p.stat + first + size_t(h) * p.splits;
        float mx = -INFINITY, sum = 0.0f;
        for (uint32_t i = lane; i < splits; i += 32) mx = fmaxf(mx, st[i].x);
#pragma unroll
        for (int o = 16; o; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
        for (uint32_t i = lane; i < splits; i += 32)
            sum = fmaf(st[i].y, st[i].x == -INFINITY ? 1.0f : kv4_ex2(st[i].x - mx), sum);
#pragma unroll
        for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        if (lane == 0) lse[h] = mx + log2f(sum);
        if (is_out) {
            const float inv = 1.0f / sum;
            for (uint32_t i = lane; i < splits; i += 32) wgt[i] = st[i].x == -INFINITY ? sum * 0.0f : kv4_ex2(st[i].x - mx) * inv;
        }
    }
    __syncthreads();
    if (is_out) {
        const uint32_t q = tid / kKjOuts, d = (blockIdx.x * kKjOuts + tid % kKjOuts) % HD;
        const float* src = p.part + (first + size_t(h_lo) * p.splits) * HD + d;
        float v = 0.0f;
#pragma unroll 8
        for (uint32_t j = q; j < splits; j += kKjThreads / kKjOuts) v = fmaf(src[size_t(j) * HD], wgt[j], v);
        part_sum[tid] = v;
        __syncthreads();
        if (tid < kKjOuts) {
            v = (part_sum[tid] + part_sum[tid + kKjOuts]) + (part_sum[tid + 2 * kKjOuts] + part_sum[tid + 3 * kKjOuts]);
            const size_t at = s * p.t.out_row + (kvh * p.group + h_lo) * HD + d;
            if (p.t.dtype == SMOE_DTYPE_F32) static_cast<float*>(p.t.out)[at] = v;
            else static_cast<__nv_bfloat16*>(p.t.out)[at] = __float2bfloat16_rn(v);
        }
        return;
    }
    const float* row = p.logits + (size_t(s) * c.num_kv_heads + kvh) * p.rows * p.gs;
    float w[4], old[4];
    size_t at[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const uint32_t e = e0 + k * kKjThreads + tid, page = e < n ? kv4_page(c, s, e, p.a.err) : ~0u;
        at[k] = page == ~0u ? ~size_t(0) : (size_t(page) * c.num_kv_heads + kvh) * kKvPage + e % kKvPage;
        old[k] = page != ~0u && c.score && p.t.decay != 0.0f ? c.score[at[k]] * p.t.decay : 0.0f;
        w[k] = 0.0f;
    }
    uint32_t h = 0;
    if (p.gs % 4 == 0)
        for (; h + 4 <= p.group; h += 4) {
            float4 y[4];
#pragma unroll
            for (int k = 0; k < 4; ++k)
                y[k] = at[k] == ~size_t(0) ? make_float4(0.f, 0.f, 0.f, 0.f)
                                           : *reinterpret_cast<const float4*>(row + size_t(e0 + k * kKjThreads + tid) * p.gs + h);
#pragma unroll
            for (int k = 0; k < 4; ++k)
                w[k] += (kv4_ex2(y[k].x - lse[h]) + kv4_ex2(y[k].y - lse[h + 1])) + (kv4_ex2(y[k].z - lse[h + 2]) + kv4_ex2(y[k].w - lse[h + 3]));
        }
    for (; h < p.group; ++h)
#pragma unroll
        for (int k = 0; k < 4; ++k)
            if (at[k] != ~size_t(0)) w[k] += kv4_ex2(row[size_t(e0 + k * kKjThreads + tid) * p.gs + h] - lse[h]);
#pragma unroll
    for (int k = 0; k < 4; ++k)
        if (at[k] != ~size_t(0)) p.t.score_out[at[k]] = old[k] + w[k];
}

// ----------------------------------------------------------------- eviction
struct Kv4Evict {
    Kv4Args a;
    uint32_t keep, recent, max_len;
    uint32_t* pos_out;                           // null: in place
    float* score_out;
    uint32_t* lists;                             // per (sequence, KV head): moved count, then targets, then sources
    uint32_t cap, stride;                        // moves a pair can have, u32s of one pair's list
};

// Order of the scores as unsigned integers, NaN lowest; -0 and 0 are equal.
SMOE_DEVINL uint32_t kv4_rank_key(float x) {
    if (x != x) return 0u;
    const uint32_t b = __float_as_uint(x + 0.0f);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
constexpr uint32_t kKvLate = 0xffffffffu;        // key of an entry that stays for its position (above +inf's)

constexpr int kEvThreads = 1024;

// One CTA per (KV head, sequence). The keep-th largest key comes out of four
// passes over histograms of its bytes; the entries above it stay, and of
// those equal to it the lowest. Then each warp walks its own stretch of
// entries 32 at a time (ballots and population counts give the ranks) and
// lists free entries below `keep` and kept ones past it, both ascending.
__global__ void __launch_bounds__(kEvThreads) k_kv4_evict_select(Kv4Evict p) {
    pdl_release();
    pdl_acquire();
    __shared__ uint32_t hist[256], wsum[32], wsum2[32], pick[2];
    const SmoeKv4Cache& c = p.a.c;
    const uint32_t kvh = blockIdx.x, s = blockIdx.y, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    uint32_t* list = p.lists + (size_t(s) * c.num_kv_heads + kvh) * p.stride;
    uint32_t n = ld_plain(c.len + s);
    if (n > p.max_len) {
        if (tid == 0) serve_err(p.a.err, SMOE_DEVERR_BAD_RANGE);
        n = p.max_len;
    }
    if (n <= p.keep) {
        if (tid == 0) list[0] = 0;
        return;
    }
    const uint32_t seen = ld_plain((c.seen ? c.seen : c.len) + s);
    auto key_of = [&](uint32_t e) -> uint32_t {
        const uint32_t page = kv4_page(c, s, e, p.a.err);
        if (page == ~0u) return 0u;
        const size_t i = (size_t(page) * c.num_kv_heads + kvh) * kKvPage + e % kKvPage;
        return uint64_t(c.pos[i]) + p.recent >= seen ? kKvLate : kv4_rank_key(c.score[i]);
    };
    uint32_t prefix = 0, need = p.keep;          // need: kept entries among those that share the prefix
    for (int shift = 24; shift >= 0; shift -= 8) {
        for (uint32_t i = tid; i < 256; i += kEvThreads) hist[i] = 0;
        __syncthreads();
        for (uint32_t e = tid; e < n; e += kEvThreads) {
            const uint32_t k = key_of(e);
            if (shift == 24 || (k ^ prefix) >> (shift + 8) == 0) atomicAdd(&hist[k >> shift & 255u], 1u);
        }
        __syncthreads();
        if (tid == 0) {
            uint32_t left = need, b = 255;
            while (b && hist[b] < left) left -= hist[b--];
            pick[0] = b;
            pick[1] = left;
        }
        __syncthreads();
        prefix |= pick[0] << shift;
        need = pick[1];
        __syncthreads();
    }
    // the warp's stretch of entries, whole words of 32
    const uint32_t words = (n + 31) / 32, per = (words + 31) / 32, w0 = min(words, warp * per), w1 = min(words, w0 + per);
    uint32_t equal = 0;
    for (uint32_t w = w0; w < w1; ++w) {
        const uint32_t e = w * 32 + lane;
        equal += __popc(__ballot_sync(0xffffffffu, e < n && key_of(e) == prefix));
    }
    if (lane == 0) wsum[warp] = equal;
    __syncthreads();
    uint32_t before = 0;
    for (uint32_t i = 0; i < warp; ++i) before += wsum[i];
    __syncthreads();
    for (int pass = 0; pass < 2; ++pass) {       // 0: counts of the stretch, 1: the lists
        uint32_t eq = before, nfree = 0, nfar = 0, free0 = 0, far0 = 0;
        if (pass) {
            for (uint32_t i = 0; i < warp; ++i) {
                free0 += wsum[i];
                far0 += wsum2[i];
            }
            if (tid == 0) {
                uint32_t all = 0;
                for (uint32_t i = 0; i < 32; ++i) all += wsum2[i];
                list[0] = min(all, p.cap);
            }
        }
        for (uint32_t w = w0; w < w1; ++w) {
            const uint32_t e = w * 32 + lane, k = e < n ? key_of(e) : 0u;
            const uint32_t eqs = __ballot_sync(0xffffffffu, e < n && k == prefix), low = (1u << lane) - 1u;
            const bool stays = e < n && (k > prefix || (k == prefix && eq + __popc(eqs & low) < need));
            eq += __popc(eqs);
            const bool is_free = e < n && e < p.keep && !stays, is_far = stays && e >= p.keep;
            const uint32_t frees = __ballot_sync(0xffffffffu, is_free), fars = __ballot_sync(0xffffffffu, is_far);
            if (pass) {
                const uint32_t i = free0 + nfree + __popc(frees & low), j = far0 + nfar + __popc(fars & low);
                if (is_free && i < p.cap) list[1 + i] = e;
                if (is_far && j < p.cap) list[1 + p.cap + j] = e;
            }
            nfree += __popc(frees);
            nfar += __popc(fars);
        }
        if (!pass) {
            if (lane == 0) {
                wsum[warp] = nfree;
                wsum2[warp] = nfar;
            }
            __syncthreads();
        }
    }
}

// The moves of a (KV head, sequence): one warp a pair, 128 bytes of codes as
// one word a lane (head_dim 128), scales and biases, pos and score by the
// lanes after. Sources are past `keep` and targets below it, so no move reads
// what another writes. With separate outputs, pos and score of every entry
// below min(len, keep) are written: first all, then the moved ones by the
// warps that move them - of an entry only one of the two.
__global__ void __launch_bounds__(256) k_kv4_evict_move(Kv4Evict p) {
    pdl_release();
    pdl_acquire();
    const SmoeKv4Cache& c = p.a.c;
    const Kv4Geom G(c.head_dim);
    const uint32_t kvh = blockIdx.y, s = blockIdx.z, lane = threadIdx.x & 31;
    const uint32_t* list = p.lists + (size_t(s) * c.num_kv_heads + kvh) * p.stride;
    const uint32_t moves = list[0], warps = gridDim.x * 8;
    auto index = [&](uint32_t e, uint32_t page) { return (size_t(page) * c.num_kv_heads + kvh) * kKvPage + e % kKvPage; };
    float* score_out = p.score_out ? p.score_out : c.score;
    uint32_t* pos_out = p.pos_out ? p.pos_out : c.pos;
    for (uint32_t m = blockIdx.x * 8 + (threadIdx.x >> 5); m < moves; m += warps) {
        const uint32_t to = list[1 + m], from = list[1 + p.cap + m];
        const uint32_t pt = kv4_page(c, s, to, p.a.err), pf = kv4_page(c, s, from, p.a.err);
        if (pt == ~0u || pf == ~0u) continue;
        uint8_t* bt = c.blocks + (size_t(pt) * c.num_kv_heads + kvh) * G.block;
        const uint8_t* bf = c.blocks + (size_t(pf) * c.num_kv_heads + kvh) * G.block;
        const uint32_t st = to % kKvPage, sf = from % kKvPage;
        if (lane < G.ng * 16)                    // plane lane / 8, word lane % 8 of its 32 bytes
            *reinterpret_cast<uint32_t*>(bt + lane / 8 * kKvPlane + st * 32 + lane % 8 * 4) =
                *reinterpret_cast<const uint32_t*>(bf + lane / 8 * kKvPlane + sf * 32 + lane % 8 * 4);
        if (lane < G.ng * 2)
            *reinterpret_cast<uint32_t*>(bt + G.sb(0, 0) + lane * kKvPage * 4 + st * 4) =
                *reinterpret_cast<const uint32_t*>(bf + G.sb(0, 0) + lane * kKvPage * 4 + sf * 4);
        if (lane == 8) pos_out[index(to, pt)] = c.pos[index(from, pf)];
        if (lane == 9) score_out[index(to, pt)] = c.score[index(from, pf)];
    }
    if (!p.pos_out) return;
    uint32_t n = min(ld_plain(c.len + s), min(p.max_len, p.keep));
    for (uint32_t e = blockIdx.x * 256 + threadIdx.x; e < n; e += gridDim.x * 256) {
        uint32_t lo = 0, hi = moves;             // is e a target? (targets ascend)
        while (lo < hi) {
            const uint32_t mid = (lo + hi) / 2;
            if (list[1 + mid] < e) lo = mid + 1;
            else hi = mid;
        }
        if (lo < moves && list[1 + lo] == e) continue;
        const uint32_t page = kv4_page(c, s, e, p.a.err);
        if (page == ~0u) continue;
        pos_out[index(e, page)] = c.pos[index(e, page)];
        score_out[index(e, page)] = c.score[index(e, page)];
    }
}

__global__ void __launch_bounds__(256) k_kv4_advance(uint32_t* len, uint32_t* seen, uint32_t n_seqs, const uint32_t* cu,
                                                     uint32_t n_each, uint32_t keep) {
    pdl_release();
    pdl_acquire();
    const uint32_t s = blockIdx.x * 256 + threadIdx.x;
    if (s >= n_seqs) return;
    const uint32_t n = cu ? cu[s + 1] - cu[s] : n_each, l = len[s] + n;
    len[s] = keep && l > keep ? keep : l;
    if (seen) seen[s] += n;
}

}  // namespace smoe
