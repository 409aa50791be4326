// kv4.cuh - the paged 4-bit KV cache: quantised append, read-back, attention
// of one query token per sequence, eviction by accumulated attention weight.
#pragma once
#include <cooperative_groups.h>

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
// A CTA takes 8 rows: a warp finds each one's entry (sequence, page, slot), and
// four lanes do a unit - a group of 64 values of a row, KV head and side - 16
// values a lane: the group's 32 bytes of codes are 8 a lane, its minimum and
// maximum two shuffles. Values are fetched before the entries are known, and
// two units a lane are in flight. Bound by the chain of look-ups (bounds,
// length, page table) for a step's rows (256 fp32 rows of 4 heads of 128: 7 us,
// their read-back 6, both cold) and by that chain and the instructions that
// find the codes for a prompt's (5,800 bf16 rows: 14 us cold, 54% of the issue
// slots used; 14,400 entries read back: 16 us). With a division for each code
// and two lanes a unit the first took 10 us, the third 26. (16 or 32 rows a
// CTA, so that all CTAs fit the GPU at once, took 1.1 and 1.3 times as long.)
constexpr int kKwRows = 8, kKwThreads = 256;

struct Kv4RowPlace {
    uint32_t page, slot, pos;                    // page ~0: nowhere
};
// The units of a CTA's rows that a group of four lanes takes, every
// kKwThreads / 4th.
struct Kv4Units {
    uint32_t units, rows, lg, dr, du;            // per row; rows here; log2 of the groups; a step in rows and units
    uint32_t row, u;
    SMOE_DEVINL Kv4Units(const Kv4Geom& G, uint32_t heads, uint32_t total) {
        constexpr uint32_t step = kKwThreads / 4;
        units = heads * 2 * G.ng;
        rows = min(uint32_t(kKwRows), total - blockIdx.x * kKwRows);
        lg = G.ng >> 1;                          // (1 or 2 groups)
        dr = step / units;
        du = step % units;
        row = (threadIdx.x >> 2) / units;
        u = (threadIdx.x >> 2) % units;
    }
    SMOE_DEVINL bool more() const { return row < rows; }
    SMOE_DEVINL uint32_t g() const { return u & ((1u << lg) - 1u); }
    SMOE_DEVINL uint32_t kv() const { return u >> lg & 1u; }
    SMOE_DEVINL uint32_t h() const { return u >> (lg + 1); }
    // element of the row's k or v where this lane's 16 values start
    SMOE_DEVINL size_t at(const SmoeKv4Rows& r) const {
        const size_t w = blockIdx.x * kKwRows + row;
        return (kv() ? w * r.v_row + h() * r.v_head : w * r.k_row + h() * r.k_head) + g() * 64 + (threadIdx.x & 3) * 16;
    }
    SMOE_DEVINL void next() {
        row += dr;
        u += du;
        if (u >= units) {
            u -= units;
            ++row;
        }
    }
};
// Sequence of a row where seq_of_row finds none: past the last one's rows, or
// starts that do not ascend, of which it may miss the row's. By one warp.
static __device__ __noinline__ uint32_t kv4_seq_by_scan(const uint32_t* cu, uint32_t n, uint32_t row, uint32_t lane) {
    for (uint32_t b = 0; b < n; b += 32) {
        const uint32_t s = b + lane;
        const uint32_t hit = __ballot_sync(0xffffffffu, s < n && ld_plain(cu + s) <= row && row < ld_plain(cu + s + 1));
        if (hit) return b + __ffs(hit) - 1;
    }
    return n;
}
// The places of the CTA's rows, a warp a row; entry = base[s] + index in the sequence.
SMOE_DEVINL void kv4_places(const Kv4Args& a, const SmoeKv4Rows& r, const uint32_t* base, Kv4RowPlace* places) {
    const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5, row = blockIdx.x * kKwRows + warp, ns = a.c.n_seqs;
    Kv4RowPlace p{~0u, 0u, 0u};
    // Each CTA reports on some of the sequences' ranges (one that is bad may have no row here): fetched first, looked at last
    const uint32_t mine = blockIdx.x * kKwThreads + threadIdx.x;
    const uint32_t from = mine < ns ? ld_plain(r.cu + mine) : 0u, to = mine < ns ? ld_plain(r.cu + mine + 1) : 0u;
    if (row < r.total) {
        // (a decode step has a row a sequence: look there first)
        uint32_t s = row, lo = row < ns ? ld_plain(r.cu + row) : ~0u, hi = row < ns ? ld_plain(r.cu + row + 1) : 0u;
        if (lo > row || row >= hi) {
            s = seq_of_row(r.cu, ns, row, lane);
            if (s >= ns) s = kv4_seq_by_scan(r.cu, ns, row, lane);
            lo = s < ns ? ld_plain(r.cu + s) : 0u;
            hi = s < ns ? ld_plain(r.cu + s + 1) : 0u;
        }
        if (s < ns && hi <= r.total) {           // (no sequence: a row past the last one's)
            const uint32_t t = row - lo;
            const uint64_t e = uint64_t(base ? ld_plain(base + s) : 0u) + t;
            if (a.c.pos) p.pos = ld_plain((a.c.seen ? a.c.seen : a.c.len) + s) + t;
            p.page = kv4_page(a.c, s, e, a.err);
            p.slot = uint32_t(e % kKvPage);
        }
    }
    if (lane == 0) places[warp] = p;
    bool bad = from > to || to > r.total;
#pragma unroll 1
    for (uint32_t s = mine + gridDim.x * kKwThreads; s < ns; s += gridDim.x * kKwThreads)
        bad |= ld_plain(r.cu + s) > ld_plain(r.cu + s + 1) || ld_plain(r.cu + s + 1) > r.total;
    if (bad) serve_err(a.err, SMOE_DEVERR_BAD_RANGE);
    __syncthreads();
}

// 16 values of a row, in pieces of 16 bytes, or of 8 where a bf16 row may start between two such.
template <int DTYPE, bool WIDE>
SMOE_DEVINL void kv4_load16(const void* p, size_t at, float* x) {
    if (DTYPE == SMOE_DTYPE_F32) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float4 v = ld_plain(reinterpret_cast<const float4*>(static_cast<const float*>(p) + at) + i);
            x[4 * i] = v.x;
            x[4 * i + 1] = v.y;
            x[4 * i + 2] = v.z;
            x[4 * i + 3] = v.w;
        }
        return;
    }
    uint32_t w[8];
    if (WIDE) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const uint4 v = ld_plain(reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(p) + at) + i);
            w[4 * i] = v.x;
            w[4 * i + 1] = v.y;
            w[4 * i + 2] = v.z;
            w[4 * i + 3] = v.w;
        }
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint2 v = ld_plain(reinterpret_cast<const uint2*>(static_cast<const uint16_t*>(p) + at) + i);
            w[2 * i] = v.x;
            w[2 * i + 1] = v.y;
        }
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        x[2 * i] = __uint_as_float(w[i] << 16);
        x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
}

// Minimum and maximum that a NaN passes through (fminf and fmaxf drop it): a
// group with a NaN has a NaN as its scale and bias, and reads back as NaN.
SMOE_DEVINL float kv4_min(float a, float b) {
    float d;
    asm("min.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
    return d;
}
SMOE_DEVINL float kv4_max(float a, float b) {
    float d;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
    return d;
}
// The code of one value by the definition.
static __device__ __noinline__ uint32_t kv4_code(float x, float bias, float scale) {
    const float q = scale > 0.0f ? rintf(__fdiv_rn(__fsub_rn(x, bias), scale)) : 0.0f;
    return uint32_t(fminf(fmaxf(q, 0.0f), 15.0f));
}
// Those of 16 values, without dividing: with d = x - bias, the whole number r
// nearest to d / scale by way of the reciprocal is right or off by one. For r
// of -1 .. 16 (others are cut to 0 or 15) r scale (5 + 8 bits) and
// u = d - r scale are exact, so |u| against scale / 2 says which, ties
// included: fl(d / scale) is exactly half-way only where d is (2 r + 1) scale / 2
// - neighbours of that number in fp32 are further from it than half a unit of
// the quotient. (bf16 values hit ties often: some in every second warp.) |u|
// and scale / 2 are compared as integers, |u| one unit up where r is odd, which
// moves ties to even. Infinities and NaN: d / scale is infinite or NaN then,
// which r takes to a value past 15 or (NaN too) to -1.
SMOE_DEVINL void kv4_codes16(const float* y, float bias, float scale, uint32_t* code) {
    code[0] = code[1] = 0u;
    if (!(scale >= 1e-37f && scale <= 3e38f)) {  // no finite reciprocal, or no positive scale
        if (scale > 0.0f)
#pragma unroll 1
            for (int k = 0; k < 2; ++k)
#pragma unroll
                for (int i = 0; i < 8; ++i) code[k] |= kv4_code(k ? y[8 + i] : y[i], bias, scale) << (4 * i);
        return;
    }
    const float inv = 1.0f / scale, magic = 12582912.0f;         // 1.5 x 2^23: adding it rounds to a whole number, in the low bits
    const uint64_t off = pack2(-bias, -bias), inv2 = pack2(inv, inv), up = pack2(magic, magic), down = pack2(-magic, -magic), step = pack2(-scale, -scale);
    const int half = __float_as_int(0.5f * scale);
#pragma unroll
    for (int w = 0; w < 2; ++w)
#pragma unroll
        for (int k = 6; k >= 0; k -= 2) {
            const uint64_t d = add2(pack2(y[8 * w + k], y[8 * w + k + 1]), off);
            float t[2], u[2];
            unpack2(fma2(d, inv2, up), t[0], t[1]);
            int c[2];
#pragma unroll
            for (int i = 0; i < 2; ++i) t[i] = fmaxf(t[i], magic - 1.0f);
            unpack2(fma2(add2(pack2(t[0], t[1]), down), step, d), u[0], u[1]);
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                c[i] = __float_as_int(t[i]) - __float_as_int(magic);
                const int v = (__float_as_int(u[i]) & 0x7fffffff) + (c[i] & 1);
                if (v > half) c[i] += __float_as_int(u[i]) >> 31 | 1;
            }
            // (cut to 0 .. 15 and put below the pairs so far)
            asm("cvt.pack.sat.u4.s32.b32 %0, %1, %2, %3;" : "=r"(code[w]) : "r"(c[1]), "r"(c[0]), "r"(code[w]));
        }
}

template <int DTYPE, bool WIDE>
__global__ void __launch_bounds__(kKwThreads, 4) k_kv4_append(Kv4Args a, SmoeKv4Rows r) {
    __shared__ Kv4RowPlace places[kKwRows];
    pdl_release();
    pdl_acquire();
    const Kv4Geom G(a.c.head_dim);
    const uint32_t j = threadIdx.x & 3;
    float x[2][16];
    auto load = [&](const Kv4Units& w, float* y) { kv4_load16<DTYPE, WIDE>(w.kv() ? r.v : r.k, w.at(r), y); };
    auto store = [&](const Kv4Units& w, const float* y) {
        const uint32_t g = w.g(), kv = w.kv(), h = w.h();
        const Kv4RowPlace p = places[w.row];
        float lo = y[0], hi = y[0];
#pragma unroll
        for (int k = 1; k < 16; ++k) {
            lo = kv4_min(lo, y[k]);
            hi = kv4_max(hi, y[k]);
        }
        const uint32_t mask = 0xfu << (threadIdx.x & 28);
#pragma unroll
        for (int o = 1; o < 4; o <<= 1) {
            lo = kv4_min(lo, __shfl_xor_sync(mask, lo, o));
            hi = kv4_max(hi, __shfl_xor_sync(mask, hi, o));
        }
        if (p.page == ~0u) return;
        const __nv_bfloat16 bb = __float2bfloat16_rn(lo);
        const __nv_bfloat16 sb = __float2bfloat16_rn(__fmul_rn(__fsub_rn(hi, lo), 1.0f / 15.0f));
        const float bias = __bfloat162float(bb), scale = __bfloat162float(sb);
        uint32_t code[2];
        kv4_codes16(y, bias, scale, code);
        uint8_t* blk = a.c.blocks + (size_t(p.page) * a.c.num_kv_heads + h) * G.block;
        *reinterpret_cast<uint2*>(blk + G.codes(kv, g) + p.slot * 32 + j * 8) = make_uint2(code[0], code[1]);
        if (j == 0) {
            *reinterpret_cast<uint32_t*>(blk + G.sb(kv, g) + p.slot * 4) =
                uint32_t(__bfloat16_as_ushort(sb)) | uint32_t(__bfloat16_as_ushort(bb)) << 16;
            if (kv == 0 && g == 0) {
                const size_t at = (size_t(p.page) * a.c.num_kv_heads + h) * kKvPage + p.slot;
                if (a.c.pos) a.c.pos[at] = p.pos;
                if (a.c.score) a.c.score[at] = 0.0f;
            }
        }
    };
    Kv4Units w(G, a.c.num_kv_heads, r.total), ahead = w;
    if (w.more()) load(w, x[0]);
    ahead.next();
    if (ahead.more()) load(ahead, x[1]);
    kv4_places(a, r, a.c.len, places);
#pragma unroll 1
    for (; w.more(); w.next()) {
        store(w, x[0]);
#pragma unroll
        for (int k = 0; k < 16; ++k) x[0][k] = x[1][k];
        ahead.next();
        if (ahead.more()) load(ahead, x[1]);
    }
}

template <int DTYPE, bool WIDE>
__global__ void __launch_bounds__(kKwThreads) k_kv4_read(Kv4Args a, const uint32_t* first, SmoeKv4Rows r) {
    __shared__ Kv4RowPlace places[kKwRows];
    pdl_release();
    pdl_acquire();
    const Kv4Geom G(a.c.head_dim);
    const uint32_t j = threadIdx.x & 3;
    kv4_places(a, r, first, places);
    Kv4Units w(G, a.c.num_kv_heads, r.total);
#pragma unroll 1
    while (w.more()) {
        Kv4Units at[2] = {w, w};
        at[1].next();
        w = at[1];
        w.next();
        uint2 code[2];
        uint32_t sb[2];
#pragma unroll
        for (int q = 0; q < 2; ++q) {
            const uint32_t g = at[q].g(), kv = at[q].kv(), h = at[q].h();
            code[q] = make_uint2(0u, 0u);
            sb[q] = 0u;
            if (!at[q].more()) continue;
            const Kv4RowPlace p = places[at[q].row];
            if (p.page == ~0u) continue;
            const uint8_t* blk = a.c.blocks + (size_t(p.page) * a.c.num_kv_heads + h) * G.block;
            code[q] = ld_plain(reinterpret_cast<const uint2*>(blk + G.codes(kv, g) + p.slot * 32 + j * 8));
            sb[q] = ld_plain(reinterpret_cast<const uint32_t*>(blk + G.sb(kv, g) + p.slot * 4));
        }
#pragma unroll
        for (int q = 0; q < 2; ++q) {
            if (!at[q].more() || places[at[q].row].page == ~0u) continue;
            const float scale = __uint_as_float(sb[q] << 16), bias = __uint_as_float(sb[q] & 0xffff0000u);
            float v[16];
#pragma unroll
            for (int k = 0; k < 16; ++k)
                v[k] = __fadd_rn(__fmul_rn(float((k < 8 ? code[q].x : code[q].y) >> (4 * (k % 8)) & 15u), scale), bias);
            const size_t to = at[q].at(r);
            void* dst = at[q].kv() ? r.v : r.k;
            if (DTYPE == SMOE_DTYPE_F32) {
                float4* d = reinterpret_cast<float4*>(static_cast<float*>(dst) + to);
#pragma unroll
                for (int k = 0; k < 4; ++k) d[k] = make_float4(v[4 * k], v[4 * k + 1], v[4 * k + 2], v[4 * k + 3]);
                continue;
            }
            uint32_t w[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) w[k] = pack_bf16x2(v[2 * k], v[2 * k + 1]);
            if (WIDE) {
                uint4* d = reinterpret_cast<uint4*>(static_cast<uint16_t*>(dst) + to);
                d[0] = make_uint4(w[0], w[1], w[2], w[3]);
                d[1] = make_uint4(w[4], w[5], w[6], w[7]);
            } else {
                uint2* d = reinterpret_cast<uint2*>(static_cast<uint16_t*>(dst) + to);
#pragma unroll
                for (int k = 0; k < 4; ++k) d[k] = make_uint2(w[2 * k], w[2 * k + 1]);
            }
        }
    }
}

// ---------------------------------------------------------------- attention
// One query token per sequence. With a group's codes c (0..15), scales s and
// biases b, and c' = c - 8, b' = b + 8 s:
//   q . k = sum_g s_g (q_g . c'_g) + b'_g sum(q_g)
//   sum_j p_j v_j = sum_j (p_j s_j) c'_j + sum_j p_j b'_j        (per group)
// so the codes are the tensor cores' operands (exact in fp16) and scales and
// biases stay in fp32. (c' and not c: the two sums then do not cancel - fp32
// results were four times as far from 64 bits with c.) q goes in as one (bf16 q) or two fp16 pieces, each
// head scaled by a power of two so that its largest value is near 2^14; p s
// as two fp16 pieces (22 bits), times a power of two per group and head that
// follows the largest products. (bf16 pieces need no such power, but three
// more instructions for every 16 codes.)
// The entries are the M rows of both products and 8 of a KV head's query
// heads the N columns. (16 at a time halve the unpacking of wide groups, but
// need 255 registers: 8 warps an SM instead of 12, and 1.2 times the time.)
//
// All pages of all (sequence, KV head) pairs, in one line, are cut into equal
// stretches, one a warp of a grid that fills the GPU once: ragged lengths do
// not matter, and no warp waits for another. A warp copies its pages' keys and
// values, by turns, into a ring of three of its own (166 KB an SM), and for
// each pair that its stretch touches it keeps a running maximum, sums and
// accumulators. A pair inside one stretch is done (unless weights are
// wanted); the parts of the others are stored and joined by k_kv4_join. The
// part of (warp, pair) has the number warp + pair: along the line at least
// one of the two grows from a part to the next, so no two share one.
//
// Bound by each warp's chain: 16 entries cost about 400 warp instructions (the
// codes' unpacking on the integer units, the probabilities' pieces), a page
// takes a warp 5 us, and the 12 warps an SM that their registers allow use 53%
// of the issue slots. Two contexts of 125,000 (head_dim 128, 32 / 4 heads,
// bf16, weights): 64 us with the join for 156 MB, 2.4 TB/s (3.9 TB/s once the
// rings run; the first pages come in after 7 us, warps end between 37 and 56).
// 32 contexts of 512 to 8,192: 33 us with the join; one of 300: 11 us, of
// which most is the two launches. (A power of two per group alone, by the
// largest scale whatever its weight, is 1 to 2% faster, and wrong in the first
// digit where a value 2^30 times the others has no weight.)
constexpr int kKaWarps = 4, kKaStages = 3;
constexpr uint32_t kKaCtas = 3, kKaGrid = 148 * kKaCtas, kKaHeads = 8;

struct Kv4Attn {
    Kv4Args a;
    SmoeKv4AttnArgs t;
    uint32_t group, chunks;                      // query heads per KV head; rounds of 8 heads that makes
    uint32_t warps;                              // of the grid
    float* part;                                 // [warps + pairs][8 heads][head_dim] weighted sums
    float2* stat;                                // [warps + pairs][8 heads] maximum, sum
    uint2* meta;                                 // [pairs] first warp of a pair with entries, number of its parts
    uint32_t lanes;                              // k_kv4_join: threads that share an output's parts (a power of two)
    float* logits;                               // [n_seqs][num_heads][rows] log2-scaled scores, with weights
    uint32_t rows;                               // max_len rounded up to a page
    float scale_log2;                            // positive
    int most_e;                                  // largest power of two that q may go in with
};

// Entries of sequence s that the token attends to.
SMOE_DEVINL uint32_t kv4_valid(const Kv4Attn& p, uint32_t s) {
    const uint64_t n = uint64_t(ld_plain(p.a.c.len + s)) + p.t.extra;
    if (n > p.t.max_len) {
        serve_err(p.a.err, SMOE_DEVERR_BAD_RANGE);
        return p.t.max_len;
    }
    return uint32_t(n);
}
SMOE_DEVINL uint32_t kv4_pages(uint32_t n) { return (n + kKvPage - 1) / kKvPage; }

// The line of pages: sequence s starts at heads * (pages of the sequences
// before it), `heads` pairs of equal length each. (Below 2^31 pages: the host
// refuses more.)
// Stretches are equal up to a page. Those below 3 pages are all rounded up
// instead, which leaves some warps without: they cut fewer pairs. 2, 32 and 100
// contexts, head_dim 128, call after call: rounding takes 2 to 8% less at 1.5
// pages a warp, from 1.5% less to 4% more at 3.5 and 4.9, and 2 to 5% more at
// 6.5 to 14.5.
struct Kv4Line {
    uint32_t total, each, more;                  // pages; pages of a stretch, the first `more` of them have one more
    SMOE_DEVINL Kv4Line(uint32_t pages, uint32_t warps) : total(pages), each(pages / warps), more(pages % warps) {
        if (each < 3) {
            each = max(1u, each + (more != 0));
            more = 0;
        }
    }
    SMOE_DEVINL uint32_t first(uint32_t w) const { return uint32_t(min(uint64_t(total), uint64_t(w) * each + min(w, more))); }
    SMOE_DEVINL uint32_t warp_of(uint32_t page) const {
        const uint32_t longer = more * (each + 1);
        return page < longer ? page / (each + 1) : more + (page - longer) / each;
    }
};
// By a whole warp: the line, and the sequence that holds warp w's first page
// with the page of the line that it starts at.
SMOE_DEVINL Kv4Line kv4_line(const Kv4Attn& p, uint32_t heads, uint32_t lane, uint32_t w, uint32_t& seq, uint32_t& start) {
    const uint32_t ns = p.a.c.n_seqs;
    uint32_t total = 0, before = 0, n = 0;
#pragma unroll 1
    for (uint32_t b = 0; b < ns; b += 32) {
        const uint32_t s = b + lane;
        n = s < ns ? kv4_pages(kv4_valid(p, s)) : 0u;
        total += __reduce_add_sync(0xffffffffu, n);
    }
    const Kv4Line L(total * heads, p.warps);
    const uint32_t want = L.first(w);
    seq = ns;
    start = 0;
    if (want >= L.total) return L;
#pragma unroll 1
    for (uint32_t b = 0; b < ns; b += 32) {
        const uint32_t s = b + lane;
        if (ns > 32) n = s < ns ? kv4_pages(kv4_valid(p, s)) : 0u;             // (else they are still at hand)
        uint32_t incl = n;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const uint32_t v = __shfl_up_sync(0xffffffffu, incl, o);
            if (lane >= uint32_t(o)) incl += v;
        }
        const uint32_t hit = __ballot_sync(0xffffffffu, (before + incl) * heads > want);
        if (hit) {
            const int l = __ffs(hit) - 1;
            seq = b + l;
            start = (before + __shfl_sync(0xffffffffu, incl - n, l)) * heads;
            return L;
        }
        before += __shfl_sync(0xffffffffu, incl, 31);
    }
    return L;
}

// 8 codes less 8 as fp16 pairs (code n, code n + 4): 1024 + c and 1024 + 16 c
// are exact, and so is what the subtraction or the multiply-add makes of them.
SMOE_DEVINL void kv4_half_codes(uint32_t w, uint32_t* r) {
    constexpr uint32_t M0 = 0x000F000Fu, M1 = 0x00F000F0u, ONE = 0x64006400u;
    const uint32_t w8 = w >> 8;
    asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(r[0]) : "r"(lop3_and_or(w, M0, ONE)), "r"(0x64086408u));
    asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(r[1]) : "r"(lop3_and_or(w, M1, ONE)), "r"(0x2C002C00u), "r"(0xD480D480u));
    asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(r[2]) : "r"(lop3_and_or(w8, M0, ONE)), "r"(0x64086408u));
    asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(r[3]) : "r"(lop3_and_or(w8, M1, ONE)), "r"(0x2C002C00u), "r"(0xD480D480u));
}
SMOE_DEVINL void mma_f16f32_16816(float* d, const uint32_t* a, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
SMOE_DEVINL void mma_f16f32_16816_z(float* d, const uint32_t* a, uint32_t b0, uint32_t b1) {      // from zero
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.0f));
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

// 16 consecutive values of a head's group.
SMOE_DEVINL void kv4_load_q(const void* q, size_t at, int dtype, float* x) {
    if (dtype == SMOE_DTYPE_F32) {
        const float4* src = reinterpret_cast<const float4*>(static_cast<const float*>(q) + at);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float4 v = src[i];
            x[4 * i] = v.x;
            x[4 * i + 1] = v.y;
            x[4 * i + 2] = v.z;
            x[4 * i + 3] = v.w;
        }
    } else {                                     // (q's rows are 8-byte aligned: strides are multiples of 4)
        const uint2* src = reinterpret_cast<const uint2*>(static_cast<const uint16_t*>(q) + at);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint2 v = src[i];
            x[4 * i] = lo_f(v.x);
            x[4 * i + 1] = hi_f(v.x);
            x[4 * i + 2] = lo_f(v.y);
            x[4 * i + 3] = hi_f(v.y);
        }
    }
}

// New powers of two of a group's sums o (heads 2 cl, 2 cl + 1 of this lane),
// where the page's scales do not fit the old ones: the larger of its largest
// p s and an eighth of the largest sum so far goes near 2^8. (What is lost
// stays below 2^-32 of the larger one; sums in fp32 have room above.) Bounded
// so that no scale of the page, the largest being `big`, and no factor of the
// sums passes fp32.
SMOE_DEVINL void kv4_new_up(const uint8_t* scales, uint32_t big, uint32_t gr, const float (&x)[4][4], float (&o)[4][4], float (&up)[2]) {
    float y[2] = {0.0f, 0.0f}, sum[2] = {0.0f, 0.0f};
#pragma unroll
    for (int mt = 0; mt < 4; ++mt) {
        const float s0 = fabsf(lo_f(*reinterpret_cast<const uint32_t*>(scales + (mt * 16 + gr) * 4)));
        const float s1 = fabsf(lo_f(*reinterpret_cast<const uint32_t*>(scales + (mt * 16 + 8 + gr) * 4)));
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            y[k] = fmaxf(y[k], fmaxf(x[mt][k] * s0, x[mt][2 + k] * s1));
            sum[k] = fmaxf(sum[k], fmaxf(fabsf(o[mt][k]), fabsf(o[mt][2 + k])));
        }
    }
#pragma unroll
    for (int k = 0; k < 2; ++k) {
#pragma unroll
        for (int d = 4; d < 32; d <<= 1) {
            y[k] = fmaxf(y[k], __shfl_xor_sync(0xffffffffu, y[k], d));
            sum[k] = fmaxf(sum[k], __shfl_xor_sync(0xffffffffu, sum[k], d));
        }
        const int was = int(__float_as_uint(up[k]) >> 23);       // biased exponents; 0: none yet
        const float top = fmaxf(y[k], was ? sum[k] * 0.125f / up[k] : 0.0f);
        int now = min(262 - int(__float_as_uint(top) >> 23), 373 - int(big >> 7));
        if (was) now = min(now, was + 100);
        now = max(1, min(227, now));
        const float next = __uint_as_float(uint32_t(now) << 23), r = was ? next / up[k] : 0.0f;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            o[j][k] *= r;
            o[j][2 + k] *= r;
        }
        up[k] = next;
    }
}

template <int NG>
constexpr uint32_t kv4_attn_smem() { return kKaWarps * kKaStages * (NG * 2304 + 8); }

// NG groups of 64 (head_dim / 64), QP pieces of q.
template <int NG, int QP>
__global__ void __launch_bounds__(kKaWarps * 32, kKaCtas) k_kv4_attention(const Kv4Attn p) {
    constexpr uint32_t HD = NG * 64, UNIT = NG * 2304, SB = NG * kKvPlane;     // a unit: a page's keys or values, codes then scales
    extern __shared__ __align__(128) uint8_t kv4_smem[];
    const SmoeKv4Cache& c = p.a.c;
    const uint32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, gr = lane >> 2, cl = lane & 3;
    const uint32_t me = blockIdx.x * kKaWarps + warp, nheads = c.num_kv_heads * p.chunks;        // pairs of a sequence
    uint8_t* ring = kv4_smem + warp * kKaStages * UNIT;
    uint64_t* bars = reinterpret_cast<uint64_t*>(kv4_smem + kKaWarps * kKaStages * UNIT) + warp * kKaStages;
    if (lane == 0) {
        for (int i = 0; i < kKaStages; ++i) mbar_init(bars + i, 1);
        fence_mbar_init();
    }
    __syncwarp();
    pdl_acquire();
    uint32_t seq;
    uint32_t start;
    const Kv4Line L = kv4_line(p, nheads, lane, me, seq, start);
    const uint32_t t0 = L.first(me), t1 = L.first(me + 1);
    if (t0 >= t1) return;
    const uint32_t mine = t1 - t0;

    // where the stretch starts, and the next unit to send for (ahead of the one in work)
    uint32_t n = kv4_valid(p, seq), np = kv4_pages(n), hc = (t0 - start) / np, pg = (t0 - start) % np;
    uint32_t a_seq = seq, a_np = np, a_hc = hc, a_pg = pg, sent = 0;
    uint32_t a_page = 0, good = 0, slot = 0, phase = 0;          // good: bit i % 2, page i can be read; slot, phase: of the unit in work
    auto send = [&](uint32_t st) {               // unit `sent`, into slot st
        if (sent % 2 == 0) {
            a_page = kv4_page(c, a_seq, uint64_t(a_pg) * kKvPage, p.a.err);
            good = (good & ~(1u << (sent / 2 % 2))) | uint32_t(a_page != ~0u) << (sent / 2 % 2);
        }
        if (elect_one()) {
            if (a_page != ~0u) {
                const uint8_t* blk = c.blocks + (size_t(a_page) * c.num_kv_heads + a_hc / p.chunks) * (2 * UNIT);
                mbar_arrive_expect_tx(bars + st, UNIT);
                bulk_g2s(ring + st * UNIT, blk + sent % 2 * SB, SB, bars + st);
                bulk_g2s(ring + st * UNIT + SB, blk + 2 * SB + sent % 2 * (UNIT - SB), UNIT - SB, bars + st);
            } else {
                mbar_arrive(bars + st);          // nothing to wait for; its entries are masked
            }
        }
        if (++sent % 2 == 0 && sent < 2 * mine && ++a_pg == a_np) {
            a_pg = 0;
            if (++a_hc == nheads) {
                a_hc = 0;
                do a_np = kv4_pages(kv4_valid(p, ++a_seq));
                while (a_np == 0);               // (a page is still to come, so there is a sequence that has it)
            }
        }
    };
    for (int i = 0; i < kKaStages; ++i)
        if (sent < 2 * mine) send(i);

    uint32_t qf[NG][4][QP][2];                   // fragments of q: head gr, dimensions in the order kv4_half_codes gives the codes
    float qsm[NG][2], sc[2];                     // of the heads 2 cl, 2 cl + 1: the groups' sums; scale_log2 over the head's power of two
    float m[2], l[2], bacc[NG][2], o[NG][4][4], up[NG][2];       // up: the power of two of the group's sums in o, for each head
    bool failed = false, fresh = true;           // fresh: the pair starts with this page
    uint32_t heads = 0, head0 = 0;               // of the pair: query heads and the first of them
    float* lrow = nullptr;
    auto arrived = [&]() {
        if (!failed && !mbar_wait_bounded(bars + slot, phase)) {
            failed = true;                       // (the results are void, the error word says so)
            atomicCAS(p.a.err, 0u, uint32_t(SMOE_DEVERR_MBAR_TIMEOUT));
        }
    };
    auto read = [&]() {                          // the unit in work has been read: its slot for the one three further on
        __syncwarp();
        if (sent < 2 * mine) send(slot);
        if (++slot == uint32_t(kKaStages)) {
            slot = 0;
            phase ^= 1u;
        }
    };
#pragma unroll 1
    for (uint32_t i = 0; i < mine; ++i) {
        if (fresh) {
            fresh = false;
            if (pg == 0 && lane == 0)            // this warp is the pair's first one
                p.meta[uint64_t(seq) * nheads + hc] = make_uint2(me, L.warp_of(t0 + i + np - 1) - me + 1);
            const uint32_t kvh = hc / p.chunks, h0 = hc % p.chunks * kKaHeads;
            heads = min(kKaHeads, p.group - h0);
            head0 = kvh * p.group + h0;
            lrow = p.logits ? p.logits + (size_t(seq) * p.t.num_heads + head0 + 2 * cl) * p.rows + gr : nullptr;
            float x[NG][16], mx = 0.0f, sum[NG];
#pragma unroll
            for (int g = 0; g < NG; ++g) {
                if (gr < heads) kv4_load_q(p.t.q, seq * p.t.q_row + size_t(head0 + gr) * HD + g * 64 + cl * 16, p.t.dtype, x[g]);
#pragma unroll
                for (int d = 0; d < 16; ++d) {
                    if (gr >= heads) x[g][d] = 0.0f;
                    mx = fmaxf(mx, fabsf(x[g][d]));
                }
            }
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
            // 2^e with mx 2^e in [2^14, 2^15), kept within what fp32 can invert (an infinity or NaN in q stays one) and
            // low enough for scale_log2 / 2^e to be a normal number: at 0 it would make NaN of the masked scores
            const int e = max(-100, min(p.most_e, 14 - (int(__float_as_uint(mx) >> 23) - 127)));
            const float by = __uint_as_float(uint32_t(127 + e) << 23), inv = p.scale_log2 * __uint_as_float(uint32_t(127 - e) << 23);
#pragma unroll
            for (int g = 0; g < NG; ++g) {
                sum[g] = 0.0f;
#pragma unroll
                for (int st = 0; st < 4; ++st)
#pragma unroll
                    for (int b = 0; b < 2; ++b) {
                        const int d = st / 2 * 8 + st % 2 * 2 + b;
                        const float y0 = x[g][d] * by, y1 = x[g][d + 4] * by;
                        const uint32_t hi = cvt_f16x2(y0, y1);
                        qf[g][st][0][b] = hi;
                        sum[g] += half_lo(hi) + half_hi(hi);
                        if (QP == 2) {
                            const uint32_t lo = cvt_f16x2(y0 - half_lo(hi), y1 - half_hi(hi));
                            qf[g][st][QP - 1][b] = lo;
                            sum[g] += half_lo(lo) + half_hi(lo);
                        }
                    }
                sum[g] += __shfl_xor_sync(0xffffffffu, sum[g], 1);
                sum[g] += __shfl_xor_sync(0xffffffffu, sum[g], 2);
                up[g][0] = up[g][1] = 0.0f;
            }
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                const int from = (2 * cl + k) * 4;
                sc[k] = __shfl_sync(0xffffffffu, inv, from);
                m[k] = -INFINITY;
                l[k] = 0.0f;
#pragma unroll
                for (int g = 0; g < NG; ++g) {
                    qsm[g][k] = __shfl_sync(0xffffffffu, sum[g], from);
                    bacc[g][k] = 0.0f;
#pragma unroll
                    for (int j = 0; j < 4; ++j) o[g][j][k] = o[g][j][2 + k] = 0.0f;
                }
            }
        }
        const uint32_t e0 = pg * kKvPage;
        const uint32_t have = good >> (i % 2) & 1u ? min(kKvPage, n - e0) : 0u;                // entries of this page
        const uint8_t* blk = ring + slot * UNIT;
        arrived();
        float x[4][4];                           // scores: entry 16 mt + gr (0, 1) and + 8 (2, 3), heads 2 cl, 2 cl + 1
#pragma unroll
        for (int mt = 0; mt < 4; ++mt) {
            const uint32_t ka = mt * 16 + gr, kb = ka + 8;
            uint2 wa[NG], wb[NG];
            uint32_t sa[NG], sb[NG];
            float d[NG][4];
#pragma unroll
            for (int g = 0; g < NG; ++g) {
                wa[g] = *reinterpret_cast<const uint2*>(blk + g * kKvPlane + ka * 32 + cl * 8);
                wb[g] = *reinterpret_cast<const uint2*>(blk + g * kKvPlane + kb * 32 + cl * 8);
                sa[g] = *reinterpret_cast<const uint32_t*>(blk + SB + g * 256 + ka * 4);
                sb[g] = *reinterpret_cast<const uint32_t*>(blk + SB + g * 256 + kb * 4);
            }
#pragma unroll
            for (int w = 0; w < 2; ++w) {        // (the groups' chains of products side by side)
                uint32_t ra[NG][4], rb[NG][4];
#pragma unroll
                for (int g = 0; g < NG; ++g) {
                    kv4_half_codes(w ? wa[g].y : wa[g].x, ra[g]);
                    kv4_half_codes(w ? wb[g].y : wb[g].x, rb[g]);
                }
#pragma unroll
                for (int h = 0; h < 2; ++h)
#pragma unroll
                    for (int q = 0; q < QP; ++q)
#pragma unroll
                        for (int g = 0; g < NG; ++g) {
                            const uint32_t af[4] = {ra[g][2 * h], rb[g][2 * h], ra[g][2 * h + 1], rb[g][2 * h + 1]};
                            if (w + h + q == 0) mma_f16f32_16816_z(d[g], af, qf[g][0][0][0], qf[g][0][0][1]);
                            else mma_f16f32_16816(d[g], af, qf[g][w * 2 + h][q][0], qf[g][w * 2 + h][q][1]);
                        }
            }
#pragma unroll
            for (int g = 0; g < NG; ++g) {
                const float s0 = lo_f(sa[g]), b0 = fmaf(8.0f, s0, hi_f(sa[g])), s1 = lo_f(sb[g]), b1 = fmaf(8.0f, s1, hi_f(sb[g]));
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    x[mt][k] = fmaf(s0, d[g][k], g ? fmaf(b0, qsm[g][k], x[mt][k]) : b0 * qsm[g][k]);
                    x[mt][2 + k] = fmaf(s1, d[g][2 + k], g ? fmaf(b1, qsm[g][k], x[mt][2 + k]) : b1 * qsm[g][k]);
                }
            }
        }
        read();
        if (have < kKvPage)
#pragma unroll
            for (int mt = 0; mt < 4; ++mt)
#pragma unroll
                for (int k = 0; k < 4; ++k)
                    if (mt * 16 + gr + (k < 2 ? 0 : 8) >= have) x[mt][k] = -INFINITY;
        if (lrow) {
#pragma unroll
            for (int k = 0; k < 2; ++k)
                if (2 * cl + k < heads) {        // (the last page's rows are there, whatever its entries)
                    float* at = lrow + size_t(k) * p.rows + e0;
#pragma unroll
                    for (int mt = 0; mt < 4; ++mt) {
                        at[mt * 16] = x[mt][k] * sc[k];
                        at[mt * 16 + 8] = x[mt][2 + k] * sc[k];
                    }
                }
        }
        // running maximum (of the scaled scores); moved only when it is 2^8 too low
        float f[2];
        bool move = false;
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            float mx = x[0][k];
#pragma unroll
            for (int mt = 0; mt < 4; ++mt) mx = fmaxf(fmaxf(mx, x[mt][k]), x[mt][2 + k]);
#pragma unroll
            for (int d = 4; d < 32; d <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, d));
            mx *= sc[k];                         // (the scale is positive)
            f[k] = 1.0f;
            if (mx > m[k] + 8.0f || (mx > m[k] && m[k] == -INFINITY)) {
                f[k] = m[k] == -INFINITY ? 0.0f : kv4_ex2(m[k] - mx);
                m[k] = mx;
                move = true;
            }
        }
        if (__any_sync(0xffffffffu, move)) {
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                l[k] *= f[k];
#pragma unroll
                for (int g = 0; g < NG; ++g) {
                    bacc[g][k] *= f[k];
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        o[g][j][k] *= f[k];
                        o[g][j][2 + k] *= f[k];
                    }
                }
            }
        }
        const float mm[2] = {m[0] == -INFINITY ? 0.0f : m[0], m[1] == -INFINITY ? 0.0f : m[1]};
#pragma unroll
        for (int mt = 0; mt < 4; ++mt)
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                x[mt][k] = kv4_ex2(fmaf(x[mt][k], sc[k & 1], -mm[k & 1]));
                l[k & 1] += x[mt][k];
            }
        blk = ring + slot * UNIT;
        arrived();
        if (have < kKvPage) {                    // entries past the last one may hold anything: their scales and biases become 0
#pragma unroll
            for (int g = 0; g < NG; ++g)
#pragma unroll
                for (uint32_t e = lane; e < kKvPage; e += 32)
                    if (e >= have) *reinterpret_cast<uint32_t*>(ring + slot * UNIT + SB + g * 256 + e * 4) = 0u;
            __syncwarp();
            fence_proxy_async();                 // (the slot goes to a bulk copy next)
        }
        // The power of two of a group's p s for a head. While the page's scales
        // times it lie in [2^-2, 2^7] nothing passes fp16's range (p <= 2^8), and
        // what the pieces lose, 2^-25, is below 2^-22 of the entry with p = 1. A
        // pair's first page puts its largest scale near 2^3; where scales differ
        // more, kv4_new_up goes by the products themselves, for a large scale may
        // have no weight.
#pragma unroll
        for (int g = 0; g < NG; ++g) {
            const uint2 w = *reinterpret_cast<const uint2*>(blk + SB + g * 256 + lane * 8);
            const uint32_t s0 = w.x & 0x7fffu, s1 = w.y & 0x7fffu, big = __reduce_max_sync(0xffffffffu, max(s0, s1));
            const uint32_t low = __reduce_min_sync(0xffffffffu, min(s0 - 1, s1 - 1)) + 1;        // (of those that are not 0)
            const float hi = __uint_as_float(big << 16), lo = __uint_as_float(min(big, low) << 16);
            const bool fits = hi * fmaxf(up[g][0], up[g][1]) <= 128.0f && lo * fminf(up[g][0], up[g][1]) >= 0.25f;
            if (!__all_sync(0xffffffffu, fits || big == 0)) {
                if (up[g][0] == 0.0f && hi <= 32.0f * lo) {      // (a pair's first page: no head has one yet)
                    up[g][0] = up[g][1] = __uint_as_float(uint32_t(max(1, min(227, 257 - int(big >> 7)))) << 23);
                } else {
                    kv4_new_up(blk + SB + g * 256, big, gr, x, o[g], up[g]);
                }
            }
        }
#pragma unroll
        for (int mt = 0; mt < 4; ++mt) {
            const uint32_t ka = mt * 16 + gr, kb = ka + 8;
#pragma unroll
            for (int g = 0; g < NG; ++g) {
                const uint32_t sa = *reinterpret_cast<const uint32_t*>(blk + SB + g * 256 + ka * 4);
                const uint32_t sb = *reinterpret_cast<const uint32_t*>(blk + SB + g * 256 + kb * 4);
                const float b0 = fmaf(8.0f, lo_f(sa), hi_f(sa)), b1 = fmaf(8.0f, lo_f(sb), hi_f(sb));
                const float s0[2] = {lo_f(sa) * up[g][0], lo_f(sa) * up[g][1]}, s1[2] = {lo_f(sb) * up[g][0], lo_f(sb) * up[g][1]};
                // codes of this lane's 8 dimensions (8 gr ..) of the entries 2 cl, 2 cl + 1, 2 cl + 8, 2 cl + 9 of the tile;
                // lanes cl >= 2 load the pair the other way round (the four entries of a load then lie in different banks)
                uint32_t w[4];
#pragma unroll
                for (int k = 0; k < 4; ++k)
                    w[k] = *reinterpret_cast<const uint32_t*>(blk + g * kKvPlane + (mt * 16 + 2 * cl + ((k & 1) ^ (cl >> 1)) + (k >> 1) * 8) * 32 + gr * 4);
                // halves of the pair's words side by side, so that a register's halves are the two entries' codes of one dimension
                const uint32_t p_lo = cl < 2 ? 0x5410u : 0x1054u, p_hi = cl < 2 ? 0x7632u : 0x3276u;
                uint32_t c0[8], c1[8];           // dimension n: entries (2 cl, 2 cl + 1), and + 8
                kv4_half_codes(__byte_perm(w[0], w[1], p_lo), c0);
                kv4_half_codes(__byte_perm(w[0], w[1], p_hi), c0 + 4);
                kv4_half_codes(__byte_perm(w[2], w[3], p_lo), c1);
                kv4_half_codes(__byte_perm(w[2], w[3], p_hi), c1 + 4);
                bacc[g][0] = fmaf(x[mt][0], b0, fmaf(x[mt][2], b1, bacc[g][0]));
                bacc[g][1] = fmaf(x[mt][1], b0, fmaf(x[mt][3], b1, bacc[g][1]));
                const float y0 = x[mt][0] * s0[0], y1 = x[mt][1] * s0[1], y2 = x[mt][2] * s1[0], y3 = x[mt][3] * s1[1];
                const uint32_t u0 = cvt_f16x2(y0, y1), u1 = cvt_f16x2(y2, y3);
                const uint32_t v0 = movm_trans(cvt_f16x2(y0 - half_lo(u0), y1 - half_hi(u0)));
                const uint32_t v1 = movm_trans(cvt_f16x2(y2 - half_lo(u1), y3 - half_hi(u1)));
                const uint32_t z0 = movm_trans(u0), z1 = movm_trans(u1);
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const uint32_t af[4] = {c0[2 * j], c0[2 * j + 1], c1[2 * j], c1[2 * j + 1]};
                    mma_f16f32_16816(o[g][j], af, z0, z1);
                }
#pragma unroll
                for (int j = 0; j < 4; ++j) {    // (apart from the first pieces': those of one accumulator wait for one another)
                    const uint32_t af[4] = {c0[2 * j], c0[2 * j + 1], c1[2 * j], c1[2 * j + 1]};
                    mma_f16f32_16816(o[g][j], af, v0, v1);
                }
            }
        }
        read();
        const bool whole = pg + 1 == np;         // the pair's last page
        if (whole || i + 1 == mine) {
            fresh = true;
            const uint64_t pair = uint64_t(seq) * nheads + hc;
            const bool alone = whole && i + 1 >= np && !p.logits;               // its first page was in this stretch, too
#pragma unroll
            for (int d = 4; d < 32; d <<= 1)
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    l[k] += __shfl_xor_sync(0xffffffffu, l[k], d);
#pragma unroll
                    for (int g = 0; g < NG; ++g) bacc[g][k] += __shfl_xor_sync(0xffffffffu, bacc[g][k], d);
                }
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                const uint32_t h = 2 * cl + k;
                const float inv = 1.0f / l[k];
#pragma unroll
                for (int g = 0; g < NG; ++g) {
                    const float down = up[g][k] == 0.0f ? 0.0f : 1.0f / up[g][k];                // (exact: a power of two)
                    float v[8];                  // dimensions 8 gr .. of the group
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        v[2 * j] = fmaf(o[g][j][k], down, bacc[g][k]);
                        v[2 * j + 1] = fmaf(o[g][j][2 + k], down, bacc[g][k]);
                    }
                    if (!alone) {
                        float4* dst = reinterpret_cast<float4*>(p.part + ((me + pair) * kKaHeads + h) * HD + g * 64 + gr * 8);
                        dst[0] = make_float4(v[0], v[1], v[2], v[3]);
                        dst[1] = make_float4(v[4], v[5], v[6], v[7]);
                    } else if (h < heads) {
                        const size_t at = seq * p.t.out_row + size_t(head0 + h) * HD + g * 64 + gr * 8;
#pragma unroll
                        for (int j = 0; j < 8; ++j) v[j] *= inv;
                        if (p.t.dtype == SMOE_DTYPE_F32) {
                            float4* dst = reinterpret_cast<float4*>(static_cast<float*>(p.t.out) + at);
                            dst[0] = make_float4(v[0], v[1], v[2], v[3]);
                            dst[1] = make_float4(v[4], v[5], v[6], v[7]);
                        } else {                 // (rows are 8-byte aligned: strides are multiples of 4)
                            uint2* dst = reinterpret_cast<uint2*>(static_cast<uint16_t*>(p.t.out) + at);
                            dst[0] = make_uint2(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]));
                            dst[1] = make_uint2(pack_bf16x2(v[4], v[5]), pack_bf16x2(v[6], v[7]));
                        }
                    }
                }
                if (!alone && gr == 0) p.stat[(me + pair) * kKaHeads + h] = make_float2(m[k], l[k]);
            }
        }
        if (i + 1 < mine && ++pg == np) {
            pg = 0;
            if (++hc == nheads) {
                hc = 0;
                do n = kv4_valid(p, ++seq), np = kv4_pages(n);
                while (np == 0);
            }
        }
    }
    // Released here, and by k_kv4_join not before its end: CTAs of the next call
    // that are resident beside those of this one or of the join end up two and
    // not three on some SMs, and the rest run after all others (32 contexts, 14
    // pages a warp, no weights: 112 us a call instead of 80).
    pdl_release();
    if (failed)                                  // no copy may be in flight when the CTA ends
        for (uint32_t u = 2 * mine > uint32_t(kKaStages) ? 2 * mine - kKaStages : 0u; u < 2 * mine; ++u)
            mbar_wait_bounded(bars + u % kKaStages, (u / kKaStages) & 1);
}

// The parts of the pairs joined in their order, and with weights each entry's
// new weight from the stored scores. grid (x, KV head, sequence): the first
// `outs` CTAs take 1024 / lanes outputs each, 4 a thread, `lanes` threads
// sharing the parts of an output (many parts, few outputs: the chain of loads
// stays short); the others 1024 entries each, 4 a thread. Every CTA first
// forms the maxima and sums of the heads that it needs from the parts'
// (contiguous: a thread a head and every 32nd part). Bound by that chain of
// loads: 4 us for a short sequence, 8 to 12 us where 260,000 entries get
// weights (their stored scores pass at 2 to 3 TB/s).
constexpr int kKjThreads = 256, kKjEntries = 4 * kKjThreads;
__global__ void __launch_bounds__(kKjThreads) k_kv4_join(const Kv4Attn p, uint32_t outs) {
    constexpr uint32_t heads = kKaHeads;
    extern __shared__ float2 kv4_stat[];         // [chunks][heads] maximum; 1 / sum (outputs) or log2 of the sum (weights)
    __shared__ float2 red[kKjThreads];
    __shared__ float4 part_v[kKjThreads];
    pdl_acquire();
    const SmoeKv4Cache& c = p.a.c;
    const uint32_t kvh = blockIdx.y, s = blockIdx.z, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, HD = c.head_dim;
    const bool is_out = blockIdx.x < outs;
    const uint32_t quads = kKjThreads / p.lanes, at = (blockIdx.x * quads + tid % quads) * 4, h = at / HD, d = at % HD;
    // a CTA's outputs belong to one round of heads: 1024 / lanes divides heads x HD (lanes >= 2 at HD 64)
    const uint32_t ch0 = is_out ? blockIdx.x * quads * 4 / HD / heads : 0u, ch1 = is_out ? ch0 + 1 : p.chunks;
    const uint64_t pair0 = (uint64_t(s) * c.num_kv_heads + kvh) * p.chunks;
    uint2 mt = p.meta[pair0 + ch0];              // (of a sequence without entries: anything)
    const uint32_t n = kv4_valid(p, s), e = (blockIdx.x - outs) * kKjEntries + tid * 4;
    if (!is_out && (blockIdx.x - outs) * kKjEntries >= n) return;
    if (is_out && n && mt.y == 1 && !p.logits) return;           // one part: its warp has written the outputs
    // the entries' page and old weights, fetched while the statistics come in
    uint32_t page = ~0u;
    size_t to = 0;
    float old[4] = {0.f, 0.f, 0.f, 0.f};
    if (!is_out && e < n) {
        page = kv4_page(c, s, e, p.a.err);       // (4 entries lie in one page)
        to = (size_t(page) * c.num_kv_heads + kvh) * kKvPage + e % kKvPage;
        if (page != ~0u && c.score && p.t.decay != 0.0f)
#pragma unroll
            for (int k = 0; k < 4; ++k)
                if (e + k < n) old[k] = c.score[to + k] * p.t.decay;
    }
    for (uint32_t ch = ch0; ch < ch1; ++ch) {
        if (ch > ch0) mt = p.meta[pair0 + ch];
        const uint32_t parts = n ? mt.y : 0u;
        const float2* st = p.stat + (mt.x + pair0 + ch) * heads + tid % heads;
        float mx = -INFINITY, sum = 0.0f;
        for (uint32_t j0 = tid / heads; j0 < parts; j0 += 8 * kKjThreads / heads) {
            float2 t[8];
            float now = mx;
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                const uint32_t j = j0 + k * (kKjThreads / heads);
                t[k] = j < parts ? st[uint64_t(j) * heads] : make_float2(-INFINITY, 0.0f);
                now = fmaxf(now, t[k].x);
            }
            sum *= mx == -INFINITY ? 1.0f : kv4_ex2(mx - now);
#pragma unroll
            for (int k = 0; k < 8; ++k) sum = fmaf(t[k].y, t[k].x == -INFINITY ? 1.0f : kv4_ex2(t[k].x - now), sum);
            mx = now;
        }
        red[tid] = make_float2(mx, sum);
        __syncthreads();
        for (uint32_t k = warp; k < heads; k += kKjThreads / 32) {
            const float2 t = lane < kKjThreads / heads ? red[lane * heads + k] : make_float2(-INFINITY, 0.0f);
            float top = t.x;
#pragma unroll
            for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
            float all = t.y * (t.x == -INFINITY ? 1.0f : kv4_ex2(t.x - top));
#pragma unroll
            for (int o = 16; o; o >>= 1) all += __shfl_xor_sync(0xffffffffu, all, o);
            if (lane == 0) kv4_stat[(ch - ch0) * heads + k] = make_float2(top, is_out ? 1.0f / all : top + log2f(all));
        }
        __syncthreads();
    }
    if (is_out) {
        const uint32_t q = tid / quads, parts = n && h < p.group ? mt.y : 0u;
        const uint64_t first = (mt.x + pair0 + ch0) * heads + h % heads;
        const float2 all = kv4_stat[h % heads];
        float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
        for (uint32_t j = q; j < parts; j += p.lanes) {
            const uint64_t row = first + uint64_t(j) * heads;
            const float4 x = *reinterpret_cast<const float4*>(p.part + row * HD + d);
            const float mj = p.stat[row].x, f = mj == -INFINITY ? 0.0f : kv4_ex2(mj - all.x);
            v.x = fmaf(x.x, f, v.x);
            v.y = fmaf(x.y, f, v.y);
            v.z = fmaf(x.z, f, v.z);
            v.w = fmaf(x.w, f, v.w);
        }
        if (p.lanes > 1) {
            part_v[tid] = v;
            __syncthreads();
        }
        if (q != 0 || h >= p.group) return;
        for (uint32_t i = 1; i < p.lanes; ++i) {
            const float4 x = part_v[tid + i * quads];
            v.x += x.x;
            v.y += x.y;
            v.z += x.z;
            v.w += x.w;
        }
        const float inv = n ? all.y : 0.0f;
        const size_t dst = s * p.t.out_row + size_t(kvh * p.group + h) * HD + d;
        if (p.t.dtype == SMOE_DTYPE_F32)
            *reinterpret_cast<float4*>(static_cast<float*>(p.t.out) + dst) = make_float4(v.x * inv, v.y * inv, v.z * inv, v.w * inv);
        else
            *reinterpret_cast<uint2*>(static_cast<uint16_t*>(p.t.out) + dst) =
                make_uint2(pack_bf16x2(v.x * inv, v.y * inv), pack_bf16x2(v.z * inv, v.w * inv));
        return;
    }
    if (page == ~0u) return;
    float4 w = make_float4(old[0], old[1], old[2], old[3]);
    const float* x = p.logits + (size_t(s) * p.t.num_heads + kvh * p.group) * p.rows + e;
#pragma unroll 8
    for (uint32_t k = 0; k < p.group; ++k) {
        const float4 y = *reinterpret_cast<const float4*>(x + size_t(k) * p.rows);
        const float l = kv4_stat[k].y;           // (rounds of heads follow one another)
        w.x += kv4_ex2(y.x - l);
        w.y += kv4_ex2(y.y - l);
        w.z += kv4_ex2(y.z - l);
        w.w += kv4_ex2(y.w - l);
    }
    float* dst = p.t.score_out + to;
    if (e + 4 <= n && (reinterpret_cast<uintptr_t>(dst) & 15u) == 0) {
        *reinterpret_cast<float4*>(dst) = w;
    } else {
        dst[0] = w.x;
        if (e + 1 < n) dst[1] = w.y;
        if (e + 2 < n) dst[2] = w.z;
        if (e + 3 < n) dst[3] = w.w;
    }
}

// ----------------------------------------------------------------- eviction
struct Kv4Evict {
    Kv4Args a;
    uint32_t keep, recent, max_len;
    uint32_t* pos_out;                           // null: in place
    float* score_out;
    uint32_t* lists;                             // per (sequence, KV head): targets, then sources
    uint32_t cap;                                // moves that a pair can have
    uint32_t cached;                             // keys that a CTA's shared memory holds
};

// Order of the scores as unsigned integers, NaN lowest; -0 and 0 are equal.
SMOE_DEVINL uint32_t kv4_rank_key(float x) {
    if (x != x) return 0u;
    const uint32_t b = __float_as_uint(x + 0.0f);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
constexpr uint32_t kKvLate = 0xffffffffu;        // key of an entry that stays for its position (above +inf's)

// A cluster of CTAs per (KV head, sequence), each CTA a stretch of the
// entries, a warp a stretch of those.
//  1. Keys (a score's order, or kKvLate) into shared memory; the first of
//     three histograms - 11, 11 and 10 bits of the key - with them.
//  2. The keep-th largest key: after each histogram every CTA adds up all of
//     the cluster's and finds the digit; the next one counts the keys that
//     share the digits so far. Entries above the key stay, and of those
//     equal to it the lowest.
//  3. Each warp turns its words of 32 entries into masks of those that stay
//     (a ballot each, lane i keeps the i-th), counts free entries below `keep`
//     and kept ones past it, and - with what the warps and CTAs before it
//     counted - lists both, ascending.
//  4. The j-th kept entry goes to the j-th free one: a warp takes up to 32
//     moves (few moves go to many warps, eight each), looks up their pages a
//     lane each, and copies eight at a time, 128 bytes
//     of codes as a word a lane, scales, biases, pos and score another.
//     Sources are past `keep` and targets below it: no move reads what
//     another writes. (Separate outputs have pos and score of all entries
//     below `keep` from step 1, before the moved ones' overwrite them.)
// Bound by the chain of steps for short sequences (8 of 1,100 entries cut to
// 1,024, 4 KV heads: 10.3 us; 12.7 with 32 moves a warp) and by the moves for
// long ones (16 of 6,000 to 32,768 cut to 4,096: 56 us, of which the selection
// takes 15; the moves' 32-byte sectors pass at about 6 TB/s, as far as memory
// goes). One launch: with a launch a step the first took 37 us, the second 244.
constexpr int kEvThreads = 512, kEvWarps = kEvThreads / 32, kEvDigits = 3;
constexpr uint32_t kEvBins = 2048, kEvCtas = 8;  // of a cluster, at most
__host__ __device__ constexpr uint32_t kv4_evict_smem(uint32_t cached) { return (kEvDigits * kEvBins + cached) * 4; }

// Exclusive sum over the threads of a CTA of two counts at once; totals in `all`.
SMOE_DEVINL uint2 ev_scan(uint2 v, uint2* warp_sums, uint32_t warp, uint32_t lane, uint2& all) {
    uint2 incl = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const uint32_t x = __shfl_up_sync(0xffffffffu, incl.x, o), y = __shfl_up_sync(0xffffffffu, incl.y, o);
        if (lane >= uint32_t(o)) incl.x += x, incl.y += y;
    }
    __syncthreads();
    if (lane == 31) warp_sums[warp] = incl;
    __syncthreads();
    const uint2 w = lane < uint32_t(kEvWarps) ? warp_sums[lane] : make_uint2(0u, 0u);
    uint2 wi = w;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const uint32_t x = __shfl_up_sync(0xffffffffu, wi.x, o), y = __shfl_up_sync(0xffffffffu, wi.y, o);
        if (lane >= uint32_t(o)) wi.x += x, wi.y += y;
    }
    all = make_uint2(__shfl_sync(0xffffffffu, wi.x, 31), __shfl_sync(0xffffffffu, wi.y, 31));
    const uint32_t bx = __shfl_sync(0xffffffffu, wi.x - w.x, warp), by = __shfl_sync(0xffffffffu, wi.y - w.y, warp);
    return make_uint2(bx + incl.x - v.x, by + incl.y - v.y);
}

__global__ void __launch_bounds__(kEvThreads) k_kv4_evict(const Kv4Evict p) {
    namespace cg = cooperative_groups;
    extern __shared__ uint32_t ev_smem[];
    __shared__ uint2 warp_sums[32], counts[2];
    __shared__ uint32_t pick[3];
    cg::cluster_group cluster = cg::this_cluster();
    pdl_release();
    const SmoeKv4Cache& c = p.a.c;
    const uint32_t ctas = cluster.num_blocks(), rank = cluster.block_rank();
    const uint32_t kvh = blockIdx.x / ctas, s = blockIdx.y, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    uint32_t *hist = ev_smem, *keys = ev_smem + kEvDigits * kEvBins;
    for (uint32_t i = tid; i < kEvDigits * kEvBins; i += kEvThreads) hist[i] = 0;
    __syncthreads();
    pdl_acquire();
    uint32_t* to_list = p.lists + (size_t(s) * c.num_kv_heads + kvh) * 2 * p.cap;
    uint32_t* from_list = to_list + p.cap;
    uint32_t n = ld_plain(c.len + s);
    if (n > p.max_len) {
        if (tid == 0) serve_err(p.a.err, SMOE_DEVERR_BAD_RANGE);
        n = p.max_len;
    }
    const uint32_t seen = ld_plain((c.seen ? c.seen : c.len) + s);
    // this CTA's entries: whole words of 32
    const uint32_t words = (n + 31) / 32, wper = (words + ctas - 1) / ctas;
    const uint32_t e0 = min(n, rank * wper * 32), e1 = min(n, e0 + wper * 32);
    auto place = [&](uint32_t e) -> size_t {     // index of entry e in pos and score, ~0 when it has none
        const uint32_t page = kv4_page(c, s, e, p.a.err);
        return page == ~0u ? ~size_t(0) : (size_t(page) * c.num_kv_heads + kvh) * kKvPage + e % kKvPage;
    };
    if (n <= p.keep) {                           // all stay (the whole cluster returns)
        if (p.pos_out)
            for (uint32_t e = e0 + tid; e < e1; e += kEvThreads) {
                const size_t i = place(e);
                if (i != ~size_t(0)) p.pos_out[i] = c.pos[i], p.score_out[i] = c.score[i];
            }
        return;
    }
    auto key = [&](uint32_t pos, float score) { return uint64_t(pos) + p.recent >= seen ? kKvLate : kv4_rank_key(score); };
    auto key_of = [&](uint32_t e) -> uint32_t {
        if (e - e0 < p.cached) return keys[e - e0];
        const size_t i = place(e);
        return i == ~size_t(0) ? 0u : key(c.pos[i], c.score[i]);
    };

    uint32_t prefix = 0, need = p.keep;          // need: kept entries among those that share the digits so far
#pragma unroll
    for (int d = 0; d < kEvDigits; ++d) {
        constexpr int kShift[kEvDigits] = {21, 10, 0};
        const int shift = kShift[d], up = d == 0 ? 32 : kShift[d > 0 ? d - 1 : 0];
        const uint32_t mask = d == 2 ? 1023u : 2047u;
        uint32_t* h = hist + d * kEvBins;
        if (d == 0) {                            // four entries a thread at a time - they share a page - and two such at once
            for (uint32_t eb = e0 + tid * 4; eb < e1; eb += 8 * kEvThreads) {
                size_t at[2];
                uint4 ps[2];
                float4 sc[2];
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    const uint32_t e = eb + u * 4 * kEvThreads;
                    at[u] = e < e1 ? place(e) : ~size_t(0);
                }
#pragma unroll
                for (int u = 0; u < 2; ++u)
                    if (at[u] != ~size_t(0)) {   // (whole quads: past the last entry the page goes on)
                        ps[u] = *reinterpret_cast<const uint4*>(c.pos + at[u]);
                        sc[u] = *reinterpret_cast<const float4*>(c.score + at[u]);
                    }
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    const uint32_t e = eb + u * 4 * kEvThreads, m = e < e1 ? min(4u, e1 - e) : 0u;
                    const bool ok = at[u] != ~size_t(0);
                    const uint32_t k[4] = {ok ? key(ps[u].x, sc[u].x) : 0u, ok ? key(ps[u].y, sc[u].y) : 0u,
                                           ok ? key(ps[u].z, sc[u].z) : 0u, ok ? key(ps[u].w, sc[u].w) : 0u};
#pragma unroll
                    for (int q = 0; q < 4; ++q)
                        if (q < m) {
                            if (e + q - e0 < p.cached) keys[e + q - e0] = k[q];
                            atomicAdd(h + (k[q] >> shift), 1u);
                        }
                    if (p.pos_out && ok && e < p.keep) {
                        if (e + 4 <= p.keep) {   // (n > keep: the whole quad is there)
                            *reinterpret_cast<uint4*>(p.pos_out + at[u]) = ps[u];
                            *reinterpret_cast<float4*>(p.score_out + at[u]) = sc[u];
                        } else {
                            const uint32_t pq[3] = {ps[u].x, ps[u].y, ps[u].z};
                            const float sq[3] = {sc[u].x, sc[u].y, sc[u].z};
#pragma unroll
                            for (int q = 0; q < 3; ++q)
                                if (e + q < p.keep) p.pos_out[at[u] + q] = pq[q], p.score_out[at[u] + q] = sq[q];
                        }
                    }
                }
            }
        } else {
            for (uint32_t e = e0 + tid; e < e1; e += kEvThreads) {
                const uint32_t k = key_of(e);
                if ((k ^ prefix) >> up == 0) atomicAdd(h + (k >> shift & mask), 1u);
            }
        }
        cluster.sync();
        // bins from the top, four a thread: where the sum passes `need`
        uint32_t mine[4] = {0u, 0u, 0u, 0u};
        const uint32_t b = kEvBins - 4 - 4 * tid;
        static_assert(kEvBins == 4 * kEvThreads, "four bins a thread");
        uint4 theirs[kEvCtas];                   // (all of them on their way at once)
#pragma unroll
        for (uint32_t r = 0; r < kEvCtas; ++r)
            theirs[r] = r < ctas ? *reinterpret_cast<const uint4*>(cluster.map_shared_rank(h, r) + b) : make_uint4(0u, 0u, 0u, 0u);
#pragma unroll
        for (uint32_t r = 0; r < kEvCtas; ++r) {
            mine[0] += theirs[r].x;
            mine[1] += theirs[r].y;
            mine[2] += theirs[r].z;
            mine[3] += theirs[r].w;
        }
        uint2 all;
        uint32_t above = ev_scan(make_uint2(mine[0] + mine[1] + mine[2] + mine[3], 0u), warp_sums, warp, lane, all).x;
#pragma unroll
        for (int q = 3; q >= 0; --q) {
            if (above < need && above + mine[q] >= need) {
                pick[0] = b + q;
                pick[1] = need - above;
                pick[2] = mine[q];
            }
            above += mine[q];
        }
        __syncthreads();
        prefix |= pick[0] << shift;
        need = pick[1];
    }
    // the warp's words of the CTA's
    const uint32_t cw = (e1 - e0 + 31) / 32, per = (cw + kEvWarps - 1) / kEvWarps, w0 = min(cw, warp * per), w1 = min(cw, w0 + per);
    const uint32_t low = (1u << lane) - 1u;
    uint2 all;
    uint32_t eq0 = 0;                            // entries with the key before this warp's
    const bool some = pick[2] > need;            // not all entries with the key stay
    if (some) {
        uint32_t equal = 0;
        for (uint32_t w = w0; w < w1; ++w) {
            const uint32_t e = e0 + w * 32 + lane;
            equal += __popc(__ballot_sync(0xffffffffu, e < e1 && key_of(e) == prefix));
        }
        eq0 = __shfl_sync(0xffffffffu, ev_scan(make_uint2(lane == 0 ? equal : 0u, 0u), warp_sums, warp, lane, all).x, 0);
        if (tid == 0) counts[0] = all;
        cluster.sync();
#pragma unroll
        for (uint32_t r = 0; r < kEvCtas; ++r) eq0 += r < rank ? cluster.map_shared_rank(counts, r)[0].x : 0u;
    }
    // masks of the words wb, wb + 1, .. that stay: lane i's of word wb + i
    uint32_t eq = eq0;
    auto masks = [&](uint32_t wb) -> uint32_t {
        uint32_t mine = 0;
        for (uint32_t i = 0; i < 32 && wb + i < w1; ++i) {
            const uint32_t e = e0 + (wb + i) * 32 + lane, k = e < e1 ? key_of(e) : 0u;
            uint32_t m = __ballot_sync(0xffffffffu, e < e1 && k >= prefix);
            if (some) {
                const uint32_t eqs = __ballot_sync(0xffffffffu, e < e1 && k == prefix);
                m = __ballot_sync(0xffffffffu, (m >> lane & 1u) && (k > prefix || eq + __popc(eqs & low) < need));
                eq += __popc(eqs);
            }
            if (lane == i) mine = m;
        }
        return mine;
    };
    auto upto = [](uint32_t e, uint32_t end) -> uint32_t {       // bits of the entries e .. e + 31 that lie below `end`
        return e >= end ? 0u : end - e >= 32 ? 0xffffffffu : (1u << (end - e)) - 1u;
    };
    // this lane's word: its free entries below `keep` (x), its kept ones past it (y)
    auto split = [&](uint32_t wb, uint32_t m) -> uint2 {
        if (wb + lane >= w1) return make_uint2(0u, 0u);
        const uint32_t e = e0 + (wb + lane) * 32, k = upto(e, p.keep);
        return make_uint2(~m & k & upto(e, e1), m & ~k);
    };
    uint32_t kept = 0;
    uint2 mine = make_uint2(0u, 0u);
    for (uint32_t wb = w0; wb < w1; wb += 32) {
        kept = masks(wb);
        const uint2 f = split(wb, kept);
        mine.x += __popc(f.x);
        mine.y += __popc(f.y);
    }
    uint2 first = ev_scan(mine, warp_sums, warp, lane, all);     // before this lane's words (if they are one)
    if (tid == 0) counts[1] = all;
    cluster.sync();
    uint32_t moves = 0;
#pragma unroll
    for (uint32_t r = 0; r < kEvCtas; ++r) {
        const uint2 v = r < ctas ? cluster.map_shared_rank(counts, r)[1] : make_uint2(0u, 0u);
        if (r < rank) first.x += v.x, first.y += v.y;
        moves += v.y;
    }
    moves = min(moves, p.cap);
    const bool once = w1 - w0 <= 32;
    if (!once) {                                 // several words a lane: from the warp's first entry on
        first.x = __shfl_sync(0xffffffffu, first.x, 0);
        first.y = __shfl_sync(0xffffffffu, first.y, 0);
        eq = eq0;
    }
    for (uint32_t wb = w0; wb < w1; wb += 32) {
        if (!once) kept = masks(wb);
        const uint2 f = split(wb, kept);
        uint2 at = first;
        if (!once) {
            uint2 incl = make_uint2(__popc(f.x), __popc(f.y));
            const uint2 v = incl;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const uint32_t x = __shfl_up_sync(0xffffffffu, incl.x, o), y = __shfl_up_sync(0xffffffffu, incl.y, o);
                if (lane >= uint32_t(o)) incl.x += x, incl.y += y;
            }
            at.x += incl.x - v.x;
            at.y += incl.y - v.y;
            first.x += __shfl_sync(0xffffffffu, incl.x, 31);
            first.y += __shfl_sync(0xffffffffu, incl.y, 31);
        }
        for (uint32_t i = 0; i < 32 && wb + i < w1; ++i) {
            const uint32_t fx = __shfl_sync(0xffffffffu, f.x, i), fy = __shfl_sync(0xffffffffu, f.y, i);
            const uint32_t ax = __shfl_sync(0xffffffffu, at.x, i) + __popc(fx & low), ay = __shfl_sync(0xffffffffu, at.y, i) + __popc(fy & low);
            const uint32_t e = e0 + (wb + i) * 32 + lane;
            if ((fx >> lane & 1u) && ax < p.cap) to_list[ax] = e;
            if ((fy >> lane & 1u) && ay < p.cap) from_list[ay] = e;
        }
    }
    cluster.sync();                              // the lists are written (and no CTA reads another's memory after this)

    // What a lane copies of a move, at base + (page and KV head) * step + slot * width: a word of codes (plane lane / 8,
    // word lane % 8 of its 32 bytes), and from lane 31 downwards the scale and bias pairs, pos and score.
    const Kv4Geom G(c.head_dim);
    const uint32_t x = 31 - lane;
    const bool codes = lane < G.ng * 16, rest = x < G.ng * 2 + 2;
    uint8_t* const code_base = c.blocks + lane / 8 * kKvPlane + lane % 8 * 4;
    const uint32_t step = x < G.ng * 2 ? G.block : kKvPage * 4;
    const uint8_t* rest_from = x < G.ng * 2 ? c.blocks + G.sb(0, 0) + x * kKvPage * 4
                               : x == G.ng * 2 ? reinterpret_cast<const uint8_t*>(c.pos) : reinterpret_cast<const uint8_t*>(c.score);
    uint8_t* rest_to = x < G.ng * 2 ? c.blocks + G.sb(0, 0) + x * kKvPage * 4
                       : x == G.ng * 2 ? reinterpret_cast<uint8_t*>(p.pos_out ? p.pos_out : c.pos)
                                       : reinterpret_cast<uint8_t*>(p.score_out ? p.score_out : c.score);
    const uint32_t warps = ctas * kEvWarps, some_moves = min(32u, ((moves + warps - 1) / warps + 7) / 8 * 8);     // a warp's at a time
    for (uint32_t m0 = (rank * kEvWarps + warp) * some_moves; m0 < moves; m0 += warps * some_moves) {
        uint32_t te = 0, fe = 0, tb = 0, fb = 0;
        bool ok = lane < some_moves && m0 + lane < moves;
        if (ok) {
            te = to_list[m0 + lane];
            fe = from_list[m0 + lane];
            const uint32_t tp = kv4_page(c, s, te, p.a.err), fp = kv4_page(c, s, fe, p.a.err);
            ok = tp != ~0u && fp != ~0u;
            tb = tp;
            fb = fp;
        }
        const uint32_t oks = __ballot_sync(0xffffffffu, ok);
#pragma unroll 1
        for (uint32_t q0 = 0; q0 < 32 && oks >> q0; q0 += 8) {
            uint32_t code[8], word[8];
#pragma unroll
            for (int q = 0; q < 8; ++q) {
                const uint32_t e = __shfl_sync(0xffffffffu, fe, q0 + q), page = __shfl_sync(0xffffffffu, fb, q0 + q);
                const bool has = oks >> (q0 + q) & 1u;
                const size_t at = size_t(page) * c.num_kv_heads + kvh;
                code[q] = word[q] = 0u;
                if (has && codes) code[q] = *reinterpret_cast<const uint32_t*>(code_base + at * G.block + e % kKvPage * 32);
                if (has && rest) word[q] = *reinterpret_cast<const uint32_t*>(rest_from + at * step + e % kKvPage * 4);
            }
#pragma unroll
            for (int q = 0; q < 8; ++q) {
                const uint32_t e = __shfl_sync(0xffffffffu, te, q0 + q), page = __shfl_sync(0xffffffffu, tb, q0 + q);
                const bool has = oks >> (q0 + q) & 1u;
                const size_t at = size_t(page) * c.num_kv_heads + kvh;
                if (has && codes) *reinterpret_cast<uint32_t*>(code_base + at * G.block + e % kKvPage * 32) = code[q];
                if (has && rest) *reinterpret_cast<uint32_t*>(rest_to + at * step + e % kKvPage * 4) = word[q];
            }
        }
    }
}

__global__ void __launch_bounds__(256) k_kv4_advance(uint32_t* len, uint32_t* seen, uint32_t n_seqs, const uint32_t* cu,
                                                     uint32_t n_each, uint32_t keep, uint32_t* err) {
    pdl_release();
    pdl_acquire();
    const uint32_t s = blockIdx.x * 256 + threadIdx.x;
    if (s >= n_seqs) return;
    uint32_t n = n_each;
    if (cu) {
        const uint32_t from = cu[s], to = cu[s + 1];
        if (from > to) serve_err(err, SMOE_DEVERR_BAD_RANGE);
        n = from > to ? 0u : to - from;
    }
    const uint32_t l = len[s] + n;
    len[s] = keep && l > keep ? keep : l;
    if (seen) seen[s] += n;
}

}  // namespace smoe
