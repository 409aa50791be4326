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
    const uint32_t p = __ldg(c.table + size_t(s) * c.table_stride + e / kKvPage);
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
    if (dtype == SMOE_DTYPE_F32) return __ldg(reinterpret_cast<const float4*>(static_cast<const float*>(p) + at));
    const uint2 u = __ldg(reinterpret_cast<const uint2*>(static_cast<const uint16_t*>(p) + at));
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
    const uint32_t t = row - __ldg(r.cu + s);
    const uint64_t e = uint64_t(__ldg(a.c.len + s)) + t;
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
                if (a.c.pos) a.c.pos[i] = __ldg((a.c.seen ? a.c.seen : a.c.len) + s) + t;
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
    const uint64_t e = uint64_t(first ? __ldg(first + s) : 0u) + (row - __ldg(r.cu + s));
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
struct Kv4Attn {
    Kv4Args a;
    SmoeKv4AttnArgs t;
    float* logits;                               // [n_seqs][num_heads][max_len rounded up to pages]
    uint32_t stride;                             // floats of a logits row
};

// Entries of sequence s that the token attends to.
SMOE_DEVINL uint32_t kv4_valid(const Kv4Attn& p, uint32_t s) {
    const uint64_t n = uint64_t(__ldg(p.a.c.len + s)) + p.t.extra;
    if (n > p.t.max_len) {
        if (threadIdx.x == 0) serve_err(p.a.err, SMOE_DEVERR_BAD_RANGE);
        return p.t.max_len;
    }
    return uint32_t(n);
}

SMOE_DEVINL float kv4_value(const uint8_t* blk, const Kv4Geom& G, uint32_t kv, uint32_t slot, uint32_t d) {
    const uint32_t g = d >> 6, i = d & 63;
    const uint32_t code = blk[G.codes(kv, g) + slot * 32 + (i >> 1)] >> (4 * (i & 1)) & 15u;
    const uint32_t sb = *reinterpret_cast<const uint32_t*>(blk + G.sb(kv, g) + slot * 4);
    return fmaf(float(code), __uint_as_float(sb << 16), __uint_as_float(sb & 0xffff0000u));
}

// One CTA per (KV head, sequence), its query heads one after the other:
// scores of all entries, their maximum and sum, the weighted values.
__global__ void __launch_bounds__(256) k_kv4_attention(Kv4Attn p) {
    pdl_release();
    pdl_acquire();
    __shared__ float q[128], red[256];
    const SmoeKv4Cache& c = p.a.c;
    const Kv4Geom G(c.head_dim);
    const uint32_t kvh = blockIdx.x, s = blockIdx.y, tid = threadIdx.x, hd = c.head_dim;
    const uint32_t group = p.t.num_heads / c.num_kv_heads, n = kv4_valid(p, s);
    auto block_of = [&](uint32_t e) -> const uint8_t* {
        const uint32_t page = kv4_page(c, s, e, p.a.err);
        return page == ~0u ? nullptr : c.blocks + (size_t(page) * c.num_kv_heads + kvh) * G.block;
    };
    for (uint32_t j = 0; j < group; ++j) {
        const uint32_t h = kvh * group + j;
        float* l = p.logits + (size_t(s) * p.t.num_heads + h) * p.stride;
        __syncthreads();
        if (tid < hd)
            q[tid] = p.t.dtype == SMOE_DTYPE_F32
                         ? static_cast<const float*>(p.t.q)[s * p.t.q_row + h * hd + tid]
                         : bf16_bits_to_f32(static_cast<const uint16_t*>(p.t.q)[s * p.t.q_row + h * hd + tid]);
        __syncthreads();
        float m = -INFINITY;
        for (uint32_t e = tid; e < n; e += 256) {
            const uint8_t* blk = block_of(e);
            float x = 0.0f;
            for (uint32_t d = 0; blk && d < hd; ++d) x = fmaf(q[d], kv4_value(blk, G, 0, e % kKvPage, d), x);
            x = blk ? x * p.t.scale : -INFINITY;
            l[e] = x;
            m = fmaxf(m, x);
        }
        red[tid] = m;
        for (uint32_t o = 128; o; o >>= 1) {
            __syncthreads();
            if (tid < o) red[tid] = fmaxf(red[tid], red[tid + o]);
        }
        __syncthreads();
        m = red[0];
        __syncthreads();
        float sum = 0.0f;
        for (uint32_t e = tid; e < n; e += 256) {
            const float x = expf(l[e] - m);
            l[e] = x;
            sum += x;
        }
        red[tid] = sum;
        for (uint32_t o = 128; o; o >>= 1) {
            __syncthreads();
            if (tid < o) red[tid] += red[tid + o];
        }
        __syncthreads();
        const float inv = n ? 1.0f / red[0] : 0.0f;
        __syncthreads();
        float acc = 0.0f;
        const uint32_t d = tid % hd, part = tid / hd, parts = 256 / hd;
        for (uint32_t e = part; e < n; e += parts) {
            const uint8_t* blk = block_of(e);
            if (blk) acc = fmaf(l[e], kv4_value(blk, G, 1, e % kKvPage, d), acc);
        }
        red[tid] = acc;
        __syncthreads();
        if (tid < hd) {
            for (uint32_t i = 1; i < parts; ++i) acc += red[tid + i * hd];
            acc *= inv;
            if (p.t.dtype == SMOE_DTYPE_F32) static_cast<float*>(p.t.out)[s * p.t.out_row + h * hd + tid] = acc;
            else static_cast<__nv_bfloat16*>(p.t.out)[s * p.t.out_row + h * hd + tid] = __float2bfloat16_rn(acc);
        }
        for (uint32_t e = tid; p.t.score_out && e < n; e += 256) l[e] *= inv;
    }
    __syncthreads();
    for (uint32_t e = tid; p.t.score_out && e < n; e += 256) {
        const uint32_t page = kv4_page(c, s, e, p.a.err);
        if (page == ~0u) continue;
        const size_t i = (size_t(page) * c.num_kv_heads + kvh) * kKvPage + e % kKvPage;
        float w = 0.0f;
        for (uint32_t j = 0; j < group; ++j)
            w += p.logits[(size_t(s) * p.t.num_heads + kvh * group + j) * p.stride + e];
        p.t.score_out[i] = c.score && p.t.decay != 0.0f ? fmaf(p.t.decay, c.score[i], w) : w;
    }
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
    uint32_t n = __ldg(c.len + s);
    if (n > p.max_len) {
        if (tid == 0) serve_err(p.a.err, SMOE_DEVERR_BAD_RANGE);
        n = p.max_len;
    }
    if (n <= p.keep) {
        if (tid == 0) list[0] = 0;
        return;
    }
    const uint32_t seen = __ldg((c.seen ? c.seen : c.len) + s);
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
    uint32_t n = min(__ldg(c.len + s), min(p.max_len, p.keep));
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
