// prompt_attn.cuh - attention over packed prompts: causal, grouped heads,
// sequences of different lengths in one launch.
#pragma once
#include "serve.cuh"

namespace smoe {

// The keys [lo, hi) that row i of a sequence of len_q rows over len_k keys
// attends to.
struct PackedSeq {
    uint32_t q0, k0, len_q, len_k, causal, window;
    SMOE_DEVINL uint32_t hi(uint32_t i) const {
        if (!causal) return len_k;
        const int64_t h = int64_t(i) + 1 + int64_t(len_k) - int64_t(len_q);
        return h < 0 ? 0u : uint32_t(h);                 // (h <= len_k)
    }
    SMOE_DEVINL uint32_t lo(uint32_t i) const {
        const uint32_t h = hi(i);
        return window && h > window ? h - window : 0u;
    }
};

// One warp per (row, head): online softmax, 4 dimensions a lane.
__global__ void __launch_bounds__(256) k_attention_packed(SmoeCudaPackedAttnArgs a, uint32_t* err) {
    pdl_release();
    pdl_acquire();
    const uint32_t lane = threadIdx.x & 31, row = blockIdx.x * 8 + (threadIdx.x >> 5), h = blockIdx.y;
    if (row >= a.total_q) return;
    const uint32_t s = seq_of_row(a.cu_q, a.n_seqs, row, lane);
    if (s >= a.n_seqs) return;
    const uint32_t* ck = a.cu_k ? a.cu_k : a.cu_q;
    PackedSeq S{a.cu_q[s], ck[s], a.cu_q[s + 1] - a.cu_q[s], ck[s + 1] - ck[s], a.causal, a.window};
    if (a.cu_q[s + 1] > a.total_q || ck[s + 1] < ck[s] || ck[s + 1] > a.total_k) {
        if (lane == 0) serve_err(err, SMOE_DEVERR_BAD_RANGE);
        return;
    }
    const uint32_t kvh = h / (a.num_heads / a.num_kv_heads), d = lane * 4;
    auto load = [&](const uint16_t* p, float* x) {
        const uint2 u = d < a.head_dim ? *reinterpret_cast<const uint2*>(p + d) : make_uint2(0u, 0u);
        x[0] = __uint_as_float(u.x << 16);
        x[1] = __uint_as_float(u.x & 0xffff0000u);
        x[2] = __uint_as_float(u.y << 16);
        x[3] = __uint_as_float(u.y & 0xffff0000u);
    };
    float q[4], acc[4] = {0.f, 0.f, 0.f, 0.f}, m = -INFINITY, l = 0.f;
    load(a.q + row * a.q_row + h * a.q_head, q);
    const uint32_t i = row - S.q0, hi = S.hi(i), lo = S.lo(i);
    for (uint32_t j = lo; j < hi; ++j) {
        float k[4], v[4];
        load(a.k + (S.k0 + j) * a.k_row + kvh * a.k_head, k);
        load(a.v + (S.k0 + j) * a.v_row + kvh * a.v_head, v);
        float x = q[0] * k[0] + q[1] * k[1] + q[2] * k[2] + q[3] * k[3];
        for (int o = 16; o; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
        x *= a.scale;
        const float mn = fmaxf(m, x), r = expf(m - mn), w = expf(x - mn);
        l = l * r + w;
        for (int c = 0; c < 4; ++c) acc[c] = fmaf(w, v[c], acc[c] * r);
        m = mn;
    }
    const float inv = hi > lo ? 1.0f / l : 0.0f;
    if (d < a.head_dim)
        *reinterpret_cast<uint2*>(a.out + row * a.out_row + h * a.out_head + d) =
            make_uint2(pack_bf16x2(acc[0] * inv, acc[1] * inv), pack_bf16x2(acc[2] * inv, acc[3] * inv));
    if (a.lse && lane == 0) a.lse[size_t(row) * a.num_heads + h] = hi > lo ? m + logf(l) : -INFINITY;
}

}  // namespace smoe
