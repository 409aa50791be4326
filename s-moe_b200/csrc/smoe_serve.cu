// smoe_serve.cu - the long-context serving entries of include/smoe_cuda.h:
// packed prompt attention and the 4-bit KV cache. Kernels live in
// prompt_attn.cuh and kv4.cuh.
#include <cuda.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cmath>

#include "serve.cuh"
#include "kv4.cuh"
#include "prompt_attn.cuh"

namespace {

using smoe::ctx_fail;
using smoe::CtxView;

bool aligned(const void* p, uintptr_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

template <typename... KArgs, typename... Args>
int launch_cluster(const CtxView& c, void (*kern)(KArgs...), dim3 grid, dim3 block, size_t smem, uint32_t cluster, Args... args) {
    cudaLaunchConfig_t lc{};
    cudaLaunchAttribute at[2];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    at[1].id = cudaLaunchAttributeClusterDimension;
    at[1].val.clusterDim.x = cluster;
    at[1].val.clusterDim.y = at[1].val.clusterDim.z = 1;
    lc.gridDim = grid;
    lc.blockDim = block;
    lc.dynamicSmemBytes = smem;
    lc.stream = c.stream;
    lc.attrs = at;
    lc.numAttrs = cluster > 1 ? 2 : 1;
    const cudaError_t e = cudaLaunchKernelEx(&lc, kern, KArgs(args)...);
    if (e != cudaSuccess) return ctx_fail(SMOE_ERR_CUDA, cudaGetErrorString(e), long(e));
    *c.dispatches += 1;
    return SMOE_OK;
}
template <typename... KArgs, typename... Args>
int launch(const CtxView& c, void (*kern)(KArgs...), dim3 grid, dim3 block, size_t smem, Args... args) {
    return launch_cluster(c, kern, grid, block, smem, 1u, args...);
}

// Raise a kernel's shared-memory limit once per (kernel, device); a call
// inside a stream capture then makes no attribute call.
template <typename K>
int smem_limit(const CtxView& c, K kern, size_t smem) {
    if (smem > c.smem_optin) return ctx_fail(SMOE_ERR_UNSUPPORTED, "kernel needs more shared memory than the device has", long(smem));
    static thread_local struct { const void* f; int dev; } seen[32];
    static thread_local int nseen = 0;
    for (int i = 0; i < nseen; ++i)
        if (seen[i].f == reinterpret_cast<const void*>(kern) && seen[i].dev == c.device) return SMOE_OK;
    const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, int(smem));
    if (e != cudaSuccess) return ctx_fail(SMOE_ERR_CUDA, cudaGetErrorString(e), long(e));
    if (nseen < 32) seen[nseen++] = {reinterpret_cast<const void*>(kern), c.device};
    return SMOE_OK;
}

// No two rows or heads of an output share an element: either all heads of a
// row lie before the next row starts, or all rows of a head before the next head.
bool apart(uint64_t row, uint64_t head, uint64_t rows, uint64_t heads, uint64_t head_dim) {
    const auto span = [](uint64_t stride, uint64_t n, uint64_t inner) { return static_cast<unsigned __int128>(stride) * (n - 1) + inner; };
    const bool heads_inside = (heads <= 1 || head >= head_dim) && (rows <= 1 || row >= span(head, heads, head_dim));
    const bool rows_inside = (rows <= 1 || row >= head_dim) && (heads <= 1 || head >= span(row, rows, head_dim));
    return heads_inside || rows_inside;
}

// bf16 rows whose groups all start on 16 bytes.
bool wide_rows(const SmoeKv4Rows* r) { return (r->k_row | r->k_head | r->v_row | r->v_head) % 8 == 0; }

using EncodeTiled = decltype(&cuTensorMapEncodeTiled);
EncodeTiled encode_tiled() {
    static const EncodeTiled fn = [] {
        void* p = nullptr;
        cudaDriverEntryPointQueryResult q{};
        if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &p, 12000, cudaEnableDefault, &q) != cudaSuccess ||
            q != cudaDriverEntryPointSuccess)
            p = nullptr;
        return reinterpret_cast<EncodeTiled>(p);
    }();
    return fn;
}

// bf16 [rows][heads][head_dim] with the given strides (elements; of a dimension
// of one element any, of another not 0), read in boxes of 64 columns x
// box_heads x box_rows, 128-byte swizzle, zeros outside.
int map_rows(CUtensorMap* m, const void* base, uint32_t head_dim, uint32_t heads, uint32_t rows, uint64_t row, uint64_t head,
             uint32_t box_heads, uint32_t box_rows) {
    const EncodeTiled enc = encode_tiled();
    if (!enc) return ctx_fail(SMOE_ERR_CUDA, "cuTensorMapEncodeTiled is missing", 0);
    const cuuint64_t dims[3] = {head_dim, heads, rows};
    const cuuint64_t strides[2] = {heads > 1 ? head * 2 : 16, rows > 1 ? row * 2 : 16};
    const cuuint32_t box[3] = {64, box_heads, box_rows}, one[3] = {1, 1, 1};
    const CUresult r = enc(m, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void*>(base), dims, strides, box, one,
                           CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                           CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return r == CUDA_SUCCESS ? SMOE_OK : ctx_fail(SMOE_ERR_ARG, "tensor map refused (strides too large?)", long(r));
}

// The cache a call names: shape, pointers and alignment.
int check_cache(const SmoeKv4Cache* c, const char* what) {
    if (!c || !c->blocks || !c->table || !c->len || c->n_pages == 0 || c->n_seqs == 0 || c->table_stride == 0 ||
        c->num_kv_heads == 0)
        return ctx_fail(SMOE_ERR_ARG, what, 0);
    if (!smoe_cuda_kv4_block_bytes(c->head_dim))
        return ctx_fail(SMOE_ERR_UNSUPPORTED, "the 4-bit cache takes head_dim 64 or 128", c->head_dim);
    if (!aligned(c->blocks, 16) || !aligned(c->pos, 16) || !aligned(c->score, 16))
        return ctx_fail(SMOE_ERR_ARG, "cache blocks, pos and score must be 16-byte aligned", 0);
    if (c->n_seqs > 65535 || c->num_kv_heads > 65535)
        return ctx_fail(SMOE_ERR_ARG, "at most 65535 sequences and KV heads", c->n_seqs);
    return SMOE_OK;
}

int check_rows(const SmoeKv4Rows* r, const SmoeKv4Cache* c, bool written, const char* what) {
    if (!r || !r->cu || (r->total && (!r->k || !r->v))) return ctx_fail(SMOE_ERR_ARG, what, 0);
    if (written && (!apart(r->k_row, r->k_head, r->total, c->num_kv_heads, c->head_dim) ||
                    !apart(r->v_row, r->v_head, r->total, c->num_kv_heads, c->head_dim)))
        return ctx_fail(SMOE_ERR_ARG, "rows or heads of the rows to write overlap", long(r->k_row));
    if (r->dtype != SMOE_DTYPE_F32 && r->dtype != SMOE_DTYPE_BF16)
        return ctx_fail(SMOE_ERR_ARG, "rows are fp32 or bf16", r->dtype);
    if (!aligned(r->k, 16) || !aligned(r->v, 16) || (r->k_row | r->k_head | r->v_row | r->v_head) % 4)
        return ctx_fail(SMOE_ERR_ARG, "rows need 16-byte aligned bases and strides that are multiples of 4", 0);
    return SMOE_OK;
}

// Offsets in the context's scratch for packed attention.
struct PackedScratch {
    size_t cost, place, list, part, stat, bytes;
    explicit PackedScratch(int num_sms) {
        const size_t rows = size_t(2) * num_sms * 256;
        cost = 65536;                            // (the plan: 16 bytes a CTA and one more)
        place = cost + size_t(smoe::kPaMaxPairs) * 4;
        list = place + size_t(smoe::kPaMaxPairs) * 8;
        part = list + size_t(smoe::kPaMaxPairs) * 8;
        stat = part + rows * 128 * 4;
        bytes = stat + rows * 8;
    }
};

// A 4-bit attention call's launch and workspace, from its arguments alone
// (the workspace is asked for without a context).
struct AttnPlan {
    uint32_t group, chunks, rows;
    uint64_t parts, part_bytes, stat_bytes, meta_bytes, logit_bytes;
    AttnPlan(const SmoeKv4Cache& c, const SmoeKv4AttnArgs& t) {
        group = t.num_heads / c.num_kv_heads;
        chunks = (group + smoe::kKaHeads - 1) / smoe::kKaHeads;
        rows = (t.max_len + SMOE_KV4_PAGE - 1) / SMOE_KV4_PAGE * SMOE_KV4_PAGE;
        const uint64_t pairs = uint64_t(c.n_seqs) * c.num_kv_heads * chunks, all_heads = uint64_t(c.n_seqs) * t.num_heads;
        auto up = [](uint64_t n) { return (n + 255) / 256 * 256; };
        parts = uint64_t(smoe::kKaGrid) * smoe::kKaWarps + pairs;
        part_bytes = up(parts * smoe::kKaHeads * c.head_dim * 4);
        stat_bytes = up(parts * smoe::kKaHeads * 8);
        meta_bytes = up(pairs * 8);
        logit_bytes = t.score_out ? all_heads * rows * 4 : 0;
    }
    uint64_t bytes() const { return part_bytes + stat_bytes + meta_bytes + logit_bytes; }
};

}  // namespace

size_t smoe::packed_scratch_bytes(int num_sms) { return PackedScratch(num_sms).bytes; }

extern "C" {

int smoe_cuda_attention_packed(SmoeCudaCtx* ctx, const SmoeCudaPackedAttnArgs* a) {
    if (!ctx || !a || !a->cu_q || a->num_heads == 0 || a->num_kv_heads == 0 || a->num_heads % a->num_kv_heads ||
        (a->window && !a->causal))
        return ctx_fail(SMOE_ERR_ARG, "bad packed attention arguments", 0);
    if (a->total_q == 0 || a->n_seqs == 0) return SMOE_OK;
    if (!a->q || !a->out || (a->total_k && (!a->k || !a->v)))
        return ctx_fail(SMOE_ERR_ARG, "packed attention: null operand", 0);
    if (a->head_dim == 0 || a->head_dim > 128 || a->head_dim % 8)
        return ctx_fail(SMOE_ERR_UNSUPPORTED, "packed attention takes head_dim <= 128, a multiple of 8", a->head_dim);
    if (a->num_heads / a->num_kv_heads > 128)
        return ctx_fail(SMOE_ERR_UNSUPPORTED, "at most 128 query heads per KV head", a->num_heads / a->num_kv_heads);
    // (a dimension of one element has no stride)
    const uint64_t rows[] = {a->q_row, a->out_row, a->k_row, a->v_row}, heads[] = {a->q_head, a->out_head, a->k_head, a->v_head};
    uint64_t all_strides = 0;
    for (int i = 0; i < 4; ++i) {
        const uint32_t n = i < 2 ? a->total_q : a->total_k, h = i < 2 ? a->num_heads : a->num_kv_heads;
        all_strides |= (n > 1 ? rows[i] : 0) | (h > 1 ? heads[i] : 0);
        if ((n > 1 && rows[i] == 0) || (h > 1 && heads[i] == 0 && i < 2))
            return ctx_fail(SMOE_ERR_ARG, "packed attention: a stride of 0 is taken for the heads of k and v only", i);
    }
    if (!aligned(a->q, 16) || !aligned(a->k, 16) || !aligned(a->v, 16) || !aligned(a->out, 16) || all_strides % 8)
        return ctx_fail(SMOE_ERR_ARG, "packed attention needs 16-byte aligned bases and strides that are multiples of 8", 0);
    if (!apart(a->out_row, a->out_head, a->total_q, a->num_heads, a->head_dim))
        return ctx_fail(SMOE_ERR_ARG, "packed attention: rows or heads of out overlap", long(a->out_row));
    if (!(a->scale >= 0.0f) || std::isinf(a->scale)) return ctx_fail(SMOE_ERR_ARG, "packed attention needs a finite scale >= 0", 0);
    const CtxView c = smoe::ctx_view(ctx);
    smoe::PackedArgs p{};
    p.a = *a;
    p.group = a->num_heads / a->num_kv_heads;
    p.scale_log2 = std::max(a->scale * 1.4426950408889634f, 1e-35f);
    p.err = c.err;
    // (a scale of 0 must still keep the masked scores' -inf: 1e-35 times any finite score is 0 to the exponential)
    p.tokens = smoe::kPaRows / p.group;
    CUtensorMap mq, mk, mv;
    int rc = map_rows(&mq, a->q, a->head_dim, a->num_heads, a->total_q, a->q_row, a->q_head, p.group, p.tokens);
    if (rc) return rc;
    // (KV heads that share their rows are one head of the map)
    p.k_step = a->k_head != 0;
    p.v_step = a->v_head != 0;
    if (a->total_k) {
        if ((rc = map_rows(&mk, a->k, a->head_dim, p.k_step ? a->num_kv_heads : 1, a->total_k, a->k_row, a->k_head, 1, smoe::kPaKeys)) ||
            (rc = map_rows(&mv, a->v, a->head_dim, p.v_step ? a->num_kv_heads : 1, a->total_k, a->v_row, a->v_head, 1, smoe::kPaKeys)))
            return rc;
    } else {
        mk = mv = mq;                            // no row has a key: never read
    }
    // at most one partial tile pair a sequence; the kernels count them
    const uint64_t pairs = uint64_t(a->total_q) / (2 * p.tokens) + std::min(a->n_seqs, a->total_q), ctas = pairs * a->num_kv_heads;
    if (ctas > 0x7fffffffu) return ctx_fail(SMOE_ERR_UNSUPPORTED, "packed attention: more than 2^31 tile pairs", long(ctas));
    const uint64_t most = pairs * (uint64_t(a->total_k) / smoe::kPaKeys + 3);
    // A CTA per pair when all of them fit the GPU at once and the keys of the whole call are few - the sequences' own lengths
    // are on the device - so that no pair can be long: the plan and the joining of cut pairs cost some 6 us. (Above 65,536
    // pairs, or 2^31 blocks, too.)
    const bool direct = (ctas <= uint64_t(c.num_sms) && a->total_k <= 16 * smoe::kPaKeys) || pairs > smoe::kPaMaxPairs || most >= (uint64_t(1) << 31);
    const bool sorted = !direct && ctas >= uint64_t(4) * c.num_sms;
    const PackedScratch sc(c.num_sms);
    uint8_t* ws = static_cast<uint8_t*>(c.packed);
    const uint32_t grid = direct ? uint32_t(ctas) : uint32_t(c.num_sms);
    if (!direct) {
        smoe::PaPlace* plan = nullptr;
        uint2* list = nullptr;
        if (sorted) {
            p.list = list = reinterpret_cast<uint2*>(ws + sc.list);
            p.taken = reinterpret_cast<uint32_t*>(ws);
        } else {
            p.plan = plan = reinterpret_cast<smoe::PaPlace*>(ws);
            p.part = reinterpret_cast<float*>(ws + sc.part);
            p.stat = reinterpret_cast<float2*>(ws + sc.stat);
        }
        if ((rc = launch(c, smoe::k_packed_plan, dim3(1), dim3(smoe::kPlThreads), 0, p, plan, grid,
                         reinterpret_cast<uint32_t*>(ws + sc.cost), reinterpret_cast<uint2*>(ws + sc.place), list)))
            return rc;
    }
    auto run = [&](auto kern, size_t smem, auto join) -> int {
        int r = smem_limit(c, kern, smem);
        if (r || (r = launch(c, kern, dim3(grid), dim3(smoe::kPaThreads), smem, mq, mk, mv, p)) || !p.plan) return r;
        return launch(c, join, dim3(grid, 8), dim3(256), 0, p);
    };
    return a->head_dim <= 64 ? run(smoe::k_attention_packed<64>, smoe::PackedSmem<64>::bytes(), smoe::k_packed_join<64>)
                             : run(smoe::k_attention_packed<128>, smoe::PackedSmem<128>::bytes(), smoe::k_packed_join<128>);
}

uint64_t smoe_cuda_kv4_block_bytes(uint32_t head_dim) {
    return head_dim == 64 || head_dim == 128 ? smoe::Kv4Geom(head_dim).block : 0;
}

int smoe_cuda_kv4_append(SmoeCudaCtx* ctx, const SmoeKv4Cache* cache, const SmoeKv4Rows* rows) {
    if (!ctx) return ctx_fail(SMOE_ERR_ARG, "null context", 0);
    int rc = check_cache(cache, "kv4_append: bad cache");
    if (rc || (rc = check_rows(rows, cache, false, "kv4_append: bad rows"))) return rc;
    if (rows->total == 0) return SMOE_OK;
    const CtxView c = smoe::ctx_view(ctx);
    using namespace smoe;
    auto run = [&](auto kern) {
        return launch(c, kern, dim3((rows->total - 1) / kKwRows + 1), dim3(kKwThreads), 0, Kv4Args{*cache, c.err}, *rows);
    };
    if (rows->dtype == SMOE_DTYPE_F32) return run(k_kv4_append<SMOE_DTYPE_F32, true>);
    return wide_rows(rows) ? run(k_kv4_append<SMOE_DTYPE_BF16, true>) : run(k_kv4_append<SMOE_DTYPE_BF16, false>);
}

int smoe_cuda_kv4_read(SmoeCudaCtx* ctx, const SmoeKv4Cache* cache, const uint32_t* first, const SmoeKv4Rows* rows) {
    if (!ctx) return ctx_fail(SMOE_ERR_ARG, "null context", 0);
    int rc = check_cache(cache, "kv4_read: bad cache");
    if (rc || (rc = check_rows(rows, cache, true, "kv4_read: bad rows"))) return rc;
    if (rows->total == 0) return SMOE_OK;
    const CtxView c = smoe::ctx_view(ctx);
    using namespace smoe;
    auto run = [&](auto kern) {
        return launch(c, kern, dim3((rows->total - 1) / kKwRows + 1), dim3(kKwThreads), 0, Kv4Args{*cache, c.err}, first, *rows);
    };
    if (rows->dtype == SMOE_DTYPE_F32) return run(k_kv4_read<SMOE_DTYPE_F32, true>);
    return wide_rows(rows) ? run(k_kv4_read<SMOE_DTYPE_BF16, true>) : run(k_kv4_read<SMOE_DTYPE_BF16, false>);
}

uint64_t smoe_cuda_kv4_attention_workspace(const SmoeKv4Cache* cache, const SmoeKv4AttnArgs* t) {
    if (!cache || !t || cache->num_kv_heads == 0) return 0;
    return AttnPlan(*cache, *t).bytes();
}

int smoe_cuda_kv4_attention(SmoeCudaCtx* ctx, const SmoeKv4Cache* cache, const SmoeKv4AttnArgs* t) {
    if (!ctx || !t) return ctx_fail(SMOE_ERR_ARG, "kv4_attention: null argument", 0);
    int rc = check_cache(cache, "kv4_attention: bad cache");
    if (rc) return rc;
    if (!t->q || !t->out || t->num_heads == 0 || t->num_heads % cache->num_kv_heads || t->max_len > 0x7fffffffu)
        return ctx_fail(SMOE_ERR_ARG, "kv4_attention: bad arguments", t->num_heads);
    if (!(t->scale >= 0.0f) || std::isinf(t->scale)) return ctx_fail(SMOE_ERR_ARG, "kv4_attention needs a finite scale >= 0", 0);
    if (t->dtype != SMOE_DTYPE_F32 && t->dtype != SMOE_DTYPE_BF16)
        return ctx_fail(SMOE_ERR_ARG, "kv4_attention: q and out are fp32 or bf16", t->dtype);
    if (!aligned(t->q, 16) || !aligned(t->out, 16) || (t->q_row | t->out_row) % 4)
        return ctx_fail(SMOE_ERR_ARG, "kv4_attention needs 16-byte aligned q and out and strides that are multiples of 4", 0);
    if (cache->n_seqs > 1 && t->out_row < uint64_t(t->num_heads) * cache->head_dim)
        return ctx_fail(SMOE_ERR_ARG, "kv4_attention: rows of out overlap", long(t->out_row));
    if (uint64_t(cache->n_seqs) * t->num_heads * ((uint64_t(t->max_len) + SMOE_KV4_PAGE - 1) / SMOE_KV4_PAGE) >= (uint64_t(1) << 31))
        return ctx_fail(SMOE_ERR_UNSUPPORTED, "kv4_attention: more than 2^31 pages to read", long(t->max_len));
    if (t->num_heads / cache->num_kv_heads > 6144)                // (the joining kernel takes 8 bytes of shared memory for each)
        return ctx_fail(SMOE_ERR_UNSUPPORTED, "kv4_attention: at most 6144 query heads per KV head", t->num_heads);
    const uint64_t need = smoe_cuda_kv4_attention_workspace(cache, t);
    if (need && (!t->workspace || t->workspace_bytes < need || !aligned(t->workspace, 16)))
        return ctx_fail(SMOE_ERR_ARG, "kv4_attention: workspace missing, too small or unaligned; bytes needed", long(need));
    const CtxView c = smoe::ctx_view(ctx);
    const AttnPlan plan(*cache, *t);
    smoe::Kv4Attn p{};
    p.a = {*cache, c.err};
    p.t = *t;
    p.group = t->num_heads / cache->num_kv_heads;
    p.chunks = plan.chunks;
    p.warps = smoe::kKaGrid * smoe::kKaWarps;
    uint8_t* ws = static_cast<uint8_t*>(t->workspace);
    p.part = reinterpret_cast<float*>(ws);
    p.stat = reinterpret_cast<float2*>(ws + plan.part_bytes);
    p.meta = reinterpret_cast<uint2*>(ws + plan.part_bytes + plan.stat_bytes);
    p.logits = plan.logit_bytes ? reinterpret_cast<float*>(ws + plan.part_bytes + plan.stat_bytes + plan.meta_bytes) : nullptr;
    p.rows = plan.rows;
    // (a scale of 0 must still keep the masked scores' -inf: 1e-35 times any finite score is 0 to the exponential)
    p.scale_log2 = std::max(t->scale * 1.4426950408889634f, 1e-35f);
    p.most_e = std::min(100, std::ilogb(std::min(p.scale_log2, 1e30f)) + 126);
    auto run = [&](auto kern, uint32_t smem) -> int {
        const int r = smem_limit(c, kern, smem);
        return r ? r : launch(c, kern, dim3(smoe::kKaGrid), dim3(smoe::kKaWarps * 32), smem, p);
    };
    using namespace smoe;
    const bool f32 = t->dtype == SMOE_DTYPE_F32;
    if (cache->head_dim == 64) rc = f32 ? run(k_kv4_attention<1, 2>, kv4_attn_smem<1>()) : run(k_kv4_attention<1, 1>, kv4_attn_smem<1>());
    else rc = f32 ? run(k_kv4_attention<2, 2>, kv4_attn_smem<2>()) : run(k_kv4_attention<2, 1>, kv4_attn_smem<2>());
    if (rc) return rc;
    // threads an output: about a quarter of the parts that a pair has when all are equally long
    const uint32_t pages = (t->max_len + SMOE_KV4_PAGE - 1) / SMOE_KV4_PAGE;
    const uint64_t pairs = uint64_t(cache->n_seqs) * cache->num_kv_heads * plan.chunks;
    const uint64_t usual = std::min<uint64_t>(p.warps / pairs + 2, pages);
    p.lanes = cache->head_dim == 64 ? 2 : 1;                      // (1024 / lanes outputs: within one round of heads)
    while (p.lanes < 64 && p.lanes * 4 < usual) p.lanes *= 2;
    const uint32_t per = 4 * kKjThreads / p.lanes, outs = (p.group * cache->head_dim + per - 1) / per;
    const uint32_t entries = p.logits ? (t->max_len + kKjEntries - 1) / kKjEntries : 0u;
    // (past 5,000 heads more than a launch has without asking, with the kernel's own arrays)
    if (p.group > 5000 && (rc = smem_limit(c, k_kv4_join, 6144 * 8))) return rc;
    return launch(c, k_kv4_join, dim3(outs + entries, cache->num_kv_heads, cache->n_seqs), dim3(kKjThreads),
                  size_t(plan.chunks) * kKaHeads * 8, p, outs);
}

uint64_t smoe_cuda_kv4_evict_workspace(const SmoeKv4Cache* cache, uint32_t max_len) {
    // a pair moves at most min(keep, len - keep) <= len / 2 entries
    return cache ? uint64_t(cache->n_seqs) * cache->num_kv_heads * (uint64_t(max_len / 2) * 2 + 2) * 4 : 0;
}

int smoe_cuda_kv4_evict(SmoeCudaCtx* ctx, const SmoeKv4Cache* cache, uint32_t keep, uint32_t recent, uint32_t max_len,
                        uint32_t* pos_out, float* score_out, void* workspace, uint64_t workspace_bytes) {
    if (!ctx) return ctx_fail(SMOE_ERR_ARG, "null context", 0);
    int rc = check_cache(cache, "kv4_evict: bad cache");
    if (rc) return rc;
    if (!cache->pos || !cache->score) return ctx_fail(SMOE_ERR_ARG, "kv4_evict needs the cache's pos and score", 0);
    if (keep == 0 || max_len > 0x7fffffffu) return ctx_fail(SMOE_ERR_ARG, "kv4_evict: bad keep or max_len", keep);
    if (!pos_out != !score_out || pos_out == cache->pos || score_out == cache->score) {
        // one of the two alone, or the cache's own array: in place is asked for with NULL
        return ctx_fail(SMOE_ERR_ARG, "kv4_evict: pos_out and score_out are both NULL or both separate arrays", 0);
    }
    if (!aligned(pos_out, 16) || !aligned(score_out, 16))
        return ctx_fail(SMOE_ERR_ARG, "kv4_evict: pos_out and score_out must be 16-byte aligned", 0);
    const uint64_t need = smoe_cuda_kv4_evict_workspace(cache, max_len);
    if (!workspace || workspace_bytes < need || !aligned(workspace, 16))
        return ctx_fail(SMOE_ERR_ARG, "kv4_evict: workspace missing, too small or unaligned; bytes needed", long(need));
    const CtxView c = smoe::ctx_view(ctx);
    // CTAs of a pair: 8192 entries each, 8 at most; past what their shared memory holds keys are read again each time
    uint32_t ctas = 1;
    while (ctas < smoe::kEvCtas && uint64_t(ctas) * 8192 < max_len) ctas *= 2;
    const uint32_t cached = std::min<uint32_t>(49152, (max_len / ctas + 64 + 31) / 32 * 32);
    if (uint64_t(cache->num_kv_heads) * ctas > 0x7fffffffu) return ctx_fail(SMOE_ERR_ARG, "kv4_evict: too many KV heads", cache->num_kv_heads);
    if ((rc = smem_limit(c, smoe::k_kv4_evict, smoe::kv4_evict_smem(49152)))) return rc;
    smoe::Kv4Evict p{{*cache, c.err}, keep, recent, max_len, pos_out, score_out, static_cast<uint32_t*>(workspace),
                     std::max(1u, max_len / 2), cached};
    return launch_cluster(c, smoe::k_kv4_evict, dim3(cache->num_kv_heads * ctas, cache->n_seqs), dim3(smoe::kEvThreads),
                          smoe::kv4_evict_smem(cached), ctas, p);
}

int smoe_cuda_kv4_advance(SmoeCudaCtx* ctx, uint32_t* len, uint32_t* seen, uint32_t n_seqs, const uint32_t* cu,
                          uint32_t n_each, uint32_t keep) {
    if (!ctx || !len || n_seqs == 0) return ctx_fail(SMOE_ERR_ARG, "bad kv4_advance arguments", n_seqs);
    const CtxView c = smoe::ctx_view(ctx);
    return launch(c, smoe::k_kv4_advance, dim3((n_seqs - 1) / 256 + 1), dim3(256), 0, len, seen, n_seqs, cu, n_each, keep, c.err);
}

}  // extern "C"
