// serve.cuh - what the long-context serving entries (smoe_serve.cu) share:
// the parts of the context they use, their launches, and the look-up of a
// packed row's sequence.
#pragma once
#include <atomic>
#include <cuda_runtime.h>

#include "../../include/smoe_cuda.h"
#include "smoe_common.cuh"

namespace smoe {

struct CtxView {
    int device, num_sms;
    size_t smem_optin;
    cudaStream_t stream;
    uint32_t* err;                       // device error word
    std::atomic<uint64_t>* dispatches;
    void* packed;                        // packed attention: plan and parts of cut tile pairs (packed_scratch_bytes)
};
size_t packed_scratch_bytes(int num_sms);                // smoe_serve.cu
CtxView ctx_view(SmoeCudaCtx* c);                        // smoe_cuda.cu
int ctx_fail(int code, const char* msg, long v);         // sets the message of the failure, returns code

// Programmatic dependent launch: the next kernel of the stream may start its
// set-up while this one runs; it waits for this one's end before it touches
// memory. Every kernel of these entries waits, and all release their dependents
// at once but the cache attention (at its end) and its join (by its end).
SMOE_DEVINL void pdl_release() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
SMOE_DEVINL void pdl_acquire() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

// Every global read of these kernels is an ordinary load, never __ldg: a
// dependent launch is resident before its predecessors end, so the read-only
// path may hold lines that they have since rewritten (len, for one, is read
// by every kernel of a step and advanced at its end), and only ordinary loads
// are ordered by pdl_acquire.
template <typename T>
SMOE_DEVINL T ld_plain(const T* p) { return *p; }

// One lane of a converged warp. Bulk copies and tensor-core instructions take
// their operands from uniform registers: under this predicate the compiler
// moves them there once, under `lane == 0` it adds a loop over the lanes'
// values to each (some 40 instructions a copy).
SMOE_DEVINL bool elect_one() {
    uint32_t p;
    asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.u32 %0, 1, 0, p;\n}\n" : "=r"(p));
    return p != 0;
}

static __device__ __noinline__ void serve_err(uint32_t* err, uint32_t code) { atomicCAS(err, 0u, code); }

// The sequence s with cu[s] <= row < cu[s + 1] (cu ascending, cu[0] = 0), by
// one warp together: each step looks at 32 bounds, so 1024 sequences take
// two dependent loads. n when there is none.
SMOE_DEVINL uint32_t seq_of_row(const uint32_t* cu, uint32_t n, uint32_t row, uint32_t lane) {
    uint32_t lo = 0, span = n;           // the answer is in [lo, lo + span)
#pragma unroll 1
    while (span > 1) {
        const uint32_t step = (span + 31) / 32, at = lo + min((lane + 1) * step, span);
        const uint32_t past = __ballot_sync(0xffffffffu, ld_plain(cu + at) <= row);   // bounds at or below the row
        const uint32_t k = __popc(past);
        if (k * step >= span) return n;
        lo += k * step;
        span = min(step, span - k * step);
    }
    return (span == 1 && ld_plain(cu + lo) <= row && row < ld_plain(cu + lo + 1)) ? lo : n;
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

}  // namespace smoe
