// sjk_kv16.cuh - what the kernels of the 16-bit layers share: element types, table look-ups, programmatic launches.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <atomic>

#include "sjk_common.cuh"

namespace sjk16 {

SJK_HD size_t type_bytes(int type) { return type == SJK_F32 ? 4u : 2u; }
static inline bool type_ok(int type) { return type == SJK_F32 || type == SJK_F16 || type == SJK_BF16; }
static inline bool aligned(const void * p, size_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

// rows whose address is a multiple of an element's size; a list of int32 (NULL passes)
static inline bool rows_ok(const sjk_rows & r) { return aligned(r.p, type_bytes(r.type)); }
static inline bool list_ok(const void * p) { return aligned(p, 4); }
// no byte of `na` from a is one of `nb` from b (NULL passes): what one CTA writes while others still read
static inline bool apart(const void * a, size_t na, const void * b, size_t nb) {
    const uintptr_t x = reinterpret_cast<uintptr_t>(a), y = reinterpret_cast<uintptr_t>(b);
    return !a || !b || !na || !nb || (x < y ? y - x >= na : x - y >= nb);
}

// two 16-bit values of a word, widened; two floats rounded to nearest even and packed
template <int TYPE>
SJK_DEV float2 widen2(uint32_t w) {
    if constexpr (TYPE == SJK_F16) return __half22float2(*reinterpret_cast<const __half2 *>(&w));
    else return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xFFFF0000u));
}
template <int TYPE>
SJK_DEV uint32_t pack2(float a, float b) {
    if constexpr (TYPE == SJK_F16) { const __half2 h = __floats2half2_rn(a, b); return *reinterpret_cast<const uint32_t *>(&h); }
    else { const __nv_bfloat162 h = __floats2bfloat162_rn(a, b); return *reinterpret_cast<const uint32_t *>(&h); }
}

SJK_DEV float load1(const void * p, int64_t i, int type) {
    if (type == SJK_F32) return static_cast<const float *>(p)[i];
    if (type == SJK_F16) return __half2float(static_cast<const __half *>(p)[i]);
    return __bfloat162float(static_cast<const __nv_bfloat16 *>(p)[i]);
}
SJK_DEV void store1(void * p, int64_t i, int type, float x) {
    if (type == SJK_F32) static_cast<float *>(p)[i] = x;
    else if (type == SJK_F16) static_cast<__half *>(p)[i] = __float2half_rn(x);
    else static_cast<__nv_bfloat16 *>(p)[i] = __float2bfloat16_rn(x);
}

SJK_DEV void pdl_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
SJK_DEV void pdl_release() { asm volatile("griddepcontrol.launch_dependents;"); }

// The kernels of this family are programmatic dependents of what precedes them in the stream: each waits for its
// predecessors (griddepcontrol.wait) before it touches memory, so only the launch itself overlaps them.
template <typename... Params, typename... Args>
static inline int launch(void (*kernel)(Params...), dim3 grid, dim3 block, size_t smem, sjk_stream st, Args &&... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = block;
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    return sjk_check(cudaLaunchKernelEx(&cfg, kernel, static_cast<Params>(args)...));
}

// A kernel's dynamic shared memory limit, raised to `bytes` on the current device at the first call there.
template <auto KERNEL>
static inline int smem_limit(size_t bytes) {
    static std::atomic<uint64_t> done{0};
    int dev = 0;
    if (sjk_check(cudaGetDevice(&dev))) return SJK_ERR_DEVICE;
    const uint64_t bit = dev < 64 ? 1ull << dev : 0ull;
    if (done.load(std::memory_order_relaxed) & bit) return 0;
    if (sjk_check(cudaFuncSetAttribute(KERNEL, cudaFuncAttributeMaxDynamicSharedMemorySize, (int) bytes))) return SJK_ERR_DEVICE;
    done.fetch_or(bit, std::memory_order_relaxed);
    return 0;
}

}  // namespace sjk16
