// Device and launch helpers shared by the attention-side kernels: 16-element
// row pieces of fp16 / bf16 tensors, programmatic dependent launch, the status
// words of these translation units.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cstdint>

#include "gemv_common.cuh"

namespace clb {

template <bool kBf16>
__device__ __forceinline__ float2 unpack2(uint32_t v) {
    if (kBf16) return __bfloat1622float2(*reinterpret_cast<__nv_bfloat162*>(&v));
    return __half22float2(*reinterpret_cast<__half2*>(&v));
}

template <bool kBf16>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
    if (kBf16) {
        __nv_bfloat162 r = __floats2bfloat162_rn(lo, hi);
        return *reinterpret_cast<uint32_t*>(&r);
    }
    __half2 r = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<uint32_t*>(&r);
}

// 8 consecutive elements starting at element `at`; kVec: 16-byte aligned.
template <bool kBf16, bool kVec>
__device__ __forceinline__ uint4 load8(const void* p, int64_t at) {
    const uint16_t* e = static_cast<const uint16_t*>(p) + at;
    if constexpr (kVec) {
        return *reinterpret_cast<const uint4*>(e);
    } else {
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = (uint32_t)e[2 * i] | ((uint32_t)e[2 * i + 1] << 16);
        return make_uint4(w[0], w[1], w[2], w[3]);
    }
}

template <bool kVec>
__device__ __forceinline__ void store8(void* p, int64_t at, uint4 v) {
    uint16_t* e = static_cast<uint16_t*>(p) + at;
    if (kVec) {
        *reinterpret_cast<uint4*>(e) = v;
        return;
    }
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        e[2 * i] = (uint16_t)w[i];
        e[2 * i + 1] = (uint16_t)(w[i] >> 16);
    }
}

template <bool kBf16>
__device__ __forceinline__ void unpack8(uint4 v, float* x) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 f = unpack2<kBf16>(w[i]);
        x[2 * i] = f.x;
        x[2 * i + 1] = f.y;
    }
}

template <bool kBf16>
__device__ __forceinline__ uint4 pack8(const float* x) {
    return make_uint4(pack2<kBf16>(x[0], x[1]), pack2<kBf16>(x[2], x[3]),
                      pack2<kBf16>(x[4], x[5]), pack2<kBf16>(x[6], x[7]));
}

// n / d for 0 <= n < 2^31 by a multiplication, d fixed at launch.
struct FastDiv {
    uint32_t d, mul, shift;
    FastDiv() = default;
    explicit FastDiv(uint32_t divisor) : d(divisor), mul(0), shift(0) {
        while (((uint64_t)1 << shift) < d) ++shift;
        mul = (uint32_t)((((uint64_t)1 << 32) * (((uint64_t)1 << shift) - d)) / d + 1);
    }
    __device__ __forceinline__ int div(int n) const {
        return (int)((__umulhi((uint32_t)n, mul) + (uint32_t)n) >> shift);
    }
    __device__ __forceinline__ int mod(int n) const { return n - div(n) * (int)d; }
};

// Rows of 16-bit elements that 16-byte accesses may be used on.
inline bool aligned16(const void* p, int64_t stride0, int64_t stride1) {
    return (reinterpret_cast<uintptr_t>(p) & 15u) == 0 && stride0 % 8 == 0 && stride1 % 8 == 0;
}

// 16-byte asynchronous copies to shared memory, in groups.
__device__ __forceinline__ void copy16(void* to, const void* from, bool go) {
    if (go)
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(to)), "l"(from)
                     : "memory");
}
__device__ __forceinline__ void copies_end_group() {
    asm volatile("cp.async.commit_group;" ::: "memory");
}
template <int kLeft>
__device__ __forceinline__ void copies_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(kLeft) : "memory");
}

// One poll of an mbarrier phase that the hardware may hold for up to `hold_ns`
// before it answers no: a warp that waits then issues next to nothing (plain
// polls took half of the issue slots of the prefix kernel).
__device__ __forceinline__ bool mbar_try_wait_held(uint32_t bar, uint32_t parity, uint32_t hold_ns) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(bar), "r"(parity), "r"(hold_ns)
        : "memory");
    return ok != 0;
}
constexpr uint32_t kHoldNs = 20000;
// Nanoseconds for which a wait bounded by `budget` SM cycles (about half a
// nanosecond each) is held.
inline uint32_t hold_within(long long budget) {
    return budget < 2 ? 1 : budget / 2 < kHoldNs ? (uint32_t)(budget / 2) : kHoldNs;
}

// Bounded wait on one phase, at most `budget` SM cycles and one poll more.
__device__ __forceinline__ bool mbar_wait_held(uint32_t bar, uint32_t parity, long long budget) {
    if (mbar_try_wait_held(bar, parity, kHoldNs)) return true;
    const long long t0 = clock64();
#pragma unroll 1
    while (!mbar_try_wait_held(bar, parity, kHoldNs)) {
        if (clock64() - t0 > budget) return false;
    }
    return true;
}

// Programmatic dependent launch: the kernel waits (griddepcontrol.wait) before
// its first global access, so the launch latency is hidden and stream order kept.
template <typename... P, typename... A>
cudaError_t launch_pdl(void (*kernel)(P...), dim3 grid, dim3 block, size_t smem,
                       cudaStream_t stream, const A&... args) {
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = grid;
    cfg.blockDim = block;
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kernel, args...);
}

// Reads (optionally clears) a status word of the calling translation unit.
template <typename Symbol>
cudaError_t read_status_symbol(Symbol& symbol, int clear, int* status) {
    cudaError_t e = cudaMemcpyFromSymbol(status, symbol, sizeof(int));
    const int zero = 0;
    if (e == cudaSuccess && clear) e = cudaMemcpyToSymbol(symbol, &zero, sizeof(int));
    return e;
}

}  // namespace clb
