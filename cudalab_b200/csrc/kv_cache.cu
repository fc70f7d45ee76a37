// Quantisation of K and V as they are written into the paged cache
// (kv_layout.cuh), and reading tokens back.
//
// Per token and head: s = fp16(min(max|x| / top, 65504)), top = 127 (int8) or
// 7 (int4); q = clamp(rint(x * (1 / s)), -top, top) with the stored s, so the
// rounding of s to fp16 costs no accuracy; s = 0 gives q = 0, NaN is stored
// as 0 and infinities saturate.  Every step is one IEEE operation in fp32.
// x * (1 / s) instead of x / s: one division per row instead of one per
// element, which at the instruction count of an IEEE division would bound the
// kernel; it can differ from x / s only where x lies within an fp32 rounding
// of the middle between two steps, where both are as near.
//
// Both kernels are bound by memory: the write reads 2 B and writes bits / 8 B
// per element, the read the reverse.  head_dim / 16 lanes share a row; a lane
// holds 8 elements in each half of it, so that the lanes touch the 16-bit
// elements in whole lines (with 16 neighbours a lane every access was one of
// half sectors: 37 us for the 33 below), and takes K and V, so that four
// loads are in flight.  8 heads of 128: reading 32768 tokens, int8, 33.3 us (33.5 to
// 34.1 in a loop of calls), 6.1 TB/s, 0.93 of a copy; writing 8192 tokens as int4
// and reading them back 17.2 us (18.4), 4.9 TB/s, for two kernels of 6.5 us' bytes
// each and their ramps.  (The write's
// instructions show as well: 16 for each element took 21 us where 13 took 20.)
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cstdint>

#include "gemv_common.cuh"
#include "kv_device.cuh"
#include "kv_layout.cuh"

namespace clb {
namespace {

__device__ int g_kv_status;

constexpr int kThreads = 128;

// Place of a slot: its page's block, and the token's row j in the block.
struct Place {
    const uint8_t* block;
    int j;
};

__device__ __forceinline__ bool find_slot(const KvCacheArgs& a, const FastDiv& page_size,
                                          int64_t slot, int head, int block_bytes, Place* p) {
    if (slot < 0) return false;
    int64_t page;
    int off;
    if (slot <= 0x7fffffff) {
        page = page_size.div((int)slot);
        off = page_size.mod((int)slot);
    } else {
        page = slot / a.page_size;
        off = (int)(slot % a.page_size);
    }
    if (page >= a.num_pages) {
        atomicCAS(&g_kv_status, 0, kStatusKvIndex);
        return false;
    }
    const int blocks = a.page_size / kKvBlock;
    p->block = a.pages + ((page * a.kv_heads + head) * blocks + off / kKvBlock) * block_bytes;
    p->j = off % kKvBlock;
    return true;
}

// Two elements' larger magnitudes, NaN where one is.
template <bool kBf16>
__device__ __forceinline__ uint32_t larger2(uint32_t a, uint32_t b) {
    uint32_t r;
    b &= 0x7fff7fffu;
    if (kBf16)
        asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    else
        asm("max.NaN.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
}

// Largest magnitude of 16 elements, NaN if one of them is.
template <bool kBf16>
__device__ __forceinline__ float max16(const uint32_t (&w)[8]) {
    uint32_t m = w[0] & 0x7fff7fffu;
#pragma unroll
    for (int i = 1; i < 8; ++i) m = larger2<kBf16>(m, w[i]);
    const float2 f = unpack2<kBf16>(m);
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(f.x), "f"(f.y));
    return r;
}

// m / kTop, correctly rounded, for m of a 16-bit type: the product with the
// rounded reciprocal and one step on its remainder, which is exact (Markstein,
// IBM J. Res. Dev. 34, 1990).  A general division is three times as long.
template <int kTop>
__device__ __forceinline__ float over_top(float m) {
    constexpr float top = kTop, inv = 1.f / top;
    const float q = __fmul_rn(m, inv);
    return fmaf(fmaf(-q, top, m), inv, q);
}

// rint(x * inv) as two's complement fields, for |x * inv| < top + 1/2.  Adding
// 1.5 * 2^23 rounds to the nearest even integer and leaves it in the low bits,
// without the quarter-rate conversion.
template <int kBits>
__device__ __forceinline__ void quantise16(const float (&x)[16], float inv, uint32_t* out) {
    uint32_t q[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) q[i] = __float_as_uint(__fmul_rn(x[i], inv) + 12582912.f);
    if (kBits == 8) {
#pragma unroll
        for (int w = 0; w < 4; ++w)
            out[w] = prmt_i<0x5410u>(prmt_i<0x0040u>(q[4 * w], q[4 * w + 1]),
                                     prmt_i<0x0040u>(q[4 * w + 2], q[4 * w + 3]));
    } else {
        // sum_i 16^i (q_i + 8), whose digits 1 to 15 do not carry; then the
        // sign bit of every digit flipped back
        constexpr uint32_t kMagic = 0x4b400000u, kDigits = 0x11111111u;
#pragma unroll
        for (int w = 0; w < 2; ++w) {
            uint32_t r = q[8 * w + 7];
#pragma unroll
            for (int i = 6; i >= 0; --i) r = 16u * r + q[8 * w + i];
            out[w] = (r + kDigits * (8u - kMagic)) ^ 0x88888888u;
        }
    }
}

// 16 fields as floats: the field, its sign bit flipped, in the mantissa of
// 2^23, less 2^23 and the flip (exact).
template <int kBits>
__device__ __forceinline__ void expand16(const uint32_t (&raw)[4], float (&x)[16]) {
    if (kBits == 8) {
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            const uint32_t u = raw[w] ^ 0x80808080u;
            x[4 * w] = __uint_as_float(prmt_i<0x7650u>(u, 0x4b000000u)) - 8388736.f;
            x[4 * w + 1] = __uint_as_float(prmt_i<0x7651u>(u, 0x4b000000u)) - 8388736.f;
            x[4 * w + 2] = __uint_as_float(prmt_i<0x7652u>(u, 0x4b000000u)) - 8388736.f;
            x[4 * w + 3] = __uint_as_float(prmt_i<0x7653u>(u, 0x4b000000u)) - 8388736.f;
        }
    } else {
#pragma unroll
        for (int i = 0; i < 16; ++i)
            x[i] = __uint_as_float(lop3_sel_xor(raw[i / 8] >> (4 * (i % 8)), 0xFu, 0x4b000008u)) -
                   8388616.f;
    }
}

// 12 CTAs an SM, 40 registers (17.2 us for the 8192 tokens above, by 10 17.7, by
// 16 18.3).
template <int kDim, int kBits, bool kBf16, bool kVec>
__global__ void __launch_bounds__(kThreads, 12)
    kv_write_kernel(const KvCacheArgs a, const FastDiv heads, const FastDiv page_size) {
    constexpr int kRow = kDim * kBits / 8, kLanes = kDim / 16, kTop = kBits == 8 ? 127 : 7;
    constexpr int kBlockBytes = kv_block_bytes(kRow);
    pdl_allow_dependents();
    pdl_wait_prior_grids();
    const int row = (int)(blockIdx.x * (kThreads / kLanes) + threadIdx.x / kLanes);
    const int l = threadIdx.x % kLanes;
    const int64_t token = heads.div(row);
    const int head = heads.mod(row);
    const bool in = token < a.tokens;
    const int64_t slot = in ? a.slots[token] : -1;
    uint32_t w[2][8] = {};
    if (in) {
#pragma unroll
        for (int part = 0; part < 2; ++part) {
            const void* from = part ? a.v : a.k;
            const int64_t at = 8 * l + (part ? token * a.v_token + head * a.v_head
                                             : token * a.k_token + head * a.k_head);
            const uint4 x = load8<kBf16, kVec>(from, at);
            const uint4 y = load8<kBf16, kVec>(from, at + kDim / 2);
            w[part][0] = x.x, w[part][1] = x.y, w[part][2] = x.z, w[part][3] = x.w;
            w[part][4] = y.x, w[part][5] = y.y, w[part][6] = y.z, w[part][7] = y.w;
        }
    }
    Place p;
    const bool put = find_slot(a, page_size, slot, head, kBlockBytes, &p);
#pragma unroll
    for (int part = 0; part < 2; ++part) {
        float m = max16<kBf16>(w[part]);
        if (!(m == m)) {  // NaN is stored as 0
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float2 f = unpack2<kBf16>(w[part][i]);
                w[part][i] &= (f.x == f.x ? 0xffffu : 0u) | (f.y == f.y ? 0xffff0000u : 0u);
            }
            m = max16<kBf16>(w[part]);
        }
#pragma unroll
        for (int o = kLanes / 2; o > 0; o >>= 1)
            m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
        // at most 65504 = 2^16 - 32 with m limited to kTop of it
        const __half s = __float2half_rn(over_top<kTop>(fminf(m, 65504.f * kTop)));
        if (!put) continue;
        float x[16];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float2 f = unpack2<kBf16>(w[part][i]);
            x[2 * i] = f.x;
            x[2 * i + 1] = f.y;
        }
        const uint32_t bits = __half_as_ushort(s);
        float inv = bits ? __frcp_rn(__half2float(s)) : 0.f;
        // A normal s is within 2^-11 of m / kTop, so |x / s| < kTop + 1/2; one
        // that is subnormal or at its limit need not be.
        if (bits - 1u < 0x3ffu || bits >= 0x7bffu) {
#pragma unroll
            for (int i = 0; i < 16; ++i)
                x[i] = fminf(fmaxf(__fmul_rn(x[i], inv), -(float)kTop), (float)kTop);
            inv = 1.f;
        }
        uint32_t q[4];
        quantise16<kBits>(x, inv, q);
        uint8_t* rows = const_cast<uint8_t*>(p.block) + part * kKvBlock * kRow;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            uint8_t* to = rows + kv_offset<kRow>(p.j, kBits * l + i * (kRow / 2));
            if (kBits == 8)
                *reinterpret_cast<uint2*>(to) = make_uint2(q[2 * i], q[2 * i + 1]);
            else
                *reinterpret_cast<uint32_t*>(to) = q[i];
        }
        if (l == 0)
            reinterpret_cast<__half*>(const_cast<uint8_t*>(p.block) +
                                      2 * kKvBlock * kRow)[part * kKvBlock + p.j] = s;
    }
}

template <int kDim, int kBits, bool kBf16, bool kVec>
__global__ void __launch_bounds__(kThreads) kv_read_kernel(const KvCacheArgs a, const FastDiv heads,
                                                           const FastDiv page_size) {
    constexpr int kRow = kDim * kBits / 8, kLanes = kDim / 16;
    constexpr int kBlockBytes = kv_block_bytes(kRow);
    pdl_allow_dependents();
    pdl_wait_prior_grids();
    const int row = (int)(blockIdx.x * (kThreads / kLanes) + threadIdx.x / kLanes);
    const int l = threadIdx.x % kLanes;
    const int64_t token = heads.div(row);
    const int head = heads.mod(row);
    if (token >= a.tokens) return;
    Place p;
    const bool have = find_slot(a, page_size, a.slots[token], head, kBlockBytes, &p);
    uint32_t raw[2][4] = {};
    float s[2] = {0.f, 0.f};
    if (have) {
#pragma unroll
        for (int part = 0; part < 2; ++part) {
            const uint8_t* rows = p.block + part * kKvBlock * kRow;
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const uint8_t* from = rows + kv_offset<kRow>(p.j, kBits * l + i * (kRow / 2));
                if (kBits == 8) {
                    const uint2 r = *reinterpret_cast<const uint2*>(from);
                    raw[part][2 * i] = r.x, raw[part][2 * i + 1] = r.y;
                } else {
                    raw[part][i] = *reinterpret_cast<const uint32_t*>(from);
                }
            }
            s[part] = __half2float(reinterpret_cast<const __half*>(
                p.block + 2 * kKvBlock * kRow)[part * kKvBlock + p.j]);
        }
    }
#pragma unroll
    for (int part = 0; part < 2; ++part) {
        float x[16];
        expand16<kBits>(raw[part], x);
#pragma unroll
        for (int i = 0; i < 16; ++i) x[i] = __fmul_rn(x[i], s[part]);
        void* y = part ? a.v : a.k;
        const int64_t at = part ? token * a.v_token + head * a.v_head
                                : token * a.k_token + head * a.k_head;
        store8<kVec>(y, at + 8 * l, pack8<kBf16>(x));
        store8<kVec>(y, at + 8 * l + kDim / 2, pack8<kBf16>(x + 8));
    }
}

using Kernel = void (*)(KvCacheArgs, FastDiv, FastDiv);

template <bool kWrite, int kDim, int kBits>
Kernel pick(bool bf16, bool vec) {
    if constexpr (kWrite)
        return bf16 ? (vec ? kv_write_kernel<kDim, kBits, true, true>
                           : kv_write_kernel<kDim, kBits, true, false>)
                    : (vec ? kv_write_kernel<kDim, kBits, false, true>
                           : kv_write_kernel<kDim, kBits, false, false>);
    else
        return bf16 ? (vec ? kv_read_kernel<kDim, kBits, true, true>
                           : kv_read_kernel<kDim, kBits, true, false>)
                    : (vec ? kv_read_kernel<kDim, kBits, false, true>
                           : kv_read_kernel<kDim, kBits, false, false>);
}

template <bool kWrite>
cudaError_t launch(const KvCacheArgs& a, cudaStream_t stream) {
    if (a.tokens == 0) return cudaSuccess;
    const bool vec = aligned16(a.k, a.k_token, a.k_head) && aligned16(a.v, a.v_token, a.v_head);
    const bool bf16 = a.type == kTypeBf16;
    Kernel k = nullptr;
    if (a.head_dim == 64)
        k = a.bits == 8 ? pick<kWrite, 64, 8>(bf16, vec) : pick<kWrite, 64, 4>(bf16, vec);
    else if (a.head_dim == 128)
        k = a.bits == 8 ? pick<kWrite, 128, 8>(bf16, vec) : pick<kWrite, 128, 4>(bf16, vec);
    else
        k = a.bits == 8 ? pick<kWrite, 256, 8>(bf16, vec) : pick<kWrite, 256, 4>(bf16, vec);
    const int64_t threads = a.tokens * a.kv_heads * (a.head_dim / 16);
    return launch_pdl(k, dim3((unsigned)((threads + kThreads - 1) / kThreads)), dim3(kThreads), 0,
                      stream, a, FastDiv((uint32_t)a.kv_heads), FastDiv((uint32_t)a.page_size));
}

}  // namespace

cudaError_t launch_kv_write(const KvCacheArgs& a, cudaStream_t s) { return launch<true>(a, s); }
cudaError_t launch_kv_read(const KvCacheArgs& a, cudaStream_t s) { return launch<false>(a, s); }

cudaError_t read_kv_status(int clear, int* status) {
    return read_status_symbol(g_kv_status, clear, status);
}

}  // namespace clb
