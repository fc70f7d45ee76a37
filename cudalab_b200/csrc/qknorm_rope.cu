// RMSNorm of every head of q and k and the rotation by position, in one pass.
//
//   y = x * rsqrt(mean(x^2) + eps) * w      (w given; without it y = x)
//   pairs (a, b) = (y_i, y_{i + R/2}) or (y_2i, y_{2i+1}), i < R/2:
//   a' = a c_i - b s_i,  b' = b c_i + a s_i;  the other head_dim - R elements pass.
//
// fp32 throughout, one rounding at the end.  Bound by memory: every element is
// read and written once.  A lane holds two 8-element pieces (16-byte loads) of
// a head; with pairs of halves they are the two pieces that rotate against
// each other, so the rotation needs no exchange between lanes and the mean
// three shuffles at head_dim 128.  The lanes of a head take kHeads heads of
// one token, so the token's cosines and sines are loaded once for them.
#include <cuda_runtime.h>

#include <cstdint>

#include "gemv_common.cuh"
#include "kv_device.cuh"
#include "kv_layout.cuh"

namespace clb {
namespace {

__device__ int g_rope_status;

constexpr int kThreads = 256;
constexpr int kHeads = 2;  // heads per lane group

__device__ __forceinline__ void rotate(float& p, float& q, float c, float s) {
    const float y = p * c - q * s;
    q = q * c + p * s;
    p = y;
}

template <int kLanes, bool kBf16, bool kVec>
__global__ void __launch_bounds__(kThreads) qknorm_rope_kernel(const QkRopeArgs a, int tasks) {
    pdl_allow_dependents();
    pdl_wait_prior_grids();
    const int64_t group = ((int64_t)blockIdx.x * kThreads + threadIdx.x) / kLanes;
    const int l = threadIdx.x % kLanes;
    const int64_t token = group / tasks;
    const int first = (int)(group % tasks) * kHeads;
    const int total = a.heads[0] + a.heads[1];
    const bool have = token < a.tokens && 16 * l < a.head_dim;
    // The two pieces of this lane: rotating lanes come first.
    const int turning = a.rotary / 16;
    const bool turn = l < turning;
    int d0, d1, i0;
    if (turn && !a.interleaved) {
        d0 = 8 * l;
        d1 = d0 + a.rotary / 2;
        i0 = d0;
    } else {
        d0 = 16 * l;
        d1 = d0 + 8;
        i0 = 8 * l;
    }
    uint4 raw[kHeads][2];
    int which[kHeads], head[kHeads];
#pragma unroll
    for (int n = 0; n < kHeads; ++n) {
        const int h = first + n;
        which[n] = h >= a.heads[0];
        head[n] = which[n] ? h - a.heads[0] : h;
        raw[n][0] = raw[n][1] = make_uint4(0, 0, 0, 0);
        if (have && h < total) {
            const int64_t at = token * a.x_token[which[n]] + head[n] * a.x_head[which[n]];
            raw[n][0] = load8<kBf16, kVec>(a.x[which[n]], at + d0);
            raw[n][1] = load8<kBf16, kVec>(a.x[which[n]], at + d1);
        }
    }
    float c[8], s[8];
    if (have && turn) {
        int64_t pos = a.positions64 ? static_cast<const int64_t*>(a.positions)[token]
                                    : static_cast<const int32_t*>(a.positions)[token];
        if (pos < 0 || pos >= a.table_rows) {
            atomicCAS(&g_rope_status, 0, kStatusKvIndex);
            pos = pos < 0 ? 0 : a.table_rows - 1;
        }
        const float4* t = reinterpret_cast<const float4*>(a.table + pos * a.rotary + i0);
        const float4* u = reinterpret_cast<const float4*>(a.table + pos * a.rotary + a.rotary / 2 + i0);
        const float4 c0 = t[0], c1 = t[1], s0 = u[0], s1 = u[1];
        c[0] = c0.x, c[1] = c0.y, c[2] = c0.z, c[3] = c0.w;
        c[4] = c1.x, c[5] = c1.y, c[6] = c1.z, c[7] = c1.w;
        s[0] = s0.x, s[1] = s0.y, s[2] = s0.z, s[3] = s0.w;
        s[4] = s1.x, s[5] = s1.y, s[6] = s1.z, s[7] = s1.w;
    }
#pragma unroll
    for (int n = 0; n < kHeads; ++n) {
        float x[16];
        unpack8<kBf16>(raw[n][0], x);
        unpack8<kBf16>(raw[n][1], x + 8);
        if (a.w[0] != nullptr) {
            float sum = 0.f;
#pragma unroll
            for (int i = 0; i < 16; ++i) sum = fmaf(x[i], x[i], sum);
#pragma unroll
            for (int o = kLanes / 2; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
            if (have) {
                const float r = rsqrtf(sum / (float)a.head_dim + a.eps);
                float w[16];
                unpack8<kBf16>(load8<kBf16, kVec>(a.w[which[n]], d0), w);
                unpack8<kBf16>(load8<kBf16, kVec>(a.w[which[n]], d1), w + 8);
#pragma unroll
                for (int i = 0; i < 16; ++i) x[i] = x[i] * r * w[i];
            }
        }
        if (!have || first + n >= total) continue;
        if (turn && a.interleaved) {
#pragma unroll
            for (int i = 0; i < 8; ++i) rotate(x[2 * i], x[2 * i + 1], c[i], s[i]);
        } else if (turn) {
#pragma unroll
            for (int i = 0; i < 8; ++i) rotate(x[i], x[i + 8], c[i], s[i]);
        }
        const int64_t at = token * a.y_token[which[n]] + head[n] * a.y_head[which[n]];
        store8<kVec>(a.y[which[n]], at + d0, pack8<kBf16>(x));
        store8<kVec>(a.y[which[n]], at + d1, pack8<kBf16>(x + 8));
    }
}

using Kernel = void (*)(QkRopeArgs, int);

template <int kLanes>
Kernel pick(bool bf16, bool vec) {
    return bf16 ? (vec ? qknorm_rope_kernel<kLanes, true, true>
                       : qknorm_rope_kernel<kLanes, true, false>)
                : (vec ? qknorm_rope_kernel<kLanes, false, true>
                       : qknorm_rope_kernel<kLanes, false, false>);
}

}  // namespace

cudaError_t launch_qknorm_rope(const QkRopeArgs& a, cudaStream_t stream) {
    if (a.tokens == 0) return cudaSuccess;
    bool vec = true;
    for (int i = 0; i < 2; ++i)
        vec = vec && aligned16(a.x[i], a.x_token[i], a.x_head[i]) &&
              aligned16(a.y[i], a.y_token[i], a.y_head[i]) &&
              (reinterpret_cast<uintptr_t>(a.w[i]) & 15u) == 0;
    const bool bf16 = a.type == kTypeBf16;
    const int lanes = a.head_dim <= 64 ? 4 : a.head_dim <= 128 ? 8 : 16;
    const Kernel k = lanes == 4 ? pick<4>(bf16, vec) : lanes == 8 ? pick<8>(bf16, vec)
                                                                  : pick<16>(bf16, vec);
    const int tasks = (a.heads[0] + a.heads[1] + kHeads - 1) / kHeads;
    const int64_t threads = a.tokens * tasks * lanes;
    return launch_pdl(k, dim3((unsigned)((threads + kThreads - 1) / kThreads)), dim3(kThreads), 0,
                      stream, a, tasks);
}

cudaError_t read_qknorm_rope_status(int clear, int* status) {
    return read_status_symbol(g_rope_status, clear, status);
}

}  // namespace clb
