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
// three shuffles at head_dim 128.  The lanes of a head walk over `per` heads of
// one token and of one of q and k, so cosines, sines and weights are loaded
// once for them and multiplied into the four factors of each pair.  A lane's
// pieces of the next kDepth heads are on their way to its own places in shared
// memory (16-byte asynchronous copies) while it computes: what a lane waits for
// is held by no register.  8192 tokens of 64 + 8 heads of 128 (bf16): 49 us,
// 6.25 TB/s, 0.96 of a copy (61 us with weights and rotation applied one after
// the other under 64 registers, 80 us with loads into registers).
#include <cuda_runtime.h>

#include <cstdint>

#include "gemv_common.cuh"
#include "kv_device.cuh"
#include "kv_layout.cuh"

namespace clb {
namespace {

__device__ int g_rope_status;

constexpr int kThreads = 256;
constexpr int kDepth = 4;

struct Tasks {
    int per;         // heads of a task
    int q_tasks;     // tasks of a token's q; the rest are of its k
    FastDiv tasks;   // of a token
};

// kPartial: the rotation ends before the head does (lanes without a partner).
template <int kLanes, bool kBf16, bool kVec, bool kInterleaved, bool kPartial>
__global__ void __launch_bounds__(kThreads, 3) qknorm_rope_kernel(const QkRopeArgs a,
                                                                  const Tasks tasks) {
    pdl_allow_dependents();
    pdl_wait_prior_grids();
    const int task = (int)(blockIdx.x * (kThreads / kLanes) + threadIdx.x / kLanes);
    const int l = threadIdx.x % kLanes;
    const int64_t token = tasks.tasks.div(task);
    const int in_token = tasks.tasks.mod(task);
    const int which = in_token >= tasks.q_tasks;
    const int first = (which ? in_token - tasks.q_tasks : in_token) * tasks.per;
    const bool have = token < a.tokens && 16 * l < a.head_dim;
    const int count = have ? min(tasks.per, a.heads[which] - first) : 0;
    // The two pieces of this lane: rotating lanes come first.
    const bool turn = l < a.rotary / 16;
    int d0 = 16 * l, d1 = d0 + 8, i0 = 8 * l;
    if (!kInterleaved && turn) {
        d0 = i0;
        d1 = d0 + a.rotary / 2;
    }
    const uint16_t* x0 = static_cast<const uint16_t*>(a.x[which]) + token * a.x_token[which] +
                         first * a.x_head[which];
    uint16_t* y0 = static_cast<uint16_t*>(a.y[which]) + token * a.y_token[which] +
                   first * a.y_head[which];
    __shared__ uint4 ring[kVec ? kDepth : 1][2][kVec ? kThreads : 1];
    const int tid = threadIdx.x;
    if (kVec) {
#pragma unroll
        for (int n = 0; n < kDepth - 1; ++n) {
            copy16(&ring[n][0][tid], x0 + n * a.x_head[which] + d0, n < count);
            copy16(&ring[n][1][tid], x0 + n * a.x_head[which] + d1, n < count);
            copies_end_group();
        }
    }
    // What a pair (p, q) of the lane turns into, the weights and the rotation in
    // one: p' = pp p + pq q, q' = qp p + qq q (times the row's 1 / rms).  Lanes
    // past `rotary` only scale.
    float pp[8], pq[8], qp[8], qq[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) pp[i] = qq[i] = 1.f, pq[i] = qp[i] = 0.f;
    if (have) {
        float c[8], s[8], w[16];
#pragma unroll
        for (int i = 0; i < 8; ++i) c[i] = 1.f, s[i] = 0.f;
#pragma unroll
        for (int i = 0; i < 16; ++i) w[i] = 1.f;
        if (turn) {
            int64_t pos = a.positions64 ? static_cast<const int64_t*>(a.positions)[token]
                                        : static_cast<const int32_t*>(a.positions)[token];
            if (pos < 0 || pos >= a.table_rows) {
                atomicCAS(&g_rope_status, 0, kStatusKvIndex);
                pos = pos < 0 ? 0 : a.table_rows - 1;
            }
            const float4* t = reinterpret_cast<const float4*>(a.table + pos * a.rotary + i0);
            const float4* u = t + a.rotary / 8;
            const float4 c0 = t[0], c1 = t[1], s0 = u[0], s1 = u[1];
            c[0] = c0.x, c[1] = c0.y, c[2] = c0.z, c[3] = c0.w;
            c[4] = c1.x, c[5] = c1.y, c[6] = c1.z, c[7] = c1.w;
            s[0] = s0.x, s[1] = s0.y, s[2] = s0.z, s[3] = s0.w;
            s[4] = s1.x, s[5] = s1.y, s[6] = s1.z, s[7] = s1.w;
        }
        if (a.w[0] != nullptr) {
            unpack8<kBf16>(load8<kBf16, kVec>(a.w[which], d0), w);
            unpack8<kBf16>(load8<kBf16, kVec>(a.w[which], d1), w + 8);
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float wp = kInterleaved ? w[2 * i] : w[i], wq = kInterleaved ? w[2 * i + 1] : w[i + 8];
            pp[i] = wp * c[i], pq[i] = -wq * s[i], qp[i] = wp * s[i], qq[i] = wq * c[i];
        }
    }
    const float inv_dim = 1.f / (float)a.head_dim;
#pragma unroll 1
    for (int n = 0; n < tasks.per; ++n) {  // the same count for all lanes of a warp
        float x[16];
        if (kVec) {
            const int ahead = n + kDepth - 1;
            copy16(&ring[ahead % kDepth][0][tid], x0 + ahead * a.x_head[which] + d0, ahead < count);
            copy16(&ring[ahead % kDepth][1][tid], x0 + ahead * a.x_head[which] + d1, ahead < count);
            copies_end_group();
            copies_wait<kDepth - 1>();
        }
        uint4 raw[2] = {};
        if (n < count) {
            raw[0] = kVec ? ring[n % kDepth][0][tid] : load8<kBf16, false>(x0 + n * a.x_head[which], d0);
            raw[1] = kVec ? ring[n % kDepth][1][tid] : load8<kBf16, false>(x0 + n * a.x_head[which], d1);
        }
        unpack8<kBf16>(raw[0], x);
        unpack8<kBf16>(raw[1], x + 8);
        float r = 1.f;
        if (a.w[0] != nullptr) {
            float sum = 0.f;
#pragma unroll
            for (int i = 0; i < 16; ++i) sum = fmaf(x[i], x[i], sum);
#pragma unroll
            for (int o = kLanes / 2; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
            r = rsqrtf(fmaf(sum, inv_dim, a.eps));
        }
        if (n >= count) continue;
        if (!kPartial || turn) {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                float& p = kInterleaved ? x[2 * i] : x[i];
                float& q = kInterleaved ? x[2 * i + 1] : x[i + 8];
                const float y = fmaf(pp[i], p, pq[i] * q) * r;
                q = fmaf(qq[i], q, qp[i] * p) * r;
                p = y;
            }
        } else {  // no partner: an infinity stays its own
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                x[kInterleaved ? 2 * i : i] *= pp[i] * r;
                x[kInterleaved ? 2 * i + 1 : i + 8] *= qq[i] * r;
            }
        }
        store8<kVec>(y0 + n * a.y_head[which], d0, pack8<kBf16>(x));
        store8<kVec>(y0 + n * a.y_head[which], d1, pack8<kBf16>(x + 8));
    }
}

using Kernel = void (*)(QkRopeArgs, Tasks);

template <int kLanes, bool kInterleaved, bool kPartial>
Kernel pick(bool bf16, bool vec) {
    return bf16 ? (vec ? qknorm_rope_kernel<kLanes, true, true, kInterleaved, kPartial>
                       : qknorm_rope_kernel<kLanes, true, false, kInterleaved, kPartial>)
                : (vec ? qknorm_rope_kernel<kLanes, false, true, kInterleaved, kPartial>
                       : qknorm_rope_kernel<kLanes, false, false, kInterleaved, kPartial>);
}

template <bool kInterleaved, bool kPartial>
Kernel pick_lanes(int lanes, bool bf16, bool vec) {
    return lanes == 4 ? pick<4, kInterleaved, kPartial>(bf16, vec)
                      : lanes == 8 ? pick<8, kInterleaved, kPartial>(bf16, vec)
                                   : pick<16, kInterleaved, kPartial>(bf16, vec);
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
    const bool partial = a.rotary < a.head_dim;
    const Kernel k =
        a.interleaved ? (partial ? pick_lanes<true, true>(lanes, bf16, vec)
                                 : pick_lanes<true, false>(lanes, bf16, vec))
                      : (partial ? pick_lanes<false, true>(lanes, bf16, vec)
                                 : pick_lanes<false, false>(lanes, bf16, vec));
    // Heads per task: as many as leave every SM its 32 warps, at most 8.
    const int64_t rows = a.tokens * (a.heads[0] + a.heads[1]);
    Tasks t;
    t.per = 1;
    while (t.per < 8 && rows * lanes / (2 * t.per) >= (int64_t)148 * 32 * 32) t.per *= 2;
    t.q_tasks = (a.heads[0] + t.per - 1) / t.per;
    const int tasks = t.q_tasks + (a.heads[1] + t.per - 1) / t.per;
    t.tasks = FastDiv((uint32_t)tasks);
    const int64_t threads = a.tokens * tasks * lanes;
    return launch_pdl(k, dim3((unsigned)((threads + kThreads - 1) / kThreads)), dim3(kThreads), 0,
                      stream, a, t);
}

cudaError_t read_qknorm_rope_status(int clear, int* status) {
    return read_status_symbol(g_rope_status, clear, status);
}

}  // namespace clb
