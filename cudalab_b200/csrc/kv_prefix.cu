// Attention of many query rows over one run of cached tokens that all of them
// see: the prefix that a batch shares (layout of the cache: kv_layout.cuh).
//
//   s_j = scale * ks_j * (q . k_j),  o = sum_j e^(s_j) vs_j v_j / sum_j e^(s_j)
//
// With a batch's worth of rows per cache head the operation is bound by
// arithmetic, 4 rows tokens head_dim operations per head against tokens
// (2 head_dim bits / 8 + 4) bytes, so it runs on the 5th-generation tensor
// cores.  A CTA takes 128 rows (lanes of Tensor Memory) and a range of tokens,
// 128 at a time:
//   * 8 warps expand the tile's 8 cache blocks, one block a warp, to exact fp16
//     whole values in shared memory (rows of tokens, 64 elements wide, 128-byte
//     swizzle), read a tile ahead into registers; the scales become two
//     numbers per token in fp32;
//   * one thread issues the MMAs (M = N = 128, K = 16, fp32 accumulators): S =
//     Q K^T with Q in Tensor Memory and K as stored (K-major), O += P V with P in
//     Tensor Memory and the same layout of V read across (MN-major);
//   * 8 warps, half a row's tokens a thread, do the softmax as in
//     kv_attention.cu: p_j = 2^(s_j - m) summed in fp32, weights p_j vs_j in
//     fp16 (what the MMA takes beside V), one lazy reference m per row near the
//     maximum of s_j + log2 vs_j,
//     O is only rescaled when a weight exceeds kMostWeight,
//     which the two warps of a row find out with one barrier a tile.
// S is double-buffered: the tensor cores compute tile i + 1's S and tile i -
// 1's O while the softmax of tile i runs.
//
// Tensor Memory (512 columns): S 2 x 128, O head_dim, P 64, Q head_dim / 2.
// int4: a byte's nibbles leave their word as pairs (0, 4) (1, 5) (2, 6) (3, 7),
// so K, Q and V all keep that order of the 8 elements of a 16-byte piece; the
// sum over them does not mind, and O's columns are put back when it is written.
//
// The tokens are cut so that heads x row tiles x parts fill the SMs; each part
// writes a normalised fp32 result and its lse, joined by the launch over the
// sequences' own tokens.  Every wait is bounded (status 8 on expiry).
//
// Measured (8 heads of 128, int8): 16384 tokens for 512 rows a head with the
// launch over 64 sequences' own tokens 90 us, 0.39 PFLOP/s; a tile takes a CTA
// 1.6 us, of which its MMAs need 0.74 at the measured peak.  The rest is
// instructions: 7700 of a warp per tile (softmax and expansion about halves),
// 0.55 a cycle and scheduler.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cstdint>

#include "gemv_common.cuh"
#include "gemv_launch.h"
#include "kv_device.cuh"
#include "kv_layout.cuh"

namespace clb {
namespace {

__device__ int g_kv_prefix_status;

constexpr int kRows = 128, kTile = 128;  // query rows and tokens of a tile
constexpr int kSoftWarps = 8, kFillWarps = 8;
constexpr int kMmaWarp = kSoftWarps + kFillWarps;
constexpr int kThreads = 32 * (kMmaWarp + 1);
// Weights are fp16: the row's largest is 2^7 when its reference is taken, so that
// a tail of far smaller ones keeps its bits, and stays below fp16's 65504.
constexpr float kLift = 7.f, kMostWeight = 32768.f;
constexpr uint32_t kColS = 0, kColO = 256, kColP = 384, kColQ = 448, kColumns = 512;

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float lg2(float x) {
    float y;
    asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ void fence_before() {
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
}
__device__ __forceinline__ void fence_after() {
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
}
__device__ __forceinline__ void wait_st() {
    asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void commit(uint32_t bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(
                     bar)
                 : "memory");
}

// D[tmem] (+)= A[tmem] x B[smem].
__device__ __forceinline__ void mma(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc,
                                    uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %3, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %4, {%5, %5, %5, %5}, p;\n\t}"
        ::"r"(d), "r"(a), "l"(b), "r"(accumulate), "r"(idesc), "r"(0u)
        : "memory");
}

// Instruction descriptor of kind::f16: D fp32 (bits 4-5 = 1), A and B fp16, A
// K-major, B K-major or MN-major (bit 16), N >> 3 at bit 17, M >> 4 at bit 24.
__host__ __device__ constexpr uint32_t instruction(int n, bool b_mn_major) {
    return (1u << 4) | ((uint32_t)b_mn_major << 16) | ((uint32_t)(n >> 3) << 17) |
           ((uint32_t)(kRows >> 4) << 24);
}
// Shared-memory descriptor of a 128-byte swizzled operand: 8-row groups of 1024
// bytes (stride 1024 at bit 32), the next 64 columns `wide` bytes on (bit 16;
// MN-major only), version 1 (bit 46), 128-byte swizzle (2 at bit 61).
__device__ __forceinline__ uint64_t operand(uint32_t addr, uint32_t wide) {
    return (uint64_t)((addr >> 4) & 0x3FFFu) | ((uint64_t)((wide >> 4) & 0x3FFFu) << 16) |
           ((uint64_t)(1024 >> 4) << 32) | (1ull << 46) | (2ull << 61);
}

// 16 bytes of the cache, asked for here and not where they are used (a plain
// load may be moved down to its use, which costs the whole latency).
__device__ __forceinline__ uint4 load_now(const uint8_t* p) {
    uint4 v;
    asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
                 : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
    return v;
}

// 32 columns of this thread's lane: issue, and the wait that makes them valid.
__device__ __forceinline__ void ld32(uint32_t addr, uint32_t (&r)[32]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, "
        "%12, %13, %14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, "
        "%30, %31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]),
          "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]),
          "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]),
          "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]),
          "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(addr)
        : "memory");
}
__device__ __forceinline__ void ld_wait(uint32_t (&r)[32]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]),
                   "+r"(r[6]), "+r"(r[7]), "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]),
                   "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]), "+r"(r[16]), "+r"(r[17]),
                   "+r"(r[18]), "+r"(r[19]), "+r"(r[20]), "+r"(r[21]), "+r"(r[22]), "+r"(r[23]),
                   "+r"(r[24]), "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]), "+r"(r[29]),
                   "+r"(r[30]), "+r"(r[31])
                 :
                 : "memory");
}
__device__ __forceinline__ void ld16(uint32_t addr, uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, "
        "%12, %13, %14, %15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]),
          "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]),
          "=r"(r[14]), "=r"(r[15])
        : "r"(addr)
        : "memory");
}
__device__ __forceinline__ void ld_wait(uint32_t (&r)[16]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]),
                   "+r"(r[6]), "+r"(r[7]), "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]),
                   "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15])
                 :
                 : "memory");
}
__device__ __forceinline__ void st32(uint32_t addr, const uint32_t (&r)[32]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, "
        "%12, %13, %14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, "
        "%30, %31, %32};" ::"r"(addr),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
        "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]),
        "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]),
        "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]),
        "r"(r[29]), "r"(r[30]), "r"(r[31])
        : "memory");
}
__device__ __forceinline__ void st16(uint32_t addr, const uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, "
        "%12, %13, %14, %15, %16};" ::"r"(addr),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
        "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]),
        "r"(r[15])
        : "memory");
}

// Barrier of the 64 threads that share 32 rows, and whether any of them says so.
__device__ __forceinline__ bool any_of_rows(int id, bool say) {
    uint32_t r;
    asm volatile(
        "{\n\t.reg .pred p, q;\n\t"
        "setp.ne.u32 p, %1, 0;\n\t"
        "barrier.cta.red.or.pred q, %2, 64, p;\n\t"
        "selp.u32 %0, 1, 0, q;\n\t}"
        : "=r"(r) : "r"((uint32_t)say), "r"(id) : "memory");
    return r != 0;
}

struct PrefixParams {
    KvAttentionArgs a;
    FastDiv group, page_blocks;
    int rows;        // per cache head
    int row_tiles, parts, part_tiles, tiles;
    int q_vec;
    long long wait_cycles;
    uint32_t hold_ns;
};

template <int kDim, int kBits>
struct PrefixShape {
    static constexpr int kRow = kDim * kBits / 8;
    static constexpr int kBlockBytes = kv_block_bytes(kRow);
    static constexpr int kHalfBytes = kTile * 128;        // 64 elements wide
    static constexpr int kOperandBytes = kDim / 64 * kHalfBytes;
    static constexpr int kLoads = kRow / 32;              // 16-byte pieces per lane of a part
    static constexpr int kOutStride = kDim * 4 + 16;      // bytes of a staged output row
    // K and V twice each (the output is staged there at the end), per-token
    // numbers, barriers; at least 120 KB, so that one CTA has an SM and its
    // Tensor Memory.
    static constexpr int kNumbers = 4 * kOperandBytes;
    static constexpr int kTops = kNumbers + 4 * 2 * kTile * 4;  // [2][kRows] exchanged by row halves
    static constexpr int kBars = kTops + 2 * kRows * 4;
    static constexpr int kGone = kBars + 136;  // [4][kFillWarps] bytes: the block is missing
    static constexpr int kEnd = kGone + 4 * kFillWarps;
    static constexpr int kSmem = (kEnd < 120 * 1024 ? 120 * 1024 : kEnd) + 1024;
    static_assert(kRows * kOutStride <= 4 * kOperandBytes, "room for the output");
};

// The 16-byte pieces of a block's part that a lane expands: load n is of token
// row 8 (n / halves) + lane / 4 (int8) or lane / 2 (int4), and lanes that store
// together (8) fall on different banks.  Both swizzles are exclusive ors of
// address bits that the loads do not carry into, so a place is one number per
// lane, exclusive or a constant, plus a constant:
template <int kDim, int kBits>
struct Pieces {
    static constexpr int kRow = kDim * kBits / 8, kHalves = kDim / 64;
    int from, to;  // place of piece 0 in the cache's part and in the operand
    __device__ explicit Pieces(int lane) {
        const int row = kBits == 8 ? lane >> 2 : lane >> 1, piece = kBits == 8 ? lane & 3 : lane & 1;
        from = kv_offset<kRow>(row, 16 * piece);
        to = row * 128 + (((kBits == 8 ? 2 : 4) * piece) ^ (row & 7)) * 16;
    }
    // load n: 64 elements on (another half of the operand), or 8 rows on (int8)
    __device__ static constexpr int column(int n) { return n % kHalves; }
    __device__ static constexpr int rows(int n) { return n / kHalves * 8; }
    __device__ int source(int n) const {  // `from` of a half: kRow / kHalves bytes on
        return (from ^ (column(n) * (kRow / kHalves))) + rows(n) * kRow;
    }
    __device__ int target(int n, int s) const {
        return (to ^ (16 * s)) + column(n) * (kTile * 128) + rows(n) * 128;
    }
};

// One 16-byte piece of whole values -> output piece s of 2 (int8) or 4 (int4).
template <int kBits>
__device__ __forceinline__ uint4 expand(const uint4& raw, int s) {
    const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
    __half2 q[4];
    if (kBits == 8) {
        __half2 lo[2], hi[2];
        int8x4_to_h2(w[2 * s], lo);
        int8x4_to_h2(w[2 * s + 1], hi);
        q[0] = lo[0], q[1] = lo[1], q[2] = hi[0], q[3] = hi[1];
    } else {
        const uint32_t up = w[s] >> 8;
        q[0] = __hadd2(u32_as_h2(lop3_sel_xor_i<0x000F000Fu, 0x64086408u>(w[s])), h2_const(kH_m1032));
        q[1] = __hadd2(u32_as_h2(lop3_sel_xor_i<0x00F000F0u, 0x54805480u>(w[s])), h2_const(kH_m72));
        q[2] = __hadd2(u32_as_h2(lop3_sel_xor_i<0x000F000Fu, 0x64086408u>(up)), h2_const(kH_m1032));
        q[3] = __hadd2(u32_as_h2(lop3_sel_xor_i<0x00F000F0u, 0x54805480u>(up)), h2_const(kH_m72));
    }
    return *reinterpret_cast<const uint4*>(q);
}

template <int kDim, int kBits, bool kBf16>
__global__ void __launch_bounds__(kThreads, 1) kv_prefix_kernel(const PrefixParams p) {
    using S = PrefixShape<kDim, kBits>;
    extern __shared__ uint8_t smem_raw[];
    // aligned for the swizzle by an offset, so that the compiler still knows the
    // accesses for shared memory
    uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
    uint8_t* kbuf = smem;                          // [2] K operands
    uint8_t* vbuf = smem + 2 * S::kOperandBytes;   // [2] V operands
    float* numbers = reinterpret_cast<float*>(smem + S::kNumbers);  // [4][2][kTile]
    float* tops = reinterpret_cast<float*>(smem + S::kTops);
    const uint32_t bars = smem_u32(smem + S::kBars);
    const uint32_t kfull = bars, vfull = bars + 16, kempty = bars + 32, vempty = bars + 48,
                   sfull = bars + 64, pfull = bars + 80, nfull = bars + 88, drained = bars + 128;
    uint8_t* gone = smem + S::kGone;
    volatile uint32_t* s_tmem = reinterpret_cast<volatile uint32_t*>(smem + S::kBars + 120);
    volatile int* s_fail = reinterpret_cast<volatile int*>(smem + S::kBars + 124);

    const KvAttentionArgs& a = p.a;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int part = (int)blockIdx.x % p.parts, rest = (int)blockIdx.x / p.parts;
    const int head = rest % a.kv_heads, row0 = rest / a.kv_heads * kRows;
    const int tile0 = part * p.part_tiles;
    const int tiles = min(p.part_tiles, p.tiles - tile0);
    const int length = a.fixed_length;

    if (tid == 0) {
        for (int i = 0; i < 2; ++i) {
            mbar_init(kfull + 8 * i, kFillWarps);
            mbar_init(vfull + 8 * i, kFillWarps);
            mbar_init(kempty + 8 * i, 1);
            mbar_init(vempty + 8 * i, 1);
            mbar_init(sfull + 8 * i, 1);
        }
        for (int i = 0; i < 4; ++i) mbar_init(nfull + 8 * i, kFillWarps);
        mbar_init(pfull, kSoftWarps);
        mbar_init(drained, 1);
        *s_fail = 0;
        fence_barrier_init();
    }
    // The launch over the sequences' own tokens may begin once every CTA here has
    // seen the preceding kernel complete: it then waits for this grid only
    // before it joins the results (KvAttentionArgs::front_by_tensor_cores).
    pdl_wait_prior_grids();
    pdl_allow_dependents();
    if (warp == 0) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                         smem_u32(const_cast<uint32_t*>(s_tmem))),
                     "r"(kColumns)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    fence_before();
    __syncthreads();
    fence_after();
    const uint32_t tmem = *s_tmem;

    // A bounded wait; false once it or any other of the CTA has run out.
    auto wait = [&](uint32_t bar, int phase) -> bool {
        if (mbar_try_wait_held(bar, (uint32_t)phase & 1u, p.hold_ns)) return true;
        const long long t0 = clock64();
        while (!mbar_try_wait_held(bar, (uint32_t)phase & 1u, p.hold_ns)) {
            if (*s_fail) return false;
            if (clock64() - t0 > p.wait_cycles) {
                atomicCAS(&g_kv_prefix_status, 0, kStatusTimeoutKv);
                *s_fail = 1;
                return false;
            }
        }
        return true;
    };

    float sum_l = 0.f;  // of this thread's row (and half of the tokens)
    // The row's reference, kLift below its largest s_j + log2 vs_j; -inf until it has
    // seen a token with a score (a page can be missing, a row NaN), and what stands
    // for it in the arithmetic.
    float known = -INFINITY, ref = 0.f;
    bool finished = false;               // softmax warps: all tiles done
    const int quarter = warp & 3, half = warp >> 2 & 1;  // of the softmax warps
    const uint32_t lane_base = tmem + ((uint32_t)(32 * quarter) << 16);

    if (warp < kSoftWarps) {
        // ---------------- softmax: half a row's tokens a thread ----------------
        const int in_tile = 32 * quarter + lane, r = row0 + in_tile;
        float unit = 1.f;  // what the row was divided by (a power of two)
        {
            // this half of the row, all of it on its way at once
            const int i0 = p.group.div(r);
            const uint16_t* src = static_cast<const uint16_t*>(a.q) + i0 * a.q_new +
                                  ((head - i0) * a.group + r) * a.q_head + half * (kDim / 2);
            uint4 raw[kDim / 16];
#pragma unroll
            for (int c = 0; c < kDim / 16; ++c) {
                raw[c] = make_uint4(0, 0, 0, 0);
                if (r < p.rows)
                    raw[c] = p.q_vec ? load8<kBf16, true>(src, 8 * c) : load8<kBf16, false>(src, 8 * c);
            }
            // A bf16 row that fp16 does not hold exactly is brought to [2^15, 2^16), where
            // it does down to 2^-32 of the row's largest.  (Few are: rows in fp16's range
            // without elements below 2^-17 need no multiplication of their scores.)
            float factor = 1.f;
            if (kBf16) {
                float top = 0.f;
                bool exact = true;
#pragma unroll
                for (int c = 0; c < kDim / 16; ++c) {
                    float x[8];
                    unpack8<kBf16>(raw[c], x);
#pragma unroll
                    for (int i = 0; i < 8; i += 2) {
                        top = fmaxf(top, fmaxf(fabsf(x[i]), fabsf(x[i + 1])));
                        const float2 h = __half22float2(__floats2half2_rn(x[i], x[i + 1]));
                        exact &= h.x == x[i] && h.y == x[i + 1];
                    }
                }
                tops[half * kRows + in_tile] = top;
                exact = !any_of_rows(1 + quarter, !exact);
                top = fmaxf(top, tops[(half ^ 1) * kRows + in_tile]);
                any_of_rows(1 + quarter, false);  // read before it is written again
                const int e = (int)(__float_as_uint(top) >> 23) - 127;
                if (!exact && e < 128) {  // rows with an infinity stay as they are
                    const int up = min(15 - e, 126);
                    factor = __uint_as_float((uint32_t)(127 + up) << 23);
                    unit = __uint_as_float((uint32_t)(127 - up) << 23);
                }
            }
#pragma unroll
            for (int d = 0; d < kDim / 2; d += 32) {
                uint32_t packed[16];
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    float x[8];
                    unpack8<kBf16>(raw[d / 8 + c], x);
#pragma unroll
                    for (int i = 0; i < 8; ++i) x[i] *= factor;
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        packed[4 * c + i] = kBits == 8 ? pack2<false>(x[2 * i], x[2 * i + 1])
                                                       : pack2<false>(x[i], x[i + 4]);
                }
                st16(lane_base + kColQ + (half * (kDim / 2) + d) / 2, packed);
            }
            wait_st();
            fence_before();
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(pfull);  // phase 0: Q is there

        const bool scaled = __any_sync(0xffffffffu, unit != 1.f);
        float l2[2] = {0.f, 0.f};
        bool ok = true;
        for (int i = 0; i < tiles && ok; ++i) {
            const int b = i & 1;
            bool good = __all_sync(0xffffffffu, wait(nfull + 8 * (i & 3), i >> 2) &&
                                                    wait(sfull + 8 * b, i >> 1));
            fence_after();
            const uint32_t s_at = lane_base + kColS + 128 * b + 64 * half;
            const float* num = numbers + (i & 3) * 2 * kTile + 64 * half;
            // columns of this half that hold tokens, and a byte for each of its 16-column
            // blocks: not 0 if its page is not there
            const int live = length - (tile0 + i) * kTile - 64 * half;
            const uint32_t missing =
                *reinterpret_cast<const uint32_t*>(gone + (i & 3) * kFillWarps + 4 * half);
            // 16 columns of S have come; columns past the end, or of no page, at -inf
            auto take_s = [&](int c, uint32_t (&s)[16]) {
                ld_wait(s);
                if (kBf16 && scaled) {
#pragma unroll
                    for (int j = 0; j < 16; ++j) s[j] = __float_as_uint(__uint_as_float(s[j]) * unit);
                }
                if (live < 16 * c + 16 || missing != 0) {
                    const int from = (missing >> (8 * c) & 0xffu) != 0 ? 0 : live - 16 * c;
#pragma unroll
                    for (int j = 0; j < 16; ++j)
                        if (j >= from) s[j] = 0xff800000u;
                }
            };
            // base-2 logit of a column, less the reference
            auto logit = [&](uint32_t s, float ks, float nref) {
                return fmaf(__uint_as_float(s), ks, nref);
            };
            bool waited = i == 0;  // for the MMAs of tile i - 1, which read P and write O
            auto previous_done = [&]() {
                if (!waited) {
                    good = __all_sync(0xffffffffu, wait(vempty + 8 * ((i - 1) & 1), (i - 1) >> 1));
                    fence_after();
                }
                waited = true;
                return good;
            };
            // Until the weights fit the reference: usually once.  The first tile
            // with a score has none yet.  What the two warps of a row do next is decided by
            // their barrier alone, so neither can wait for the other in vain.
            bool fresh = __any_sync(0xffffffffu, known == -INFINITY);
            for (int tries = 0;; ++tries, fresh = false) {
                float try_l[2] = {l2[0], l2[1]};
                __half2 most = __half2half2(__half(0.f));
                if (good && !fresh) {
                    uint32_t s[2][16], packed[16];
                    ld16(s_at, s[0]);
#pragma unroll
                    for (int c = 0; c < 4; ++c) {
                        take_s(c, s[c & 1]);
                        if (c < 3) ld16(s_at + 16 * (c + 1), s[(c + 1) & 1]);  // under the arithmetic
#pragma unroll
                        for (int j = 0; j < 16; j += 4) {
                            const uint32_t* t = s[c & 1] + j;
                            const float4 ks = *reinterpret_cast<const float4*>(num + 16 * c + j);
                            const float4 vs = *reinterpret_cast<const float4*>(num + kTile + 16 * c + j);
                            const float x = ex2(logit(t[0], ks.x, -ref)), y = ex2(logit(t[1], ks.y, -ref));
                            const float z = ex2(logit(t[2], ks.z, -ref)), w = ex2(logit(t[3], ks.w, -ref));
                            try_l[0] += x, try_l[1] += y, try_l[0] += z, try_l[1] += w;
                            uint32_t* to = packed + 8 * (c & 1) + j / 2;
                            to[0] = pack2<false>(x * vs.x, y * vs.y);
                            to[1] = pack2<false>(z * vs.z, w * vs.w);
                            most = __hmax2(most, __hmax2(u32_as_h2(to[0]), u32_as_h2(to[1])));
                        }
                        if (c & 1) {
                            if (c == 1 && !previous_done()) break;
                            st16(lane_base + kColP + 32 * half + 8 * (c - 1), packed);
                        }
                    }
                }
                const float2 m2 = __half22float2(most);
                // (a second reference always fits; the bound is for the loop's sake)
                const bool over = fresh || (tries < 3 && fmaxf(m2.x, m2.y) > kMostWeight);
                if (!any_of_rows(1 + quarter, over || !good)) {
                    l2[0] = try_l[0], l2[1] = try_l[1];
                    break;
                }
                if (any_of_rows(1 + quarter, !good)) {
                    ok = false;
                    break;
                }
                // The reference from the tile's own scores, under which what there
                // is of O is rescaled; then the tile again.
                float top = -INFINITY;
#pragma unroll 1
                for (int c = 0; c < 4; ++c) {
                    uint32_t s[16];
                    ld16(s_at + 16 * c, s);
                    take_s(c, s);
#pragma unroll
                    for (int j = 0; j < 16; j += 4) {
                        const float4 ks = *reinterpret_cast<const float4*>(num + 16 * c + j);
                        const float4 vs = *reinterpret_cast<const float4*>(num + kTile + 16 * c + j);
                        const float x = logit(s[j], ks.x, lg2(vs.x));
                        const float y = logit(s[j + 1], ks.y, lg2(vs.y));
                        const float z = logit(s[j + 2], ks.z, lg2(vs.z));
                        const float w = logit(s[j + 3], ks.w, lg2(vs.w));
                        top = fmaxf(fmaxf(fmaxf(top, x), y), fmaxf(z, w));
                    }
                }
                tops[half * kRows + in_tile] = top;
                wait_st();
                if (any_of_rows(1 + quarter, !previous_done())) {
                    ok = false;
                    break;
                }
                top = fmaxf(top, tops[(half ^ 1) * kRows + in_tile]);
                top = fmaxf(top - kLift, known);
                ref = top == -INFINITY ? 0.f : top;
                const float f = ex2(known - ref);  // 0 while nothing has been seen
                known = top;
                l2[0] *= f, l2[1] *= f;
                if (i > 0) {
#pragma unroll 1
                    for (int c = half * (kDim / 2); c < (half + 1) * (kDim / 2); c += 32) {
                        uint32_t o[32];
                        ld32(lane_base + kColO + c, o);
                        ld_wait(o);
#pragma unroll
                        for (int j = 0; j < 32; ++j) o[j] = __float_as_uint(__uint_as_float(o[j]) * f);
                        st32(lane_base + kColO + c, o);
                    }
                    wait_st();
                }
            }
            if (!ok) break;
            wait_st();
            fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(pfull);
        }
        if (ok && __all_sync(0xffffffffu, wait(vempty + 8 * ((tiles - 1) & 1), (tiles - 1) >> 1))) {
            fence_after();
            finished = true;
            sum_l = l2[0] + l2[1];
            tops[half * kRows + in_tile] = sum_l;
        }
        // nothing of this thread is in flight when the memory is freed
        asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
        wait_st();
    } else if (warp < kMmaWarp) {
        // ---------------- expansion: one cache block a warp ----------------
        const int w = warp - kSoftWarps;
        constexpr uint32_t kAbsent = 0xffffffffu, kInvalid = 0xfffffffeu;
        uint32_t where = kAbsent;  // lane i: the block of the 32-tile batch's i-th tile
        const Pieces<kDim, kBits> pieces(lane);
        uint4 raw[2][S::kLoads];       // a block's K and V on their way
        __half scale = __half(0.f);
        uint32_t at = kAbsent;
        auto find = [&](int i) {  // tile i's block
            if (i >= tiles) return;
            if ((i & 31) == 0) {
                const int blk = (tile0 + i + lane) * 8 + w;
                where = kAbsent;
                if (i + lane < tiles && blk * kKvBlock < length) {
                    const int index = p.page_blocks.div(blk);
                    const int page = __ldg(a.table + index);
                    if (page < 0 || page >= a.num_pages) {  // recorded, its tokens left out
                        atomicCAS(&g_kv_prefix_status, 0, kStatusKvIndex);
                        where = kInvalid;
                    } else {
                        where = ((uint32_t)page * a.kv_heads + head) * p.page_blocks.d +
                                (blk - index * p.page_blocks.d);
                    }
                }
            }
            at = __shfl_sync(0xffffffffu, where, i & 31);
        };
        auto fetch = [&](int x, int i) {  // its K (0, with the scales) or V (1)
            if (i >= tiles) return;
            if (at >= kInvalid) {
#pragma unroll
                for (int n = 0; n < S::kLoads; ++n) raw[x][n] = make_uint4(0, 0, 0, 0);
                if (x == 0) scale = __half(0.f);
                return;
            }
            const uint8_t* block = a.pages + (int64_t)at * S::kBlockBytes;
#pragma unroll
            for (int n = 0; n < S::kLoads; ++n)
                raw[x][n] = load_now(block + x * kKvBlock * S::kRow + pieces.source(n));
            if (x == 0) scale = reinterpret_cast<const __half*>(block + 2 * kKvBlock * S::kRow)[lane];
        };
        auto store = [&](int x, uint8_t* to) {
#pragma unroll
            for (int n = 0; n < S::kLoads; ++n)
#pragma unroll
                for (int o = 0; o < 16 / kBits; ++o)
                    *reinterpret_cast<uint4*>(to + kKvBlock * w * 128 + pieces.target(n, o)) =
                        expand<kBits>(raw[x][n], o);
        };
        auto arrive = [&](uint32_t bar) {
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            if (lane == 0) mbar_arrive(bar);
        };
        const float log2_scale = a.scale * 1.4426950408889634f;
        find(0);
        fetch(0, 0);
        fetch(1, 0);
        for (int i = 0; i < tiles; ++i) {
            const int b = i & 1;
            if (i >= 2 && !__all_sync(0xffffffffu, wait(kempty + 8 * b, (i - 2) >> 1))) break;
            // K's scale (lanes 0-15) and V's (16-31) of token lane & 15, 0 past
            // the end; that S(i - 2) is done says that softmax i - 4 is
            const bool seen = at < kInvalid &&
                              (tile0 + i) * kTile + kKvBlock * w + (lane & 15) < length;
            const float s = seen ? __half2float(scale) : 0.f;
            // A zero scale has all-zero values, so any other does as well: with fp16's
            // smallest, a weight shows when the token's score passes the reference.
            numbers[(i & 3) * 2 * kTile + (lane >> 4) * kTile + kKvBlock * w + (lane & 15)] =
                lane < 16 ? (seen ? s * log2_scale : 1.f) : (seen ? fmaxf(s, 0x1p-24f) : 0.f);
            if (lane == 0) gone[(i & 3) * kFillWarps + w] = at == kInvalid;
            store(0, kbuf + b * S::kOperandBytes);
            arrive(kfull + 8 * b);
            if (lane == 0) mbar_arrive(nfull + 8 * (i & 3));
            find(i + 1);
            fetch(0, i + 1);
            if (i >= 2 && !__all_sync(0xffffffffu, wait(vempty + 8 * b, (i - 2) >> 1))) break;
            store(1, vbuf + b * S::kOperandBytes);
            arrive(vfull + 8 * b);
            fetch(1, i + 1);
        }
    } else if (lane == 0) {
        // ---------------- MMAs ----------------
        constexpr uint32_t kIdescS = instruction(kTile, false), kIdescO = instruction(kDim, true);
        bool ok = wait(pfull, 0);  // Q
        for (int i = 0; i <= tiles && ok; ++i) {
            if (i < tiles) {
                const int b = i & 1;
                ok = wait(kfull + 8 * b, i >> 1);
                if (!ok) break;
                fence_after();
                const uint32_t kb = smem_u32(kbuf) + b * S::kOperandBytes;
#pragma unroll
                for (int k = 0; k < kDim / 16; ++k)
                    mma(tmem + kColS + 128 * b, tmem + kColQ + 8 * k,
                        operand(kb + (k >> 2) * S::kHalfBytes + (k & 3) * 32, 16), kIdescS, k > 0);
                commit(sfull + 8 * b);
                commit(kempty + 8 * b);
            }
            if (i > 0) {
                const int b = (i - 1) & 1;
                ok = wait(pfull, i) && wait(vfull + 8 * b, (i - 1) >> 1);
                if (!ok) break;
                fence_after();
                const uint32_t vb = smem_u32(vbuf) + b * S::kOperandBytes;
#pragma unroll
                for (int k = 0; k < kTile / 16; ++k)
                    mma(tmem + kColO, tmem + kColP + 8 * k, operand(vb + k * 2048, S::kHalfBytes),
                        kIdescO, i > 1 || k > 0);
                commit(vempty + 8 * b);
            }
        }
        if (!ok) {
            // every MMA issued so far (the last ones have made S for a tile that nobody
            // takes up) ends before the memory it uses is given up
            commit(drained);
            mbar_wait_held(drained, 0, kWaitTimeoutCycles);
        }
    }

    __syncthreads();
    fence_after();
    // ---------------- the output, through shared memory ----------------
    if (finished) {
        sum_l += tops[(half ^ 1) * kRows + 32 * quarter + lane];
        const float inv = sum_l > 0.f ? 1.f / sum_l : sum_l;  // 0: no token; NaN stays
        float* row = reinterpret_cast<float*>(smem + (32 * quarter + lane) * S::kOutStride);
#pragma unroll 1
        for (int c = half * (kDim / 2); c < (half + 1) * (kDim / 2); c += 32) {
            uint32_t o[32];
            ld32(lane_base + kColO + c, o);
            ld_wait(o);
#pragma unroll
            for (int j = 0; j < 32; j += 4) {
                // int4: columns (0..7) hold elements 0 4 1 5 2 6 3 7
                const int g8 = j & ~7, odd = (j >> 2) & 1;
                float v[4];
#pragma unroll
                for (int x = 0; x < 4; ++x)
                    v[x] = __uint_as_float(kBits == 8 ? o[j + x] : o[g8 + 2 * x + odd]) * inv;
                *reinterpret_cast<float4*>(row + c + j) = make_float4(v[0], v[1], v[2], v[3]);
            }
        }
        if (half == 0) row[kDim] = (ref + lg2(sum_l)) * 0.6931471805599453f;
    }
    fence_before();
    __syncthreads();
    if (warp == 0) {
        fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kColumns)
                     : "memory");
    }
    if (*s_fail) return;
    const int heads = a.kv_heads * a.group;
    const int64_t all = (int64_t)(p.rows / a.group) * heads;  // rows of one part's result
    const int valid = min(kRows, p.rows - row0);
    for (int i = tid; i < valid * (kDim / 4); i += kThreads) {
        const int rr = i / (kDim / 4), d = i % (kDim / 4) * 4;
        const int i0 = p.group.div(row0 + rr);
        const int64_t at = part * all + (int64_t)i0 * heads + (head - i0) * a.group + row0 + rr;
        const float* row = reinterpret_cast<const float*>(smem + rr * S::kOutStride);
        *reinterpret_cast<float4*>(a.out_f32 + at * kDim + d) = *reinterpret_cast<const float4*>(row + d);
        if (d == 0) a.lse[at] = row[kDim];
    }
}

template <int kDim, int kBits, bool kBf16>
cudaError_t run(const PrefixParams& p, cudaStream_t stream) {
    using S = PrefixShape<kDim, kBits>;
    const auto kernel = kv_prefix_kernel<kDim, kBits, kBf16>;
    cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, S::kSmem);
    if (e != cudaSuccess) return e;
    return launch_pdl(kernel, dim3((unsigned)(p.a.kv_heads * p.row_tiles * p.parts)), dim3(kThreads),
                      S::kSmem, stream, p);
}

// Parts of the tokens: the cut that needs the fewest tile times, with a CTA's
// set-up and output at about kSetUp tiles and one CTA per SM.
int cut(int items, int tiles) {
    constexpr int kSetUp = 5, kSms = 148, kMostParts = 16;
    int best = 1;
    int64_t cost = INT64_MAX;
    for (int parts = 1; parts <= std::min(kMostParts, tiles); ++parts) {
        const int per = (tiles + parts - 1) / parts, used = (tiles + per - 1) / per;
        const int waves = (items * used + kSms - 1) / kSms;
        const int64_t tile_times = (int64_t)waves * (per + kSetUp);
        if (tile_times < cost) cost = tile_times, best = used;
    }
    return best;
}

}  // namespace

bool kv_prefix_takes(const KvAttentionArgs& a) {
    // Both kernels with the launch that joins them, us, here / register-fed, at 16, 300,
    // 1024 and 8192 tokens:
    //                     8 rows a head                        9 rows
    //   8 x 128 int8   9.5/9.1 10.2/12.1 10.2/12.4 18.4/17.7   9.6/12.0 10.2/15.3
    //   2 x 64 int4    7.9/7.1  8.5/9.3   8.6/9.6  14.0/12.0   8.0/9.0   8.3/11.7
    //                     32 (16, 300: 24) rows                 256 rows
    //   8 x 128 int8  10.6/12.9 11.8/16.7 12.0/18.1 21.6/31.6  12.8/14.4 16.3/18.8 17.1/25.2 28.6/71.5
    //   1 x 128 int8  10.2/12.1 11.1/15.4 11.4/16.6 18.4/23.7  12.3/13.0 13.5/16.8 13.5/17.6 20.3/31.3
    //   2 x 64 int4    8.1/9.1   8.8/11.8  8.8/12.4 14.3/17.0   9.4/9.7  10.0/12.2 10.0/13.3 15.5/22.2
    // From 9 rows on (two column tiles there) this one; 512 rows of 8 heads lose 3 to 8 %
    // below 256 tokens, and up to 8 rows gain between 256 and some 2000 only.
    const int64_t rows = (int64_t)a.new_tokens * a.group;
    return a.head_dim <= 128 && rows > 8 && rows < (1 << 24);
}

int kv_prefix_parts(const KvAttentionArgs& a) {
    const int rows = a.new_tokens * a.group, row_tiles = (rows + kRows - 1) / kRows;
    return cut(a.kv_heads * row_tiles, (a.fixed_length + kTile - 1) / kTile);
}

cudaError_t launch_kv_prefix(const KvAttentionArgs& a, cudaStream_t stream) {
    PrefixParams p{};
    p.a = a;
    p.group = FastDiv((uint32_t)a.group);
    p.page_blocks = FastDiv((uint32_t)(a.page_size / kKvBlock));
    p.rows = a.new_tokens * a.group;
    p.row_tiles = (p.rows + kRows - 1) / kRows;
    p.tiles = (a.fixed_length + kTile - 1) / kTile;
    p.parts = kv_prefix_parts(a);
    p.part_tiles = (p.tiles + p.parts - 1) / p.parts;
    p.q_vec = aligned16(a.q, a.q_new, a.q_head);
    p.wait_cycles = wait_budget();
    p.hold_ns = hold_within(p.wait_cycles);
    const bool bf16 = a.type == kTypeBf16;
    if (a.head_dim == 64)
        return a.bits == 8 ? (bf16 ? run<64, 8, true>(p, stream) : run<64, 8, false>(p, stream))
                           : (bf16 ? run<64, 4, true>(p, stream) : run<64, 4, false>(p, stream));
    return a.bits == 8 ? (bf16 ? run<128, 8, true>(p, stream) : run<128, 8, false>(p, stream))
                       : (bf16 ? run<128, 4, true>(p, stream) : run<128, 4, false>(p, stream));
}

cudaError_t read_kv_prefix_status(int clear, int* status) {
    return read_status_symbol(g_kv_prefix_status, clear, status);
}

}  // namespace clb
