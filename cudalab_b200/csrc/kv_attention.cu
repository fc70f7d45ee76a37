// Attention of a few new tokens per sequence over the paged quantised cache
// (layout: kv_layout.cuh).
//
//   s_j = scale * ks_j * (q . k_j)            k_j, v_j whole values, ks_j, vs_j scales
//   o = sum_j exp(s_j) vs_j v_j / sum_j exp(s_j),   lse = ln sum_j exp(s_j)
//
// Bound by the cache's bytes: every byte is read once per row tile, the whole
// values are exact in fp16 and go to the tensor cores unscaled, the scales are
// applied to the scores (K) and to the weights of the softmax (V).
//
// One pass, rows in columns.  The scores are computed transposed, S^T = K Q^T,
// with 16 tokens of a block as the 16 rows of an mma.m16n8k16 and the query
// rows (new tokens x heads of the group) as its 8 columns: a single token of
// up to 8 grouped heads wastes nothing, and K's fragments come from one token
// per lane group, straight from the row-major cache.  The weights go back as
// the B operand of O^T = V^T P^T after a transposing movmatrix; V's fragments
// need two tokens per register, which two byte permutes interleave.  The order
// of k inside an mma is free, so a lane takes contiguous bytes and q is loaded
// in the same order.
//
// Softmax.  Each row keeps one reference m, kLift below the running maximum of
// s_j + log2 vs_j (base 2): the V weights w_j = 2^(s_j + log2 vs_j - m) then lie in
// the range fp16 represents whatever the scales are, and the denominator sums
// w_j / vs_j in fp32 under the same reference.  The weights round to fp16 (2^-11
// of each, 2^-25 of one below 2^-14) because the tensor cores take them in V's
// type; a second product with what the rounding left would double O's
// instructions.  m only moves when a score exceeds the maximum it was taken from
// by more than kSlack, so the usual block pays one vote instead of a reduction
// and a rescale.
//
// Split.  The 16-token blocks of all (sequence, head, row tile) segments form
// one line that is cut into equal ranges, one per CTA of a persistent grid, so
// ragged batches balance whatever their lengths; few segments are instead cut
// into equal chunks that no CTA shares with another segment.  The four warps
// of a CTA take its blocks in turn.  Each warp has its own ring of block buffers filled by
// bulk copies (one per block) and never waits for another warp until a segment
// ends.  A segment cut over several CTAs leaves partial results in the
// workspace; the CTA that arrives last at a group's counter adds the group's
// partials in order (groups of kFan, then the groups), so the sum order, and
// with it every bit of the result, does not depend on timing.
//
// Measured (8 heads of 128, a replayed graph; two boxes within 1 %): 64 sequences
// with 64 query heads, int8 of 2048 to 4096 tokens 70 us = 5.9 TB/s, 0.90 of a
// copy; int4 of 4096 to 8192 tokens 96 us = 4.35 TB/s, 0.66; 16 ragged sequences
// to 4096, int8 20.7 us, of which the bytes are 10.5; one sequence of 77 tokens 4.5.
// int8 is its copies (alone 67 us).  int4 has twice the elements a byte at three
// warps a scheduler: copies alone 69, without the sum over V 72, without the
// expansion of V's fields 88, of K's 90, of both 81, so what remains is the
// length of a step's chain, reads, expansion, products and softmax one after the
// other, which three warps do not cover (0.58 instructions a cycle and scheduler,
// no pipe above 51 %).  With 16 rows a head (two column tiles, two CTAs an SM)
// the same holds for both: 49 us for 31.6 (int8), 77 for 32 (int4).  The short ones
// are launch, plan, first bytes and join in a row.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <atomic>
#include <cstdint>

#include "gemv_common.cuh"
#include "gemv_launch.h"
#include "kv_device.cuh"
#include "kv_layout.cuh"

namespace clb {
namespace {

__device__ int g_kv_attention_status;

constexpr int kWarps = 4, kThreads = 32 * kWarps;
constexpr int kMaxBatch = 4096;  // lengths and their running sum are kept in shared memory
constexpr int kMaxGrid = 148 * 5;
constexpr int kFan = 16;         // partial results added by one CTA at a time
// What a CTA pays for a segment besides its units (loading q, joining its
// warps' results, latencies), in units: about 4000 cycles against 400 to 700 a
// unit.  Without it the CTA that gets the shortest sequences of a ragged batch
// ends last (64 sequences of 1 to 1024 tokens: 52 us, with it 25).
constexpr int kSegmentCost = 8;
// A row's weights are fp16: with its reference kLift below the largest logit the
// largest weight is 2^7, one far smaller keeps 7 bits more than under a largest
// of 1 (a long tail of them counts: 16384 tokens 2^-25.5 of the largest each were
// lost whole), and with kSlack more before the reference moves it stays below 2^15.
constexpr float kLift = 7.f, kSlack = 8.f;
constexpr int kPartialFloats = 16 * 128 + 2 * 16;  // O, m and l of one partial result
constexpr size_t kCounterBytes = (size_t)kMaxGrid * 3 * sizeof(int);

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

__device__ __forceinline__ void mma_16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0,
                                          uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
        "{%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

__device__ __forceinline__ uint32_t transpose8x8(uint32_t v) {
    uint32_t r;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
    return r;
}

// Fields as exact halves: under an exponent of 1024 or 64, less that and the flip
// of the sign bit.  The subtraction belongs before the products.  A score or an
// output taken with the bias on (128 or 8) and rid of bias times sum(q), or times the
// softmax's denominator, afterwards is a small difference of large sums: with a
// strong channel in K and a q that does not average to zero a logit was off by
// 3e-4, and it saved no time (the additions run beside the logic instructions).
__device__ __forceinline__ uint32_t h2_add(uint32_t v, unsigned short bias) {
    const __half2 r = __hadd2(u32_as_h2(v), h2_const(bias));
    return *reinterpret_cast<const uint32_t*>(&r);
}
__device__ __forceinline__ uint32_t bytes02(uint32_t w) {
    return h2_add(lop3_sel_xor_i<0x00FF00FFu, 0x64806480u>(w), kH_m1152);
}
__device__ __forceinline__ uint32_t nibbles04(uint32_t w) {
    return h2_add(lop3_sel_xor_i<0x000F000Fu, 0x64086408u>(w), kH_m1032);
}
__device__ __forceinline__ uint32_t nibbles15(uint32_t w) {
    return h2_add(lop3_sel_xor_i<0x00F000F0u, 0x54805480u>(w), kH_m72);
}

// kWords words of a row from shared memory: one 4-, 8- or 16-byte access.
template <int kWords>
__device__ __forceinline__ void lds_words(const uint8_t* at, uint32_t* w) {
    if constexpr (kWords == 4) {
        const uint4 v = *reinterpret_cast<const uint4*>(at);
        w[0] = v.x, w[1] = v.y, w[2] = v.z, w[3] = v.w;
    } else if constexpr (kWords == 2) {
        const uint2 v = *reinterpret_cast<const uint2*>(at);
        w[0] = v.x, w[1] = v.y;
    } else {
        w[0] = *reinterpret_cast<const uint32_t*>(at);
    }
}
__device__ __forceinline__ float lds_half(const uint8_t* at) {
    return __half2float(*reinterpret_cast<const __half*>(at));
}

// 8 elements of a q that 16-byte loads cannot take (a call, off the main path).
__device__ __noinline__ uint4 load8_apart(const uint16_t* p) { return load8<false, false>(p, 0); }

// ceil(n / d) for 0 <= n < 2^22, inv = 1 / d within 2 ulp: (n - 1/2) / d keeps
// half a step from the integers, more than the products' rounding.  The plan
// runs once per launch, on cold instructions, where an integer division costs
// more than its result.
__device__ __forceinline__ int ceil_div(int n, float inv) {
    return __float2int_ru(((float)n - 0.5f) * inv);
}

// n / d for quotients below kMostQuotient: an estimate, right to one, and its
// correction (beyond, 24 bits leave it two and more off).
constexpr int kMostQuotient = 1 << 21;
__device__ __forceinline__ int quotient(int n, int d) {
    int q = __float2int_rz(__fdividef((float)n, (float)d));
    const int r = n - q * d;
    return q - (r < 0) + (r >= d);
}

struct Params {
    KvAttentionArgs a;
    float* partial;
    int* counters;
    FastDiv row_tiles;   // of kCols rows each, per (sequence, head)
    FastDiv page_blocks; // blocks of a page
    FastDiv group;       // query heads per cache head
    int min_units;       // smallest range of a CTA
    int every_chunk;     // the grid holds every chunk of min_units of the longest lengths:
    FastDiv seg_chunks;  // a segment has this many CTAs
    FastDiv min_chunk;   // division by min_units
    int may_chunk;       // lengths are short enough for ceil_div
    float inv_grid;
    int q_vec;
    long long wait_cycles;
    uint32_t hold_ns;
};

template <int kDim, int kBits, int kNB>
struct Shape {
    static constexpr int kRow = kDim * kBits / 8;
    static constexpr int kBlockBytes = kv_block_bytes(kRow);
    static constexpr int kCols = 8 * kNB;
    // Blocks that a warp takes at a time: two give its instruction stream two
    // independent chains and halve what is paid per step.
    static constexpr int kU = kDim == 256 ? 1 : 2;
    // CTAs per SM that the registers allow, and the ring depth per warp that
    // the shared memory allows beside them.
    static constexpr int kPerSm = kDim == 256 || (kDim == 128 && kNB == 2) ? 2 : 3;
    static constexpr int kStageBytes = kU * kBlockBytes;
    static constexpr int kRedBytes = kWarps * 8 * kDim * 4;
    static constexpr int kStatBytes = kWarps * kCols * 2 * 4;
    static constexpr int kSpare = 227 * 1024 / kPerSm - 4096 - kRedBytes - kStatBytes;
    static constexpr int kFit = kSpare / (kWarps * kStageBytes);
    static constexpr int kStages = kFit < 2 ? 2 : kFit > 6 ? 6 : kFit;
    static constexpr int kRingBytes = kWarps * kStages * kStageBytes;
};

// A segment of the line: its units are [begin, begin + units).
struct Segment {
    int seq, part;  // sequence; head * row_tiles + row tile
    int begin, units;
};

template <int kDim, int kBits, int kNB, bool kBf16>
__global__ void __launch_bounds__(kThreads, Shape<kDim, kBits, kNB>::kPerSm)
    kv_attention_kernel(const Params p) {
    using S = Shape<kDim, kBits, kNB>;
    constexpr int kRow = S::kRow, kStages = S::kStages, kBlockBytes = S::kBlockBytes;
    constexpr int kU = S::kU, kStageBytes = S::kStageBytes;
    constexpr int kSteps = kDim / 16;  // mma steps of q . k, and 16-row blocks of O^T
    extern __shared__ __align__(128) uint8_t smem[];
    uint8_t* ring = smem;
    float* red = reinterpret_cast<float*>(smem + S::kRingBytes);
    float* stat = reinterpret_cast<float*>(smem + S::kRingBytes + S::kRedBytes);
    uint64_t* bars = reinterpret_cast<uint64_t*>(smem + S::kRingBytes + S::kRedBytes + S::kStatBytes);
    int* flag = reinterpret_cast<int*>(bars + kWarps * kStages);
    int* s_len = flag + 4;                 // [batch]
    int* s_cum = s_len + p.a.batch;        // [batch + 1] cells in front of a sequence
    int* s_cost = s_cum + p.a.batch + 1;   // [batch + 1] the same with kSegmentCost a segment

    const KvAttentionArgs& a = p.a;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int g = lane >> 2, t = lane & 3;
    const int heads_tiles = a.kv_heads * (int)p.row_tiles.d;  // segments of a sequence
    const int rows = a.new_tokens * a.group;

    pdl_allow_dependents();
    uint8_t* my_ring = ring + warp * kStages * kStageBytes;
    const uint32_t my_bars = smem_u32(bars) + warp * kStages * 8;
    if (lane == 0) {
        for (int i = 0; i < kStages; ++i) mbar_init(my_bars + 8 * i, 1);
        fence_barrier_init();
    }
    // Over a prefix's tensor-core launch everything up to the first result runs
    // beside it: that launch lets this one begin only after the kernel before
    // it has completed, and writes nothing but what `front` points to.  Before
    // a result is written (and the front read, or the workspace used by a
    // launch further back) `settle` waits for it.
    if (!a.front_by_tensor_cores) pdl_wait_prior_grids();
    auto settle = [&]() {
        if (a.front_by_tensor_cores) pdl_wait_prior_grids();
    };

    // Units of each sequence (a window drops the blocks in front of the first
    // token that any row sees), and how the line of all segments is cut.
    auto first_block = [&](int len) {
        // len - new + 1 - window, of which no step passes 32 bits
        const int behind = len - a.window;
        return a.window > 0 && behind >= a.new_tokens ? (behind - a.new_tokens + 1) / kKvBlock : 0;
    };
    auto units_of = [&](int len) {
        return ((len + kKvBlock - 1) / kKvBlock - first_block(len) + kU - 1) / kU;
    };
    const int most = a.max_pages * a.page_size, grid = (int)gridDim.x;
    auto length_of = [&](int b) {
        int len = a.fixed_length >= 0 ? a.fixed_length : __ldg(a.lengths + b);
        if (len > most || len < 0) {
            atomicCAS(&g_kv_attention_status, 0, kStatusKvIndex);
            len = len < 0 ? 0 : most;
        }
        return len;
    };
    // Up to 32 sequences every warp plans for itself (all write the same values
    // and read their own), more are planned by the first warp.
    const bool few = a.batch <= 32;
    int cell = 1;   // units of a cell of the line (s_cum counts cells)
    int share = 1;  // cells of a CTA
    if (!p.every_chunk) {
        for (int b = few ? lane : tid; b < a.batch; b += few ? 32 : kThreads) s_len[b] = length_of(b);
        if (few) __syncwarp(); else __syncthreads();
        if (few || warp == 0) {
            int units = 0, segments = 0;
            for (int b = lane; b < a.batch; b += 32) {
                const int n = units_of(s_len[b]);
                units += n;
                segments += n > 0;
            }
            units = __reduce_add_sync(0xffffffffu, units) * heads_tiles;
            segments = __reduce_add_sync(0xffffffffu, segments) * heads_tiles;
            // equal ranges of the line (the estimate may be short on very long ones)
            const int cost = units + kSegmentCost * segments;
            share = max(p.min_units, ceil_div(cost, p.inv_grid));
            if (share * (int64_t)grid < cost) share += 1 + (share >> 20);
            if (2 * segments <= grid && p.may_chunk) {
                // Few segments: each is cut into chunks of its own, one per CTA,
                // so that a CTA works on one segment.  Eight sizes between the
                // equal range and the one that must fit, four lanes on each; the
                // smallest with which the grid holds all chunks is taken.
                share = max(p.min_units, ceil_div(units, p.inv_grid));
                const int more = max(0, ceil_div(units, __fdividef(1.f, (float)(grid - segments))) + 1 - share);
                const int mine = share + (more * (lane >> 2) * 37 >> 8);  // 37/256 > 1/7
                const float inv = __fdividef(1.f, (float)mine);
                int chunks = 0;
                for (int b = lane & 3; b < a.batch; b += 4) chunks += ceil_div(units_of(s_len[b]), inv);
                chunks += __shfl_xor_sync(0xffffffffu, chunks, 1);
                chunks += __shfl_xor_sync(0xffffffffu, chunks, 2);
                const uint32_t ok = __ballot_sync(0xffffffffu, chunks * heads_tiles <= grid);
                cell = __shfl_sync(0xffffffffu, mine, __ffs(ok | 0x80000000u) - 1);
                share = 1;
            }
            const float inv = __fdividef(1.f, (float)cell);
            int before = 0, filled = 0;
            for (int b0 = 0; b0 < a.batch; b0 += 32) {
                const int b = b0 + lane;
                int n = b < a.batch ? units_of(s_len[b]) : 0;
                if (cell > 1) n = ceil_div(n, inv);
                const uint32_t some = __ballot_sync(0xffffffffu, n > 0);
                int scan = n;
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) {
                    const int v = __shfl_up_sync(0xffffffffu, scan, o);
                    if (lane >= o) scan += v;
                }
                if (b < a.batch) {
                    s_cum[b] = before + scan - n;
                    s_cost[b] = before + scan - n +
                                kSegmentCost * (filled + __popc(some & ((1u << lane) - 1)));
                }
                before += __shfl_sync(0xffffffffu, scan, 31);
                filled += __popc(some);
            }
            if (lane == 0) {
                s_cum[a.batch] = before;
                s_cost[a.batch] = before + kSegmentCost * filled;
                flag[1] = cell, flag[2] = share;
            }
        }
        if (few) {
            __syncwarp();
        } else {
            __syncthreads();
            cell = flag[1];
            share = flag[2];
        }
    }
    const bool chunked = p.every_chunk || cell > 1;

    // Row `r` of a tile of sequence `seq`: where it is in the outputs.
    auto out_row = [&](int seq, int head, int r) {
        const int i = p.group.div(r);
        return ((int64_t)seq * a.new_tokens + i) * (a.kv_heads * a.group) + (head - i) * a.group + r;
    };
    // One normalised output: 4 elements d.. of row `row`; `front` joins the
    // result over the tokens in front.
    auto write_out = [&](int64_t row, int d, float4 o, float m, float l, bool first) {
        float lse2 = l > 0.f ? m + lg2(l) : (l == l ? -INFINITY : l);
        const float inv = l > 0.f ? 1.f / l : (l == l ? 0.f : l);
        o.x *= inv, o.y *= inv, o.z *= inv, o.w *= inv;
        if (a.front != nullptr) {
            constexpr float kLog2e = 1.4426950408889634f;
            const int64_t all = (int64_t)a.batch * a.new_tokens * a.kv_heads * a.group;
            float sum = lse2 == -INFINITY ? 0.f : 1.f, top = lse2;
#pragma unroll 4
            for (int f = 0; f < a.front_parts; ++f) {
                const int64_t at = f * all + row;
                const float4 x = __ldcg(reinterpret_cast<const float4*>(a.front + at * kDim + d));
                const float fl = __ldcg(a.front_lse + at) * kLog2e;
                const float next = fmaxf(top, fl);
                const float ref = next == -INFINITY ? 0.f : next;
                const float wo = ex2(top - ref), wf = ex2(fl - ref);
                top = next;
                sum = sum * wo + wf;
                o.x = o.x * wo + x.x * wf, o.y = o.y * wo + x.y * wf;
                o.z = o.z * wo + x.z * wf, o.w = o.w * wo + x.w * wf;
            }
            const float i2 = sum > 0.f ? 1.f / sum : (sum == sum ? 0.f : sum);
            o.x *= i2, o.y *= i2, o.z *= i2, o.w *= i2;
            lse2 = sum > 0.f ? top + lg2(sum) : (sum == sum ? -INFINITY : sum);
        }
        if (a.out_f32 != nullptr)
            *reinterpret_cast<float4*>(a.out_f32 + row * kDim + d) = o;
        else
            *reinterpret_cast<uint2*>(static_cast<uint16_t*>(a.out) + row * kDim + d) =
                make_uint2(pack2<kBf16>(o.x, o.y), pack2<kBf16>(o.z, o.w));
        if (first && a.lse != nullptr) a.lse[row] = lse2 * 0.6931471805599453f;
    };

    // A row tile with nothing to read (its rows see no cached token).
    auto write_empty = [&](int b, int part) {
        settle();
        const int h = p.row_tiles.div(part), r0 = p.row_tiles.mod(part) * S::kCols;
        const int n = min(S::kCols, rows - r0) * (kDim / 4);
        for (int i = tid; i < n; i += kThreads) {
            const int d = i % (kDim / 4) * 4;
            write_out(out_row(b, h, r0 + i / (kDim / 4)), d, make_float4(0.f, 0.f, 0.f, 0.f),
                      -INFINITY, 0.f, d == 0);
        }
    };

    // The CTA's range [u0, u1) and its first segment.  Chunked, the line is the
    // units of the one segment; else the units of all segments.
    Segment start;
    int u0, u1, c0 = 0, parts = 0;  // chunked: first CTA and CTAs of the segment
    int len0;                       // length of the first segment's sequence
    if (p.every_chunk) {
        const int segment = p.seg_chunks.div((int)blockIdx.x);
        c0 = segment * (int)p.seg_chunks.d;
        start.seq = quotient(segment, heads_tiles);
        start.part = segment - start.seq * heads_tiles;
        len0 = length_of(start.seq);
        start.begin = 0;
        start.units = units_of(len0);
        u0 = ((int)blockIdx.x - c0) * p.min_units;
        u1 = min(u0 + p.min_units, start.units);
        parts = p.min_chunk.div(start.units + p.min_units - 1);
        if (u0 >= u1) {
            if (start.units == 0 && u0 == 0) write_empty(start.seq, start.part);
            return;
        }
    } else {
        for (int i = blockIdx.x; i < a.batch * heads_tiles; i += grid) {
            const int b = i / heads_tiles;
            if (s_cum[b + 1] == s_cum[b]) write_empty(b, i - b * heads_tiles);
        }
        // last sequence whose cells (`sums`) begin at or before x, by the whole warp
        auto find = [&](const int* sums, int x) {
            int count = 0;
            for (int b0 = 0; b0 < a.batch; b0 += 32) {
                const int b = b0 + lane;
                const uint32_t at_or_before =
                    __ballot_sync(0xffffffffu, b < a.batch && sums[min(b, a.batch)] * heads_tiles <= x);
                count += __popc(at_or_before);
                if (at_or_before != 0xffffffffu) break;
            }
            return count - 1;
        };
        // Equal ranges are cut in cost; the unit at which a cost begins:
        const int total_cost = s_cost[a.batch] * heads_tiles;
        auto unit_at = [&](int cost) {
            if (cost >= total_cost) return s_cum[a.batch] * heads_tiles;
            const int b = find(s_cost, cost);
            const int n = s_cum[b + 1] - s_cum[b], in = cost - s_cost[b] * heads_tiles;
            const int part = quotient(in, n + kSegmentCost);
            return s_cum[b] * heads_tiles + part * n + min(n, in - part * (n + kSegmentCost));
        };
        const int64_t x0 = (int64_t)blockIdx.x * share;
        if (chunked) {
            u0 = (int)min(x0, (int64_t)s_cum[a.batch] * heads_tiles);
            u1 = min(u0 + 1, s_cum[a.batch] * heads_tiles);
        } else {
            u0 = unit_at((int)min(x0, (int64_t)total_cost));
            u1 = unit_at((int)min(x0 + share, (int64_t)total_cost));
        }
        if (u0 >= u1) return;
        const int lo = find(s_cum, u0);
        const int cells = s_cum[lo + 1] - s_cum[lo], in = u0 - s_cum[lo] * heads_tiles;
        start.seq = lo;
        start.part = quotient(in, cells);
        start.units = cells;
        start.begin = s_cum[lo] * heads_tiles + start.part * cells;
        len0 = s_len[lo];
        if (chunked) {
            const int chunk = in - start.part * cells;
            c0 = (int)blockIdx.x - chunk;
            parts = cells;
            start.begin = 0;
            start.units = units_of(len0);
            u0 = chunk * cell;
            u1 = min(u0 + cell, start.units);
        }
    }
    auto next_segment = [&](Segment& c) {
        c.begin += c.units;
        if (!chunked && ++c.part == heads_tiles) {
            c.part = 0;
            do ++c.seq; while (c.seq < a.batch && s_cum[c.seq + 1] == s_cum[c.seq]);
            if (c.seq < a.batch) c.units = s_cum[c.seq + 1] - s_cum[c.seq];
        }
    };

    // q of a segment's rows g + 8 n, this lane's pieces, as stored.
    constexpr int kKWords = kRow / 16, kKPer = kKWords < 4 ? kKWords : 4;
    constexpr int kVWords = kRow / 32, kVPer = kVWords < 4 ? kVWords : 4;
    constexpr int kKAccess = kKWords / kKPer, kVAccess = kVWords / kVPer;
    auto k_byte = [&](int i) {  // byte offset of the i-th access of a quarter row
        return kRow == 256 ? (i >> 1) * 128 + 32 * t + 16 * (i & 1)
                           : kRow == 128 ? 32 * t + 16 * i : (kRow / 4) * t;
    };
    uint4 qraw[kNB][kDim / 32];
    auto load_q = [&](const Segment& c) {
        const int head = p.row_tiles.div(c.part), first = p.row_tiles.mod(c.part) * S::kCols;
#pragma unroll
        for (int n = 0; n < kNB; ++n) {
            const int r = first + 8 * n + g;
            const int i0 = p.group.div(r);
            const uint16_t* at = static_cast<const uint16_t*>(a.q) + c.seq * a.q_batch +
                                 i0 * a.q_new + ((head - i0) * a.group + r) * a.q_head;
            constexpr int kElements = kKPer * 32 / kBits;  // of an access of the cache
#pragma unroll
            for (int i = 0; i < kDim / 32; ++i) {
                qraw[n][i] = make_uint4(0, 0, 0, 0);
                const int e = k_byte(8 * i / kElements) * 8 / kBits + 8 * i % kElements;
                if (r < rows) qraw[n][i] = p.q_vec ? load8<kBf16, true>(at, e) : load8_apart(at + e);
            }
        }
    };
    load_q(start);

    // The warp's copies run kStages units ahead of its arithmetic.  The blocks
    // are looked up 32 units at a time, one unit per lane, and the lane that
    // holds a unit issues its copies, so the walk over segments and pages costs
    // a step a compare.
    constexpr uint32_t kAbsent = 0xffffffffu, kInvalid = 0xfffffffeu;
    const uint64_t policy = policy_evict_first();
    auto look_up = [&](int u, int seq, uint32_t (&at)[kU]) {
#pragma unroll
        for (int k = 0; k < kU; ++k) at[k] = kAbsent;
        if (u >= u1) return;
        int part = start.part, in = u;
        if (!chunked) {
            int next = s_cum[seq + 1];
            while (next * heads_tiles <= u) next = s_cum[++seq + 1];
            const int units = next - s_cum[seq];
            in = u - s_cum[seq] * heads_tiles;
            part = quotient(in, units);
            in -= part * units;
        }
        const int len = chunked ? len0 : s_len[seq];
        const uint32_t head = p.row_tiles.div(part);
#pragma unroll
        for (int k = 0; k < kU; ++k) {
            const int blk = in * kU + k + first_block(len);
            if (k > 0 && blk * kKvBlock >= len) break;
            const int index = p.page_blocks.div(blk);
            const int page = __ldg(a.table + seq * a.table_stride + index);
            if (page < 0 || page >= a.num_pages) {
                atomicCAS(&g_kv_attention_status, 0, kStatusKvIndex);
                at[k] = kInvalid;
            } else {
                at[k] = ((uint32_t)page * a.kv_heads + head) * p.page_blocks.d +
                        (blk - index * p.page_blocks.d);
            }
        }
    };
    auto copy = [&](int stage, const uint32_t (&at)[kU]) {
        const uint32_t bar = my_bars + 8 * stage, to = smem_u32(my_ring) + stage * kStageBytes;
        if (kU == 2 && at[0] < kInvalid && at[kU - 1] == at[0] + 1) {  // one stretch of memory
            mbar_arrive_expect_tx(bar, kStageBytes);
            bulk_g2s(to, a.pages + (int64_t)at[0] * kBlockBytes, kStageBytes, bar, policy);
            return;
        }
        uint32_t bytes = 0;
#pragma unroll
        for (int k = 0; k < kU; ++k) bytes += at[k] < kInvalid ? kBlockBytes : 0;
        mbar_arrive_expect_tx(bar, bytes);  // none: the phase completes at once
#pragma unroll
        for (int k = 0; k < kU; ++k)
            if (at[k] < kInvalid)
                bulk_g2s(to + k * kBlockBytes, a.pages + (int64_t)at[k] * kBlockBytes, kBlockBytes,
                         bar, policy);
    };
    int issued = kStages, done = 0;  // of this warp's units
    const int mine = u0 + warp < u1 ? (u1 - u0 - warp + kWarps - 1) / kWarps : 0;
    uint32_t at[kU];
    look_up(u0 + warp + kWarps * lane, start.seq, at);
    // units with an invalid page, of the batch in use and of the one being issued
    uint32_t bad[kU], bad_next[kU];
#pragma unroll
    for (int k = 0; k < kU; ++k) bad[k] = bad_next[k] = __ballot_sync(0xffffffffu, at[k] == kInvalid);
    if (lane < min(kStages, mine)) copy(lane, at);

    // Places of this lane's pieces inside a block.
    int k_at[kKAccess], v_at[2][kVAccess];
#pragma unroll
    for (int i = 0; i < kKAccess; ++i) k_at[i] = kv_offset<kRow>(g, k_byte(i));
#pragma unroll
    for (int i = 0; i < kVAccess; ++i)
#pragma unroll
        for (int x = 0; x < 2; ++x)
            v_at[x][i] = kKvBlock * kRow +
                         kv_offset<kRow>(2 * t + x, kRow == 256 ? 128 * i + 16 * g : (kRow / 8) * g);
    const int scale_at = 2 * kKvBlock * kRow + 2 * g;

    int stage = 0;
    uint32_t phase = 0;
    bool failed = false;
    int cu = u0 + warp;
    Segment seg = start;
    while (seg.begin < u1) {
        const int sa = max(seg.begin, u0), sb = min(seg.begin + seg.units, u1);
        const int head = p.row_tiles.div(seg.part), row0 = p.row_tiles.mod(seg.part) * S::kCols;
        const int len = chunked ? len0 : s_len[seg.seq];
        const int token0 = first_block(len) * kKvBlock;

        // q as B fragments, in fp16.  Rows are brought to [2^15, 2^16) by a power of two,
        // which holds fp16 elements exactly and bf16 ones down to 2^-32 of their row's
        // largest.  rs brings a score to base-2 logits.
        uint32_t qf[kNB][kSteps][2];
        float rs[kNB][2];
#pragma unroll
        for (int n = 0; n < kNB; ++n) {
            float x[kDim / 4], top = 0.f;
#pragma unroll
            for (int i = 0; i < kDim / 32; ++i) unpack8<kBf16>(qraw[n][i], x + 8 * i);
#pragma unroll
            for (int i = 0; i < kDim / 4; ++i) top = fmaxf(top, fabsf(x[i]));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
            const int e = (int)(__float_as_uint(top) >> 23) - 127;
            float unit = a.scale * 1.4426950408889634f;
            if (e < 128) {  // rows with an infinity stay as they are
                const int up = min(15 - e, 126);
                const float factor = __uint_as_float((uint32_t)(127 + up) << 23);
#pragma unroll
                for (int i = 0; i < kDim / 4; ++i) x[i] *= factor;
                unit *= __uint_as_float((uint32_t)(127 - up) << 23);
            }
#pragma unroll
            for (int c = 0; c < 2; ++c) rs[n][c] = __shfl_sync(0xffffffffu, unit, 8 * t + 4 * c);
#pragma unroll
            for (int w = 0; w < kKWords; ++w) {
                if (kBits == 8) {
                    qf[n][w][0] = pack2<false>(x[4 * w], x[4 * w + 2]);
                    qf[n][w][1] = pack2<false>(x[4 * w + 1], x[4 * w + 3]);
                } else {
                    qf[n][2 * w][0] = pack2<false>(x[8 * w], x[8 * w + 4]);
                    qf[n][2 * w][1] = pack2<false>(x[8 * w + 1], x[8 * w + 5]);
                    qf[n][2 * w + 1][0] = pack2<false>(x[8 * w + 2], x[8 * w + 6]);
                    qf[n][2 * w + 1][1] = pack2<false>(x[8 * w + 3], x[8 * w + 7]);
                }
            }
        }
        // Tokens [lo, hi) that every row of the sequence sees.
        const int all_hi = a.causal ? len - a.new_tokens + 1 : len;
        const int all_lo = a.window > 0 ? len - a.window : 0;

        float o[kSteps][kNB][4];
        // the reference, 0 in its place while it is -inf, and what a score may reach under it
        float m[kNB][2], ref[kNB][2], limit[kNB][2], l[kNB][2];
#pragma unroll
        for (int n = 0; n < kNB; ++n) {
#pragma unroll
            for (int i = 0; i < kSteps; ++i) o[i][n][0] = o[i][n][1] = o[i][n][2] = o[i][n][3] = 0.f;
            m[n][0] = m[n][1] = limit[n][0] = limit[n][1] = -INFINITY;
            l[n][0] = l[n][1] = ref[n][0] = ref[n][1] = 0.f;
        }

#pragma unroll 1
        for (; cu < sb; cu += kWarps) {
            // every lane leaves the wait with the same answer
            if (!failed && !__all_sync(0xffffffffu, mbar_try_wait_held(my_bars + 8 * stage, phase >> stage & 1u, p.hold_ns))) {
                const long long t0 = clock64();
                do
                    failed = __any_sync(0xffffffffu, clock64() - t0 > p.wait_cycles);
                while (!failed && !__all_sync(0xffffffffu, mbar_try_wait_held(my_bars + 8 * stage, phase >> stage & 1u, p.hold_ns)));
                if (failed && lane == 0) atomicCAS(&g_kv_attention_status, 0, kStatusTimeoutKv);
            }
            if (!failed) {
                phase ^= 1u << stage;
                const uint8_t* base = my_ring + stage * kStageBytes;
                float s[kU][kNB][4];
#pragma unroll
                for (int k = 0; k < kU; ++k)
#pragma unroll
                    for (int n = 0; n < kNB; ++n) s[k][n][0] = s[k][n][1] = s[k][n][2] = s[k][n][3] = 0.f;
#pragma unroll
                for (int i = 0; i < kKAccess; ++i)
#pragma unroll
                    for (int k = 0; k < kU; ++k) {
                        const uint8_t* kb = base + k * kBlockBytes + k_at[i];
                        uint32_t w0[kKPer], w1[kKPer];
                        lds_words<kKPer>(kb, w0);
                        lds_words<kKPer>(kb + 8 * kRow, w1);
#pragma unroll
                        for (int w = 0; w < kKPer; ++w) {
                            const int x = i * kKPer + w;
                            const uint32_t u0 = w0[w] >> 8, u1 = w1[w] >> 8;
                            if (kBits == 8) {
                                const uint32_t f[4] = {bytes02(w0[w]), bytes02(w1[w]), bytes02(u0),
                                                       bytes02(u1)};
#pragma unroll
                                for (int n = 0; n < kNB; ++n)
                                    mma_16816(s[k][n], f, qf[n][x][0], qf[n][x][1]);
                            } else {
                                const uint32_t e[4] = {nibbles04(w0[w]), nibbles04(w1[w]),
                                                       nibbles15(w0[w]), nibbles15(w1[w])};
                                const uint32_t f[4] = {nibbles04(u0), nibbles04(u1), nibbles15(u0),
                                                       nibbles15(u1)};
#pragma unroll
                                for (int n = 0; n < kNB; ++n) {
                                    mma_16816(s[k][n], e, qf[n][2 * x][0], qf[n][2 * x][1]);
                                    mma_16816(s[k][n], f, qf[n][2 * x + 1][0], qf[n][2 * x + 1][1]);
                                }
                            }
                        }
                    }
                // Scores of tokens j0 + g (0, 1) and j0 + g + 8 (2, 3) of each block,
                // log2 of V's scale added (a zero scale has all-zero values: any will do).
                float iv[kU][2];
                bool over = false;
#pragma unroll
                for (int k = 0; k < kU; ++k) {
                    const uint8_t* sc = base + k * kBlockBytes + scale_at;
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const float ks = lds_half(sc + 16 * h);
                        const float lv = fmaxf(lg2(lds_half(sc + 32 + 16 * h)), -24.f);
                        iv[k][h] = ex2(-lv);  // finite whatever a masked token's scale holds
#pragma unroll
                        for (int n = 0; n < kNB; ++n)
#pragma unroll
                            for (int c = 0; c < 2; ++c)
                                s[k][n][2 * h + c] = fmaf(s[k][n][2 * h + c], ks * rs[n][c], lv);
                    }
                }
                const int j0 = (cu - seg.begin) * (kU * kKvBlock) + token0;
                bool cut = j0 + kU * kKvBlock > all_hi || j0 < all_lo;
#pragma unroll
                for (int k = 0; k < kU; ++k) cut |= (bad[k] >> (done & 31)) & 1u;
                if (cut) {
#pragma unroll
                    for (int n = 0; n < kNB; ++n)
#pragma unroll
                        for (int c = 0; c < 2; ++c) {
                            const int r = row0 + 8 * n + 2 * t + c;
                            const int end = len - a.new_tokens + p.group.div(r) + 1;
                            const int hi = a.causal ? min(end, len) : len;
                            // (a row in front of the sequence sees nothing, by hi)
                            const int lo = a.window > 0 ? max(end, 0) - a.window : 0;
#pragma unroll
                            for (int k = 0; k < kU; ++k)
#pragma unroll
                                for (int h = 0; h < 2; ++h) {
                                    const int j = j0 + k * kKvBlock + g + 8 * h;
                                    if (j >= hi || j < lo || ((bad[k] >> (done & 31)) & 1u))
                                        s[k][n][2 * h + c] = -INFINITY;
                                }
                        }
                }
#pragma unroll
                for (int k = 0; k < kU; ++k)
#pragma unroll
                    for (int n = 0; n < kNB; ++n) {
                        over |= fmaxf(s[k][n][0], s[k][n][2]) > limit[n][0];
                        over |= fmaxf(s[k][n][1], s[k][n][3]) > limit[n][1];
                    }
                if (__any_sync(0xffffffffu, over)) {
#pragma unroll
                    for (int n = 0; n < kNB; ++n)
#pragma unroll
                        for (int c = 0; c < 2; ++c) {
                            float top = fmaxf(s[0][n][c], s[0][n][c + 2]);
                            if (kU == 2)
                                top = fmaxf(top, fmaxf(s[kU - 1][n][c], s[kU - 1][n][c + 2]));
#pragma unroll
                            for (int x = 4; x < 32; x <<= 1)
                                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, x));
                            top = fmaxf(top - kLift, m[n][c]);
                            // a row that has seen nothing keeps -inf and zeros
                            const float f = top == -INFINITY ? 1.f : ex2(m[n][c] - top);
                            m[n][c] = top;
                            ref[n][c] = top == -INFINITY ? 0.f : top;
                            limit[n][c] = top + (kLift + kSlack);
                            l[n][c] *= f;
#pragma unroll
                            for (int i = 0; i < kSteps; ++i) {
                                o[i][n][c] *= f;
                                o[i][n][c + 2] *= f;
                            }
                        }
                }
                uint32_t pf[kU][kNB][2];
#pragma unroll
                for (int k = 0; k < kU; ++k)
#pragma unroll
                    for (int n = 0; n < kNB; ++n)
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            const float w0 = ex2(s[k][n][2 * h] - ref[n][0]);
                            const float w1 = ex2(s[k][n][2 * h + 1] - ref[n][1]);
                            l[n][0] = fmaf(w0, iv[k][h], l[n][0]);
                            l[n][1] = fmaf(w1, iv[k][h], l[n][1]);
                            pf[k][n][h] = transpose8x8(pack2<false>(w0, w1));
                        }
                // O^T += V^T P^T: tokens 2t, 2t + 1, 2t + 8, 2t + 9 of each block.
#pragma unroll
                for (int k = 0; k < kU; ++k)
#pragma unroll
                    for (int i = 0; i < kVAccess; ++i) {
                        const uint8_t* vb = base + k * kBlockBytes;
                        uint32_t w[4][kVPer];
#pragma unroll
                        for (int x = 0; x < 4; ++x)
                            lds_words<kVPer>(vb + v_at[x & 1][i] + (x >> 1) * 8 * kRow, w[x]);
#pragma unroll
                        for (int y = 0; y < kVPer; ++y)
#pragma unroll
                            for (int h = 0; h < 2; ++h) {  // low and high half of the words
                                const uint32_t d0 = h ? prmt_i<0x7632u>(w[0][y], w[1][y])
                                                      : prmt_i<0x5410u>(w[0][y], w[1][y]);
                                const uint32_t d1 = h ? prmt_i<0x7632u>(w[2][y], w[3][y])
                                                      : prmt_i<0x5410u>(w[2][y], w[3][y]);
                                const uint32_t e0 = d0 >> 8, e1 = d1 >> 8;
                                const int x = 2 * (i * kVPer + y) + h;
                                if (kBits == 8) {
                                    const uint32_t f[4] = {bytes02(d0), bytes02(e0), bytes02(d1),
                                                           bytes02(e1)};
#pragma unroll
                                    for (int n = 0; n < kNB; ++n)
                                        mma_16816(o[x][n], f, pf[k][n][0], pf[k][n][1]);
                                } else {
                                    const uint32_t e[4] = {nibbles04(d0), nibbles15(d0),
                                                           nibbles04(d1), nibbles15(d1)};
                                    const uint32_t f[4] = {nibbles04(e0), nibbles15(e0),
                                                           nibbles04(e1), nibbles15(e1)};
#pragma unroll
                                    for (int n = 0; n < kNB; ++n) {
                                        mma_16816(o[2 * x][n], e, pf[k][n][0], pf[k][n][1]);
                                        mma_16816(o[2 * x + 1][n], f, pf[k][n][0], pf[k][n][1]);
                                    }
                                }
                            }
                    }
                __syncwarp();  // every lane has read the stage before it is filled again
                if (issued < mine) {
                    const int i = issued & 31;
                    if (i == 0) {
                        look_up(u0 + warp + kWarps * (issued + lane), seg.seq, at);
#pragma unroll
                        for (int k = 0; k < kU; ++k)
                            bad_next[k] = __ballot_sync(0xffffffffu, at[k] == kInvalid);
                    }
                    if (lane == i) copy(stage, at);
                    ++issued;
                }
                if ((++done & 31) == 0) {
#pragma unroll
                    for (int k = 0; k < kU; ++k) bad[k] = bad_next[k];
                }
            }
            stage = stage + 1 == kStages ? 0 : stage + 1;
        }

        // ---- the segment's end: the warps' results meet in shared memory ----
        // Value v of a lane: 4 elements of row 2t + v / (kSteps / 2) (+ 8 n),
        // stored lane by lane; warp w joins and writes the values w, w + 4, ...
        settle();
        const Segment now = seg;
        next_segment(seg);
        const bool whole = sa == now.begin && sb == now.begin + now.units;
        float* slot = p.partial + ((int64_t)blockIdx.x * 2 + (now.begin >= u0)) * kPartialFloats;
        auto value_row = [&](int v) { return 2 * t + v / (kSteps / 2); };
        auto value_d = [&](int v) {
            const int i = v % (kSteps / 2) * 2;  // its first 16-row block of O^T
            return kRow == 256 ? (i / 8) * 128 + 16 * g + 2 * (i % 8) : (kDim / 8) * g + 2 * i;
        };
#pragma unroll
        for (int n = 0; n < kNB; ++n) {
#pragma unroll
            for (int c = 0; c < 2; ++c) {
#pragma unroll
                for (int x = 4; x < 32; x <<= 1) l[n][c] += __shfl_xor_sync(0xffffffffu, l[n][c], x);
                if (g == 0)
                    *reinterpret_cast<float2*>(stat + (warp * S::kCols + 8 * n + 2 * t + c) * 2) =
                        make_float2(m[n][c], l[n][c]);
#pragma unroll
                for (int i = 0; i < kSteps; i += 2)
                    reinterpret_cast<float4*>(red)[(warp * kSteps + c * (kSteps / 2) + i / 2) * 32 + lane] =
                        make_float4(o[i][n][c], o[i][n][c + 2], o[i + 1][n][c], o[i + 1][n][c + 2]);
            }
            __syncthreads();
#pragma unroll
            for (int v0 = 0; v0 < kSteps; v0 += kWarps) {
                const int v = v0 + warp, col = 8 * n + value_row(v), d = value_d(v);
                float2 ml[kWarps];
                float top = -INFINITY, sum = 0.f;
#pragma unroll
                for (int w = 0; w < kWarps; ++w) {
                    ml[w] = *reinterpret_cast<const float2*>(stat + (w * S::kCols + col) * 2);
                    top = fmaxf(top, ml[w].x);
                }
                float4 r = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
                for (int w = 0; w < kWarps; ++w) {
                    // a warp that saw nothing has zeros here (or the NaN of its q)
                    const float f = ml[w].x == -INFINITY ? 0.f : ex2(ml[w].x - top);
                    const float4 x = reinterpret_cast<const float4*>(red)[(w * kSteps + v) * 32 + lane];
                    sum = fmaf(f, ml[w].y, sum);
                    r.x = fmaf(f, x.x, r.x), r.y = fmaf(f, x.y, r.y);
                    r.z = fmaf(f, x.z, r.z), r.w = fmaf(f, x.w, r.w);
                }
                if (!whole) {
                    reinterpret_cast<float4*>(slot)[(n * kSteps + v) * 32 + lane] = r;
                    if (d == 0)
                        *reinterpret_cast<float2*>(slot + 16 * 128 + 2 * col) = make_float2(top, sum);
                } else if (row0 + col < rows) {
                    write_out(out_row(now.seq, head, row0 + col), d, r, top, sum, d == 0);
                }
            }
            __syncthreads();
        }
        if (seg.begin < u1) load_q(seg);

        if (!whole) {
            if (!chunked) {
                const int cost = s_cost[now.seq] * heads_tiles + now.part * (now.units + kSegmentCost);
                c0 = quotient(cost, share);
                parts = quotient(cost + now.units - 1, share) - c0 + 1;
            }
            const int me = (int)blockIdx.x - c0;
            auto slot_of = [&](int i) {  // of the segment's i-th CTA
                return p.partial + ((int64_t)(c0 + i) * 2 + (i == 0)) * kPartialFloats;
            };
            auto arrive = [&](int* counter, int count) {
                __syncthreads();
                if (tid == 0) {
                    // releases this CTA's stores (ordered by the barrier) and
                    // acquires those of the CTAs that came before
                    int old;
                    asm volatile("atom.add.acq_rel.gpu.global.s32 %0, [%1], 1;"
                                 : "=r"(old) : "l"(counter) : "memory");
                    *flag = old == count - 1;
                    if (old == count - 1) *counter = 0;  // ready for the next launch
                }
                __syncthreads();
                return *flag != 0;
            };
            // Adds the `count` partial results first, first + step, ... in order;
            // eight are in flight at a time.
            auto add = [&](int first, int step, int count, float* to) {
#pragma unroll 1
                for (int nv = warp; nv < kNB * kSteps; nv += kWarps) {
                    const int v = nv % kSteps, d = value_d(v);
                    const int col = nv / kSteps * 8 + value_row(v);
                    float top = -INFINITY, sum = 0.f;
                    float4 r = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 1
                    for (int k0 = 0; k0 < count; k0 += 8) {
                        float2 ml[8];
                        float4 x[8];
                        float best = top;
#pragma unroll
                        for (int k = 0; k < 8; ++k) {
                            ml[k] = make_float2(-INFINITY, 0.f);
                            x[k] = make_float4(0.f, 0.f, 0.f, 0.f);
                            if (k0 + k < count) {
                                const float* src = slot_of(first + (k0 + k) * step);
                                ml[k] = __ldcg(reinterpret_cast<const float2*>(src + 16 * 128 + 2 * col));
                                x[k] = __ldcg(reinterpret_cast<const float4*>(src) + nv * 32 + lane);
                            }
                        }
#pragma unroll
                        for (int k = 0; k < 8; ++k) best = fmaxf(best, ml[k].x);
                        const float ref = best == -INFINITY ? 0.f : best;
                        const float old = ex2(top - ref);
                        top = best;
                        sum *= old, r.x *= old, r.y *= old, r.z *= old, r.w *= old;
#pragma unroll
                        for (int k = 0; k < 8; ++k) {
                            const float f = ex2(ml[k].x - ref);
                            sum = fmaf(ml[k].y, f, sum);
                            r.x = fmaf(x[k].x, f, r.x), r.y = fmaf(x[k].y, f, r.y);
                            r.z = fmaf(x[k].z, f, r.z), r.w = fmaf(x[k].w, f, r.w);
                        }
                    }
                    if (to == nullptr) {
                        if (row0 + col < rows)
                            write_out(out_row(now.seq, head, row0 + col), d, r, top, sum, d == 0);
                    } else {
                        // over the leader's own partial result, whose O this lane alone has
                        // read; m and l go elsewhere until every warp has read them
                        reinterpret_cast<float4*>(to)[nv * 32 + lane] = r;
                        if (d == 0)
                            *reinterpret_cast<float2*>(stat + 2 * col) = make_float2(top, sum);
                    }
                }
                if (to != nullptr) {
                    __syncthreads();
                    if (tid < 2 * S::kCols) to[16 * 128 + tid] = stat[tid];
                }
            };
            const int groups = (parts + kFan - 1) / kFan, mine_group = me / kFan;
            const int lead = mine_group * kFan, size = min(kFan, parts - lead);
            // Counters: a CTA can lead the first group of the segment it
            // begins and a later group of the segment it is inside of.
            if (arrive(p.counters + (mine_group == 0 ? 0 : kMaxGrid) + c0 + lead, size)) {
                if (groups == 1) {
                    add(0, 1, parts, nullptr);
                } else {
                    add(lead, 1, size, slot_of(lead));
                    if (arrive(p.counters + 2 * kMaxGrid + c0, groups))
                        add(0, kFan, groups, nullptr);
                }
            }
            __syncthreads();
        }
    }

    if (failed) {
        // Copies in flight must land before the CTA's shared memory is given up:
        // the units issued and not done are in the next stages of the ring.
        for (int i = 0; i < min(issued, mine) - done; ++i) {
            const int at_stage = (done + i) % kStages;
            mbar_wait_held(my_bars + 8 * at_stage, phase >> at_stage & 1u, kWaitTimeoutCycles);
        }
    }
}

// Blocks of all segments if every sequence were as long as its page table (or
// reached back as far as the window lets its rows see).
int64_t longest_line(const KvAttentionArgs& a, int64_t row_tiles) {
    int64_t blocks = a.fixed_length >= 0 ? (a.fixed_length + kKvBlock - 1) / kKvBlock
                                         : (int64_t)a.max_pages * (a.page_size / kKvBlock);
    if (a.window > 0)
        blocks = std::min(blocks, ((int64_t)a.window + a.new_tokens - 2) / kKvBlock + 2);
    return blocks * a.batch * a.kv_heads * row_tiles;
}

template <int kDim, int kBits, int kNB, bool kBf16>
cudaError_t run(Params& p, cudaStream_t stream) {
    using S = Shape<kDim, kBits, kNB>;
    const auto kernel = kv_attention_kernel<kDim, kBits, kNB, kBf16>;
    const KvAttentionArgs& a = p.a;
    const size_t fixed = S::kRingBytes + S::kRedBytes + S::kStatBytes +
                         kWarps * S::kStages * 8 + 16;
    const size_t smem = fixed + (3 * (size_t)a.batch + 2) * sizeof(int);
    const size_t smem_max = fixed + (3 * (size_t)kMaxBatch + 2) * sizeof(int);
    static std::atomic<int> resident[64];  // CTAs the device holds at once, 0: not asked yet
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    if (dev < 0 || dev >= 64) return cudaErrorInvalidDevice;
    int ctas = resident[dev].load(std::memory_order_acquire);
    if (ctas == 0) {
        if ((e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                      (int)smem_max)) != cudaSuccess)
            return e;
        int n = 0, sms = 0;
        if ((e = cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, kernel, kThreads,
                                                               fixed + 1028)) != cudaSuccess)
            return e;
        if ((e = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev)) != cudaSuccess)
            return e;
        ctas = std::min(std::max(1, n) * sms, kMaxGrid);
        resident[dev].store(ctas, std::memory_order_release);
    }
    p.row_tiles = FastDiv((a.new_tokens * a.group + S::kCols - 1) / S::kCols);
    const int64_t line = longest_line(a, p.row_tiles.d);
    // Never more CTAs than chunks of min_units in segments of the greatest length.
    const int64_t segments = (int64_t)a.batch * a.kv_heads * p.row_tiles.d;
    const int64_t unit_chunk = (int64_t)p.min_units * S::kU;  // blocks
    const int64_t per = std::max<int64_t>(1, (line / segments + unit_chunk - 1) / unit_chunk);
    const int64_t grid = std::min<int64_t>(ctas, segments * per);
    p.every_chunk = grid == segments * per;
    p.seg_chunks = FastDiv((uint32_t)per);
    p.min_chunk = FastDiv((uint32_t)p.min_units);
    // blocks of all segments below 2^21: every count that the plan divides is
    p.may_chunk = line < (int64_t)1 << 21;
    p.inv_grid = 1.f / (float)grid;
    return launch_pdl(kernel, dim3((unsigned)grid), dim3(kThreads), smem, stream, p);
}

// Rows of a tile: 16 where a head has more than 8 and the registers hold them.
int tile_rows(const KvAttentionArgs& a) {
    return a.head_dim < 256 && (int64_t)a.new_tokens * a.group > 8 ? 16 : 8;
}

template <int kDim, int kBits>
cudaError_t run_dim(Params& p, bool two, bool bf16, cudaStream_t s) {
    if constexpr (kDim < 256) {
        if (two)
            return bf16 ? run<kDim, kBits, 2, true>(p, s) : run<kDim, kBits, 2, false>(p, s);
    }
    return bf16 ? run<kDim, kBits, 1, true>(p, s) : run<kDim, kBits, 1, false>(p, s);
}

}  // namespace

size_t kv_attention_workspace() {
    return kCounterBytes + (size_t)kMaxGrid * 2 * kPartialFloats * sizeof(float);
}

bool kv_attention_fits(const KvAttentionArgs& a) {
    const int64_t rows = (int64_t)a.new_tokens * a.group;
    const int64_t per = a.page_size / kKvBlock;
    return longest_line(a, (rows + 7) / 8) +
                   (int64_t)kSegmentCost * a.batch * a.kv_heads * ((rows + 7) / 8) <
               ((int64_t)1 << 31) - ((int64_t)1 << 21) &&
           a.num_pages * a.kv_heads * per < ((int64_t)1 << 32) - 2;  // blocks are numbered
}

bool kv_attention_tiles_fit(const KvAttentionArgs& a) {
    const int64_t rows = (int64_t)a.new_tokens * a.group;
    const int tile = tile_rows(a);
    return (rows + tile - 1) / tile * a.kv_heads < kMostQuotient;
}

cudaError_t launch_kv_attention(const KvAttentionArgs& a, cudaStream_t stream) {
    if (a.batch == 0) return cudaSuccess;
    Params p{};
    p.a = a;
    p.counters = static_cast<int*>(a.workspace);
    p.partial = reinterpret_cast<float*>(static_cast<uint8_t*>(a.workspace) + kCounterBytes);
    p.page_blocks = FastDiv(a.page_size / kKvBlock);
    p.group = FastDiv(a.group);
    p.min_units = 2 * kWarps;
    p.q_vec = (reinterpret_cast<uintptr_t>(a.q) & 15u) == 0 && a.q_batch % 8 == 0 &&
              a.q_new % 8 == 0 && a.q_head % 8 == 0;
    p.wait_cycles = wait_budget();
    p.hold_ns = hold_within(p.wait_cycles);
    const bool two = tile_rows(a) == 16, bf16 = a.type == kTypeBf16;
    if (a.head_dim == 64)
        return a.bits == 8 ? run_dim<64, 8>(p, two, bf16, stream)
                           : run_dim<64, 4>(p, two, bf16, stream);
    if (a.head_dim == 128)
        return a.bits == 8 ? run_dim<128, 8>(p, two, bf16, stream)
                           : run_dim<128, 4>(p, two, bf16, stream);
    return a.bits == 8 ? run_dim<256, 8>(p, two, bf16, stream)
                       : run_dim<256, 4>(p, two, bf16, stream);
}

cudaError_t read_kv_attention_status(int clear, int* status) {
    return read_status_symbol(g_kv_attention_status, clear, status);
}

}  // namespace clb
