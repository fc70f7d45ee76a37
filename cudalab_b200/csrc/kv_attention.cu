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
// Softmax.  Each row keeps one reference m, the running maximum of s_j + log2
// vs_j (base 2): the V weights w_j = 2^(s_j + log2 vs_j - m) then lie in the
// range fp16 represents with full relative precision whatever the scales are,
// and the denominator sums w_j / vs_j in fp32 under the same reference.  m
// only moves when a score exceeds it by more than kSlack, so the usual block
// pays one vote instead of a reduction and a rescale.
//
// Split.  The 16-token blocks of all (sequence, head, row tile) segments form
// one line that is cut into equal ranges, one per CTA of a persistent grid, so
// ragged batches balance whatever their lengths; the four warps of a CTA take
// its blocks in turn.  Each warp has its own ring of block buffers filled by
// bulk copies (one per block) and never waits for another warp until a segment
// ends.  A segment cut over several CTAs leaves partial results in the
// workspace; the CTA that arrives last at a group's counter adds the group's
// partials in order (groups of kFan, then the groups), so the sum order, and
// with it every bit of the result, does not depend on timing.
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
constexpr int kMaxGrid = 148 * 8;
constexpr int kFan = 16;         // partial results added by one CTA
constexpr float kSlack = 8.f;    // weights stay below 2^8, far inside fp16
constexpr int kPartialFloats = 16 * 128 + 2 * 16;  // O, m and l of one partial result
constexpr size_t kCounterBytes = (size_t)kMaxGrid * 3 * sizeof(int);

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float lg2(float x) {
    float y;
    asm("lg2.approx.f32 %0, %1;" : "=f"(y) : "f"(x));
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

__device__ __forceinline__ uint32_t h2_add(uint32_t v, unsigned short bias) {
    const __half2 r = __hadd2(u32_as_h2(v), h2_const(bias));
    return *reinterpret_cast<const uint32_t*>(&r);
}

// Bytes 0 and 2 of w as a pair of halves (two's complement, exact); the pair
// 1 and 3 is the same of w >> 8.
__device__ __forceinline__ uint32_t bytes02(uint32_t w) {
    return h2_add(lop3_sel_xor_i<0x00FF00FFu, 0x64806480u>(w), kH_m1152);
}
// Nibbles 0 and 4, and 1 and 5, of w; 2, 6 and 3, 7 are the same of w >> 8.
__device__ __forceinline__ uint32_t nibbles04(uint32_t w) {
    return h2_add(lop3_sel_xor_i<0x000F000Fu, 0x64086408u>(w), kH_m1032);
}
__device__ __forceinline__ uint32_t nibbles15(uint32_t w) {
    return h2_add(lop3_sel_xor_i<0x00F000F0u, 0x54805480u>(w), kH_m72);
}

// kWords words of a row from shared memory, at byte offset `at` of its part:
// one 4-, 8- or 16-byte access.
template <int kWords>
__device__ __forceinline__ void lds_words(uint32_t addr, uint32_t* w) {
    if constexpr (kWords == 4) {
        const uint4 v = lds16(addr);
        w[0] = v.x, w[1] = v.y, w[2] = v.z, w[3] = v.w;
    } else if constexpr (kWords == 2) {
        asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(w[0]), "=r"(w[1]) : "r"(addr));
    } else {
        asm volatile("ld.shared.u32 %0, [%1];" : "=r"(w[0]) : "r"(addr));
    }
}
__device__ __forceinline__ float lds_half(uint32_t addr) {
    uint16_t v;
    asm volatile("ld.shared.u16 %0, [%1];" : "=h"(v) : "r"(addr));
    return __half2float(__ushort_as_half(v));
}

struct Params {
    KvAttentionArgs a;
    float* partial;
    int* counters;
    int row_tiles;       // of kCols rows each, per (sequence, head)
    int blocks_per_page;
    uint32_t page_magic; // ceil(2^32 / blocks_per_page)
    int min_blocks;      // smallest range of a CTA
    int q_vec;
    long long wait_cycles;
};

template <int kDim, int kBits, int kNB>
struct Shape {
    static constexpr int kRow = kDim * kBits / 8;
    static constexpr int kBlockBytes = kv_block_bytes(kRow);
    static constexpr int kCols = 8 * kNB;
    // Ring depth per warp: what keeps 16 KB or more in flight per warp slot of
    // an SM without taking the third CTA's shared memory.
    static constexpr int kStages = kBlockBytes <= 1088 ? 6 : kBlockBytes <= 2112 ? 5
                                   : kBlockBytes <= 4160 ? 3 : 2;
    static constexpr int kRingBytes = kWarps * kStages * kBlockBytes;
    static constexpr int kRedBytes = kWarps * 8 * kDim * 4;
    static constexpr int kStatBytes = kWarps * kCols * 2 * 4;
};

// The walk over the line of blocks: segment s covers [seg0, seg0 + blocks).
struct Cursor {
    int seq, unit;    // sequence; head * row_tiles + tile
    int seg0, blocks;
};

template <int kDim, int kBits, int kNB, bool kBf16>
__global__ void __launch_bounds__(kThreads, kDim == 256 ? 2 : 3)
    kv_attention_kernel(const Params p) {
    using S = Shape<kDim, kBits, kNB>;
    constexpr int kRow = S::kRow, kStages = S::kStages, kBlockBytes = S::kBlockBytes;
    constexpr int kSteps = kDim / 16;  // mma steps of q . k, and 16-row blocks of O^T
    extern __shared__ __align__(128) uint8_t smem[];
    uint8_t* ring = smem;
    float* red = reinterpret_cast<float*>(smem + S::kRingBytes);
    float* stat = reinterpret_cast<float*>(smem + S::kRingBytes + S::kRedBytes);
    uint64_t* bars = reinterpret_cast<uint64_t*>(smem + S::kRingBytes + S::kRedBytes + S::kStatBytes);
    int* flag = reinterpret_cast<int*>(bars + kWarps * kStages);
    int* s_len = flag + 4;                 // [batch]
    int* s_cum = s_len + p.a.batch;        // [batch + 1] blocks in front of a sequence

    const KvAttentionArgs& a = p.a;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int g = lane >> 2, t = lane & 3;
    const int units = a.kv_heads * p.row_tiles;
    const int rows = a.new_tokens * a.group;

    pdl_allow_dependents();
    const uint32_t my_ring = smem_u32(ring) + warp * kStages * kBlockBytes;
    const uint32_t my_bars = smem_u32(bars) + warp * kStages * 8;
    if (lane == 0) {
        for (int i = 0; i < kStages; ++i) mbar_init(my_bars + 8 * i, 1);
        fence_barrier_init();
    }
    pdl_wait_prior_grids();

    // Lengths, and the blocks of each sequence summed up.  A window drops the
    // blocks in front of the first token that any row sees.
    auto first_block = [&](int len) {
        if (a.window <= 0) return 0;
        const int first = len - a.new_tokens + 1 - a.window;
        return first > 0 ? first / kKvBlock : 0;
    };
    const int most = a.max_pages * a.page_size;
    {
        const int per = (a.batch + kThreads - 1) / kThreads, b0 = tid * per;
        int sum = 0;
        for (int b = b0; b < min(b0 + per, a.batch); ++b) {
            int len = a.fixed_length >= 0 ? a.fixed_length : a.lengths[b];
            if (len > most || len < 0) {
                if (blockIdx.x == 0) atomicCAS(&g_kv_attention_status, 0, kStatusKvIndex);
                len = len < 0 ? 0 : most;
            }
            s_len[b] = len;
            s_cum[b] = sum;  // of this thread's sequences, for now
            sum += (len + kKvBlock - 1) / kKvBlock - first_block(len);
        }
        int scan = sum;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int v = __shfl_up_sync(0xffffffffu, scan, o);
            if (lane >= o) scan += v;
        }
        int* tot = reinterpret_cast<int*>(red);
        if (lane == 31) tot[warp] = scan;
        __syncthreads();
        int before = scan - sum;
        for (int w = 0; w < warp; ++w) before += tot[w];
        for (int b = b0; b < min(b0 + per, a.batch); ++b) s_cum[b] += before;
        if (tid == kThreads - 1) s_cum[a.batch] = before + sum;
        __syncthreads();
    }
    const int total = s_cum[a.batch] * units;
    const int share = max(p.min_blocks, (total + (int)gridDim.x - 1) / (int)gridDim.x);
    const int u0 = min(total, (int)blockIdx.x * share), u1 = min(total, u0 + share);

    // Row `r` of a tile of sequence `seq`: where it is in q and in the outputs.
    auto out_row = [&](int seq, int head, int r) {
        return ((int64_t)seq * a.new_tokens + r / a.group) * (a.kv_heads * a.group) +
               head * a.group + r % a.group;
    };
    // One normalised output: 4 elements d.. of row `row`; `front` joins the
    // result over the tokens in front.
    auto write_out = [&](int64_t row, int d, float4 o, float m, float l, bool first) {
        float lse2 = l > 0.f ? m + lg2(l) : (l == l ? -INFINITY : l);
        const float inv = l > 0.f ? 1.f / l : (l == l ? 0.f : l);
        o.x *= inv, o.y *= inv, o.z *= inv, o.w *= inv;
        if (a.front != nullptr) {
            constexpr float kLog2e = 1.4426950408889634f;
            const float4 f = __ldcg(reinterpret_cast<const float4*>(a.front + row * kDim + d));
            const float fl = __ldcg(a.front_lse + row) * kLog2e;
            const float top = fmaxf(lse2, fl);
            const float ref = top == -INFINITY ? 0.f : top;
            const float wo = ex2(lse2 - ref), wf = ex2(fl - ref), sum = wo + wf;
            const float i2 = sum > 0.f ? 1.f / sum : (sum == sum ? 0.f : sum);
            o.x = (o.x * wo + f.x * wf) * i2;
            o.y = (o.y * wo + f.y * wf) * i2;
            o.z = (o.z * wo + f.z * wf) * i2;
            o.w = (o.w * wo + f.w * wf) * i2;
            lse2 = sum > 0.f ? ref + lg2(sum) : (sum == sum ? -INFINITY : sum);
        }
        if (a.out_f32 != nullptr)
            *reinterpret_cast<float4*>(a.out_f32 + row * kDim + d) = o;
        else
            *reinterpret_cast<uint2*>(static_cast<uint16_t*>(a.out) + row * kDim + d) =
                make_uint2(pack2<kBf16>(o.x, o.y), pack2<kBf16>(o.z, o.w));
        if (first && a.lse != nullptr) a.lse[row] = lse2 * 0.6931471805599453f;
    };

    // Sequences with nothing to read (their rows see no cached token).
    for (int b = blockIdx.x; b < a.batch; b += gridDim.x) {
        if (s_cum[b + 1] != s_cum[b]) continue;
        const int n = rows * a.kv_heads * (kDim / 4);
        for (int i = tid; i < n; i += kThreads) {
            const int d = i % (kDim / 4) * 4, r = i / (kDim / 4);
            write_out(out_row(b, r / rows, r % rows), d, make_float4(0.f, 0.f, 0.f, 0.f),
                      -INFINITY, 0.f, d == 0);
        }
    }
    if (u0 >= u1) return;

    // First segment of the range.
    Cursor start;
    {
        int lo = 0, hi = a.batch;  // last sequence whose blocks begin at or before u0
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (s_cum[mid] <= u0 / units) lo = mid; else hi = mid;
        }
        start.seq = lo;
        start.blocks = s_cum[lo + 1] - s_cum[lo];
        const int in = u0 - s_cum[lo] * units;
        start.unit = in / start.blocks;
        start.seg0 = s_cum[lo] * units + start.unit * start.blocks;
    }
    auto next_segment = [&](Cursor& c) {
        c.seg0 += c.blocks;
        if (++c.unit == units) {
            c.unit = 0;
            do ++c.seq; while (c.seq < a.batch && s_cum[c.seq + 1] == s_cum[c.seq]);
            if (c.seq < a.batch) c.blocks = s_cum[c.seq + 1] - s_cum[c.seq];
        }
    };

    // The warp's copies run kStages blocks ahead of its arithmetic.  The page
    // of a copy is loaded one step before the copy is issued.
    const uint64_t policy = policy_evict_first();
    const int64_t head_bytes = (int64_t)p.blocks_per_page * kBlockBytes;
    Cursor ic = start;   // segment of the next copy
    int iu = u0 + warp;  // its block
    int page = 0, sub = 0;
    auto load_page = [&]() {
        if (iu >= u1) return;
        while (iu >= ic.seg0 + ic.blocks) next_segment(ic);
        const int blk = iu - ic.seg0 + first_block(s_len[ic.seq]);
        const int n = (int)__umulhi((uint32_t)blk, p.page_magic);
        const int index = p.blocks_per_page == 1 ? blk : n;
        sub = blk - index * p.blocks_per_page;
        page = __ldg(a.table + ic.seq * a.table_stride + index);
    };
    uint32_t bad = 0;      // stages whose block has no valid page
    uint32_t pending = 0;  // stages with a copy that nothing has waited for
    auto issue = [&](int stage) {
        if (iu >= u1) return;
        const bool ok = page >= 0 && page < a.num_pages;
        bad = ok ? bad & ~(1u << stage) : bad | (1u << stage);
        pending |= (uint32_t)ok << stage;
        if (lane == 0) {
            if (ok) {
                const uint32_t bar = my_bars + 8 * stage;
                mbar_arrive_expect_tx(bar, kBlockBytes);
                const uint8_t* src = a.pages +
                                     ((int64_t)page * a.kv_heads + ic.unit / p.row_tiles) * head_bytes +
                                     (int64_t)sub * kBlockBytes;
                bulk_g2s(my_ring + stage * kBlockBytes, src, kBlockBytes, bar, policy);
            } else {
                atomicCAS(&g_kv_attention_status, 0, kStatusKvIndex);
            }
        }
        iu += kWarps;
    };
    load_page();
#pragma unroll 1
    for (int i = 0; i < kStages; ++i) {
        issue(i);
        load_page();
    }

    // Byte offsets of this lane's pieces inside a K part and a V part.
    constexpr int kKWords = kRow / 16, kKPer = kKWords < 4 ? kKWords : 4;
    constexpr int kVWords = kRow / 32, kVPer = kVWords < 4 ? kVWords : 4;
    auto k_byte = [&](int i) {  // i-th access of a quarter row
        return kRow == 256 ? (i >> 1) * 128 + 32 * t + 16 * (i & 1)
                           : kRow == 128 ? 32 * t + 16 * i : (kRow / 4) * t;
    };
    auto v_byte = [&](int i) { return kRow == 256 ? 128 * i + 16 * g : (kRow / 8) * g; };

    int stage = 0, phase = 0;
    bool failed = false;
    int cu = u0 + warp;
    Cursor seg = start;
    while (seg.seg0 < u1) {
        const int sa = max(seg.seg0, u0), sb = min(seg.seg0 + seg.blocks, u1);
        const int head = seg.unit / p.row_tiles, tile = seg.unit % p.row_tiles;
        const int len = s_len[seg.seq], row0 = tile * S::kCols;
        const int block0 = first_block(len) - seg.seg0;

        // q of this lane's rows g + 8 n as B fragments.  bf16 rows are brought
        // into fp16's range by a power of two (exact; elements 2^14 below
        // their row's largest lose bits that fp32 sums would not keep either).
        uint32_t qf[kNB][kSteps][2];
        float rs[kNB][2];
#pragma unroll
        for (int n = 0; n < kNB; ++n) {
            const int r = row0 + 8 * n + g;
            float x[kDim / 4];
#pragma unroll
            for (int i = 0; i < kDim / 4; ++i) x[i] = 0.f;
            if (r < rows) {
                const uint16_t* src = static_cast<const uint16_t*>(a.q) + seg.seq * a.q_batch +
                                      r / a.group * a.q_new +
                                      (head * a.group + r % a.group) * a.q_head;
                // piece i: the elements of access i, 16 bytes of q at a time
                constexpr int kAccess = kKPer * 32 / kBits;  // elements per access
#pragma unroll
                for (int i = 0; i < kKWords / kKPer; ++i) {
                    const int e0 = k_byte(i) * 8 / kBits;
#pragma unroll
                    for (int j = 0; j < kAccess; j += 8)
                        unpack8<kBf16>(p.q_vec ? load8<kBf16, true>(src, e0 + j)
                                               : load8<kBf16, false>(src, e0 + j),
                                       x + i * kAccess + j);
                }
            }
            float unit = a.scale * 1.4426950408889634f;
            if (kBf16) {
                float m = 0.f;
#pragma unroll
                for (int i = 0; i < kDim / 4; ++i) m = fmaxf(m, fabsf(x[i]));
                m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 1));
                m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 2));
                const int e = (int)(__float_as_uint(m) >> 23) - 127;
                // zero, denormal and non-finite rows stay as they are
                if (e > -126 && e < 127) {
                    const float down = __uint_as_float((uint32_t)(127 - e) << 23);
#pragma unroll
                    for (int i = 0; i < kDim / 4; ++i) x[i] *= down;
                    unit *= __uint_as_float((uint32_t)(127 + e) << 23);
                }
            }
            rs[n][0] = __shfl_sync(0xffffffffu, unit, 8 * t);
            rs[n][1] = __shfl_sync(0xffffffffu, unit, 8 * t + 4);
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
        // Tokens [lo, hi) that the rows 2t, 2t + 1 (+ 8 n) see.
        int hi[kNB][2], lo[kNB][2];
#pragma unroll
        for (int n = 0; n < kNB; ++n)
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                const int r = row0 + 8 * n + 2 * t + c;
                const int at = len - a.new_tokens + r / a.group + 1;
                hi[n][c] = a.causal ? min(at, len) : len;
                lo[n][c] = a.window > 0 ? at - a.window : 0;
            }
        const int all_hi = a.causal ? len - a.new_tokens + 1 : len;
        const int all_lo = a.window > 0 ? len - a.window : 0;

        float o[kSteps][kNB][4];
        float m[kNB][2], l[kNB][2];
#pragma unroll
        for (int n = 0; n < kNB; ++n) {
#pragma unroll
            for (int i = 0; i < kSteps; ++i) o[i][n][0] = o[i][n][1] = o[i][n][2] = o[i][n][3] = 0.f;
            m[n][0] = m[n][1] = -INFINITY;
            l[n][0] = l[n][1] = 0.f;
        }

#pragma unroll 1
        for (; cu < sb; cu += kWarps) {
            const bool have = !((bad >> stage) & 1u) && !failed;
            if (have && !mbar_wait_bounded(my_bars + 8 * stage, (uint32_t)phase >> stage & 1u,
                                           p.wait_cycles)) {
                if (lane == 0) atomicCAS(&g_kv_attention_status, 0, kStatusTimeoutKv);
                failed = true;
            }
            failed = __any_sync(0xffffffffu, failed);
            if (have && !failed) {
                phase ^= 1 << stage;
                pending &= ~(1u << stage);
                const uint32_t base = my_ring + stage * kBlockBytes;
                const int j0 = (cu + block0) * kKvBlock;
                float s[kNB][4];
#pragma unroll
                for (int n = 0; n < kNB; ++n) s[n][0] = s[n][1] = s[n][2] = s[n][3] = 0.f;
#pragma unroll
                for (int i = 0; i < kKWords / kKPer; ++i) {
                    uint32_t w0[kKPer], w1[kKPer];
                    lds_words<kKPer>(base + kv_offset<kRow>(g, k_byte(i)), w0);
                    lds_words<kKPer>(base + kv_offset<kRow>(g + 8, k_byte(i)), w1);
#pragma unroll
                    for (int w = 0; w < kKPer; ++w) {
                        const int x = i * kKPer + w;
                        if (kBits == 8) {
                            const uint32_t f[4] = {bytes02(w0[w]), bytes02(w1[w]),
                                                   bytes02(w0[w] >> 8), bytes02(w1[w] >> 8)};
#pragma unroll
                            for (int n = 0; n < kNB; ++n) mma_16816(s[n], f, qf[n][x][0], qf[n][x][1]);
                        } else {
                            const uint32_t e[4] = {nibbles04(w0[w]), nibbles04(w1[w]),
                                                   nibbles15(w0[w]), nibbles15(w1[w])};
                            const uint32_t h0 = w0[w] >> 8, h1 = w1[w] >> 8;
                            const uint32_t f[4] = {nibbles04(h0), nibbles04(h1), nibbles15(h0),
                                                   nibbles15(h1)};
#pragma unroll
                            for (int n = 0; n < kNB; ++n) {
                                mma_16816(s[n], e, qf[n][2 * x][0], qf[n][2 * x][1]);
                                mma_16816(s[n], f, qf[n][2 * x + 1][0], qf[n][2 * x + 1][1]);
                            }
                        }
                    }
                }
                // Scores of tokens j0 + g (0, 1) and j0 + g + 8 (2, 3).
                const uint32_t scales = base + 2 * kKvBlock * kRow + 2 * g;
                const float ks0 = lds_half(scales), ks1 = lds_half(scales + 16);
                // V scales; a zero scale has all-zero values, any weight will do
                const float lv0 = fmaxf(lg2(lds_half(scales + 32)), -24.f);
                const float lv1 = fmaxf(lg2(lds_half(scales + 48)), -24.f);
                bool over = false;
#pragma unroll
                for (int n = 0; n < kNB; ++n) {
                    s[n][0] = fmaf(s[n][0] * ks0, rs[n][0], lv0);
                    s[n][1] = fmaf(s[n][1] * ks0, rs[n][1], lv0);
                    s[n][2] = fmaf(s[n][2] * ks1, rs[n][0], lv1);
                    s[n][3] = fmaf(s[n][3] * ks1, rs[n][1], lv1);
                }
                if (j0 + kKvBlock > all_hi || j0 < all_lo) {
#pragma unroll
                    for (int n = 0; n < kNB; ++n)
#pragma unroll
                        for (int c = 0; c < 4; ++c) {
                            const int j = j0 + g + 8 * (c >> 1);
                            if (j >= hi[n][c & 1] || j < lo[n][c & 1]) s[n][c] = -INFINITY;
                        }
                }
#pragma unroll
                for (int n = 0; n < kNB; ++n) {
                    over |= fmaxf(s[n][0], s[n][2]) > m[n][0] + kSlack;
                    over |= fmaxf(s[n][1], s[n][3]) > m[n][1] + kSlack;
                }
                if (__any_sync(0xffffffffu, over)) {
#pragma unroll
                    for (int n = 0; n < kNB; ++n)
#pragma unroll
                        for (int c = 0; c < 2; ++c) {
                            float top = fmaxf(s[n][c], s[n][c + 2]);
#pragma unroll
                            for (int x = 4; x < 32; x <<= 1)
                                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, x));
                            top = fmaxf(top, m[n][c]);
                            // a row that has seen nothing keeps -inf and zeros
                            const float f = top == -INFINITY ? 1.f : ex2(m[n][c] - top);
                            m[n][c] = top;
                            l[n][c] *= f;
#pragma unroll
                            for (int i = 0; i < kSteps; ++i) {
                                o[i][n][c] *= f;
                                o[i][n][c + 2] *= f;
                            }
                        }
                }
                const float iv0 = ex2(-lv0), iv1 = ex2(-lv1);
                uint32_t pf[kNB][2];
#pragma unroll
                for (int n = 0; n < kNB; ++n) {
                    const float r0 = m[n][0] == -INFINITY ? 0.f : m[n][0];
                    const float r1 = m[n][1] == -INFINITY ? 0.f : m[n][1];
                    const float w0 = ex2(s[n][0] - r0), w1 = ex2(s[n][1] - r1);
                    const float w2 = ex2(s[n][2] - r0), w3 = ex2(s[n][3] - r1);
                    // masked tokens may hold any scale: 0 * inf must not reach the sum
                    l[n][0] += (s[n][0] == -INFINITY ? 0.f : w0 * iv0) +
                               (s[n][2] == -INFINITY ? 0.f : w2 * iv1);
                    l[n][1] += (s[n][1] == -INFINITY ? 0.f : w1 * iv0) +
                               (s[n][3] == -INFINITY ? 0.f : w3 * iv1);
                    pf[n][0] = transpose8x8(pack2<false>(w0, w1));
                    pf[n][1] = transpose8x8(pack2<false>(w2, w3));
                }
                // O^T += V^T P^T: tokens 2t, 2t + 1, 2t + 8, 2t + 9.
                const uint32_t vb = base + kKvBlock * kRow;
#pragma unroll
                for (int i = 0; i < kVWords / kVPer; ++i) {
                    uint32_t w[4][kVPer];
#pragma unroll
                    for (int x = 0; x < 4; ++x)
                        lds_words<kVPer>(
                            vb + kv_offset<kRow>(2 * t + (x & 1) + 8 * (x >> 1), v_byte(i)), w[x]);
#pragma unroll
                    for (int y = 0; y < kVPer; ++y)
#pragma unroll
                        for (int h = 0; h < 2; ++h) {  // low and high half of the words
                            const uint32_t c0 = h ? prmt_i<0x7632u>(w[0][y], w[1][y])
                                                  : prmt_i<0x5410u>(w[0][y], w[1][y]);
                            const uint32_t c1 = h ? prmt_i<0x7632u>(w[2][y], w[3][y])
                                                  : prmt_i<0x5410u>(w[2][y], w[3][y]);
                            const int x = 2 * (i * kVPer + y) + h;
                            if (kBits == 8) {
                                const uint32_t f[4] = {bytes02(c0), bytes02(c0 >> 8), bytes02(c1),
                                                       bytes02(c1 >> 8)};
#pragma unroll
                                for (int n = 0; n < kNB; ++n) mma_16816(o[x][n], f, pf[n][0], pf[n][1]);
                            } else {
                                const uint32_t d0 = c0 >> 8, d1 = c1 >> 8;
                                const uint32_t e[4] = {nibbles04(c0), nibbles15(c0), nibbles04(c1),
                                                       nibbles15(c1)};
                                const uint32_t f[4] = {nibbles04(d0), nibbles15(d0), nibbles04(d1),
                                                       nibbles15(d1)};
#pragma unroll
                                for (int n = 0; n < kNB; ++n) {
                                    mma_16816(o[2 * x][n], e, pf[n][0], pf[n][1]);
                                    mma_16816(o[2 * x + 1][n], f, pf[n][0], pf[n][1]);
                                }
                            }
                        }
                }
            }
            __syncwarp();  // every lane has read the stage before it is filled again
            if (!failed) {
                issue(stage);
                load_page();
            }
            stage = stage + 1 == kStages ? 0 : stage + 1;
        }

        // ---- the segment's end: the warps' results meet in shared memory ----
#pragma unroll
        for (int n = 0; n < kNB; ++n)
#pragma unroll
            for (int c = 0; c < 2; ++c) {
#pragma unroll
                for (int x = 4; x < 32; x <<= 1) l[n][c] += __shfl_xor_sync(0xffffffffu, l[n][c], x);
                if (g == 0) {
                    const int col = 8 * n + 2 * t + c;
                    stat[(warp * S::kCols + col) * 2] = m[n][c];
                    stat[(warp * S::kCols + col) * 2 + 1] = l[n][c];
                }
            }
        const bool whole = sa == seg.seg0 && sb == seg.seg0 + seg.blocks;
        float* slot = p.partial + ((int64_t)blockIdx.x * 2 + (seg.seg0 >= u0)) * kPartialFloats;
#pragma unroll
        for (int n = 0; n < kNB; ++n) {
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                float* dst = red + (warp * 8 + 2 * t + c) * kDim;
                // element of (block i, half h): contiguous in the lane's eighth of the row
#pragma unroll
                for (int i = 0; i < kSteps; i += 2) {
                    const int d = kRow == 256 ? (i / 8) * 128 + 16 * g + 2 * (i % 8)
                                              : (kDim / 8) * g + 2 * i;
                    *reinterpret_cast<float4*>(dst + d) = make_float4(
                        o[i][n][c], o[i][n][c + 2], o[i + 1][n][c], o[i + 1][n][c + 2]);
                }
            }
            __syncthreads();
            for (int i = tid; i < 8 * (kDim / 4); i += kThreads) {
                const int d = i % (kDim / 4) * 4, rr = i / (kDim / 4), col = 8 * n + rr;
                float top = -INFINITY, sum = 0.f;
#pragma unroll
                for (int w = 0; w < kWarps; ++w)
                    top = fmaxf(top, stat[(w * S::kCols + col) * 2]);
                float4 r = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
                for (int w = 0; w < kWarps; ++w) {
                    const float mw = stat[(w * S::kCols + col) * 2];
                    // a warp that saw nothing has zeros here (or the NaN of its q)
                    const float f = mw == -INFINITY ? 0.f : ex2(mw - top);
                    const float4 v = *reinterpret_cast<const float4*>(red + (w * 8 + rr) * kDim + d);
                    sum += f * stat[(w * S::kCols + col) * 2 + 1];
                    r.x += f * v.x, r.y += f * v.y, r.z += f * v.z, r.w += f * v.w;
                }
                if (whole) {
                    if (row0 + col < rows)
                        write_out(out_row(seg.seq, head, row0 + col), d, r, top, sum, d == 0);
                } else {
                    *reinterpret_cast<float4*>(slot + col * kDim + d) = r;
                    if (d == 0) {
                        slot[16 * 128 + 2 * col] = top;
                        slot[16 * 128 + 2 * col + 1] = sum;
                    }
                }
            }
            __syncthreads();
        }

        if (!whole) {
            // Adds `count` partial results at base, base + stride, ... in order.
            const int c0 = seg.seg0 / share, c1 = (seg.seg0 + seg.blocks - 1) / share;
            const int n = c1 - c0 + 1, me = (int)blockIdx.x - c0;
            auto slot_of = [&](int i) {  // of the segment's i-th CTA
                return p.partial + ((int64_t)(c0 + i) * 2 + (i == 0)) * kPartialFloats;
            };
            auto arrive = [&](int* counter, int count) {
                __threadfence();
                __syncthreads();
                if (tid == 0) {
                    const int old = atomicAdd(counter, 1);
                    *flag = old == count - 1;
                    if (old == count - 1) *counter = 0;  // ready for the next launch
                }
                __syncthreads();
                const bool last = *flag != 0;
                __threadfence();
                __syncthreads();
                return last;
            };
            auto add = [&](int first, int step, int count, float* to) {
#pragma unroll 1
                for (int i = tid; i < S::kCols * (kDim / 4); i += kThreads) {
                    const int d = i % (kDim / 4) * 4, col = i / (kDim / 4);
                    float top = -INFINITY, sum = 0.f;
                    float4 r = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 8
                    for (int k = 0; k < count; ++k) {
                        const float* src = slot_of(first + k * step);
                        const float4 v = __ldcg(reinterpret_cast<const float4*>(src + col * kDim + d));
                        const float2 ml = __ldcg(reinterpret_cast<const float2*>(src + 16 * 128 + 2 * col));
                        const float nt = fmaxf(top, ml.x);
                        const float ref = nt == -INFINITY ? 0.f : nt;
                        const float fo = ex2(top - ref), fn = ex2(ml.x - ref);
                        sum = sum * fo + ml.y * fn;
                        r.x = r.x * fo + v.x * fn, r.y = r.y * fo + v.y * fn;
                        r.z = r.z * fo + v.z * fn, r.w = r.w * fo + v.w * fn;
                        top = nt;
                    }
                    if (to == nullptr) {
                        if (row0 + col < rows)
                            write_out(out_row(seg.seq, head, row0 + col), d, r, top, sum, d == 0);
                    } else {
                        // the leader's own place, read by nobody else in this group
                        *reinterpret_cast<float4*>(to + col * kDim + d) = r;
                        if (d == 0) red[2 * col] = top, red[2 * col + 1] = sum;
                    }
                }
                if (to != nullptr) {
                    __syncthreads();
                    if (tid < 2 * S::kCols) to[16 * 128 + tid] = red[tid];
                }
            };
            const int groups = (n + kFan - 1) / kFan, mine = me / kFan;
            const int lead = mine * kFan, size = min(kFan, n - lead);
            // Counters: a CTA can lead the first group of the segment it
            // begins and a later group of the segment it is inside of.
            int* first = p.counters + (mine == 0 ? 0 : kMaxGrid) + c0 + lead;
            if (arrive(first, size)) {
                if (groups == 1) {
                    add(0, 1, n, nullptr);
                } else {
                    add(lead, 1, size, slot_of(lead));
                    if (arrive(p.counters + 2 * kMaxGrid + c0, groups))
                        add(0, kFan, groups, nullptr);
                }
            }
            __syncthreads();
        }
        next_segment(seg);
        if (seg.seq >= a.batch) break;
    }

    if (failed) {
        // Copies in flight must land before the CTA's shared memory is given up.
        for (int i = 0; i < kStages; ++i)
            if ((pending >> i) & 1u)
                mbar_wait_bounded(my_bars + 8 * i, (uint32_t)phase >> i & 1u, p.wait_cycles);
    }
}

// Blocks of all segments if every sequence were as long as its page table.
int64_t longest_line(const KvAttentionArgs& a, int64_t row_tiles) {
    const int64_t blocks = a.fixed_length >= 0
                               ? (a.fixed_length + kKvBlock - 1) / kKvBlock
                               : (int64_t)a.max_pages * (a.page_size / kKvBlock);
    return blocks * a.batch * a.kv_heads * row_tiles;
}

template <int kDim, int kBits, int kNB, bool kBf16>
cudaError_t run(Params& p, cudaStream_t stream) {
    using S = Shape<kDim, kBits, kNB>;
    const auto kernel = kv_attention_kernel<kDim, kBits, kNB, kBf16>;
    const KvAttentionArgs& a = p.a;
    const size_t fixed = S::kRingBytes + S::kRedBytes + S::kStatBytes +
                         kWarps * S::kStages * 8 + 16;
    const size_t smem = fixed + (2 * (size_t)a.batch + 1) * sizeof(int);
    const size_t smem_max = fixed + (2 * (size_t)kMaxBatch + 1) * sizeof(int);
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
    p.row_tiles = (a.new_tokens * a.group + S::kCols - 1) / S::kCols;
    const int64_t line = longest_line(a, p.row_tiles);
    const int64_t grid = std::min<int64_t>(ctas, std::max<int64_t>(line / p.min_blocks + 1, a.batch));
    return launch_pdl(kernel, dim3((unsigned)grid), dim3(kThreads), smem, stream, p);
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
    // the page division by multiplication is exact below 2^32 / blocks_per_page
    const int64_t per = a.page_size / kKvBlock;
    return longest_line(a, (rows + 7) / 8) < ((int64_t)1 << 31) - ((int64_t)1 << 21) &&
           (int64_t)a.max_pages * per * per < (int64_t)1 << 32;
}

cudaError_t launch_kv_attention(const KvAttentionArgs& a, cudaStream_t stream) {
    if (a.batch == 0) return cudaSuccess;
    Params p{};
    p.a = a;
    p.counters = static_cast<int*>(a.workspace);
    p.partial = reinterpret_cast<float*>(static_cast<uint8_t*>(a.workspace) + kCounterBytes);
    p.blocks_per_page = a.page_size / kKvBlock;
    p.page_magic = (uint32_t)((((uint64_t)1 << 32) + p.blocks_per_page - 1) / p.blocks_per_page);
    p.min_blocks = kWarps;
    p.q_vec = (reinterpret_cast<uintptr_t>(a.q) & 15u) == 0 && a.q_batch % 8 == 0 &&
              a.q_new % 8 == 0 && a.q_head % 8 == 0;
    p.wait_cycles = wait_budget();
    const bool two = a.new_tokens * a.group > 8, bf16 = a.type == kTypeBf16;
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
