// Attention over a 4-bit cache (kv4.cuh): single tokens and portions of prompts, any head size that is a multiple of 32 up
// to 256, any grouping of query heads, bfloat16 or 32-bit rows.
//
// For request r with q_len new tokens and kv_len tokens in the cache, query i sits at position p = kv_len - q_len + i and
// sees the keys at positions j <= p with j > p - window (window == 0: all) or j < first.  Rows of a kv head are its queries'
// heads, position by position: row = i * group + (head within the group).
//
// A block takes 8 or 16 rows of a kv head (NT eights) as the columns of its products and walks the chunks of 32 tokens (two tiles)
// that any of them sees, dealt to its four warps.  Either `splits` blocks, a cluster, share out a row tile's chunks and join
// over their shared memory, or (SPREAD) each of as many blocks as fit takes an equal stretch of all row tiles' chunks and a second
// kernel joins what was cut.  Both products have the cache as
// their left operand, so that a code is unpacked once for all rows and a lane's share of a tile is what it needs and
// nothing else:
//     S^T [tokens x rows]  = K Q^T        one accumulator per group of 32 dims, which times its scale is added to the scores
//     O^T [dims x rows]   += V^T (P s)^T  the scale of a token's group goes into its probability, rounded once to bfloat16
// The probabilities leave the first product with tokens down the lanes and enter the second with tokens across them: an
// 8 x 8 transposition of bfloat16 (movmatrix) per eight tokens, rows and group.
// A code becomes a number by masking it into the mantissa of a power of two.  Keys, as float16: of a word's four nibbles to a half
// two need no shift (1024 + c and 1024 + 16 c, whose row takes a sixteenth of its dim), and what is too much is taken off the
// accumulator's start, a sum over the row's dims.  So an accumulator holds up to 1,039 times the sum of the row's magnitudes in a group
// on its way to a product that may be much less, and each of a dozen additions may lose about 2^-24 of that.  (A choice of speed, and less than
// the worst by far: with scores of up to 1,400, large parts of them common to all keys, results were no further from 64 bits than
// the rounding of the result.)  Rows are scaled by a power of two for it, their largest dim to [16, 32).  Values, as bfloat16 (a probability times a scale
// has no bounds): 128 + c, and 136 times the sum of a chunk's weights (a product with ones) is taken off the sums after each
// chunk of 32 tokens, before it could add up over all of them.
// 32-bit rows: queries and probabilities are sums of three bfloat16 (24 bits), and 136 is subtracted from codes before the
// products; codes are exact in one, so three products do.
//
// A tile of a kv head is one contiguous piece of 18 hd bytes: one bulk copy, issued by one lane into the warp's own ring.
// Nothing but a warp's own barriers orders that ring; warps and blocks meet once, at the end of a row tile.
//
// Measured: 64 requests of 1,000 - 8,100 tokens, 32 / 8 heads of 128, 93 us, 3.6 TB/s of codes and scales, 55 % of what a copy
// reaches; one request of 131,072 tokens 44 us, 3.4 TB/s.  There DRAM is at 45 %, half of the issue slots and of the integer pipe are
// used, and the 12 warps that registers let an SM hold wait for their own instructions most, 320 a tile.  The loads alone, without the
// products, take 73 - 81 us of the 93 (two copies of 2,304 bytes a chunk, whatever the ring's depth).  Portions of few rows are bound by
// the same instructions, which unpack a code again for each row tile: 40 tokens behind 30,000, 125 us, DRAM at 3 %, the tensor cores
// at 37 %.  32-bit rows cost three products for one.
#pragma once

#define LSB_CLUSTER_ALONG_X            // splits are the fastest part of blockIdx.x
#include "copy_ring.h"
#include "kv4.cuh"

#include <cuda_fp16.h>

#include <type_traits>

LSB_DEFINE_STATUS()

typedef __nv_bfloat16 bf16;

constexpr int kWarps = 4;
constexpr int kThreads = 32 * kWarps;
constexpr int kMaxSpread = 256;        // row tiles (of one kv head, of all requests) whose chunks are spread evenly over a grid's blocks
constexpr int kMaxSplits = 8;         // blocks of a cluster of portable size
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kRescale = 8.f;        // a row's reference maximum moves when a score exceeds it by this (log2)
constexpr uint32_t kSpinLimit = 1u << 22;

struct Kv4Params {
    const void* qkv;                   // q of token t, head h at qkv + t * qkv_stride + h * hd
    int qkv_stride;
    const unsigned char* pages;
    const int *q_start, *kv_len, *table_rows, *block_table;
    int table_stride;
    void* out;                         // [tokens, nh * hd]
    int nh, nkv, tiles_per_page, num_pages;
    float scale;
    int window, first;
    int mode;                          // which requests: 1: those that bring one token; 2: the others
    int splits;
    float* parts;                      // spread: what blocks have of rows that others have a part of, two slots a block
    int n_requests, row_tiles;         // spread: all of them; of each request
};

// ------------------------------------------------------------------ PTX helpers
__device__ __forceinline__ uint32_t smem_u32(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void bar_init(uint64_t* bar) {
    asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" ::"r"(smem_u32(bar)));
}
__device__ __forceinline__ void bar_expect(uint64_t* bar, uint32_t bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(smem_u32(bar)), "r"(bytes) : "memory");
}
__device__ __forceinline__ void bulk_load(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
                 ::"r"(smem_u32(dst)), "l"(src), "r"(bytes), "r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ bool bar_ready(uint64_t* bar, uint32_t parity) {
    uint32_t ok;
    asm volatile("{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}"
                 : "=r"(ok) : "r"(smem_u32(bar)), "r"(parity) : "memory");
    return ok != 0;
}
// (bounded; false if the wait ran out)
__device__ __forceinline__ bool bar_wait(uint64_t* bar, uint32_t parity) {
    for (uint32_t it = 0; it < kSpinLimit; ++it) {
        if (bar_ready(bar, parity)) return true;
        if ((it & 255u) == 255u) __nanosleep(128);
    }
    return false;
}
// D = A B + C on float16, 32-bit sums
__device__ __forceinline__ void mma_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1,
                                        float c0, float c1, float c2, float c3) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%12,%13};"
                 : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(c0), "f"(c1), "f"(c2), "f"(c3));
}
// ... on bfloat16
__device__ __forceinline__ void mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1,
                                    float c0, float c1, float c2, float c3) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%12,%13};"
                 : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(c0), "f"(c1), "f"(c2), "f"(c3));
}
__device__ __forceinline__ uint32_t transposed(uint32_t a) {
    uint32_t r;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(a));
    return r;
}
__device__ __forceinline__ float fast_exp2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// nibbles 0 and 4 of x as two bfloat16 of 128 + nibble
__device__ __forceinline__ uint32_t raised(uint32_t x) {
    uint32_t r;
    asm("lop3.b32 %0, %1, 0x000f000f, 0x43004300, 0xea;" : "=r"(r) : "r"(x));
    return r;
}
// nibbles 0 and 4 of x as two float16 of 1024 + nibble; nibbles 1 and 5 of 1024 + 16 nibble
__device__ __forceinline__ uint32_t raised_low(uint32_t x) {
    uint32_t r;
    asm("lop3.b32 %0, %1, 0x000f000f, 0x64006400, 0xea;" : "=r"(r) : "r"(x));
    return r;
}
__device__ __forceinline__ uint32_t raised_high(uint32_t x) {
    uint32_t r;
    asm("lop3.b32 %0, %1, 0x00f000f0, 0x64006400, 0xea;" : "=r"(r) : "r"(x));
    return r;
}
// (of two bfloat16 of 128 + nibble) less 136: exact
__device__ __forceinline__ uint32_t lowered(uint32_t x) {
    uint32_t r;
    asm("sub.rn.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(x), "r"(0x43084308u));
    return r;
}
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
}
__device__ __forceinline__ uint32_t pack2_f16(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
__device__ __forceinline__ float low_f16(uint32_t v) { return __half2float(__ushort_as_half((unsigned short)(v & 0xffffu))); }
__device__ __forceinline__ float high_f16(uint32_t v) { return __half2float(__ushort_as_half((unsigned short)(v >> 16))); }
__device__ __forceinline__ float max3(float a, float b, float c) {
    float r;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}
__device__ __forceinline__ float low_half(uint32_t v) { return __uint_as_float(v << 16); }
__device__ __forceinline__ float high_half(uint32_t v) { return __uint_as_float(v & 0xffff0000u); }

// N consecutive 16-bit pieces at p (aligned to the largest power of two that divides 2 N, at most 16), two to a word.
template <int N>
__device__ __forceinline__ void load_halves(const unsigned char* p, uint32_t (&w)[(N + 1) / 2]) {
    if constexpr (N % 8 == 0) {
#pragma unroll
        for (int i = 0; i < N / 8; ++i) {
            const uint4 v = reinterpret_cast<const uint4*>(p)[i];
            w[4 * i] = v.x; w[4 * i + 1] = v.y; w[4 * i + 2] = v.z; w[4 * i + 3] = v.w;
        }
    } else if constexpr (N % 4 == 0) {
#pragma unroll
        for (int i = 0; i < N / 4; ++i) {
            const uint2 v = reinterpret_cast<const uint2*>(p)[i];
            w[2 * i] = v.x; w[2 * i + 1] = v.y;
        }
    } else if constexpr (N % 2 == 0) {
#pragma unroll
        for (int i = 0; i < N / 2; ++i) w[i] = reinterpret_cast<const uint32_t*>(p)[i];
    } else {
        const unsigned short* h = reinterpret_cast<const unsigned short*>(p);
#pragma unroll
        for (int i = 0; i < N / 2; ++i) w[i] = h[2 * i] | (uint32_t)h[2 * i + 1] << 16;
        w[N / 2] = h[N - 1];
    }
}

__device__ __forceinline__ void cluster_barrier() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ uint32_t peer_address(const void* own, uint32_t rank) {
    uint32_t peer;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(peer) : "r"(smem_u32(own)), "r"(rank));
    return peer;
}
__device__ __forceinline__ float peer_f32(const float* own, uint32_t rank) {
    float v;
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(peer_address(own, rank)) : "memory");
    return v;
}
__device__ __forceinline__ float4 peer_f32x4(const float4* own, uint32_t rank) {
    float4 v;
    asm volatile("ld.shared::cluster.v4.f32 {%0,%1,%2,%3}, [%4];"
                 : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(peer_address(own, rank)) : "memory");
    return v;
}

template <typename T> __device__ __forceinline__ void store_four(T* to, float4 v);
template <> __device__ __forceinline__ void store_four<float>(float* to, float4 v) { *reinterpret_cast<float4*>(to) = v; }
template <> __device__ __forceinline__ void store_four<bf16>(bf16* to, float4 v) {
    *reinterpret_cast<uint2*>(to) = make_uint2(pack2(v.x, v.y), pack2(v.z, v.w));
}

template <typename T> __device__ __forceinline__ void store_two(T* to, float a, float b);
template <> __device__ __forceinline__ void store_two<float>(float* to, float a, float b) { *reinterpret_cast<float2*>(to) = make_float2(a, b); }
template <> __device__ __forceinline__ void store_two<bf16>(bf16* to, float a, float b) { *reinterpret_cast<uint32_t*>(to) = pack2(a, b); }

// ------------------------------------------------------------------ the kernel
// G: groups of 32 dims of a head; NT: eights of rows of a block; T: type of the rows.
template <int G, int NT, typename T>
struct Kv4Shape {
    static constexpr int kHd = kKv4Group * G;
    static constexpr int kCols = 8 * NT;
    static constexpr int kParts = std::is_same<T, float>::value ? 3 : 1;
    static constexpr int kTile = kv4_tile_bytes(kHd);
    static constexpr int kChunk = 2 * kTile;                           // what a warp takes at a time
    static constexpr int kStages = G <= 2 ? 4 : 2;
    static constexpr int kRing = kWarps * kStages * kChunk;
    static constexpr int kO = kCols * kHd * 4;                         // one O
    static constexpr int kSums = kWarps / 2 * kO;                      // half of the warps' (the block's is the first of them)
    static constexpr int kQ = kParts * kCols * kHd * 2;
    static constexpr size_t kBytes = kRing + kSums + kQ;
    static constexpr int kBlocks = NT == 1 && G <= 4 && kParts == 1 ? (G == 4 ? 3 : 4) : 2;    // that an SM holds
    static constexpr int kSlot = kCols * (kHd + 2);                    // floats of a part: maxima, sums, O
};

// Chunks of 32 tokens that a row at `pos` sees of its request: tiles of first tokens in front of the window's, and those from
// `near` on.
struct Kv4Span {
    int near, early, tiles, chunks;
    __device__ __forceinline__ Kv4Span(int p_lo, int p_hi, int W, int F) {
        near = (W > 0 && p_lo - W + 1 > 0 ? p_lo - W + 1 : 0) / kKv4Tile;
        early = min((F + kKv4Tile - 1) / kKv4Tile, near);
        tiles = early + p_hi / kKv4Tile + 1 - near;
        chunks = (tiles + 1) / 2;
    }
};

// SPREAD.  The chunks of all row tiles of all requests are one list, and for each kv head as many blocks as fit take an equal stretch
// of it: whatever the lengths, all blocks end at once.  Neighbouring blocks walk the same tokens of neighbouring heads, whose
// tiles lie side by side in a page: the pieces of 18 hd bytes that memory is asked for at one time add up to whole pages.  A row
// tile that a block has from its first chunk to its last is written out by it; of others it leaves maxima, sums and O in its
// slots (one for what it begins with in the middle, one for what it ends with), which spread_merge_kernel joins.
struct Spread {
    int blocks;                                                        // for each kv head, no stretch empty (unless there is nothing to do)
    int total;
    // ends[e]: chunks of the row tiles 0 .. e, of which each request has p.row_tiles; filled by all threads of a block
    __device__ __forceinline__ Spread(const Kv4Params& p, int cols, int grid, int* ends, int* warp_sums) {
        const int tid = threadIdx.x, W = p.window, F = W > 0 ? p.first : 0, group = p.nh / p.nkv, entries = p.n_requests * p.row_tiles;
        int n[kMaxSpread / 32 / 4], sum = 0;                           // (blocks of at least 128 threads)
        const int each = kMaxSpread / (int)blockDim.x;
#pragma unroll
        for (int i = 0; i < kMaxSpread / 32 / 4; ++i) {
            if (i >= each) break;
            const int e = tid * each + i, r = e / p.row_tiles, row0 = (e - r * p.row_tiles) * cols;
            n[i] = 0;
            if (e < entries) {
                const int q_len = p.q_start[r + 1] - p.q_start[r], rows = q_len * group, base = p.kv_len[r] - q_len;
                if ((q_len == 1) == (p.mode == 1) && row0 < rows)
                    n[i] = Kv4Span(base + row0 / group, base + (min(row0 + cols, rows) - 1) / group, W, F).chunks;
            }
            sum += n[i];
        }
        int upto = sum;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int v = __shfl_up_sync(0xffffffffu, upto, o);
            if ((tid & 31) >= o) upto += v;
        }
        if ((tid & 31) == 31) warp_sums[tid >> 5] = upto;
        __syncthreads();
        for (int w = 0; w < tid >> 5; ++w) upto += warp_sums[w];
        upto -= sum;
#pragma unroll
        for (int i = 0; i < kMaxSpread / 32 / 4; ++i) {
            if (i >= each) break;
            ends[tid * each + i] = upto += n[i];
        }
        __syncthreads();
        total = ends[kMaxSpread - 1];
        // (a chunk for each warp of a block is the least that is worth joining)
        blocks = max(1, min(min(grid / p.nkv, total), max(entries, total / kWarps)));
    }
    __device__ __forceinline__ int bound(int block) const { return (int)((long long)block * total / blocks); }
};

template <int G, int NT, typename T, bool SPREAD>
__global__ void __launch_bounds__(kThreads, Kv4Shape<G, NT, T>::kBlocks) attention_kv4_kernel(const Kv4Params p) {
    using Z = Kv4Shape<G, NT, T>;
    constexpr int HD = Z::kHd, COLS = Z::kCols, PARTS = Z::kParts, ST = Z::kStages, TILE = Z::kTile;
    constexpr bool EXACT = PARTS == 3;
    extern __shared__ __align__(128) unsigned char smem[];
    float* sums = reinterpret_cast<float*>(smem + Z::kRing);
    unsigned short* sq = reinterpret_cast<unsigned short*>(smem + Z::kRing + Z::kSums);        // [PARTS][COLS][HD]
    __shared__ uint64_t bars[kWarps][ST];
    __shared__ float2 wml[kWarps / 2][NT][32][2];                      // half of the warps' maxima and sums
    __shared__ float bm[COLS], bl[COLS];                               // the block's
    __shared__ float factor[SPREAD ? 1 : kMaxSplits][COLS], inverse[COLS];
    __shared__ float unit[COLS];                                       // what a row was divided by
    __shared__ int ends[SPREAD ? kMaxSpread : 1], warp_sums[kWarps];

    lsb_pdl_launch_dependents();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, e8 = lane >> 2, t4 = lane & 3;
    const int W = p.window, F = W > 0 ? p.first : 0, group = p.nh / p.nkv;
    for (int i = tid; i < kWarps * ST; i += kThreads) bar_init(&bars[i / ST][i % ST]);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    // the step's metadata is on the device before the step's first kernel starts
    const int splits = SPREAD ? 1 : p.splits, split = SPREAD ? 0 : (int)(blockIdx.x % splits);
    int r = blockIdx.z, h = blockIdx.y, rt = 0, q_len = 0;
    int at = 0, end = 1;                                               // spread: the block's stretch of the list
    if constexpr (SPREAD) {
        const Spread list(p, COLS, gridDim.x, ends, warp_sums);
        const int part = (int)blockIdx.x / p.nkv;
        if (part >= list.blocks) return;
        h = (int)blockIdx.x - part * p.nkv;
        at = list.bound(part);
        end = list.bound(part + 1);
    } else {
        q_len = p.q_start[r + 1] - p.q_start[r];
        // (late rows see the most keys, and start first; all blocks of a cluster leave here alike)
        rt = (q_len * group + COLS - 1) / COLS - 1 - (int)(blockIdx.x / splits);
        if (rt < 0 || (q_len == 1) != (p.mode == 1)) return;
    }
    lsb_pdl_wait();
    __syncthreads();
    CopyRing<ST> turn{0};                                              // of the warp's own ring

  for (; at < end;) {
    int c0, c1;                                                        // the block's chunks of this row tile, of `span.chunks`
    if constexpr (SPREAD) {
        int lo = 0, hi = p.n_requests * p.row_tiles - 1;               // the first row tile whose chunks end behind `at`
        while (lo < hi) {
            const int mid = (lo + hi) >> 1;
            if (ends[mid] > at) hi = mid; else lo = mid + 1;
        }
        const int before = lo > 0 ? ends[lo - 1] : 0;
        c0 = at - before;
        c1 = min(ends[lo] - before, c0 + (end - at));
        r = lo / p.row_tiles;
        rt = lo - r * p.row_tiles;
        q_len = p.q_start[r + 1] - p.q_start[r];
    }
    const int qs = p.q_start[r], n_rows = q_len * group;
    const int row0 = rt * COLS, row1 = min(row0 + COLS, n_rows);
    const int base = p.kv_len[r] - q_len;                              // position of the request's first new token
    const int p_lo = base + row0 / group, p_hi = base + (row1 - 1) / group;
    const Kv4Span span(p_lo, p_hi, W, F);
    const int near = span.near, early = span.early, n_tiles = span.tiles;
    if constexpr (!SPREAD) {
        const int per = (span.chunks + splits - 1) / splits;
        c0 = min(split * per, span.chunks);
        c1 = min(c0 + per, span.chunks);
    }
    const int n_mine = (c1 - c0 - warp + kWarps - 1) / kWarps;         // chunks c0 + warp, c0 + warp + kWarps, ... (0 or less: none)

    const int* table = p.block_table + (size_t)p.table_rows[r] * p.table_stride;
    unsigned char* ring = smem + warp * ST * Z::kChunk;
    auto first_key = [&](int c) { return (c < early ? c : c - early + near) * kKv4Tile; };     // of the c-th tile of the block's list
    // Places in the pool of the tiles of 16 of the warp's chunks, one a lane.  A chunk's second tile may be missing (its first stands
    // in for it, and its keys count as too late).  A page that is none of the pool's is recorded, and the pool's first stands in.
    auto places = [&](int k) -> int {
        const int c = 2 * (c0 + warp + kWarps * (k + (lane >> 1))) + (lane & 1);
        if (k + (lane >> 1) >= n_mine) return 0;
        const int i = min(c, n_tiles - 1), tile = i < early ? i : i - early + near, pi = tile / p.tiles_per_page;
        const int page = pi < p.table_stride ? __ldcg(table + pi) : -1;
        if (page < 0 || page >= p.num_pages) {
            lsb_set_status(LSB_BAD_PAGE);
            return 0;
        }
        return (page * p.nkv + h) * p.tiles_per_page + tile % p.tiles_per_page;
    };
    int known = places(0);
    auto issue = [&](int k) {
        if (k >= n_mine) return;
        if (k > 0 && k % 16 == 0) known = places(k);
        const int place = __shfl_sync(0xffffffffu, known, 2 * (k % 16) + (lane & 1)), s = turn.stage(k);
        if (lane == 0) bar_expect(&bars[warp][s], Z::kChunk);
        if (lane < 2) bulk_load(ring + s * Z::kChunk + lane * TILE, p.pages + (size_t)place * TILE, TILE, &bars[warp][s]);
    };
#pragma unroll
    for (int k = 0; k < ST - 1; ++k) issue(k);

    // The block's rows of queries, a warp to a row; rows beyond the last are zeros.
    const T* qkv = reinterpret_cast<const T*>(p.qkv);
    for (int c = warp; c < COLS; c += kWarps) {
        const int row = row0 + c;
        const T* from = qkv + (size_t)(qs + row / group) * p.qkv_stride + (h * group + row % group) * HD;
        float x[G], top = 0.f;
#pragma unroll
        for (int g = 0; g < G; ++g) {
            x[g] = row < row1 ? lsb_to_float(from[g * 32 + lane]) : 0.f;
            top = fmaxf(top, fabsf(x[g]));
        }
        if constexpr (EXACT) {
#pragma unroll
            for (int g = 0; g < G; ++g)
#pragma unroll
                for (int part = 0; part < PARTS; ++part) {
                    const bf16 y = __float2bfloat16_rn(x[g]);
                    sq[(part * COLS + c) * HD + g * 32 + lane] = __bfloat16_as_ushort(y);
                    x[g] -= __bfloat162float(y);
                }
        } else {
            top = lsb_warp_max(top);
            // 2^n to divide by, the largest dim then in [16, 32); rows of zeros, of numbers that are none or too small for it stay
            float by = __uint_as_float((__float_as_uint(top) & 0x7f800000u)) * 0.0625f;
            if (!(by >= 1e-36f && by <= 1e37f)) by = 1.f;
            const float inv = 1.f / by;                                // (exact)
#pragma unroll
            for (int g = 0; g < G; ++g)                                // odd dims meet 16 times their codes
                sq[c * HD + g * 32 + lane] = __half_as_ushort(__float2half_rn(x[g] * ((lane & 1) ? inv * 0.0625f : inv)));
            if (lane == 0) unit[c] = by;
        }
    }
    __syncthreads();
    // Right operand of S^T: dims 32 g + 8 t + {0, 4}, {1, 5}, {2, 6}, {3, 7} of row e, as a key's nibbles unpack.
    uint32_t q[NT][PARTS][G][4];
    float start[NT][G][2];                                             // what codes that are too large add to the products of rows 2 t, 2 t + 1
    float sc[NT][2];                                                   // from a row's products to log2 of its weights
#pragma unroll
    for (int n = 0; n < NT; ++n) {
#pragma unroll
        for (int g = 0; g < G; ++g) {
            float sum = 0.f;
#pragma unroll
            for (int part = 0; part < PARTS; ++part) {
                const uint4 v = *reinterpret_cast<const uint4*>(sq + (part * COLS + n * 8 + e8) * HD + g * 32 + t4 * 8);
                const uint32_t w[4] = {v.x, v.y, v.z, v.w};
                q[n][part][g][0] = __byte_perm(w[0], w[2], 0x5410);
                q[n][part][g][1] = __byte_perm(w[0], w[2], 0x7632);
                q[n][part][g][2] = __byte_perm(w[1], w[3], 0x5410);
                q[n][part][g][3] = __byte_perm(w[1], w[3], 0x7632);
                if constexpr (!EXACT) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) sum += -1032.f * low_f16(w[i]) - 1152.f * high_f16(w[i]);      // 1024 + 8, 1024 + 16 * 8
                }
            }
            if constexpr (!EXACT) {
                sum += __shfl_xor_sync(0xffffffffu, sum, 1);
                sum += __shfl_xor_sync(0xffffffffu, sum, 2);
                start[n][g][0] = __shfl_sync(0xffffffffu, sum, 8 * t4);
                start[n][g][1] = __shfl_sync(0xffffffffu, sum, 8 * t4 + 4);
            } else {
                start[n][g][0] = start[n][g][1] = 0.f;
            }
        }
#pragma unroll
        for (int b = 0; b < 2; ++b) sc[n][b] = p.scale * kLog2e * (EXACT ? 1.f : unit[n * 8 + 2 * t4 + b]);
    }

    float o[NT][2 * G][4];
    float m[NT][2], l[NT][2];                                          // reference maxima (log2) and sums; -inf: nothing seen
#pragma unroll
    for (int n = 0; n < NT; ++n) {
        m[n][0] = m[n][1] = -INFINITY;
        l[n][0] = l[n][1] = 0.f;
#pragma unroll
        for (int i = 0; i < 2 * G; ++i) o[n][i][0] = o[n][i][1] = o[n][i][2] = o[n][i][3] = 0.f;
    }
    // One chunk; `masked`: some of its keys may be hidden from some rows.
    auto take = [&](auto masked, const unsigned char* chunk, int c) {
        constexpr bool MASKED = decltype(masked)::value;

        // ---------------------------------------------------------- products of queries and keys
        float s[2][NT][4];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const unsigned char* tile = chunk + u * TILE;
            uint32_t ka[G], kb[G], sa[(G + 1) / 2], sb[(G + 1) / 2];
            load_halves<2 * G>(tile + e8 * (HD / 2) + t4 * 4 * G, ka);
            load_halves<2 * G>(tile + (e8 + 8) * (HD / 2) + t4 * 4 * G, kb);
            load_halves<G>(tile + kv4_key_scales_at(HD) + e8 * 2 * G, sa);
            load_halves<G>(tile + kv4_key_scales_at(HD) + (e8 + 8) * 2 * G, sb);
#pragma unroll
            for (int g = 0; g < G; ++g) {
                uint32_t a[4], b[4];
                if constexpr (EXACT) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        a[i] = lowered(raised(ka[g] >> (4 * i)));
                        b[i] = lowered(raised(kb[g] >> (4 * i)));
                    }
                } else {
                    a[0] = raised_low(ka[g]); a[1] = raised_high(ka[g]);
                    b[0] = raised_low(kb[g]); b[1] = raised_high(kb[g]);
                    a[2] = raised_low(ka[g] >> 8); a[3] = raised_high(ka[g] >> 8);
                    b[2] = raised_low(kb[g] >> 8); b[3] = raised_high(kb[g] >> 8);
                }
                const float fa = g % 2 ? high_half(sa[g / 2]) : low_half(sa[g / 2]);
                const float fb = g % 2 ? high_half(sb[g / 2]) : low_half(sb[g / 2]);
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    float d[4];
                    if constexpr (EXACT) {
                        mma(d, a[0], b[0], a[1], b[1], q[n][0][g][0], q[n][0][g][1], 0.f, 0.f, 0.f, 0.f);
                        mma(d, a[2], b[2], a[3], b[3], q[n][0][g][2], q[n][0][g][3], d[0], d[1], d[2], d[3]);
#pragma unroll
                        for (int part = 1; part < PARTS; ++part) {
                            mma(d, a[0], b[0], a[1], b[1], q[n][part][g][0], q[n][part][g][1], d[0], d[1], d[2], d[3]);
                            mma(d, a[2], b[2], a[3], b[3], q[n][part][g][2], q[n][part][g][3], d[0], d[1], d[2], d[3]);
                        }
                    } else {
                        mma_f16(d, a[0], b[0], a[1], b[1], q[n][0][g][0], q[n][0][g][1], start[n][g][0], start[n][g][1], start[n][g][0], start[n][g][1]);
                        mma_f16(d, a[2], b[2], a[3], b[3], q[n][0][g][2], q[n][0][g][3], d[0], d[1], d[2], d[3]);
                    }
                    if (g == 0) {
                        s[u][n][0] = fa * d[0]; s[u][n][1] = fa * d[1]; s[u][n][2] = fb * d[2]; s[u][n][3] = fb * d[3];
                    } else {
                        s[u][n][0] = fmaf(fa, d[0], s[u][n][0]);
                        s[u][n][1] = fmaf(fa, d[1], s[u][n][1]);
                        s[u][n][2] = fmaf(fb, d[2], s[u][n][2]);
                        s[u][n][3] = fmaf(fb, d[3], s[u][n][3]);
                    }
                }
            }
        }
        // ---------------------------------------------------------- which of them count
        uint32_t seen = 0xffffffffu;                                   // bit 16 u + 4 n + i: element i of s[u][n]
        if constexpr (MASKED) {
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int b = 0; b < 2; ++b) {
                    const int pos = base + min(row0 + n * 8 + 2 * t4 + b, row1 - 1) / group;
#pragma unroll
                    for (int u = 0; u < 2; ++u)
#pragma unroll
                        for (int i = b; i < 4; i += 2) {
                            const int key = first_key(c + u) + e8 + (i >> 1) * 8;
                            if (!(key <= pos && (W <= 0 || key > pos - W || key < F))) seen &= ~(1u << (16 * u + 4 * n + i));
                        }
                }
        }
        // ---------------------------------------------------------- weights; the references move seldom
        float x[2][NT][4], top = -INFINITY;
        auto weigh = [&]() {
#pragma unroll
            for (int u = 0; u < 2; ++u)
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int i = 0; i < 4; ++i) x[u][n][i] = fmaf(s[u][n][i], sc[n][i & 1], -m[n][i & 1]);
            if constexpr (MASKED) {
#pragma unroll
                for (int u = 0; u < 2; ++u)
#pragma unroll
                    for (int n = 0; n < NT; ++n)
#pragma unroll
                        for (int i = 0; i < 4; ++i) x[u][n][i] = seen >> (16 * u + 4 * n + i) & 1u ? x[u][n][i] : -INFINITY;
            }
        };
        weigh();                                                       // (with a reference of -inf: +inf)
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int n = 0; n < NT; ++n) top = max3(max3(x[u][n][0], x[u][n][1], x[u][n][2]), x[u][n][3], top);
        if (__any_sync(0xffffffffu, top > kRescale)) {
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                float corr[2];
#pragma unroll
                for (int b = 0; b < 2; ++b) {
                    float most = -INFINITY;
#pragma unroll
                    for (int u = 0; u < 2; ++u)
#pragma unroll
                        for (int i = b; i < 4; i += 2)
                            if (!MASKED || (seen >> (16 * u + 4 * n + i) & 1u)) most = fmaxf(most, s[u][n][i] * sc[n][b]);
#pragma unroll
                    for (int y = 4; y < 32; y <<= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, y));
                    most = fmaxf(most, m[n][b]);
                    corr[b] = m[n][b] == -INFINITY ? 1.f : fast_exp2(m[n][b] - most);      // (before the first reference all is zero, or no number)
                    m[n][b] = most;
                    l[n][b] *= corr[b];
                }
#pragma unroll
                for (int i = 0; i < 2 * G; ++i) {
                    o[n][i][0] *= corr[0];
                    o[n][i][1] *= corr[1];
                    o[n][i][2] *= corr[0];
                    o[n][i][3] *= corr[1];
                }
            }
            weigh();
        }
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    x[u][n][i] = fast_exp2(x[u][n][i]);
                    l[n][i & 1] += x[u][n][i];
                }
        // ---------------------------------------------------------- values
        uint32_t va[2][(G + 1) / 2], vb[2][(G + 1) / 2], v[2][4][(G + 1) / 2];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const unsigned char* tile = chunk + u * TILE;
            load_halves<G>(tile + kv4_value_scales_at(HD) + e8 * 2 * G, va[u]);
            load_halves<G>(tile + kv4_value_scales_at(HD) + (e8 + 8) * 2 * G, vb[u]);
#pragma unroll
            for (int i = 0; i < 4; ++i)                                // tokens 2 t, 2 t + 1, 2 t + 8, 2 t + 9
                load_halves<G>(tile + kv4_values_at(HD) + (2 * t4 + (i & 1) + (i >> 1) * 8) * (HD / 2) + e8 * 2 * G, v[u][i]);
        }
#pragma unroll
        for (int g = 0; g < G; ++g) {
            [[maybe_unused]] float total[NT][4];                       // of the chunk's P s, of rows 2 t and 2 t + 1
            // (32-bit rows: the tensor cores cut their sums off rather than round them, so a chunk's are formed by themselves)
            [[maybe_unused]] float fresh[NT][2][4];
            if constexpr (EXACT) {
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int i = 0; i < 8; ++i) fresh[n][i >> 2][i & 3] = 0.f;
            }
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const float fa = g % 2 ? high_half(va[u][g / 2]) : low_half(va[u][g / 2]);
                const float fb = g % 2 ? high_half(vb[u][g / 2]) : low_half(vb[u][g / 2]);
                uint32_t b[NT][PARTS][2];
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    float y[4] = {x[u][n][0] * fa, x[u][n][1] * fa, x[u][n][2] * fb, x[u][n][3] * fb};
                    if constexpr (MASKED) {                            // (a scale that is no number stays out of rows that do not see it)
#pragma unroll
                        for (int i = 0; i < 4; ++i) y[i] = seen >> (16 * u + 4 * n + i) & 1u ? y[i] : 0.f;
                    }
#pragma unroll
                    for (int part = 0; part < PARTS; ++part) {
                        const uint32_t y0 = pack2(y[0], y[1]), y1 = pack2(y[2], y[3]);
                        b[n][part][0] = transposed(y0);
                        b[n][part][1] = transposed(y1);
                        if (part + 1 < PARTS) {
                            y[0] -= low_half(y0); y[1] -= high_half(y0);
                            y[2] -= low_half(y1); y[3] -= high_half(y1);
                        }
                    }
                    if constexpr (!EXACT) {
                        constexpr uint32_t kOnes = 0x3f803f80u;
                        if (u == 0) mma(total[n], kOnes, kOnes, kOnes, kOnes, b[n][0][0], b[n][0][1], 0.f, 0.f, 0.f, 0.f);
                        else mma(total[n], kOnes, kOnes, kOnes, kOnes, b[n][0][0], b[n][0][1], total[n][0], total[n][1], total[n][2], total[n][3]);
                    }
                }
#pragma unroll
                for (int i = 2 * g; i < 2 * g + 2; ++i) {
                    // byte i of the rows of two tokens, side by side: dims 16 i + 2 e (low nibbles) and + 1 (high ones)
                    constexpr uint32_t kPick[4] = {0x4400, 0x5511, 0x6622, 0x7733};
                    const uint32_t y = __byte_perm(v[u][0][i / 4], v[u][1][i / 4], kPick[i % 4]);
                    const uint32_t z = __byte_perm(v[u][2][i / 4], v[u][3][i / 4], kPick[i % 4]);
                    uint32_t a0 = raised(y), a1 = raised(y >> 4), a2 = raised(z), a3 = raised(z >> 4);
                    if constexpr (EXACT) { a0 = lowered(a0); a1 = lowered(a1); a2 = lowered(a2); a3 = lowered(a3); }
#pragma unroll
                    for (int n = 0; n < NT; ++n) {
                        float(&to)[4] = EXACT ? fresh[n][i - 2 * g] : o[n][i];
#pragma unroll
                        for (int part = 0; part < PARTS; ++part)
                            mma(to, a0, a1, a2, a3, b[n][part][0], b[n][part][1], to[0], to[1], to[2], to[3]);
                    }
                }
            }
            if constexpr (EXACT) {
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int i = 0; i < 8; ++i) o[n][2 * g + (i >> 2)][i & 3] += fresh[n][i >> 2][i & 3];
            } else {
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int i = 2 * g; i < 2 * g + 2; ++i) {
                        o[n][i][0] = fmaf(-136.f, total[n][0], o[n][i][0]);
                        o[n][i][1] = fmaf(-136.f, total[n][1], o[n][i][1]);
                        o[n][i][2] = fmaf(-136.f, total[n][0], o[n][i][2]);
                        o[n][i][3] = fmaf(-136.f, total[n][1], o[n][i][3]);
                    }
            }
        }
    };

    // The warp's chunks [k_lo, k_hi) hold two tiles, behind the first tokens', that all of the block's rows see whole.
    const int first_c = max(early, (W > 0 && p_hi - W >= 0 ? (p_hi - W) / kKv4Tile + 1 - near + early : 0));
    const int last_c = (p_lo + 1) / kKv4Tile - near + early;           // one past
    const int k_lo = max(0, ((first_c + 1) / 2 - c0 - warp + kWarps - 1) / kWarps);
    const int k_hi = last_c / 2 - c0 - warp <= 0 ? 0 : (last_c / 2 - c0 - warp + kWarps - 1) / kWarps;
    bool late = false;
    int k = 0;
#pragma unroll 1
    for (; k < n_mine; ++k) {
        issue(k + ST - 1);
        const int stage = turn.stage(k);
        uint64_t* bar = &bars[warp][stage];
        const uint32_t parity = turn.parity(k);
        if (__any_sync(0xffffffffu, !bar_ready(bar, parity))) {
            late = __any_sync(0xffffffffu, !bar_wait(bar, parity));
            if (late) break;
        }
        // (tiles 2 c and 2 c + 1 of the row tile's list; a missing second one is past every row)
        if (k >= k_lo && k < k_hi) take(std::false_type{}, ring + stage * Z::kChunk, 0);
        else take(std::true_type{}, ring + stage * Z::kChunk, 2 * (c0 + warp + kWarps * k));
        __syncwarp();                                                  // the stage may be written over
    }
    if (late) {
        // chunk k's copy did not arrive: it and those behind it that are under way are waited for (with the same limit) before shared
        // memory goes
        lsb_set_status(LSB_WAIT_TIMEOUT);
        for (int i = k; i < turn.issued(k, n_mine); ++i) bar_wait(&bars[warp][turn.stage(i)], turn.parity(i));
    }
    turn.used += max(n_mine, 0);

    // ------------------------------------------------------------------ the warps' sums: half of them hand theirs to the others
#pragma unroll
    for (int half = kWarps / 2; half > 0; half >>= 1) {
        if (warp >= half && warp < 2 * half) {
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                wml[warp - half][n][lane][0] = make_float2(m[n][0], l[n][0]);
                wml[warp - half][n][lane][1] = make_float2(m[n][1], l[n][1]);
#pragma unroll
                for (int i = 0; i < 2 * G; ++i)
                    reinterpret_cast<float4*>(sums)[(((warp - half) * NT + n) * 2 * G + i) * 32 + lane] =
                        make_float4(o[n][i][0], o[n][i][1], o[n][i][2], o[n][i][3]);
            }
        }
        __syncthreads();
        if (warp < half) {
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                float mine[2], theirs[2];
#pragma unroll
                for (int b = 0; b < 2; ++b) {
                    const float2 other = wml[warp][n][lane][b];
                    const float top = fmaxf(m[n][b], other.x), ref = top == -INFINITY ? 0.f : top;
                    // (a side that has seen nothing is all zeros, or no number)
                    mine[b] = m[n][b] == -INFINITY ? 1.f : fast_exp2(m[n][b] - ref);
                    theirs[b] = other.x == -INFINITY ? 1.f : fast_exp2(other.x - ref);
                    l[n][b] = l[n][b] * mine[b] + other.y * theirs[b];
                    m[n][b] = top;
                }
#pragma unroll
                for (int i = 0; i < 2 * G; ++i) {
                    const float4 x = reinterpret_cast<const float4*>(sums)[((warp * NT + n) * 2 * G + i) * 32 + lane];
                    o[n][i][0] = fmaf(x.x, theirs[0], o[n][i][0] * mine[0]);
                    o[n][i][1] = fmaf(x.y, theirs[1], o[n][i][1] * mine[1]);
                    o[n][i][2] = fmaf(x.z, theirs[0], o[n][i][2] * mine[0]);
                    o[n][i][3] = fmaf(x.w, theirs[1], o[n][i][3] * mine[1]);
                }
            }
        }
        __syncthreads();
    }
    T* out = reinterpret_cast<T*>(p.out);
    const bool complete = SPREAD ? c0 == 0 && c1 == span.chunks : splits == 1;
    if (warp == 0) {
        float* slot = nullptr;
        if constexpr (SPREAD) slot = p.parts + (size_t)(2 * blockIdx.x + (c0 == 0 ? 1 : 0)) * Z::kSlot;
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int b = 0; b < 2; ++b) {
                const int c = n * 8 + 2 * t4 + b, row = row0 + c;
                float sum = l[n][b];
#pragma unroll
                for (int x = 4; x < 32; x <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, x);
                if (complete) {
                    const float f = sum == 0.f ? 0.f : 1.f / sum;
                    if (row < row1) {
                        T* to = out + (size_t)(qs + row / group) * p.nh * HD + (h * group + row % group) * HD + 2 * e8;
#pragma unroll
                        for (int i = 0; i < 2 * G; ++i) store_two<T>(to + 16 * i, o[n][i][b] * f, o[n][i][2 + b] * f);
                    }
                } else {
                    float* to = SPREAD ? slot + 2 * COLS + c * HD : sums + c * HD;
                    if (e8 == 0) {
                        if constexpr (SPREAD) { slot[c] = m[n][b]; slot[COLS + c] = sum; }
                        else { bm[c] = m[n][b]; bl[c] = sum; }
                    }
#pragma unroll
                    for (int i = 0; i < 2 * G; ++i)
                        *reinterpret_cast<float2*>(to + 16 * i + 2 * e8) = make_float2(o[n][i][b], o[n][i][2 + b]);
                }
            }
    }
    if constexpr (SPREAD) {
        at += c1 - c0;
        if (late) return;
        continue;
    }
    if (complete) return;
    // ------------------------------------------------------------------ the blocks' sums
    constexpr int UNITS = COLS * HD / 4;
    cluster_barrier();
    if (tid < COLS) {
        float top = -INFINITY, sum = 0.f;
        for (int b = 0; b < splits; ++b) top = fmaxf(top, peer_f32(&bm[tid], b));
        for (int b = 0; b < splits; ++b) {
            const float theirs = peer_f32(&bm[tid], b);
            const float f = theirs == -INFINITY ? 1.f : fast_exp2(theirs - top);
            factor[SPREAD ? 0 : b][tid] = f;
            sum += peer_f32(&bl[tid], b) * f;
        }
        inverse[tid] = sum == 0.f ? 0.f : 1.f / sum;
    }
    __syncthreads();
    for (int u = split * kThreads + tid; u < UNITS; u += splits * kThreads) {
        const int c = u / (HD / 4), row = row0 + c;
        float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
        for (int b = 0; b < splits; ++b) {
            const float f = factor[SPREAD ? 0 : b][c];
            const float4 x = peer_f32x4(reinterpret_cast<const float4*>(sums) + u, b);
            v.x = fmaf(f, x.x, v.x); v.y = fmaf(f, x.y, v.y); v.z = fmaf(f, x.z, v.z); v.w = fmaf(f, x.w, v.w);
        }
        const float f = inverse[c];
        if (row < row1)
            store_four<T>(out + (size_t)(qs + row / group) * p.nh * HD + (h * group + row % group) * HD + (u - c * (HD / 4)) * 4,
                          make_float4(v.x * f, v.y * f, v.z * f, v.w * f));
    }
    cluster_barrier();                                                 // nobody leaves while others read its sums
    return;
  }
}

// Joins what several blocks have of one row, a block of threads for each; rows that one block had all of are done already.
template <int G, int NT, typename T>
__global__ void __launch_bounds__(128) spread_merge_kernel(const Kv4Params p, int grid) {
    using Z = Kv4Shape<G, NT, T>;
    constexpr int HD = Z::kHd, COLS = Z::kCols, UNITS = HD / 4, TEAMS = 128 / UNITS;     // fours of dims; teams that share out the parts
    __shared__ int ends[kMaxSpread], warp_sums[4];
    __shared__ float4 team_o[TEAMS][UNITS];
    __shared__ float team_m[4], team_l[4];
    lsb_pdl_launch_dependents();
    const Spread list(p, COLS, grid, ends, warp_sums);
    // (Blocks without work leave at once, but one waits: this kernel must not end before the one whose results the next reads.)
    if (blockIdx.x == 0 && blockIdx.y == 0) lsb_pdl_wait();
    const int h = blockIdx.x / COLS, c = blockIdx.x % COLS, entry = blockIdx.y, tid = threadIdx.x;
    const int before = entry > 0 ? ends[entry - 1] : 0, each = ends[entry] - before;
    const int r = entry / p.row_tiles, qs = p.q_start[r], group = p.nh / p.nkv;
    const int row = (entry - r * p.row_tiles) * COLS + c;
    if (each == 0 || row >= (p.q_start[r + 1] - qs) * group) return;   // (not of this launch; a column without a row)
    auto block_of = [&](int x) {                                       // whose stretch holds x
        int b = (int)((long long)x * list.blocks / list.total);
        while (b + 1 < list.blocks && list.bound(b + 1) <= x) ++b;
        while (b > 0 && list.bound(b) > x) --b;
        return b;
    };
    const int b0 = block_of(before), n = block_of(before + each - 1) - b0 + 1;
    if (n == 1) return;
    lsb_pdl_wait();
    auto slot_of = [&](int i) { return p.parts + (size_t)(2 * ((b0 + i) * p.nkv + h) + (i == 0 ? 1 : 0)) * Z::kSlot; };
    float top = -INFINITY;
    for (int i = tid; i < n; i += 128) top = fmaxf(top, slot_of(i)[c]);
    top = lsb_warp_max(top);
    if ((tid & 31) == 0) team_m[tid >> 5] = top;
    __syncthreads();
    top = fmaxf(fmaxf(team_m[0], team_m[1]), fmaxf(team_m[2], team_m[3]));
    const float ref = top == -INFINITY ? 0.f : top;
    float sum = 0.f;
    for (int i = tid; i < n; i += 128) {
        const float m = slot_of(i)[c];
        sum += slot_of(i)[COLS + c] * (m == -INFINITY ? 1.f : fast_exp2(m - ref));
    }
    sum = lsb_warp_sum(sum);
    if ((tid & 31) == 0) team_l[tid >> 5] = sum;
    const int team = tid / UNITS, u = tid - team * UNITS;
    if (team < TEAMS) {
        float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
        for (int i = team; i < n; i += TEAMS) {
            const float* slot = slot_of(i);
            const float m = slot[c], f = m == -INFINITY ? 1.f : fast_exp2(m - ref);
            const float4 x = *reinterpret_cast<const float4*>(slot + 2 * COLS + c * HD + 4 * u);
            v.x = fmaf(f, x.x, v.x); v.y = fmaf(f, x.y, v.y); v.z = fmaf(f, x.z, v.z); v.w = fmaf(f, x.w, v.w);
        }
        team_o[team][u] = v;
    }
    __syncthreads();
    if (tid < UNITS) {
        float4 v = team_o[0][tid];
#pragma unroll
        for (int i = 1; i < TEAMS; ++i) {
            const float4 x = team_o[i][tid];
            v.x += x.x; v.y += x.y; v.z += x.z; v.w += x.w;
        }
        sum = team_l[0] + team_l[1] + team_l[2] + team_l[3];
        const float f = sum == 0.f ? 0.f : 1.f / sum;
        store_four<T>(reinterpret_cast<T*>(p.out) + (size_t)(qs + row / group) * p.nh * HD + (size_t)(h * group + row % group) * HD + 4 * tid,
                      make_float4(v.x * f, v.y * f, v.z * f, v.w * f));
    }
}

// ------------------------------------------------------------------ host side
// What a kernel needs before its first launch on a device.
template <int G, int NT, typename T, bool SPREAD>
static int kv4_configure() {
    static bool done[64] = {};
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return (int)e;
    if (dev >= 0 && dev < 64 && done[dev]) return 0;
    auto k = attention_kv4_kernel<G, NT, T, SPREAD>;
    e = cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)Kv4Shape<G, NT, T>::kBytes);
    if (e == cudaSuccess && dev >= 0 && dev < 64) done[dev] = true;
    return (int)e;
}

struct Kv4Launch {
    const Kv4Params& p;
    dim3 grid;
    cudaStream_t stream;
    template <int G, int NT, typename T> int run() const {
        if (const int rc = kv4_configure<G, NT, T, false>()) return rc;
        return lsb_launch(attention_kv4_kernel<G, NT, T, false>, grid, dim3(kThreads), Kv4Shape<G, NT, T>::kBytes, stream, p.splits, p);
    }
};

struct Kv4SpreadLaunch {
    const Kv4Params& p;
    int blocks;
    cudaStream_t stream;
    template <int G, int NT, typename T> int run() const {
        if (const int rc = kv4_configure<G, NT, T, true>()) return rc;
        if (const int rc = lsb_launch(attention_kv4_kernel<G, NT, T, true>, dim3(blocks), dim3(kThreads), Kv4Shape<G, NT, T>::kBytes, stream, 1, p))
            return rc;
        return lsb_launch(spread_merge_kernel<G, NT, T>, dim3(p.nkv * 8 * NT, p.n_requests * p.row_tiles), dim3(128), 0, stream, 1, p, blocks);
    }
};

// What fits at once: (form 0) blocks on an SM, (1) of the kernel that spreads, or clusters of `form` blocks on the device.  The spread form has
// up to 30 registers more: with heads of 64 and 16 rows two blocks fit where three of the other do, with heads of 32 and 8 rows four where
// five do.  (Stretches for the other's number of blocks run in two rounds: one token at 131,072, 32 / 2 heads of 64, 36.9 us where it
// takes 26.6; 64 at 1,000 - 8,100, 32 / 8 of 32, 67.6 and 55.3.)  A cluster's blocks share a group of SMs, whose places clusters of 5 to 8
// blocks do not fill: of 296 blocks' places 40 clusters of 7 take two rounds (40 tokens behind 30,000, 16 / 1 heads of 128: 121 us, spread
// 72).
struct Kv4Room {
    int form;
    template <int G, int NT, typename T, bool SPREAD> static int blocks() {
        int got = 0;
        if (kv4_configure<G, NT, T, SPREAD>()) return 0;
        return cudaOccupancyMaxActiveBlocksPerMultiprocessor(&got, attention_kv4_kernel<G, NT, T, SPREAD>, kThreads,
                                                             Kv4Shape<G, NT, T>::kBytes) == cudaSuccess ? got : 0;
    }
    template <int G, int NT, typename T> int run() const {
        if (form < 2) return form ? blocks<G, NT, T, true>() : blocks<G, NT, T, false>();
        if (kv4_configure<G, NT, T, false>()) return 0;
        cudaLaunchAttribute along;
        along.id = cudaLaunchAttributeClusterDimension;
        along.val.clusterDim.x = form;
        along.val.clusterDim.y = along.val.clusterDim.z = 1;
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3(form);
        cfg.blockDim = dim3(kThreads);
        cfg.dynamicSmemBytes = Kv4Shape<G, NT, T>::kBytes;
        cfg.attrs = &along;
        cfg.numAttrs = 1;
        int got = 0;
        return cudaOccupancyMaxActiveClusters(&got, attention_kv4_kernel<G, NT, T, false>, &cfg) == cudaSuccess ? got : 0;
    }
};

struct Kv4SlotFloats {
    template <int G, int NT, typename T> int run() const { return Kv4Shape<G, NT, T>::kSlot; }
};

// The kernel for heads of `hd` and `eights` eights of rows; -1 where there is none.
template <typename T, int G, typename Op>
static int kv4_of_shape(int eights, const Op& op) {
    if constexpr (std::is_same<T, bf16>::value && G <= 4) {
        if (eights == 2) return op.template run<G, 2, T>();
    }
    return eights == 1 ? op.template run<G, 1, T>() : -1;
}
template <typename T, typename Op>
static int kv4_of(int hd, int eights, const Op& op) {
    switch (hd) {
        case 32: return kv4_of_shape<T, 1>(eights, op);
        case 64: return kv4_of_shape<T, 2>(eights, op);
        case 96: return kv4_of_shape<T, 3>(eights, op);
        case 128: return kv4_of_shape<T, 4>(eights, op);
        case 160: return kv4_of_shape<T, 5>(eights, op);
        case 192: return kv4_of_shape<T, 6>(eights, op);
        case 224: return kv4_of_shape<T, 7>(eights, op);
        case 256: return kv4_of_shape<T, 8>(eights, op);
    }
    return -1;
}

// `max_rows`: the most rows (queries times heads of a group) of a request that is taken; `eights`: eights of rows of a block;
// `spread` blocks (0: a cluster of `splits` to each row tile instead), with `parts` of two slots for each.
template <typename T>
static int kv4_attention(const void* qkv, int qkv_stride, const void* pages, const int* q_start, const int* kv_len,
                         const int* table_rows, const int* block_table, int table_stride, void* out, int n_requests,
                         long long max_rows, int nh, int nkv, int hd, int page_size, int num_pages, float scale, int window,
                         int first, int mode, int eights, int splits, int spread, float* parts, cudaStream_t stream) {
    if (n_requests <= 0 || max_rows <= 0) return 0;
    if (splits < 1 || splits > kMaxSplits || eights < 1 || nkv <= 0 || nkv > 65535 || n_requests > 65535 || page_size <= 0 ||
        page_size % kKv4Tile || (long long)num_pages * nkv * (page_size / kKv4Tile) > 0x7fffffffll ||
        (mode != 1 && mode != 2) || (spread && (spread < nkv || !parts)))
        return (int)cudaErrorInvalidValue;
    const long long row_tiles = (max_rows + 8 * eights - 1) / (8 * eights);
    if (row_tiles * splits > 0x7fffffffll || (spread && row_tiles * n_requests > kMaxSpread)) return (int)cudaErrorInvalidValue;
    Kv4Params p;
    p.qkv = qkv; p.qkv_stride = qkv_stride; p.pages = (const unsigned char*)pages;
    p.q_start = q_start; p.kv_len = kv_len; p.table_rows = table_rows; p.block_table = block_table; p.table_stride = table_stride;
    p.out = out; p.nh = nh; p.nkv = nkv; p.tiles_per_page = page_size / kKv4Tile; p.num_pages = num_pages;
    p.scale = scale; p.window = window; p.first = first; p.mode = mode; p.splits = splits;
    p.parts = parts; p.n_requests = n_requests; p.row_tiles = (int)row_tiles;
    const int rc = spread ? kv4_of<T>(hd, eights, Kv4SpreadLaunch{p, spread, stream})
                          : kv4_of<T>(hd, eights, Kv4Launch{p, dim3((unsigned)(row_tiles * splits), nkv, n_requests), stream});
    return rc < 0 ? (int)cudaErrorInvalidValue : rc;
}

#define LSB_KV4_ENTRY_POINTS(T)                                                                                              \
    LSB_API int lsb_attention_kv4(const void* qkv, int qkv_stride, const void* pages, const int* q_start, const int* kv_len, \
                                  const int* table_rows, const int* block_table, int table_stride, void* out, int n_requests, \
                                  long long max_rows, int nh, int nkv, int hd, int page_size, int num_pages, float scale,   \
                                  int window, int first, int mode, int eights, int splits, int spread,     \
                                  float* parts, cudaStream_t stream) {                                                       \
        return kv4_attention<T>(qkv, qkv_stride, pages, q_start, kv_len, table_rows, block_table, table_stride, out,         \
                                n_requests, max_rows, nh, nkv, hd, page_size, num_pages, scale, window, first, mode,         \
                                eights, splits, spread, parts, stream);                                                      \
    }                                                                                                                        \
    LSB_API int lsb_attention_kv4_room(int hd, int eights, int form) {                                                       \
        const int got = form < 0 || form > kMaxSplits ? -1 : kv4_of<T>(hd, eights, Kv4Room{form});                           \
        return got < 0 ? 0 : got;                                                                                            \
    }                                                                                                                        \
    LSB_API int lsb_attention_kv4_slot(int hd, int eights) { return kv4_of<T>(hd, eights, Kv4SlotFloats{}); }
