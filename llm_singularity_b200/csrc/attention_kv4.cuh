// Attention over a 4-bit cache (kv4.cuh): single tokens and portions of prompts, any head size that is a multiple of 32 up
// to 256, any grouping of query heads, bfloat16 or 32-bit rows.
//
// For request r with q_len new tokens and kv_len tokens in the cache, query i sits at position p = kv_len - q_len + i and
// sees the keys at positions j <= p with j > p - window (window == 0: all) or j < first.  Rows of a kv head are its queries'
// heads, position by position: row = i * group + (head within the group).
//
// A block takes kCols rows of a kv head as the columns of its products and walks the tiles of 16 tokens that any of them
// sees, dealt to its eight warps; `splits` blocks, a cluster, share out a row tile's tokens.  Both products have the cache as
// their left operand, so that a code is unpacked once for all rows and a lane's share of a tile is what it needs and
// nothing else:
//     S^T [tokens x rows]  = K Q^T        one accumulator per group of 32 dims, which times its scale is added to the scores
//     O^T [dims x rows]   += V^T (P s)^T  the scale of a token's group goes into its probability, rounded once to bfloat16
// The probabilities leave the first product with tokens down the lanes and enter the second with tokens across them: an
// 8 x 8 transposition of bfloat16 (movmatrix) per eight tokens, rows and group.
// A code becomes a bfloat16 by masking it into the mantissa of 128; keys keep the 136 that is too much (it is taken off the
// accumulator's start as 136 times the sum of the row's dims: 32 products of one group, so at most 2^-16 of the group's score
// is lost), values have it subtracted exactly before the product, where it would add up over all tokens.
// 32-bit rows: queries and probabilities are sums of three bfloat16 (24 bits), codes are exact in one, so three products do.
//
// A tile of a kv head is one contiguous piece of 18 hd bytes: one bulk copy, issued by one lane into the warp's own ring.
// Nothing but a warp's own barriers orders that ring; warps and blocks meet once, at the end, through shared memory and the
// cluster's.
#pragma once

#define LSB_CLUSTER_ALONG_X            // splits are the fastest part of blockIdx.x
#include "kv4.cuh"

#include <type_traits>

LSB_DEFINE_STATUS()

typedef __nv_bfloat16 bf16;

constexpr int kWarps = 8;
constexpr int kThreads = 32 * kWarps;
constexpr int kMaxSplits = 16;
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
    int mode;                          // 0: every request; 1: those that bring one token; 2: the others
    int splits;
};

// ------------------------------------------------------------------ PTX helpers
__device__ __forceinline__ uint32_t smem_u32(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void bar_init(uint64_t* bar) {
    asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" ::"r"(smem_u32(bar)));
}
__device__ __forceinline__ void bar_arrive(uint64_t* bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ void bulk_load(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(smem_u32(bar)), "r"(bytes) : "memory");
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
                 ::"r"(smem_u32(dst)), "l"(src), "r"(bytes), "r"(smem_u32(bar)) : "memory");
}
// (bounded; false if the wait ran out)
__device__ __forceinline__ bool bar_wait(uint64_t* bar, uint32_t parity) {
    for (uint32_t it = 0; it < kSpinLimit; ++it) {
        uint32_t ok;
        asm volatile("{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}"
                     : "=r"(ok) : "r"(smem_u32(bar)), "r"(parity) : "memory");
        if (ok) return true;
        if ((it & 255u) == 255u) __nanosleep(128);
    }
    return false;
}
// D = A B + C on bfloat16, 32-bit sums
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
// ... less 136: exact
__device__ __forceinline__ uint32_t lowered(uint32_t x) {
    uint32_t r;
    asm("sub.rn.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(x), "r"(0x43084308u));
    return r;
}
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
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

// ------------------------------------------------------------------ the kernel
// G: groups of 32 dims of a head; NT: eights of rows of a block; T: type of the rows.
template <int G, int NT, typename T>
struct Kv4Shape {
    static constexpr int kHd = kKv4Group * G;
    static constexpr int kCols = 8 * NT;
    static constexpr int kParts = std::is_same<T, float>::value ? 3 : 1;
    static constexpr int kTile = kv4_tile_bytes(kHd);
    static constexpr int kStages = G <= 2 ? 8 : 4;
    static constexpr int kRing = kWarps * kStages * kTile;
    static constexpr int kSums = kWarps * kCols * kHd * 4;             // the warps' O, in the ring's place
    static constexpr int kQ = kParts * kCols * kHd * 2;
    static constexpr int kO = kCols * kHd * 4;                         // the block's
    static constexpr size_t kBytes = (kRing > kSums ? kRing : kSums) + kQ + kO;
};

template <int G, int NT, typename T>
__global__ void __launch_bounds__(kThreads, (G <= 4 && NT == 1 && std::is_same<T, bf16>::value) ? 2 : 1)
attention_kv4_kernel(const Kv4Params p) {
    using Z = Kv4Shape<G, NT, T>;
    constexpr int HD = Z::kHd, COLS = Z::kCols, PARTS = Z::kParts, ST = Z::kStages, TILE = Z::kTile;
    constexpr bool EXACT = PARTS == 3;
    extern __shared__ __align__(128) unsigned char smem[];
    unsigned char* ring_all = smem;
    float* sums = reinterpret_cast<float*>(smem);                      // [warps][COLS][HD], when the ring is done with
    bf16* sq = reinterpret_cast<bf16*>(smem + (Z::kRing > Z::kSums ? Z::kRing : Z::kSums));   // [PARTS][COLS][HD]
    float* so = reinterpret_cast<float*>(sq + PARTS * COLS * HD);      // [COLS][HD]
    __shared__ uint64_t bars[kWarps][ST];
    __shared__ float wm[kWarps][COLS], wl[kWarps][COLS];               // the warps' maxima and sums
    __shared__ float bm[COLS], bl[COLS];                               // the block's
    __shared__ float factor[kMaxSplits][COLS], inverse[COLS];

    lsb_pdl_launch_dependents();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, e8 = lane >> 2, t4 = lane & 3;
    // the step's metadata is on the device before the step's first kernel starts
    const int splits = p.splits, split = (int)(blockIdx.x % splits), h = blockIdx.y, r = blockIdx.z;
    const int group = p.nh / p.nkv;
    const int qs = p.q_start[r], q_len = p.q_start[r + 1] - qs, n_rows = q_len * group;
    // (late rows see the most keys, and start first; all blocks of a cluster leave here alike)
    const int row_tiles = (n_rows + COLS - 1) / COLS, rt = row_tiles - 1 - (int)(blockIdx.x / splits);
    if (rt < 0 || (p.mode == 1 && q_len != 1) || (p.mode == 2 && q_len == 1)) return;
    const int row0 = rt * COLS, row1 = min(row0 + COLS, n_rows);
    const int base = p.kv_len[r] - q_len;                              // position of the request's first new token
    const int p_lo = base + row0 / group, p_hi = base + (row1 - 1) / group;
    const int W = p.window, F = W > 0 ? p.first : 0;
    const int near = (W > 0 && p_lo - W + 1 > 0 ? p_lo - W + 1 : 0) / kKv4Tile;
    const int early = min((F + kKv4Tile - 1) / kKv4Tile, near);        // tiles of first tokens in front of the window's
    const int n_tiles = early + p_hi / kKv4Tile + 1 - near;
    const int per = (n_tiles + splits - 1) / splits;
    const int c0 = min(split * per, n_tiles), c1 = min(c0 + per, n_tiles);
    const int n_mine = (c1 - c0 - warp + kWarps - 1) / kWarps;         // tiles c0 + warp, c0 + warp + kWarps, ... (0 or less: none)

    if (tid < kWarps * ST) bar_init(&bars[tid / ST][tid % ST]);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    lsb_pdl_wait();
    __syncthreads();

    const int* table = p.block_table + (size_t)p.table_rows[r] * p.table_stride;
    unsigned char* ring = ring_all + warp * ST * TILE;
    auto tile_of = [&](int k) -> int {                                 // the warp's k-th tile, counted from position 0
        const int c = c0 + warp + kWarps * k;
        return c < early ? c : c - early + near;
    };
    // Places in the pool of 32 of the warp's tiles, one a lane; -1 where the page is none of the pool's.
    auto places = [&](int k) -> int {
        if (k >= n_mine) return -1;
        const int tile = tile_of(k), pi = tile / p.tiles_per_page;
        const int page = pi < p.table_stride ? __ldcg(table + pi) : -1;
        if (page < 0 || page >= p.num_pages) {
            lsb_set_status(LSB_BAD_PAGE);
            return -1;
        }
        return (page * p.nkv + h) * p.tiles_per_page + tile % p.tiles_per_page;
    };
    int known = places(lane);
    uint32_t there = 0;                                                // which stages hold a tile (alike in all lanes)
    auto issue = [&](int k) {
        if (k >= n_mine) return;
        if (k > 0 && k % 32 == 0) known = places(k + lane);
        const int at = __shfl_sync(0xffffffffu, known, k % 32), s = k % ST;
        there = (there & ~(1u << s)) | (at >= 0 ? 1u << s : 0u);
        if (lane == 0) {
            if (at >= 0) bulk_load(ring + s * TILE, p.pages + (size_t)at * TILE, TILE, &bars[warp][s]);
            else bar_arrive(&bars[warp][s]);
        }
    };
#pragma unroll
    for (int k = 0; k < ST - 1; ++k) issue(k);

    // the block's rows of queries; rows beyond the last are zeros
    const T* qkv = reinterpret_cast<const T*>(p.qkv);
    for (int i = tid; i < COLS * HD; i += kThreads) {
        const int c = i / HD, d = i - c * HD, row = row0 + c;
        float x = 0.f;
        if (row < row1) x = lsb_to_float(qkv[(size_t)(qs + row / group) * p.qkv_stride + (h * group + row % group) * HD + d]);
#pragma unroll
        for (int part = 0; part < PARTS; ++part) {
            const bf16 y = __float2bfloat16_rn(x);
            sq[part * COLS * HD + i] = y;
            x -= __bfloat162float(y);
        }
    }
    __syncthreads();
    // Right operand of S^T: dims 32 g + 8 t + {0, 4}, {1, 5}, {2, 6}, {3, 7} of row e, as a key's nibbles unpack.
    uint32_t q[NT][PARTS][G][4];
    float start[NT][G][2];                                             // - 136 times the sum over a group, of rows 2 t and 2 t + 1
#pragma unroll
    for (int n = 0; n < NT; ++n)
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
#pragma unroll
                for (int i = 0; i < 4; ++i) sum += low_half(w[i]) + high_half(w[i]);
            }
            if constexpr (!EXACT) {
                sum += __shfl_xor_sync(0xffffffffu, sum, 1);
                sum += __shfl_xor_sync(0xffffffffu, sum, 2);
                start[n][g][0] = -136.f * __shfl_sync(0xffffffffu, sum, 8 * t4);
                start[n][g][1] = -136.f * __shfl_sync(0xffffffffu, sum, 8 * t4 + 4);
            } else {
                start[n][g][0] = start[n][g][1] = 0.f;
            }
        }
    int col_pos[NT][2];                                                // positions of rows 2 t and 2 t + 1
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int b = 0; b < 2; ++b) col_pos[n][b] = base + min(row0 + n * 8 + 2 * t4 + b, row1 - 1) / group;

    float o[NT][2 * G][4];
    float m[NT][2], l[NT][2];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
        m[n][0] = m[n][1] = -INFINITY;
        l[n][0] = l[n][1] = 0.f;
#pragma unroll
        for (int i = 0; i < 2 * G; ++i) o[n][i][0] = o[n][i][1] = o[n][i][2] = o[n][i][3] = 0.f;
    }
    const float sc = p.scale * kLog2e;
    bool ok = true;

    for (int k = 0; k < n_mine && ok; ++k) {
        issue(k + ST - 1);
        const int stage = k % ST;
        ok = __all_sync(0xffffffffu, bar_wait(&bars[warp][stage], (uint32_t)(k / ST) & 1u));
        if (!ok) break;
        if (!(there >> stage & 1u)) continue;
        const unsigned char* tile = ring + stage * TILE;
        const int key0 = tile_of(k) * kKv4Tile;

        // ---------------------------------------------------------- scores
        float s[NT][4];
        {
            uint32_t ka[G], kb[G], sa[(G + 1) / 2], sb[(G + 1) / 2];
            {
                uint32_t w[G];
                load_halves<2 * G>(tile + e8 * (HD / 2) + t4 * 4 * G, w);
#pragma unroll
                for (int g = 0; g < G; ++g) ka[g] = w[g];
                load_halves<2 * G>(tile + (e8 + 8) * (HD / 2) + t4 * 4 * G, w);
#pragma unroll
                for (int g = 0; g < G; ++g) kb[g] = w[g];
            }
            load_halves<G>(tile + kv4_key_scales_at(HD) + e8 * 2 * G, sa);
            load_halves<G>(tile + kv4_key_scales_at(HD) + (e8 + 8) * 2 * G, sb);
#pragma unroll
            for (int n = 0; n < NT; ++n) s[n][0] = s[n][1] = s[n][2] = s[n][3] = 0.f;
#pragma unroll
            for (int g = 0; g < G; ++g) {
                uint32_t a[4], b[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    a[i] = raised(ka[g] >> (4 * i));
                    b[i] = raised(kb[g] >> (4 * i));
                    if constexpr (EXACT) { a[i] = lowered(a[i]); b[i] = lowered(b[i]); }
                }
                const float fa = g % 2 ? high_half(sa[g / 2]) : low_half(sa[g / 2]);
                const float fb = g % 2 ? high_half(sb[g / 2]) : low_half(sb[g / 2]);
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    float d[4];
                    mma(d, a[0], b[0], a[1], b[1], q[n][0][g][0], q[n][0][g][1], start[n][g][0], start[n][g][1], start[n][g][0], start[n][g][1]);
                    mma(d, a[2], b[2], a[3], b[3], q[n][0][g][2], q[n][0][g][3], d[0], d[1], d[2], d[3]);
#pragma unroll
                    for (int part = 1; part < PARTS; ++part) {
                        mma(d, a[0], b[0], a[1], b[1], q[n][part][g][0], q[n][part][g][1], d[0], d[1], d[2], d[3]);
                        mma(d, a[2], b[2], a[3], b[3], q[n][part][g][2], q[n][part][g][3], d[0], d[1], d[2], d[3]);
                    }
                    s[n][0] = fmaf(fa, d[0], s[n][0]);
                    s[n][1] = fmaf(fa, d[1], s[n][1]);
                    s[n][2] = fmaf(fb, d[2], s[n][2]);
                    s[n][3] = fmaf(fb, d[3], s[n][3]);
                }
            }
        }
        // ---------------------------------------------------------- which of them count
        const bool whole = key0 + kKv4Tile - 1 <= p_lo && (W <= 0 || key0 > p_hi - W || key0 + kKv4Tile <= F);
        uint32_t seen = 0xffffffffu;                                   // bit 4 n + i: element i of s[n]
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int i = 0; i < 4; ++i) s[n][i] *= sc;
        if (!whole) {
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int key = key0 + e8 + (i >> 1) * 8, pos = col_pos[n][i & 1];
                    if (!(key <= pos && (W <= 0 || key > pos - W || key < F))) {
                        s[n][i] = -INFINITY;
                        seen &= ~(1u << (4 * n + i));
                    }
                }
        }
        // ---------------------------------------------------------- softmax: references move seldom
        bool above = false;
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int b = 0; b < 2; ++b) above = above || fmaxf(s[n][b], s[n][2 + b]) > m[n][b] + kRescale;
        if (__any_sync(0xffffffffu, above)) {
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                float corr[2];
#pragma unroll
                for (int b = 0; b < 2; ++b) {
                    float top = fmaxf(s[n][b], s[n][2 + b]);
#pragma unroll
                    for (int x = 4; x < 32; x <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, x));
                    top = fmaxf(top, m[n][b]);
                    corr[b] = top == -INFINITY ? 1.f : fast_exp2(m[n][b] - top);
                    m[n][b] = top;
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
        }
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float ref = m[n][i & 1];
                s[n][i] = fast_exp2(s[n][i] - (ref == -INFINITY ? 0.f : ref));
                l[n][i & 1] += s[n][i];
            }
        // ---------------------------------------------------------- values
        uint32_t va[(G + 1) / 2], vb[(G + 1) / 2], v[4][(G + 1) / 2];
        load_halves<G>(tile + kv4_value_scales_at(HD) + e8 * 2 * G, va);
        load_halves<G>(tile + kv4_value_scales_at(HD) + (e8 + 8) * 2 * G, vb);
#pragma unroll
        for (int i = 0; i < 4; ++i)                                    // tokens 2 t, 2 t + 1, 2 t + 8, 2 t + 9
            load_halves<G>(tile + kv4_values_at(HD) + (2 * t4 + (i & 1) + (i >> 1) * 8) * (HD / 2) + e8 * 2 * G, v[i]);
#pragma unroll
        for (int g = 0; g < G; ++g) {
            const float fa = g % 2 ? high_half(va[g / 2]) : low_half(va[g / 2]);
            const float fb = g % 2 ? high_half(vb[g / 2]) : low_half(vb[g / 2]);
            uint32_t b[NT][PARTS][2];
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                float x[4] = {s[n][0] * fa, s[n][1] * fa, s[n][2] * fb, s[n][3] * fb};
                if (!whole) {                                          // (a scale that is no number stays out of rows that do not see it)
#pragma unroll
                    for (int i = 0; i < 4; ++i) x[i] = seen >> (4 * n + i) & 1u ? x[i] : 0.f;
                }
#pragma unroll
                for (int part = 0; part < PARTS; ++part) {
                    const uint32_t y0 = pack2(x[0], x[1]), y1 = pack2(x[2], x[3]);
                    b[n][part][0] = transposed(y0);
                    b[n][part][1] = transposed(y1);
                    if (part + 1 < PARTS) {
                        x[0] -= low_half(y0); x[1] -= high_half(y0);
                        x[2] -= low_half(y1); x[3] -= high_half(y1);
                    }
                }
            }
#pragma unroll
            for (int i = 2 * g; i < 2 * g + 2; ++i) {
                // byte i of the rows of two tokens, side by side: dims 16 i + 2 e (low nibbles) and + 1 (high ones)
                constexpr uint32_t kPick[4] = {0x4400, 0x5511, 0x6622, 0x7733};
                const uint32_t x = __byte_perm(v[0][i / 4], v[1][i / 4], kPick[i % 4]);
                const uint32_t y = __byte_perm(v[2][i / 4], v[3][i / 4], kPick[i % 4]);
                const uint32_t a0 = lowered(raised(x)), a1 = lowered(raised(x >> 4));
                const uint32_t a2 = lowered(raised(y)), a3 = lowered(raised(y >> 4));
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int part = 0; part < PARTS; ++part)
                        mma(o[n][i], a0, a1, a2, a3, b[n][part][0], b[n][part][1], o[n][i][0], o[n][i][1], o[n][i][2], o[n][i][3]);
            }
        }
        __syncwarp();                                                  // the stage may be written over
    }
    if (!ok) {
        // a copy did not arrive: what is in flight is waited for (with the same limit) before shared memory goes
        lsb_set_status(LSB_WAIT_TIMEOUT);
        for (int s = 0; s < ST; ++s) {
            const int k = (n_mine - 1 - s) / ST * ST + s;              // (the last tile of stage s, whether or not it was asked for)
            if (s < n_mine) bar_wait(&bars[warp][s], (uint32_t)(k / ST) & 1u);
        }
    }
    __syncthreads();                                                   // every warp is done with its ring

    // ------------------------------------------------------------------ the warps' sums, then the blocks'
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int b = 0; b < 2; ++b) {
            float sum = l[n][b];
#pragma unroll
            for (int x = 4; x < 32; x <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, x);
            const int c = n * 8 + 2 * t4 + b;
            if (e8 == 0) {
                wm[warp][c] = m[n][b];
                wl[warp][c] = sum;
            }
#pragma unroll
            for (int i = 0; i < 2 * G; ++i)
                *reinterpret_cast<float2*>(sums + (warp * COLS + c) * HD + 16 * i + 2 * e8) = make_float2(o[n][i][b], o[n][i][2 + b]);
        }
    __syncthreads();
    if (tid < COLS) {
        float top = -INFINITY, sum = 0.f;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) top = fmaxf(top, wm[w][tid]);
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
            const float f = wm[w][tid] == -INFINITY && wl[w][tid] == 0.f ? 0.f : fast_exp2(wm[w][tid] - (top == -INFINITY ? 0.f : top));
            sum += wl[w][tid] * f;
            wm[w][tid] = f;
        }
        bm[tid] = top;
        bl[tid] = sum;
        if (splits == 1) {
            factor[0][tid] = 1.f;
            inverse[tid] = sum == 0.f ? 0.f : 1.f / sum;
        }
    }
    __syncthreads();
    constexpr int UNITS = COLS * HD / 4;
    T* out = reinterpret_cast<T*>(p.out);
    auto finish = [&](int u, float4 v) {
        const int c = u / (HD / 4), row = row0 + c;
        if (row >= row1) return;
        const float f = inverse[c];
        store_four<T>(out + (size_t)(qs + row / group) * p.nh * HD + (h * group + row % group) * HD + (u - c * (HD / 4)) * 4,
                      make_float4(v.x * f, v.y * f, v.z * f, v.w * f));
    };
    for (int u = tid; u < UNITS; u += kThreads) {
        const int c = u / (HD / 4);
        float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
            const float f = wm[w][c];
            const float4 x = reinterpret_cast<const float4*>(sums + w * COLS * HD)[u];
            v.x = fmaf(f, x.x, v.x); v.y = fmaf(f, x.y, v.y); v.z = fmaf(f, x.z, v.z); v.w = fmaf(f, x.w, v.w);
        }
        if (splits == 1) finish(u, v);
        else reinterpret_cast<float4*>(so)[u] = v;
    }
    if (splits == 1) return;
    cluster_barrier();
    if (tid < COLS) {
        float top = -INFINITY, sum = 0.f;
        for (int b = 0; b < splits; ++b) top = fmaxf(top, peer_f32(&bm[tid], b));
        for (int b = 0; b < splits; ++b) {
            const float bmx = peer_f32(&bm[tid], b), bsum = peer_f32(&bl[tid], b);
            const float f = bmx == -INFINITY && bsum == 0.f ? 0.f : fast_exp2(bmx - (top == -INFINITY ? 0.f : top));
            factor[b][tid] = f;
            sum += bsum * f;
        }
        inverse[tid] = sum == 0.f ? 0.f : 1.f / sum;
    }
    __syncthreads();
    for (int u = split * kThreads + tid; u < UNITS; u += splits * kThreads) {
        const int c = u / (HD / 4);
        float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
        for (int b = 0; b < splits; ++b) {
            const float f = factor[b][c];
            const float4 x = peer_f32x4(reinterpret_cast<const float4*>(so) + u, b);
            v.x = fmaf(f, x.x, v.x); v.y = fmaf(f, x.y, v.y); v.z = fmaf(f, x.z, v.z); v.w = fmaf(f, x.w, v.w);
        }
        finish(u, v);
    }
    cluster_barrier();                                                 // nobody leaves while others read its sums
}

// ------------------------------------------------------------------ host side
// What a kernel needs before its first launch on a device.
template <int G, int NT, typename T>
static int kv4_configure() {
    static bool done[64] = {};
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return (int)e;
    if (dev >= 0 && dev < 64 && done[dev]) return 0;
    auto k = attention_kv4_kernel<G, NT, T>;
    e = cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)Kv4Shape<G, NT, T>::kBytes);
    if (e == cudaSuccess) e = cudaFuncSetAttribute(k, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    if (e == cudaSuccess && dev >= 0 && dev < 64) done[dev] = true;
    return (int)e;
}

template <int G, int NT, typename T>
static int kv4_launch(const Kv4Params& p, dim3 grid, cudaStream_t stream) {
    if (const int rc = kv4_configure<G, NT, T>()) return rc;
    return lsb_launch(attention_kv4_kernel<G, NT, T>, grid, dim3(kThreads), Kv4Shape<G, NT, T>::kBytes, stream, p.splits, p);
}

// Blocks that an SM holds at once, and the largest cluster that can be launched (8 or 16), as blocks * 256 + cluster.
template <int G, int NT, typename T>
static int kv4_room() {
    if (kv4_configure<G, NT, T>()) return 0;
    int blocks = 0, most = 0;
    if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&blocks, attention_kv4_kernel<G, NT, T>, kThreads, Kv4Shape<G, NT, T>::kBytes) != cudaSuccess)
        return 0;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(kMaxSplits);
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = Kv4Shape<G, NT, T>::kBytes;
    if (cudaOccupancyMaxPotentialClusterSize(&most, attention_kv4_kernel<G, NT, T>, &cfg) != cudaSuccess) {
        cudaGetLastError();
        most = 8;
    }
    return blocks * 256 + (most >= 16 ? 16 : 8);
}

// `max_rows`: the most rows (queries times heads of a group) of a request that is taken; `eights`: eights of rows of a block.
template <typename T, int G, int MOST>
static int kv4_by_rows(const Kv4Params& p, int eights, dim3 grid, cudaStream_t stream) {
    if constexpr (MOST >= 2)
        if (eights == 2) return kv4_launch<G, 2, T>(p, grid, stream);
    return eights == 1 ? kv4_launch<G, 1, T>(p, grid, stream) : (int)cudaErrorInvalidValue;
}

template <typename T, int MOST>
static int kv4_attention(const void* qkv, int qkv_stride, const void* pages, const int* q_start, const int* kv_len,
                         const int* table_rows, const int* block_table, int table_stride, void* out, int n_requests,
                         long long max_rows, int nh, int nkv, int hd, int page_size, int num_pages, float scale, int window,
                         int first, int mode, int eights, int splits, cudaStream_t stream) {
    if (n_requests <= 0 || max_rows <= 0) return 0;
    if (splits < 1 || splits > kMaxSplits || nkv > 65535 || n_requests > 65535 || page_size % kKv4Tile ||
        (long long)num_pages * nkv * (page_size / kKv4Tile) > 0x7fffffffll)
        return (int)cudaErrorInvalidValue;
    const long long blocks = (max_rows + 8 * eights - 1) / (8 * eights) * splits;
    if (blocks > 0x7fffffffll) return (int)cudaErrorInvalidValue;
    Kv4Params p;
    p.qkv = qkv; p.qkv_stride = qkv_stride; p.pages = (const unsigned char*)pages;
    p.q_start = q_start; p.kv_len = kv_len; p.table_rows = table_rows; p.block_table = block_table; p.table_stride = table_stride;
    p.out = out; p.nh = nh; p.nkv = nkv; p.tiles_per_page = page_size / kKv4Tile; p.num_pages = num_pages;
    p.scale = scale; p.window = window; p.first = first; p.mode = mode; p.splits = splits;
    const dim3 grid((unsigned)blocks, nkv, n_requests);
    switch (hd) {
        case 32: return kv4_by_rows<T, 1, MOST>(p, eights, grid, stream);
        case 64: return kv4_by_rows<T, 2, MOST>(p, eights, grid, stream);
        case 96: return kv4_by_rows<T, 3, MOST>(p, eights, grid, stream);
        case 128: return kv4_by_rows<T, 4, MOST>(p, eights, grid, stream);
        case 160: return kv4_by_rows<T, 5, 1>(p, eights, grid, stream);
        case 192: return kv4_by_rows<T, 6, 1>(p, eights, grid, stream);
        case 224: return kv4_by_rows<T, 7, 1>(p, eights, grid, stream);
        case 256: return kv4_by_rows<T, 8, 1>(p, eights, grid, stream);
    }
    return (int)cudaErrorInvalidValue;
}

template <typename T, int MOST>
static int kv4_room_of(int hd, int eights) {
    if constexpr (MOST >= 2) {
        if (eights == 2) {
            switch (hd) {
                case 32: return kv4_room<1, 2, T>();
                case 64: return kv4_room<2, 2, T>();
                case 96: return kv4_room<3, 2, T>();
                case 128: return kv4_room<4, 2, T>();
            }
            return 0;
        }
    }
    switch (hd) {
        case 32: return kv4_room<1, 1, T>();
        case 64: return kv4_room<2, 1, T>();
        case 96: return kv4_room<3, 1, T>();
        case 128: return kv4_room<4, 1, T>();
        case 160: return kv4_room<5, 1, T>();
        case 192: return kv4_room<6, 1, T>();
        case 224: return kv4_room<7, 1, T>();
        case 256: return kv4_room<8, 1, T>();
    }
    return 0;
}

#define LSB_KV4_ENTRY_POINTS(T, MOST)                                                                                       \
    LSB_API int lsb_attention_kv4(const void* qkv, int qkv_stride, const void* pages, const int* q_start, const int* kv_len, \
                                  const int* table_rows, const int* block_table, int table_stride, void* out, int n_requests, \
                                  long long max_rows, int nh, int nkv, int hd, int page_size, int num_pages, float scale,   \
                                  int window, int first, int mode, int eights, int splits, cudaStream_t stream) {           \
        return kv4_attention<T, MOST>(qkv, qkv_stride, pages, q_start, kv_len, table_rows, block_table, table_stride, out,   \
                                      n_requests, max_rows, nh, nkv, hd, page_size, num_pages, scale, window, first, mode,   \
                                      eights, splits, stream);                                                               \
    }                                                                                                                        \
    LSB_API int lsb_attention_kv4_room(int hd, int eights) { return kv4_room_of<T, MOST>(hd, eights); }
