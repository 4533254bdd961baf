// Rows of prompt portions that came out as no number, once more.
//
// The tcgen05 prompt kernel multiplies first and masks by weights of zero: an infinity or NaN that a page holds at a hidden place (a key
// behind a row's own, one that its window has passed, what a page was left with by another request) makes NaN of rows that do
// not see it.  This kernel runs behind it, reads the results (bfloat16, from L2: 2,000 tokens of 32 heads of 64, 8 MB, 3 us), and where a
// (token, head) holds a NaN does that one again over the keys it sees and no others: one warp, a key at a time, 32-bit sums.  A
// true NaN comes out again.  So the price of numbers that are none is paid where they are.
//
// Query i of request r sits at p = kv_len - q_len + i and sees keys j <= p with window == 0, j > p - window, or j < first.
#include "kv4.cuh"

#include <math.h>

LSB_DEFINE_STATUS()

typedef __nv_bfloat16 bf16;

constexpr int kRepairThreads = 256;
constexpr int kItems = 64;                      // (token, head) of a block
constexpr int kMaxDims = 4;                     // of a lane: heads of up to 128

struct RepairParams {
    const bf16* q;                              // of token t, head h at q + t * q_stride + h * hd
    int q_stride;
    const int *q_start, *kv_len, *table_rows, *block_table;
    int table_stride;
    bf16* out;                                  // [tokens, nh * hd]
    int nh, nkv, hd, page_size, num_pages;
    float scale;
    int window, first;
    const void *k_pages, *v_pages;              // (a 4-bit cache: both the pages)
};

struct Plain {                                  // [page][kv head][offset][hd]
    static __device__ __forceinline__ void load(const RepairParams& p, int page, int g, int off, int d, float& k, float& v) {
        const size_t at = (((size_t)page * p.nkv + g) * p.page_size + off) * p.hd + d;
        k = __bfloat162float(reinterpret_cast<const bf16*>(p.k_pages)[at]);
        v = __bfloat162float(reinterpret_cast<const bf16*>(p.v_pages)[at]);
    }
};
struct Kv4 {
    static __device__ __forceinline__ void load(const RepairParams& p, int page, int g, int off, int d, float& k, float& v) {
        const int hd = p.hd, G = hd / kKv4Group, t = off % kKv4Tile;
        const unsigned char* tile = reinterpret_cast<const unsigned char*>(p.k_pages) +
                                    (((size_t)page * p.nkv + g) * (p.page_size / kKv4Tile) + off / kKv4Tile) * kv4_tile_bytes(hd);
        const int kc = tile[t * (hd / 2) + (d % 32 / 8 * G + d / 32) * 4 + d % 8 / 2] >> (4 * (d & 1)) & 15;
        const int vc = tile[kv4_values_at(hd) + t * (hd / 2) + d % 16 / 2 * 2 * G + d / 16] >> (4 * (d & 1)) & 15;
        k = (float)(kc - 8) * __bfloat162float(*reinterpret_cast<const bf16*>(tile + kv4_key_scales_at(hd) + (t * G + d / 32) * 2));
        v = (float)(vc - 8) * __bfloat162float(*reinterpret_cast<const bf16*>(tile + kv4_value_scales_at(hd) + (t * G + d / 32) * 2));
    }
};

template <typename Cache>
__global__ void __launch_bounds__(kRepairThreads) attention_repair_kernel(const RepairParams p) {
    __shared__ int spoilt[kItems];
    lsb_pdl_launch_dependents();
    const int r = blockIdx.z, tid = threadIdx.x, hd = p.hd;
    const int qs = p.q_start[r], q_len = p.q_start[r + 1] - qs, item0 = blockIdx.x * kItems;
    if (q_len == 1 || item0 >= q_len * p.nh) return;            // (single tokens are not the prompt kernel's)
    const int n = min(kItems, q_len * p.nh - item0), per = hd / 8;
    for (int i = tid; i < kItems; i += kRepairThreads) spoilt[i] = 0;
    __syncthreads();
    lsb_pdl_wait();
    bf16* out = p.out + (size_t)qs * p.nh * hd + (size_t)item0 * hd;
    bool any = false;
#pragma unroll 4
    for (int i = tid; i < n * per; i += kRepairThreads) {
        const uint4 x = reinterpret_cast<const uint4*>(out)[i];
        const uint32_t w[4] = {x.x, x.y, x.z, x.w};
        bool none = false;
#pragma unroll
        for (int j = 0; j < 4; ++j) none = none || (w[j] & 0x7fffu) > 0x7f80u || (w[j] >> 16 & 0x7fffu) > 0x7f80u;
        if (none) spoilt[i / per] = 1;
        any = any || none;
    }
    if (!__syncthreads_or(any)) return;
    const int lane = tid & 31;
    for (int i = tid >> 5; i < n; i += kRepairThreads / 32) {
        if (!spoilt[i]) continue;
        const int qi = (item0 + i) / p.nh, h = (item0 + i) % p.nh, g = h / (p.nh / p.nkv);
        const int pos = p.kv_len[r] - q_len + qi;
        const int lo = p.window > 0 && pos - p.window + 1 > 0 ? pos - p.window + 1 : 0, few = p.window > 0 ? min(p.first, lo) : 0;
        const int* table = p.block_table + (size_t)p.table_rows[r] * p.table_stride;
        float q[kMaxDims], o[kMaxDims], m = -INFINITY, l = 0.f;
#pragma unroll
        for (int e = 0; e < kMaxDims; ++e) {
            o[e] = 0.f;
            q[e] = lane + 32 * e < hd ? __bfloat162float(p.q[(size_t)(qs + qi) * p.q_stride + h * hd + lane + 32 * e]) : 0.f;
        }
        for (int j = 0; j < few + pos - lo + 1; ++j) {
            const int key = j < few ? j : j - few + lo, pi = key / p.page_size;
            const int page = pi < p.table_stride ? table[pi] : -1;
            if (page < 0 || page >= p.num_pages) continue;      // (recorded by the kernel before)
            float k[kMaxDims], v[kMaxDims], s = 0.f;
#pragma unroll
            for (int e = 0; e < kMaxDims; ++e) {
                k[e] = v[e] = 0.f;
                if (lane + 32 * e < hd) Cache::load(p, page, g, key % p.page_size, lane + 32 * e, k[e], v[e]);
                s = fmaf(q[e], k[e], s);
            }
            s = lsb_warp_sum(s) * p.scale;
            const float top = fmaxf(m, s), ref = top == -INFINITY ? 0.f : top;
            const float was = m == -INFINITY ? 1.f : expf(m - ref), w = expf(s - ref);      // (before the first reference all is zero, or no number)
            l = l * was + w;
            m = top;
#pragma unroll
            for (int e = 0; e < kMaxDims; ++e) o[e] = o[e] * was + w * v[e];
        }
#pragma unroll
        for (int e = 0; e < kMaxDims; ++e)
            if (lane + 32 * e < hd) out[(size_t)i * hd + lane + 32 * e] = __float2bfloat16_rn(l != 0.f ? o[e] / l : 0.f);
    }
}

// bfloat16, heads of a multiple of 8 up to 128, `out` at a multiple of 16 bytes.  kv4: the cache is one of 4 bits, `k_pages` its pages.
LSB_API int lsb_attention_repair(const void* qkv, int qkv_stride, const void* k_pages, const void* v_pages, const int* q_start,
                                 const int* kv_len, const int* table_rows, const int* block_table, int table_stride, void* out,
                                 int n_requests, int max_q_len, int nh, int nkv, int hd, int page_size, int num_pages, float scale,
                                 int window, int first, int kv4, cudaStream_t stream) {
    if (n_requests <= 0 || max_q_len <= 1) return 0;
    if (hd % 8 || hd > 32 * kMaxDims || n_requests > 65535 || (uintptr_t)out % 16) return (int)cudaErrorInvalidValue;
    const RepairParams p{(const bf16*)qkv, qkv_stride, q_start, kv_len, table_rows, block_table, table_stride, (bf16*)out, nh, nkv, hd,
                         page_size, num_pages, scale, window, first, k_pages, v_pages};
    const dim3 grid((unsigned)(((long long)max_q_len * nh + kItems - 1) / kItems), 1, n_requests);
    return kv4 ? lsb_launch(attention_repair_kernel<Kv4>, grid, dim3(kRepairThreads), 0, stream, 1, p)
               : lsb_launch(attention_repair_kernel<Plain>, grid, dim3(kRepairThreads), 0, stream, 1, p);
}
