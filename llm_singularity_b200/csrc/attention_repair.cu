// Rows of prompt portions that came out as no number, once more.
//
// The tcgen05 prompt kernel multiplies first and masks by weights of zero: an infinity or NaN that a page holds at a hidden place (a key
// behind a row's own, one that its window has passed, what a page was left with by another request) makes NaN of rows that do
// not see it.  This kernel runs behind it, reads the results (bfloat16, from L2: 2,000 tokens of 32 heads of 64, 8 MB, 3 us), and where a
// (token, head) holds a NaN does that one again over the keys it sees and no others: one warp, a key at a time, 32-bit sums.  A
// true NaN comes out again.  So the price of numbers that are none is paid where they are.
//
// One token whose key or value is no number makes true NaN of every row behind it, which need not be formed again to be known: the block
// looks for the first and the last token of its rows' kv heads whose key holds a NaN, and whose value does in a group of 32 dims, all
// threads a token each; a row that sees such a key, or whose NaN are all at dims of such values that it sees, is done.  (2,011 tokens after
// 4,096, 32 / 8 heads of 128, a NaN at token 0: 155 ms where every row walked all its keys, 0.75 ms so.
// Rows in front of such a value in their own portion, which hidden spoils them, are formed again: 904 tokens of them 43 ms.)
//
// Query i of request r sits at p = kv_len - q_len + i and sees keys j <= p with window == 0, j > p - window, or j < first.
#include "kv4.cuh"

#include <limits.h>
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

// Whether one of eight bfloat16 is a NaN.
__device__ __forceinline__ bool holds_none(const uint4& x) {
    const uint32_t w[4] = {x.x, x.y, x.z, x.w};
    bool none = false;
#pragma unroll
    for (int j = 0; j < 4; ++j) none = none || (w[j] & 0x7fffu) > 0x7f80u || (w[j] >> 16 & 0x7fffu) > 0x7f80u;
    return none;
}

struct Plain {                                  // [page][kv head][offset][hd]
    static __device__ __forceinline__ void load(const RepairParams& p, int page, int g, int off, int d, float& k, float& v) {
        const size_t at = (((size_t)page * p.nkv + g) * p.page_size + off) * p.hd + d;
        k = __bfloat162float(reinterpret_cast<const bf16*>(p.k_pages)[at]);
        v = __bfloat162float(reinterpret_cast<const bf16*>(p.v_pages)[at]);
    }
    // bit e < 4: the value holds a NaN in dims 32 e .. 32 e + 31; bit 4: the key does
    static __device__ __forceinline__ uint32_t none(const RepairParams& p, int page, int g, int off) {
        const size_t at = (((size_t)page * p.nkv + g) * p.page_size + off) * p.hd;
        const uint4 *k = reinterpret_cast<const uint4*>(reinterpret_cast<const bf16*>(p.k_pages) + at);
        const uint4 *v = reinterpret_cast<const uint4*>(reinterpret_cast<const bf16*>(p.v_pages) + at);
        uint32_t found = 0;
        for (int i = 0; i < p.hd / 8; ++i) found |= (uint32_t)holds_none(k[i]) << 4 | (uint32_t)holds_none(v[i]) << (i / 4);
        return found;
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
    static __device__ __forceinline__ uint32_t none(const RepairParams& p, int page, int g, int off) {
        const int G = p.hd / kKv4Group;
        const unsigned char* tile = reinterpret_cast<const unsigned char*>(p.k_pages) +
                                    (((size_t)page * p.nkv + g) * (p.page_size / kKv4Tile) + off / kKv4Tile) * kv4_tile_bytes(p.hd);
        const unsigned short* k = reinterpret_cast<const unsigned short*>(tile + kv4_key_scales_at(p.hd)) + off % kKv4Tile * G;
        const unsigned short* v = reinterpret_cast<const unsigned short*>(tile + kv4_value_scales_at(p.hd)) + off % kKv4Tile * G;
        uint32_t found = 0;
        for (int i = 0; i < G; ++i) found |= (uint32_t)((k[i] & 0x7fffu) > 0x7f80u) << 4 | (uint32_t)((v[i] & 0x7fffu) > 0x7f80u) << i;
        return found;
    }
};

template <typename Cache>
__global__ void __launch_bounds__(kRepairThreads) attention_repair_kernel(const RepairParams p) {
    __shared__ int spoilt[kItems], owner[kItems];
    __shared__ int none_from[kItems][kMaxDims + 1], none_to[kItems][kMaxDims + 1];      // of values in a group of dims; [kMaxDims]: of keys
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
        const bool none = holds_none(reinterpret_cast<const uint4*>(out)[i]);
        if (none) spoilt[i / per] = 1;
        any = any || none;
    }
    if (!__syncthreads_or(any)) return;
    const int lane = tid & 31, group = p.nh / p.nkv, base = p.kv_len[r] - q_len;
    const int* table = p.block_table + (size_t)p.table_rows[r] * p.table_stride;
    auto page_of = [&](int key) {                               // (one that is not held was recorded by the kernel before)
        const int pi = key / p.page_size, page = pi < p.table_stride ? table[pi] : -1;
        return page < p.num_pages ? page : -1;
    };
    // of a position: where its window begins, and how many first tokens lie in front of that
    auto window_from = [&](int pos) { return p.window > 0 && pos - p.window + 1 > 0 ? pos - p.window + 1 : 0; };
    auto few_before = [&](int lo) { return p.window > 0 ? min(p.first, lo) : 0; };
    for (int i = tid; i < n; i += kRepairThreads) {             // the first spoilt item of the same kv head looks for the others
        const int g = (item0 + i) % p.nh / group;
        int k = 0;
        while (k < i && !(spoilt[k] && (item0 + k) % p.nh / group == g)) ++k;
        owner[i] = k;
        for (int e = 0; e <= kMaxDims; ++e) {
            none_from[i][e] = INT_MAX;
            none_to[i][e] = -1;
        }
    }
    __syncthreads();
    const int lo0 = window_from(base + item0 / p.nh), few0 = few_before(lo0), last = base + (item0 + n - 1) / p.nh;
    for (int i = 0; i < n; ++i) {
        if (!spoilt[i] || owner[i] != i) continue;              // (alike for all threads)
        const int g = (item0 + i) % p.nh / group;
        for (int j = tid; j < few0 + last - lo0 + 1; j += kRepairThreads) {
            const int key = j < few0 ? j : j - few0 + lo0, page = page_of(key);
            const uint32_t found = page >= 0 ? Cache::none(p, page, g, key % p.page_size) : 0u;
            for (int e = 0; found >> e; ++e) {
                if (!(found >> e & 1u)) continue;
                atomicMin(&none_from[i][e], key);
                atomicMax(&none_to[i][e], key);
            }
        }
    }
    __syncthreads();
    for (int i = tid >> 5; i < n; i += kRepairThreads / 32) {
        if (!spoilt[i]) continue;
        const int qi = (item0 + i) / p.nh, h = (item0 + i) % p.nh, g = h / group;
        const int pos = base + qi, lo = window_from(pos), few = few_before(lo);
        auto sees = [&](int key) { return key >= 0 && key <= pos && (key >= lo || key < few); };
        const int *from = none_from[owner[i]], *to = none_to[owner[i]];
        if (sees(from[kMaxDims]) || sees(to[kMaxDims])) {
            for (int d = lane; d < hd; d += 32) out[(size_t)i * hd + d] = __ushort_as_bfloat16((unsigned short)0x7fff);
            continue;
        }
        bool open = false;                                      // a NaN of which no such value is the reason
#pragma unroll
        for (int e = 0; e < kMaxDims; ++e) {
            const int d = lane + 32 * e;
            if (d >= hd || !isnan(__bfloat162float(out[(size_t)i * hd + d]))) continue;
            bool known = false;
            for (int end = 0; end < 2; ++end) {
                const int key = end ? to[e] : from[e];
                float k = 0.f, v = 0.f;
                if (!known && sees(key)) Cache::load(p, page_of(key), g, key % p.page_size, d, k, v);
                known = known || isnan(v);
            }
            open = open || !known;
        }
        if (!__any_sync(0xffffffffu, open)) continue;
        float q[kMaxDims], o[kMaxDims], m = -INFINITY, l = 0.f;
#pragma unroll
        for (int e = 0; e < kMaxDims; ++e) {
            o[e] = 0.f;
            q[e] = lane + 32 * e < hd ? __bfloat162float(p.q[(size_t)(qs + qi) * p.q_stride + h * hd + lane + 32 * e]) : 0.f;
        }
        for (int j = 0; j < few + pos - lo + 1; ++j) {
            const int key = j < few ? j : j - few + lo, page = page_of(key);
            if (page < 0) continue;
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
            if (l != l) break;                                  // (alike in all lanes) no number, whatever follows
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
    if (hd % 8 || hd > 32 * kMaxDims || n_requests > 65535 || (uintptr_t)out % 16 || (uintptr_t)k_pages % 16) return (int)cudaErrorInvalidValue;
    const RepairParams p{(const bf16*)qkv, qkv_stride, q_start, kv_len, table_rows, block_table, table_stride, (bf16*)out, nh, nkv, hd,
                         page_size, num_pages, scale, window, first, k_pages, v_pages};
    const dim3 grid((unsigned)(((long long)max_q_len * nh + kItems - 1) / kItems), 1, n_requests);
    return kv4 ? lsb_launch(attention_repair_kernel<Kv4>, grid, dim3(kRepairThreads), 0, stream, 1, p)
               : lsb_launch(attention_repair_kernel<Plain>, grid, dim3(kRepairThreads), 0, stream, 1, p);
}
