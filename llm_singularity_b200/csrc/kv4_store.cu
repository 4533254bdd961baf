// A step's queries, keys and values on their way into a 4-bit cache, and back out of it.
//
// rope_kv4_store: for every token at position pos, each query and key head has its first `rotary_dim` dims rotated in
// split-half pairs (i, i + rotary_dim / 2) by pos * inv_freq[i]; queries go to q_out, keys (rounded to the compute type
// first, as an ordinary cache would hold them) and values are rounded to 4 bits (kv4.cuh) and written to page =
// table[row][pos / page_size].  The angle and a key's rotation are formed in 64-bit: a code flips where a value lies next to
// a border, and 32-bit angles are off by up to 2^-24 of themselves, 0.008 at position 131,072.  Queries take the 64-bit angle's
// sine and cosine in 32-bit.  The angles are shared by a token's heads.
//
// One block per token; keys and values leave as 9/32 of their bfloat16 bytes.  2,011 tokens of 32 / 8 heads of 128 take 21.5 us where
// their bytes would take 6.6: a block's start (its position, 64-bit sines, a barrier) comes before its first load, and then that load is
// waited for; 57 % of issue slots (775 instructions a warp), 54 % of an SM's warps and 13 % of DRAM are in use.  (With a head size known
// at launch only, a 64-bit division per code and keys passed through shared memory it took 27.)  A step of single tokens is a
// launch: 3 us.
#include "kv4.cuh"

LSB_DEFINE_STATUS()

constexpr int kStoreThreads = 256;
constexpr int kMaxDim = 256;

struct StoreParams {
    const void* qkv;                            // [tokens, (nh + 2 nkv) * hd]
    void* q_out;                                // [tokens, nh * hd]
    const float* inv_freq;
    int rotary_dim;
    const int *positions, *token_req, *table_rows, *block_table;
    int table_stride;
    unsigned char* pages;
    int nh, nkv, hd, page_size, num_pages, store;
    int vec;                                    // four elements at a time: addresses allow it and pairs come in fours
};

template <typename T> struct Four;
template <> struct Four<float> {
    static __device__ __forceinline__ void load(const float* p, float (&f)[4]) {
        const float4 v = *reinterpret_cast<const float4*>(p);
        f[0] = v.x; f[1] = v.y; f[2] = v.z; f[3] = v.w;
    }
    static __device__ __forceinline__ void store(float* p, const float (&f)[4]) {
        *reinterpret_cast<float4*>(p) = make_float4(f[0], f[1], f[2], f[3]);
    }
};
template <> struct Four<__nv_bfloat16> {
    static __device__ __forceinline__ void load(const __nv_bfloat16* p, float (&f)[4]) {
        const uint2 v = *reinterpret_cast<const uint2*>(p);
        f[0] = __uint_as_float(v.x << 16); f[1] = __uint_as_float(v.x & 0xffff0000u);
        f[2] = __uint_as_float(v.y << 16); f[3] = __uint_as_float(v.y & 0xffff0000u);
    }
    static __device__ __forceinline__ void store(__nv_bfloat16* p, const float (&f)[4]) {
        const __nv_bfloat162 a = __floats2bfloat162_rn(f[0], f[1]), b = __floats2bfloat162_rn(f[2], f[3]);
        *reinterpret_cast<uint2*>(p) = make_uint2(*reinterpret_cast<const uint32_t*>(&a), *reinterpret_cast<const uint32_t*>(&b));
    }
};

// One element of a head at x, rotated in 64-bit by the token's angles and rounded to the type.
template <typename T>
__device__ __forceinline__ float turned(const T* x, int d, int half, const double (*cs)[kMaxDim / 2]) {
    if (d >= 2 * half) return lsb_to_float(x[d]);
    const bool low = d < half;
    const int i = low ? d : d - half;
    const double own = (double)lsb_to_float(x[d]), other = (double)lsb_to_float(x[low ? d + half : i]);
    return lsb_to_float(lsb_from_float<T>((float)(other * (low ? -cs[1][i] : cs[1][i]) + own * cs[0][i])));
}

// A lane takes four dims of the token's keys and values, as they stand side by side in the projection, eight lanes a group; its
// codes are half a word of a key's row, or two bytes of a value's, which meet their neighbours' by a shuffle.
template <int G, typename T>
__global__ void __launch_bounds__(kStoreThreads) rope_kv4_store_kernel(const StoreParams p) {
    constexpr int HD = kKv4Group * G, TILE = kv4_tile_bytes(HD);
    __shared__ __align__(16) double cs64[2][kMaxDim / 2];
    __shared__ __align__(16) float cs[2][kMaxDim / 2];
    __shared__ long long place;                                 // tile of the token in the pool's first head, -1 for none
    __shared__ int offset;                                      // its row there
    lsb_pdl_launch_dependents();
    const int t = blockIdx.x, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int half = p.rotary_dim >> 1;
    // (positions are metadata of the step, on the device before its first kernel: the angles need not wait for the projection)
    const int pos = p.positions[t];
    for (int i = tid; i < half; i += kStoreThreads) {
        double sine, cosine;
        sincos((double)pos * (double)p.inv_freq[i], &sine, &cosine);
        cs64[0][i] = cosine;
        cs64[1][i] = sine;
        cs[0][i] = (float)cosine;
        cs[1][i] = (float)sine;
    }
    lsb_pdl_wait();
    if (tid == kStoreThreads - 1) {                             // (of the warp that has the fewest angles)
        const int pi = pos / p.page_size, within = pos - pi * p.page_size;
        int page = -1;
        if (p.store && pos >= 0 && pi < p.table_stride) page = p.block_table[(size_t)p.table_rows[p.token_req[t]] * p.table_stride + pi];
        const bool held = page >= 0 && page < p.num_pages;
        if (p.store && !held) lsb_set_status(LSB_BAD_PAGE);
        place = held ? (long long)page * p.nkv * (p.page_size / kKv4Tile) + within / kKv4Tile : -1;
        offset = within % kKv4Tile;
    }
    __syncthreads();
    const T* row = reinterpret_cast<const T*>(p.qkv) + (size_t)t * (p.nh + 2 * p.nkv) * HD;
    T* q = reinterpret_cast<T*>(p.q_out) + (size_t)t * p.nh * HD;

    if (p.vec) {
        const int quads = half >> 2, per = HD / 4 - quads;                 // per head: fours of pairs, then the fours that pass
        const int step_h = kStoreThreads / per, step_c = kStoreThreads - step_h * per;
        for (int h = tid / per, c = tid - h * per; h < p.nh; h += step_h, c += step_c) {
            if (c >= per) { c -= per; if (++h >= p.nh) break; }
            const T* from = row + h * HD;
            T* to = q + h * HD;
            float a[4], b[4];
            if (c < quads) {
                const int i = 4 * c;
                Four<T>::load(from + i, a);
                Four<T>::load(from + half + i, b);
                const float4 cosine = *reinterpret_cast<const float4*>(&cs[0][i]), sine = *reinterpret_cast<const float4*>(&cs[1][i]);
                const float c4[4] = {cosine.x, cosine.y, cosine.z, cosine.w}, s4[4] = {sine.x, sine.y, sine.z, sine.w};
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float x0 = a[e], x1 = b[e];
                    a[e] = x0 * c4[e] - x1 * s4[e];
                    b[e] = x0 * s4[e] + x1 * c4[e];
                }
                Four<T>::store(to + i, a);
                Four<T>::store(to + half + i, b);
            } else {
                Four<T>::load(from + 4 * (c + quads), a);
                Four<T>::store(to + 4 * (c + quads), a);
            }
        }
    } else {
        const int per = HD - half;
        for (int idx = tid; idx < p.nh * per; idx += kStoreThreads) {
            const int h = idx / per, c = idx - h * per;
            if (c < half) {
                const float x0 = lsb_to_float(row[h * HD + c]), x1 = lsb_to_float(row[h * HD + half + c]);
                q[h * HD + c] = lsb_from_float<T>(x0 * cs[0][c] - x1 * cs[1][c]);
                q[h * HD + half + c] = lsb_from_float<T>(x0 * cs[1][c] + x1 * cs[0][c]);
            } else {
                q[h * HD + half + c] = row[h * HD + half + c];
            }
        }
    }
    if (place < 0) return;

    const int r = offset, o = lane & 7, tiles = p.page_size / kKv4Tile, n = 2 * p.nkv * HD;
    unsigned char* tile0 = p.pages + place * TILE;
    for (int base = warp * 128; base < n; base += kStoreThreads * 4) {
        const int f = base + 4 * lane, item = f / HD, d0 = f - item * HD, g = d0 / kKv4Group;
        const bool there = f < n, value = item >= p.nkv;
        const T* x = row + (size_t)(p.nh + item) * HD;
        float y[4] = {0.f, 0.f, 0.f, 0.f};
        if (there && p.vec) {                                   // the four are of a pair's first dims, of its second ones or of none
            Four<T>::load(x + d0, y);
            if (!value && d0 < 2 * half) {
                const bool low = d0 < half;
                const int i = low ? d0 : d0 - half;
                float other[4];
                Four<T>::load(x + (low ? d0 + half : i), other);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const double sine = low ? -cs64[1][i + e] : cs64[1][i + e];
                    y[e] = lsb_to_float(lsb_from_float<T>((float)((double)other[e] * sine + (double)y[e] * cs64[0][i + e])));
                }
            }
        } else if (there) {
#pragma unroll
            for (int e = 0; e < 4; ++e) y[e] = value ? lsb_to_float(x[d0 + e]) : turned(x, d0 + e, half, cs64);
        }
        float zero = 0.f;                                       // times a number 0, times anything else NaN
#pragma unroll
        for (int e = 0; e < 4; ++e) zero = fmaf(y[e], 0.f, zero);
        bool fine = zero == 0.f;
        float top = fmaxf(fmaxf(fabsf(y[0]), fabsf(y[1])), fmaxf(fabsf(y[2]), fabsf(y[3])));
#pragma unroll
        for (int k = 1; k < 8; k <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, k));
        fine = (__ballot_sync(0xffffffffu, fine) >> (lane & 24) & 0xffu) == 0xffu;
        const float s = fine ? kv4_scale(top) : 0.f, inverse = s > 0.f ? __fdividef(1.f, s) : 0.f;
        uint32_t code = 0;
#pragma unroll
        for (int e = 0; e < 4; ++e) code |= kv4_code(s > 0.f ? y[e] : 0.f, s, inverse) << (4 * e);
        const uint32_t pair = __shfl_xor_sync(0xffffffffu, code, 1), across = __shfl_xor_sync(0xffffffffu, code, 4);
        if (!there) continue;
        unsigned char* tile = tile0 + (size_t)(value ? item - p.nkv : item) * tiles * TILE;
        if (value) {                                            // dims 16 i + 2 e and + 1: i = 2 g + o / 4, e = 2 (o % 4) and + 1
            const bool front = o < 4;
            const uint32_t two = front ? (code & 0xffu) | (across & 0xffu) << 8 : (across >> 8 & 0xffu) | (code >> 8 & 0xffu) << 8;
            *reinterpret_cast<unsigned short*>(tile + kv4_values_at(HD) + r * (HD / 2) + (2 * (o & 3) + (front ? 0 : 1)) * 2 * G + 2 * g) = (unsigned short)two;
        } else if (!(o & 1)) {                                  // dims 8 t .. 8 t + 7 of the group: t = o / 2
            *reinterpret_cast<uint32_t*>(tile + r * (HD / 2) + ((o >> 1) * G + g) * 4) = code | pair << 16;
        }
        if (o == 0)
            *reinterpret_cast<__nv_bfloat16*>(tile + (value ? kv4_value_scales_at(HD) : kv4_key_scales_at(HD)) + (r * G + g) * 2) =
                fine ? __float2bfloat16_rn(s) : __ushort_as_bfloat16((unsigned short)0x7fff);
    }
}

// What the cache holds for token i, at positions[i] of the request with block-table row token_rows[i]: keys and values
// [tokens, nkv, hd] in the compute type.  Eight dims of a head a thread.
template <typename T>
__global__ void __launch_bounds__(256) read_kv4_kernel(const unsigned char* pages, const int* token_rows, const int* positions,
                                                       const int* block_table, int table_stride, int slots, T* k_out, T* v_out,
                                                       int n, int nkv, int hd, int page_size, int num_pages) {
    lsb_pdl_launch_dependents();
    lsb_pdl_wait();
    const int per = hd / 8, G = hd / kKv4Group;
    const long long idx = (long long)blockIdx.x * blockDim.x + threadIdx.x;
    if (idx >= (long long)n * 2 * nkv * per) return;
    const int c = (int)(idx % per);
    const int item = (int)(idx / per % (2 * nkv)), i = (int)(idx / per / (2 * nkv));
    const bool value = item >= nkv;
    const int h = value ? item - nkv : item;
    const int pos = positions[i], slot = token_rows[i];
    int page = -1;
    if (slot >= 0 && slot < slots && pos >= 0 && pos / page_size < table_stride)
        page = block_table[(size_t)slot * table_stride + pos / page_size];
    T* out = (value ? v_out : k_out) + ((size_t)i * nkv + h) * hd + 8 * c;
    float f[8];
    if (page < 0 || page >= num_pages) {
        lsb_set_status(LSB_BAD_PAGE);
#pragma unroll
        for (int e = 0; e < 8; ++e) f[e] = 0.f;
    } else {
        const int within = pos % page_size, r = within % kKv4Tile, g = c / 4;
        const unsigned char* tile = pages + (((size_t)page * nkv + h) * (page_size / kKv4Tile) + within / kKv4Tile) * kv4_tile_bytes(hd);
        uint32_t word;                                          // codes of dims 8 c .. 8 c + 7, in order
        if (value) {
            const unsigned char* v = tile + kv4_values_at(hd) + r * (hd / 2) + c / 2;
            const int e = c % 2 * 4;
            word = v[e * 2 * G] | v[(e + 1) * 2 * G] << 8 | v[(e + 2) * 2 * G] << 16 | (uint32_t)v[(e + 3) * 2 * G] << 24;
        } else {
            word = *reinterpret_cast<const uint32_t*>(tile + r * (hd / 2) + (c % 4 * G + g) * 4);
        }
        const float s = __bfloat162float(*reinterpret_cast<const __nv_bfloat16*>(
            tile + (value ? kv4_value_scales_at(hd) : kv4_key_scales_at(hd)) + (r * G + g) * 2));
#pragma unroll
        for (int e = 0; e < 8; ++e) f[e] = (float)((int)(word >> (4 * e) & 15u) - 8) * s;
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) out[e] = lsb_from_float<T>(f[e]);
}

// What the portions of a step see of their 4-bit caches, as an ordinary cache in bfloat16 with pages of one tile, for the prompt
// attention that reads its tiles as tensors: exact (kv4.cuh).  The tiles of first tokens and those from the oldest row's window on
// stand side by side, so positions behind the gap are `gap` (a multiple of 16) less there: expanded[r] is the length that
// the attention is to take request r for.  Tokens that are not there yet read as zeros (their weights are zeros, and zero times
// what a page held before may be no number).
// A block for each tile of a kv head; it moves 18 hd bytes in and 64 hd out: 14 us for 6,107 tokens of 8 heads of
// 128 (32 MB, mostly written).
__global__ void __launch_bounds__(128) expand_kv4_kernel(const unsigned char* pages, const int* q_start, const int* kv_len, const int* table_rows,
                                                         const int* block_table, int table_stride, __nv_bfloat16* k_out,
                                                         __nv_bfloat16* v_out, int* table_out, int* rows_out, int* expanded,
                                                         int room, int nkv, int hd, int page_size, int num_pages, int window, int first) {
    // (No early start for the attention behind it, which reads `expanded` and rows_out before anything else: it is launched to begin
    // when this kernel has ended, lsb_prefill_attention_tc5_first's `fresh_lengths`.)
    const int c = blockIdx.x, h = blockIdx.y, r = blockIdx.z, tid = threadIdx.x;
    const int q_len = q_start[r + 1] - q_start[r], len = kv_len[r], p_lo = len - q_len;
    const int near = (window > 0 && p_lo - window + 1 > 0 ? p_lo - window + 1 : 0) / kKv4Tile;
    const int early = window > 0 ? min((first + kKv4Tile - 1) / kKv4Tile, near) : 0, gap = (near - early) * kKv4Tile;
    const int place = r * room + c;
    lsb_pdl_wait();
    if (h == 0 && tid == 0) {
        table_out[place] = place;
        if (c == 0) {
            expanded[r] = len - gap;
            rows_out[r] = r;
        }
    }
    const int pos0 = (c < early ? c : c - early + near) * kKv4Tile, pi = pos0 / page_size;
    if (q_len == 1 || pos0 >= len) return;                              // (single tokens are another kernel's)
    const int page = pi < table_stride ? block_table[(size_t)table_rows[r] * table_stride + pi] : -1;
    const bool held = page >= 0 && page < num_pages;
    if (!held && tid == 0) lsb_set_status(LSB_BAD_PAGE);
    const unsigned char* tile = pages + (((size_t)(held ? page : 0) * nkv + h) * (page_size / kKv4Tile) + pos0 % page_size / kKv4Tile) * kv4_tile_bytes(hd);
    const int per = hd / 8, G = hd / kKv4Group;
    for (int i = tid; i < 2 * kKv4Tile * per; i += 128) {
        const bool value = i >= kKv4Tile * per;
        const int j = value ? i - kKv4Tile * per : i, t = j / per, d8 = j - t * per, g = d8 / 4;
        uint4 packed = make_uint4(0, 0, 0, 0);
        if (held && pos0 + t < len) {
            uint32_t word;                                              // codes of dims 8 d8 .. 8 d8 + 7, in order
            if (value) {
                const unsigned char* v = tile + kv4_values_at(hd) + t * (hd / 2) + d8 / 2;
                const int e = d8 % 2 * 4;
                word = v[e * 2 * G] | v[(e + 1) * 2 * G] << 8 | v[(e + 2) * 2 * G] << 16 | (uint32_t)v[(e + 3) * 2 * G] << 24;
            } else {
                word = *reinterpret_cast<const uint32_t*>(tile + t * (hd / 2) + (d8 % 4 * G + g) * 4);
            }
            const float s = __bfloat162float(*reinterpret_cast<const __nv_bfloat16*>(
                tile + (value ? kv4_value_scales_at(hd) : kv4_key_scales_at(hd)) + (t * G + g) * 2));
            uint32_t w[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const __nv_bfloat162 y = __floats2bfloat162_rn((float)((int)(word >> (8 * k) & 15u) - 8) * s,
                                                               (float)((int)(word >> (8 * k + 4) & 15u) - 8) * s);
                w[k] = *reinterpret_cast<const uint32_t*>(&y);
            }
            packed = make_uint4(w[0], w[1], w[2], w[3]);
        }
        *reinterpret_cast<uint4*>((value ? v_out : k_out) + (((size_t)place * nkv + h) * kKv4Tile + t) * hd + 8 * d8) = packed;
    }
}

// `room`: tiles that each request has in k_out and v_out [requests * room, nkv, 16, hd]; table_out [requests, room].
LSB_API int lsb_expand_kv4(const void* pages, const int* q_start, const int* kv_len, const int* table_rows, const int* block_table,
                           int table_stride, void* k_out, void* v_out, int* table_out, int* rows_out, int* expanded,
                           int n_requests, int room, int nkv, int hd, int page_size, int num_pages, int window, int first,
                           cudaStream_t stream) {
    if (n_requests <= 0 || room <= 0) return 0;
    if (nkv > 65535 || n_requests > 65535) return (int)cudaErrorInvalidValue;
    return lsb_launch(expand_kv4_kernel, dim3(room, nkv, n_requests), dim3(128), 0, stream, 1, (const unsigned char*)pages, q_start, kv_len,
                      table_rows, block_table, table_stride, (__nv_bfloat16*)k_out, (__nv_bfloat16*)v_out, table_out, rows_out, expanded,
                      room, nkv, hd, page_size, num_pages, window, first);
}

LSB_API int lsb_rope_kv4_store(const void* qkv, int dtype, int n_tokens, int nh, int nkv, int hd, const int* positions,
                               const int* token_req, const int* table_rows, const int* block_table, int table_stride,
                               const float* inv_freq, int rotary_dim, void* q_out, void* pages, int page_size, int num_pages,
                               int store, cudaStream_t stream) {
    if (n_tokens <= 0) return 0;
    StoreParams p;
    p.qkv = qkv; p.q_out = q_out; p.inv_freq = inv_freq; p.rotary_dim = rotary_dim;
    p.positions = positions; p.token_req = token_req; p.table_rows = table_rows; p.block_table = block_table;
    p.table_stride = table_stride; p.pages = (unsigned char*)pages;
    p.nh = nh; p.nkv = nkv; p.hd = hd; p.page_size = page_size; p.num_pages = num_pages; p.store = store;
    p.vec = rotary_dim % 8 == 0 && (uintptr_t)qkv % 16 == 0 && (uintptr_t)q_out % 16 == 0;
    const dim3 grid(n_tokens), block(kStoreThreads);
    LSB_DISPATCH_DTYPE(dtype, {
        switch (hd) {
            case 32: return lsb_launch(rope_kv4_store_kernel<1, T>, grid, block, 0, stream, 1, p);
            case 64: return lsb_launch(rope_kv4_store_kernel<2, T>, grid, block, 0, stream, 1, p);
            case 96: return lsb_launch(rope_kv4_store_kernel<3, T>, grid, block, 0, stream, 1, p);
            case 128: return lsb_launch(rope_kv4_store_kernel<4, T>, grid, block, 0, stream, 1, p);
            case 160: return lsb_launch(rope_kv4_store_kernel<5, T>, grid, block, 0, stream, 1, p);
            case 192: return lsb_launch(rope_kv4_store_kernel<6, T>, grid, block, 0, stream, 1, p);
            case 224: return lsb_launch(rope_kv4_store_kernel<7, T>, grid, block, 0, stream, 1, p);
            case 256: return lsb_launch(rope_kv4_store_kernel<8, T>, grid, block, 0, stream, 1, p);
        }
        return (int)cudaErrorInvalidValue;
    });
}

LSB_API int lsb_read_kv4(const void* pages, const int* token_rows, const int* positions, const int* block_table, int table_stride,
                         int slots, void* k_out, void* v_out, int dtype, int n, int nkv, int hd, int page_size, int num_pages,
                         cudaStream_t stream) {
    if (n <= 0) return 0;
    const long long threads = (long long)n * 2 * nkv * (hd / 8);
    LSB_DISPATCH_DTYPE(dtype, return lsb_launch(read_kv4_kernel<T>, dim3((unsigned)((threads + 255) / 256)), dim3(256), 0, stream, 1,
                                                (const unsigned char*)pages, token_rows, positions, block_table, table_stride, slots,
                                                (T*)k_out, (T*)v_out, n, nkv, hd, page_size, num_pages));
}
