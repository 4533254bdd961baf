// A step's queries, keys and values on their way into a 4-bit cache, and back out of it.
//
// rope_kv4_store: for every token at position pos, each query and key head has its first `rotary_dim` dims rotated in
// split-half pairs (i, i + rotary_dim / 2) by pos * inv_freq[i]; queries go to q_out, keys (rounded to the compute type
// first, as an ordinary cache would hold them) and values are rounded to 4 bits (kv4.cuh) and written to page =
// table[row][pos / page_size].  The angle and a key's rotation are formed in 64-bit: a code flips where a value lies next to
// a border, and 32-bit angles are off by up to 2^-24 of themselves, 0.008 at position 131,072.  Queries take the 64-bit angle's
// sine and cosine in 32-bit.  The angles are shared by a token's heads.
//
// One block per token.  What bounds it is the projection it reads and the queries it writes; keys and values leave as 9/32
// of their bfloat16 bytes.
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

template <typename T>
__global__ void __launch_bounds__(kStoreThreads) rope_kv4_store_kernel(const StoreParams p) {
    __shared__ double cs64[2][kMaxDim / 2];
    __shared__ float cs[2][kMaxDim / 2];
    __shared__ __align__(16) unsigned char rows[kStoreThreads / 32][kMaxDim / 2];
    lsb_pdl_launch_dependents();
    const int t = blockIdx.x, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int hd = p.hd, half = p.rotary_dim >> 1;
    // (positions are metadata of the step, on the device before its first kernel: the angles need not wait for the projection)
    const int pos = p.positions[t];
    for (int i = tid; i < half; i += kStoreThreads) {
        sincos((double)pos * (double)p.inv_freq[i], &cs64[1][i], &cs64[0][i]);
        cs[0][i] = (float)cs64[0][i];
        cs[1][i] = (float)cs64[1][i];
    }
    __syncthreads();
    lsb_pdl_wait();
    const T* row = reinterpret_cast<const T*>(p.qkv) + (size_t)t * (p.nh + 2 * p.nkv) * hd;
    T* q = reinterpret_cast<T*>(p.q_out) + (size_t)t * p.nh * hd;

    if (p.vec) {
        const int quads = half >> 2, per = (hd >> 2) - quads;              // per head: fours of pairs, then the fours that pass
        for (int idx = tid; idx < p.nh * per; idx += kStoreThreads) {
            const int h = idx / per, c = idx - h * per;
            float a[4], b[4];
            if (c < quads) {
                const int i = 4 * c;
                Four<T>::load(row + h * hd + i, a);
                Four<T>::load(row + h * hd + half + i, b);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float x0 = a[e], x1 = b[e];
                    a[e] = x0 * cs[0][i + e] - x1 * cs[1][i + e];
                    b[e] = x0 * cs[1][i + e] + x1 * cs[0][i + e];
                }
                Four<T>::store(q + h * hd + i, a);
                Four<T>::store(q + h * hd + half + i, b);
            } else {
                const int i = 4 * (c + quads);
                Four<T>::load(row + h * hd + i, a);
                Four<T>::store(q + h * hd + i, a);
            }
        }
    } else {
        const int per = hd - half;
        for (int idx = tid; idx < p.nh * per; idx += kStoreThreads) {
            const int h = idx / per, c = idx - h * per;
            if (c < half) {
                const float x0 = lsb_to_float(row[h * hd + c]), x1 = lsb_to_float(row[h * hd + half + c]);
                q[h * hd + c] = lsb_from_float<T>(x0 * cs[0][c] - x1 * cs[1][c]);
                q[h * hd + half + c] = lsb_from_float<T>(x0 * cs[1][c] + x1 * cs[0][c]);
            } else {
                q[h * hd + half + c] = row[h * hd + half + c];
            }
        }
    }
    if (!p.store) return;

    int page = -1;
    if (pos / p.page_size < p.table_stride)
        page = p.block_table[(size_t)p.table_rows[p.token_req[t]] * p.table_stride + pos / p.page_size];
    if (page < 0 || page >= p.num_pages) {
        if (tid == 0) lsb_set_status(LSB_BAD_PAGE);
        return;
    }
    const int G = hd / kKv4Group, within = pos % p.page_size, r = within % kKv4Tile;
    for (int item = warp; item < 2 * p.nkv; item += kStoreThreads / 32) {
        const bool value = item >= p.nkv;
        const int h = value ? item - p.nkv : item;
        unsigned char* tile = p.pages + (((size_t)page * p.nkv + h) * (p.page_size / kKv4Tile) + within / kKv4Tile) * kv4_tile_bytes(hd);
        const T* x = row + (size_t)(p.nh + item) * hd;
        for (int base = 0; base < hd; base += 128) {            // four dims a lane, a group to eight lanes
            const int d0 = base + 4 * lane;
            float y[4] = {0.f, 0.f, 0.f, 0.f};
            if (d0 < hd) {
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int d = d0 + e;
                    y[e] = lsb_to_float(x[d]);
                    if (!value && d < 2 * half) {
                        const int i = d < half ? d : d - half;
                        const double x0 = d < half ? (double)y[e] : (double)lsb_to_float(x[i]);
                        const double x1 = d < half ? (double)lsb_to_float(x[i + half]) : (double)y[e];
                        const double z = d < half ? x0 * cs64[0][i] - x1 * cs64[1][i] : x0 * cs64[1][i] + x1 * cs64[0][i];
                        y[e] = lsb_to_float(lsb_from_float<T>((float)z));
                    }
                }
            }
            float top = 0.f;
            bool fine = true;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                fine = fine && fabsf(y[e]) <= FLT_MAX;
                top = fmaxf(top, fabsf(y[e]));
            }
#pragma unroll
            for (int o = 1; o < 8; o <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
            fine = (__ballot_sync(0xffffffffu, fine) >> (lane & 24) & 0xffu) == 0xffu;
            const float s = fine ? kv4_scale(top) : 0.f;
            uint32_t code = 0;
#pragma unroll
            for (int e = 0; e < 4; ++e) code |= (uint32_t)(kv4_code(y[e], s) + 8) << (4 * e);
            if (d0 < hd) {
                const int g = d0 / kKv4Group, o = lane & 7;
                if (value) {
                    const int i = 2 * g + (o >> 2), e = 2 * (o & 3);
                    rows[warp][e * 2 * G + i] = (unsigned char)(code & 0xffu);
                    rows[warp][(e + 1) * 2 * G + i] = (unsigned char)(code >> 8);
                } else {
                    *reinterpret_cast<unsigned short*>(&rows[warp][((o >> 1) * G + g) * 4 + (o & 1) * 2]) = (unsigned short)code;
                }
                if (o == 0) {
                    const int at = (value ? kv4_value_scales_at(hd) : kv4_key_scales_at(hd)) + (r * G + g) * 2;
                    *reinterpret_cast<__nv_bfloat16*>(tile + at) =
                        fine ? __float2bfloat16_rn(s) : __ushort_as_bfloat16((unsigned short)0x7fff);
                }
            }
        }
        __syncwarp();
        uint32_t* to = reinterpret_cast<uint32_t*>(tile + (value ? kv4_values_at(hd) : 0) + r * (hd / 2));
        for (int w = lane; w < hd / 8; w += 32) to[w] = reinterpret_cast<const uint32_t*>(rows[warp])[w];
        __syncwarp();
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
// A block for each tile of a kv head; it moves 18 hd bytes in and 64 hd out.
__global__ void __launch_bounds__(128) expand_kv4_kernel(const unsigned char* pages, const int* q_start, const int* kv_len, const int* table_rows,
                                                         const int* block_table, int table_stride, __nv_bfloat16* k_out,
                                                         __nv_bfloat16* v_out, int* table_out, int* rows_out, int* expanded,
                                                         int room, int nkv, int hd, int page_size, int num_pages, int window, int first) {
    // (The attention behind it reads lengths and rows before it waits, as a step's metadata may be read: it must not start before
    // they are there, so this kernel lets nothing start early.)
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
    LSB_DISPATCH_DTYPE(dtype, return lsb_launch(rope_kv4_store_kernel<T>, dim3(n_tokens), dim3(kStoreThreads), 0, stream, 1, p));
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
