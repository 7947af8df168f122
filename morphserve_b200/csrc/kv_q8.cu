// Into and out of the 8-bit pool: prefill scatter, decode append, and the gather back to rows of the model's type.
// HBM / latency bound; the number format is kv_q8.cuh's.
#include <string.h>

#include <algorithm>
#include <type_traits>

#include "kv_q8.cuh"

namespace mkv {

int validate_pool_q8(const mkv_pool_q8 *pool, PoolViewQ8 *out) {
    if (!pool) return MKV_ERR_NULL;
    if (pool->num_segments < 1 || pool->num_segments > MKV_MAX_SEGMENTS) return MKV_ERR_SHAPE;
    if (pool->code != MKV_Q8_INT8 && pool->code != MKV_Q8_E4M3) return MKV_ERR_DTYPE;
    if (pool->num_layers < 1 || pool->num_kv_heads < 1 || pool->block_size < 1 || pool->head_dim < 1) return MKV_ERR_SHAPE;
    if ((int64_t)pool->block_size * pool->head_dim > (1 << 24)) return MKV_ERR_SHAPE;
    if ((int64_t)pool->block_size * pool->head_dim * pool->num_kv_heads > (1 << 30)) return MKV_ERR_SHAPE;  // a page is counted in 32 bits
    if (pool->num_blocks_org < 0 || (pool->num_segments > 1 && pool->chunk_blocks < 1)) return MKV_ERR_SHAPE;
    PoolViewQ8 v;
    memset(&v, 0, sizeof(v));
    v.num_segments = pool->num_segments;
    v.code = pool->code;
    v.num_layers = pool->num_layers;
    v.num_kv_heads = pool->num_kv_heads;
    v.block_size = pool->block_size;
    v.head_dim = pool->head_dim;
    v.num_blocks_org = pool->num_blocks_org;
    v.chunk_blocks = pool->num_segments > 1 ? pool->chunk_blocks : 1;
    v.total_blocks = pool->num_blocks_org + (int64_t)(pool->num_segments - 1) * v.chunk_blocks;
    v.tile_bytes = (int64_t)pool->block_size * pool->head_dim;
    for (int i = 0; i < pool->num_segments; ++i) {
        const bool empty_org = i == 0 && pool->num_blocks_org == 0;
        if (!empty_org && (!pool->k_base[i] || !pool->v_base[i] || !pool->k_scale[i] || !pool->v_scale[i])) return MKV_ERR_NULL;
        if ((((uintptr_t)pool->k_scale[i] | (uintptr_t)pool->v_scale[i]) & 3) != 0) return MKV_ERR_ALIGN;
        v.k_base[i] = (uint8_t *)pool->k_base[i];
        v.v_base[i] = (uint8_t *)pool->v_base[i];
        v.k_scale[i] = pool->k_scale[i];
        v.v_scale[i] = pool->v_scale[i];
    }
    *out = v;
    return MKV_OK;
}

// Page of logical block `lb` of table row `row`: its tile index for (layer, head 0), or -1 if it is not there.
__device__ __forceinline__ int64_t page_of(const PoolViewQ8 &p, const int32_t *table, int64_t cols, int num_rows, int row,
                                           int lb, int layer, int &seg) {
    if (row < 0 || row >= num_rows || lb >= cols) return -1;
    const int64_t blk = __ldg(table + (int64_t)row * cols + lb);
    if (blk < 0 || blk >= p.total_blocks) return -1;
    int64_t r;
    locate_block(p, blk, seg, r);
    return tile_index(p, r, layer, 0);
}

// ------------------------------------------------------------------ access
// A thread's piece of a row: V elements of T, V codes.  V = 16: 32 bytes of a 16-bit type in one access (64 of fp32 in two), 16
// bytes of codes.  V = 1 for rows that are not so aligned.
template <typename T, int V>
struct Piece {
    static constexpr int WORDS = V * (int)sizeof(T) / 4;
    uint32_t w[WORDS];
    __device__ __forceinline__ void load(const T *src) {
#pragma unroll
        for (int i = 0; i < WORDS; i += 8)
            asm("ld.global.v8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];\n"
                         : "=r"(w[i]), "=r"(w[i + 1]), "=r"(w[i + 2]), "=r"(w[i + 3]), "=r"(w[i + 4]), "=r"(w[i + 5]), "=r"(w[i + 6]),
                           "=r"(w[i + 7])
                         : "l"(reinterpret_cast<const uint32_t *>(src) + i));
    }
    __device__ __forceinline__ void store(T *dst) const {
#pragma unroll
        for (int i = 0; i < WORDS; i += 8)
            asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};\n" ::"l"(reinterpret_cast<uint32_t *>(dst) + i), "r"(w[i]),
                         "r"(w[i + 1]), "r"(w[i + 2]), "r"(w[i + 3]), "r"(w[i + 4]), "r"(w[i + 5]), "r"(w[i + 6]), "r"(w[i + 7])
                         : "memory");
    }
    __device__ __forceinline__ float get(int i) const {
        if constexpr (sizeof(T) == 4) return __uint_as_float(w[i]);
        else if constexpr (std::is_same<T, __half>::value) {
            const __half2 h = *reinterpret_cast<const __half2 *>(&w[i >> 1]);
            return (i & 1) ? __high2float(h) : __low2float(h);
        } else
            return __uint_as_float((i & 1) ? w[i >> 1] & 0xffff0000u : w[i >> 1] << 16);
    }
    __device__ __forceinline__ void set2(int i, float a, float b) {     // elements i, i + 1
        if constexpr (sizeof(T) == 4) {
            w[i] = __float_as_uint(a);
            w[i + 1] = __float_as_uint(b);
        } else {
            struct alignas(4) Two { T x, y; } t{rounded<T>(a), rounded<T>(b)};
            w[i >> 1] = *reinterpret_cast<const uint32_t *>(&t);
        }
    }
    // Largest absolute value, as the type's own bits (16-bit types: two maxima side by side): the integer order puts
    // infinity and NaN on top.  peak_bits() makes an fp32 number's bits of it.
    __device__ __forceinline__ uint32_t peak(uint32_t most) const {
#pragma unroll
        for (int i = 0; i < WORDS; ++i)
            most = sizeof(T) == 4 ? max(most, w[i] & 0x7fffffffu) : __vmaxu2(most, w[i] & 0x7fff7fffu);
        return most;
    }
    static __device__ __forceinline__ uint32_t peak_bits(uint32_t most) {
        if constexpr (sizeof(T) == 4) return most;
        const uint32_t m = max(most & 0xffffu, most >> 16);
        if constexpr (std::is_same<T, __half>::value) return __float_as_uint(__half2float(__ushort_as_half((unsigned short)m)));
        return m << 16;
    }
    template <int CODE>
    __device__ __forceinline__ void store_codes(uint8_t *dst, float inv) const {
        uint32_t c[V / 4];
#pragma unroll
        for (int i = 0; i < V / 4; ++i)
            c[i] = inv > 0.f ? encode4<CODE>(get(4 * i), get(4 * i + 1), get(4 * i + 2), get(4 * i + 3), inv) : 0u;
        *reinterpret_cast<uint4 *>(dst) = make_uint4(c[0], c[1], c[2], c[3]);
    }
};
template <typename T>
struct Piece<T, 1> {
    T x;
    __device__ __forceinline__ void load(const T *src) { x = *src; }
    __device__ __forceinline__ uint32_t peak(uint32_t most) const { return max(most, __float_as_uint(value_of<T>(x)) & 0x7fffffffu); }
    static __device__ __forceinline__ uint32_t peak_bits(uint32_t most) { return most; }
    template <int CODE>
    __device__ __forceinline__ void store_codes(uint8_t *dst, float inv) const {
        *dst = inv > 0.f ? encode1<CODE>(value_of<T>(x), inv) : (uint8_t)0;
    }
};

struct StoreQ8Args {
    const void *k, *v;
    int64_t k_stride, v_stride, num_tokens;
    const int32_t *block_table;
    int64_t table_cols;
    const int32_t *seq_ids, *start_locs, *seq_lens;
    int num_rows, num_seqs, cur_layer;
    uint32_t vecs_magic;        // ceil(2^32 / pieces of a row)
    PoolViewQ8 pool;
};

// Threads of a block: one warp for each head of a page, up to 8 (the decode append: for each (head, K or V), up to 16);
// the grid's last dimension takes the heads behind those.
constexpr int kHeadWarps = 8, kItemWarps = 16;
constexpr int kLoadThreads = 256, kLoadFlight = 4;

// Whether a later entry with tokens names the same sequence: then that one counts.  (All threads of the block.)
__device__ __forceinline__ bool named_again(const StoreQ8Args &a, int i, int row) {
    bool again = false;
    for (int j = i + 1 + threadIdx.x; j < a.num_seqs; j += blockDim.x) again |= a.seq_ids[j] == row && a.seq_lens[j] > 0;
    return __syncthreads_or(again);
}

// ------------------------------------------------------------------ prefill scatter
// grid = (pages of the longest prompt, prompts, heads / 8).  A warp takes one head of a page, K and then V: the rows go into registers with
// every load in flight at once (NV pieces a thread; 4 KiB a warp at 16 x 128 fp16), the peak is a butterfly, the codes leave
// as one contiguous tile.  NV = 0: pages that do not fit are read twice.
// HBM bound: 64 prompts of up to 1536 tokens, 8 heads of 128 fp16, 54 us = 5.8 TB/s read and written (copy peak 6.55).  Half
// occupancy (64 registers a thread): the variants with four pieces of 16-bit rows spill 12 to 16 bytes.
template <typename T, int CODE, int V, int NV>
__device__ __forceinline__ float store_tile(const StoreQ8Args &a, const T *src, int64_t stride, uint8_t *dst, int total, int vecs, int lane) {
    uint32_t peak = 0;
    if constexpr (NV > 0) {
        Piece<T, V> x[NV];
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int e = min(lane + 32 * j, total - 1), tok = (int)__umulhi((uint32_t)e, a.vecs_magic);  // behind the end: the last one again
            x[j].load(src + tok * (int)stride + (e - tok * vecs) * V);  // (wide_ok: a page's rows are counted in 32 bits)
        }
#pragma unroll
        for (int j = 0; j < NV; ++j) peak = x[j].peak(peak);
        const float s = scale_of<CODE>(__reduce_max_sync(0xffffffffu, Piece<T, V>::peak_bits(peak))), inv = inverse_of(s);
#pragma unroll
        for (int j = 0; j < NV; ++j)
            if (lane + 32 * j < total) x[j].template store_codes<CODE>(dst + (lane + 32 * j) * V, inv);
        return s;
    } else {
        Piece<T, V> x;
        for (int e = lane; e < total; e += 32) {
            x.load(src + (e / vecs) * stride + (e % vecs) * V);
            peak = x.peak(peak);
        }
        const float s = scale_of<CODE>(__reduce_max_sync(0xffffffffu, Piece<T, V>::peak_bits(peak))), inv = inverse_of(s);
        for (int e = lane; e < total; e += 32) {
            x.load(src + (e / vecs) * stride + (e % vecs) * V);
            x.template store_codes<CODE>(dst + (int64_t)e * V, inv);
        }
        return s;
    }
}

template <typename T, int CODE, int V, int NV>
__global__ void __launch_bounds__(kHeadWarps * 32, sizeof(T) == 4 ? 2 : 4) store_q8_prefill_kernel(const __grid_constant__ StoreQ8Args a) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
    const int D = a.pool.head_dim, bs = a.pool.block_size, Hkv = a.pool.num_kv_heads, vecs = D / V;
    for (int i = blockIdx.y; i < a.num_seqs; i += gridDim.y) {
        const int row = a.seq_ids[i];
        const int64_t start = a.start_locs[i];
        const int len = (int)min((int64_t)a.seq_lens[i], start < 0 ? 0 : a.num_tokens - start);
        if ((int64_t)blockIdx.x * bs >= len) continue;
        bool again = false;
        for (int64_t lb = blockIdx.x; lb * bs < len; lb += gridDim.x) {     // (64 bits: a step may end behind what 32 count)
            int seg = 0;
            const int64_t tile0 = page_of(a.pool, a.block_table, a.table_cols, a.num_rows, row, (int)lb, a.cur_layer, seg);
            if (lb == blockIdx.x) again = named_again(a, i, row);
            if (again) break;
            if (tile0 < 0) continue;
            const int total = min(bs, (int)(len - lb * bs)) * vecs;
            for (int h = blockIdx.z * warps + warp; h < Hkv; h += gridDim.z * warps) {
                const int64_t tile = tile0 + h;
#pragma unroll 1
                for (int which = 0; which < 2; ++which) {
                    const int64_t stride = which ? a.v_stride : a.k_stride;
                    const T *src = (const T *)(which ? a.v : a.k) + (start + lb * bs) * stride + (int64_t)h * D;
                    uint8_t *dst = (which ? a.pool.v_base[seg] : a.pool.k_base[seg]) + tile * a.pool.tile_bytes;
                    const float s = store_tile<T, CODE, V, NV>(a, src, stride, dst, total, vecs, lane);
                    if (lane == 0) (which ? a.pool.v_scale[seg] : a.pool.k_scale[seg])[tile] = s;
                }
            }
        }
    }
}

// ------------------------------------------------------------------ decode append
// grid = (sequences, 2 heads / 16).  One warp for each (sequence, head, K or V): nobody else touches the tile in this launch.
// Latency bound: lengths, page, then row and scale, then the older codes where the scale grows; 3.7 us for 256 sequences of 8 heads,
// 3.0 us for 3 of 32.
template <typename T, int CODE, int V>
__global__ void __launch_bounds__(kItemWarps * 32) store_q8_decode_kernel(const __grid_constant__ StoreQ8Args a) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
    const int D = a.pool.head_dim, bs = a.pool.block_size, Hkv = a.pool.num_kv_heads;
    const int b = blockIdx.x, len = a.seq_lens[b], row = a.seq_ids[b];
    if (len <= 0) return;
    const int lb = (len - 1) / bs, slot = (len - 1) - lb * bs;
    int seg = 0;
    const int64_t tile0 = page_of(a.pool, a.block_table, a.table_cols, a.num_rows, row, lb, a.cur_layer, seg);
    if (named_again(a, b, row) || tile0 < 0) return;
    for (int item = blockIdx.y * warps + warp; item < 2 * Hkv; item += gridDim.y * warps) {
        const int h = item >> 1, which = item & 1;
        const T *src = (const T *)(which ? a.v : a.k) + b * (which ? a.v_stride : a.k_stride) + (int64_t)h * D;
        float *scale = (which ? a.pool.v_scale[seg] : a.pool.k_scale[seg]) + tile0 + h;
        uint8_t *tile = (which ? a.pool.v_base[seg] : a.pool.k_base[seg]) + (tile0 + h) * a.pool.tile_bytes;
        const float held = *scale;
        uint32_t peak = 0;
        Piece<T, V> x;
        for (int e = lane; e < D / V; e += 32) {
            x.load(src + e * V);
            peak = x.peak(peak);
        }
        const float fresh = scale_of<CODE>(__reduce_max_sync(0xffffffffu, Piece<T, V>::peak_bits(peak)));
        const float s = slot == 0 ? fresh : larger_scale(held, fresh), inv = inverse_of(s);
        for (int e = lane; e < D / V; e += 32) {
            if (D / V > 32) x.load(src + e * V);    // (a row that fits the warp is still there)
            x.template store_codes<CODE>(tile + (int64_t)slot * D + e * V, inv);
        }
        if (slot > 0 && s > held) {  // the codes before it to the new scale
            const float ratio = __fmul_rn(held, inv);
            if constexpr (V == 16) {
                constexpr int U = 4;    // 2 KiB of codes in flight: the other 15 slots of a 16 x 128 tile at once
                const int total = slot * D / 16;
                for (int e0 = lane; e0 < total; e0 += 32 * U) {
                    uint4 c[U];
#pragma unroll
                    for (int u = 0; u < U; ++u)
                        if (e0 + 32 * u < total) c[u] = reinterpret_cast<const uint4 *>(tile)[e0 + 32 * u];
#pragma unroll
                    for (int u = 0; u < U; ++u) {
                        if (e0 + 32 * u >= total) break;
                        uint32_t w[4] = {c[u].x, c[u].y, c[u].z, c[u].w};
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const float4 f = decode4<CODE>(w[i]);
                            w[i] = ratio > 0.f ? encode4<CODE>(f.x, f.y, f.z, f.w, ratio) : 0u;
                        }
                        reinterpret_cast<uint4 *>(tile)[e0 + 32 * u] = make_uint4(w[0], w[1], w[2], w[3]);
                    }
                }
            } else {
                for (int e = lane; e < slot * D; e += 32) tile[e] = ratio > 0.f ? encode1<CODE>(decode1<CODE>(tile[e]), ratio) : (uint8_t)0;
            }
        }
        if (lane == 0) *scale = s;
    }
}

// ------------------------------------------------------------------ gather
struct LoadQ8Args {
    void *k, *v;
    int64_t k_stride, v_stride, num_out_rows;
    const int32_t *block_table;
    int64_t table_cols;
    const int32_t *seq_ids, *begins, *ends, *start_locs;
    int num_rows, num_seqs, cur_layer;
    uint32_t vecs_magic;        // ceil(2^32 / pieces of a row)
    PoolViewQ8 pool;
};

// grid = (pages of the longest range, ranges, parts of a page).  A page is (head, K or V) tiles of `chunks` x 32 pieces (V codes
// each); a warp takes kLoadFlight such chunks at a time, all of their loads before the first store.
// Bound by writing: 16-bit rows are twice their codes, and the memory takes writes at 3.5-3.9 TB/s (a plain fill of 33-200 MB;
// reads and writes in equal parts go at 6.5).  32 prefixes, 65 MB written: 22.4 us, a fill of those bytes alone 17.6 us.  A third of the
// instructions (the piece's place kept over the heads) changed nothing.
template <typename T, int CODE, int V>
__global__ void __launch_bounds__(kLoadThreads, 4) load_q8_kernel(const __grid_constant__ LoadQ8Args a) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int D = a.pool.head_dim, bs = a.pool.block_size, Hkv = a.pool.num_kv_heads, vecs = D / V;
    for (int i = blockIdx.y; i < a.num_seqs; i += gridDim.y) {
        const int row = a.seq_ids[i], first_tok = a.begins[i];
        const int64_t shift = (int64_t)a.start_locs[i] - first_tok;  // output row of token t: t + shift
        const int64_t end = min((int64_t)a.ends[i], a.num_out_rows - shift);
        const int64_t begin = max((int64_t)max(first_tok, 0), -shift);   // (a negative start_locs entry reaches no row in front of the output)
        if (begin >= end) continue;
        for (int64_t lb = (int)begin / bs + (int64_t)blockIdx.x; lb * bs < end; lb += gridDim.x) {
            int seg = 0;
            const int64_t tile0 = page_of(a.pool, a.block_table, a.table_cols, a.num_rows, row, (int)lb, a.cur_layer, seg);
            if (tile0 < 0) continue;
            const int first = max((int)begin, (int)(lb * bs));
            const int total = ((int)min(end, (lb + 1) * bs) - first) * vecs, chunks = (total + 31) / 32, all = chunks * 2 * Hkv;
            const int tile_bytes = (int)a.pool.tile_bytes, skip = (int)(first - lb * bs) * D, step = gridDim.z * (kLoadThreads / 32);
            for (int c0 = blockIdx.z * (kLoadThreads / 32) + warp; c0 < all; c0 += kLoadFlight * step) {
                if constexpr (V == 16) {
                    uint4 x[kLoadFlight];
                    float s[kLoadFlight];
                    T *dst[kLoadFlight];
    #pragma unroll
                    for (int u = 0; u < kLoadFlight; ++u) {     // (behind the last piece: that one again, and nothing is written)
                        const int c = min(c0 + u * step, all - 1), item = c / chunks, e = (c - item * chunks) * 32 + lane, at = min(e, total - 1);
                        const int h = item >> 1, which = item & 1, tok = (int)__umulhi((uint32_t)at, a.vecs_magic);
                        const int64_t stride = which ? a.v_stride : a.k_stride, tile = tile0 + h;
                        x[u] = __ldg(reinterpret_cast<const uint4 *>((which ? a.pool.v_base[seg] : a.pool.k_base[seg]) + tile * tile_bytes + skip) + at);
                        s[u] = (which ? a.pool.v_scale[seg] : a.pool.k_scale[seg])[tile];
                        dst[u] = (T *)(which ? a.v : a.k) + (first + shift + tok) * stride + (int64_t)h * D + (at - tok * vecs) * V;
                        if (c0 + u * step >= all || e >= total) dst[u] = nullptr;
                    }
    #pragma unroll
                    for (int u = 0; u < kLoadFlight; ++u) {
                        if (!dst[u]) continue;
                        const uint32_t w[4] = {x[u].x, x[u].y, x[u].z, x[u].w};
                        Piece<T, V> out;
    #pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            const float4 f = decode4<CODE>(w[j]);
                            out.set2(4 * j, f.x * s[u], f.y * s[u]);
                            out.set2(4 * j + 2, f.z * s[u], f.w * s[u]);
                        }
                        out.store(dst[u]);
                    }
                } else {
                    for (int c = c0; c < min(c0 + kLoadFlight * step, all); c += step) {
                        const int item = c / chunks, e = (c - item * chunks) * 32 + lane, h = item >> 1, which = item & 1;
                        if (e >= total) continue;
                        const int64_t tile = tile0 + h;
                        const float s = (which ? a.pool.v_scale[seg] : a.pool.k_scale[seg])[tile];
                        const uint8_t code = ((which ? a.pool.v_base[seg] : a.pool.k_base[seg]) + tile * tile_bytes + skip)[e];
                        ((T *)(which ? a.v : a.k))[(first + shift + e / vecs) * (which ? a.v_stride : a.k_stride) + (int64_t)h * D + e % vecs] =
                            rounded<T>(decode1<CODE>(code) * s);
                    }
                }
            }
        }
    }
}

// Whether rows and pool allow 16 elements (32 bytes and more) and 16 codes at once.
static bool wide_ok(const PoolViewQ8 &pv, const void *k, const void *v, int64_t k_stride, int64_t v_stride, int dtype) {
    const int64_t size = dtype_bytes(dtype);
    if (std::max(k_stride, v_stride) * pv.block_size >= (1ll << 31)) return false;   // (a page's rows are addressed in 32 bits)
    if (pv.head_dim % 16 != 0 || pv.head_dim < 32) return false;
    if ((((uintptr_t)k | (uintptr_t)v | (uintptr_t)(k_stride * size) | (uintptr_t)(v_stride * size)) & 31) != 0) return false;
    for (int i = 0; i < pv.num_segments; ++i)
        if ((((uintptr_t)pv.k_base[i] | (uintptr_t)pv.v_base[i]) & 15) != 0) return false;
    return true;
}

// Calls f with (T{}, code tag, elements of a piece).
template <int N> struct Int { static constexpr int value = N; };
template <typename F>
static void dispatch(int dtype, int code, bool wide, F &&f) {
    auto with_code = [&](auto t) {
        if (code == MKV_Q8_INT8) {
            if (wide) f(t, Int<MKV_Q8_INT8>{}, Int<16>{}); else f(t, Int<MKV_Q8_INT8>{}, Int<1>{});
        } else {
            if (wide) f(t, Int<MKV_Q8_E4M3>{}, Int<16>{}); else f(t, Int<MKV_Q8_E4M3>{}, Int<1>{});
        }
    };
    if (dtype == MKV_F16) with_code(__half{});
    else if (dtype == MKV_BF16) with_code(__nv_bfloat16{});
    else with_code(float{});
}

static int check_rows(const PoolViewQ8 &pv, int64_t k_stride, int64_t v_stride, int dtype) {
    if (!dtype_ok(dtype)) return MKV_ERR_DTYPE;
    const int64_t row = (int64_t)pv.num_kv_heads * pv.head_dim;
    return k_stride < row || v_stride < row ? MKV_ERR_SHAPE : MKV_OK;
}

// Warps of a block and blocks that share `items` of a page.
static int warps_for(int items, int most) { return std::min(items, most); }
static unsigned blocks_for(int items, int most) { return (unsigned)std::min<int64_t>(ceil_div64(items, most), 65535); }
// e / n = umulhi(e, magic) for e n < 2^32: a page has at most 2^24 elements.  (n = 1 has no such factor; wide_ok keeps it out.)
static uint32_t magic_of(int n) { return n > 1 ? (uint32_t)(((1ull << 32) + n - 1) / n) : 0u; }

}  // namespace mkv

using namespace mkv;

extern "C" {

int mkv_store_kv_q8_prefill(int device, void *stream, const void *k, const void *v, int64_t k_stride, int64_t v_stride,
                            int dtype, int64_t num_tokens, const mkv_pool_q8 *pool, const int32_t *block_table,
                            int64_t table_stride, int num_rows, const int32_t *seq_ids, const int32_t *start_locs,
                            const int32_t *seq_lens, int num_seqs, int max_seq_len, int cur_layer) {
    StoreQ8Args a;
    int st = validate_pool_q8(pool, &a.pool);
    if (st) return st;
    if (num_seqs < 0 || max_seq_len < 0 || table_stride < 1 || num_rows < 0 || num_tokens < 0) return MKV_ERR_SHAPE;
    if ((st = check_rows(a.pool, k_stride, v_stride, dtype))) return st;
    if (cur_layer < 0 || cur_layer >= a.pool.num_layers) return MKV_ERR_RANGE;
    if (num_seqs == 0 || max_seq_len == 0 || num_tokens == 0) return MKV_OK;
    if (!k || !v || !block_table || !seq_ids || !seq_lens || !start_locs) return MKV_ERR_NULL;
    a.k = k; a.v = v; a.k_stride = k_stride; a.v_stride = v_stride; a.num_tokens = num_tokens;
    a.block_table = block_table; a.table_cols = table_stride; a.num_rows = num_rows;
    a.seq_ids = seq_ids; a.start_locs = start_locs; a.seq_lens = seq_lens; a.num_seqs = num_seqs; a.cur_layer = cur_layer;
    DeviceGuard guard(device);
    if (guard.err != cudaSuccess) return set_cuda_error(guard.err);
    const dim3 grid((unsigned)std::min(ceil_div64(max_seq_len, a.pool.block_size), table_stride), (unsigned)std::min(num_seqs, 65535),
                    blocks_for(a.pool.num_kv_heads, kHeadWarps));   // (no page stands behind the table's last column)
    const int threads = warps_for(a.pool.num_kv_heads, kHeadWarps) * 32;
    a.vecs_magic = magic_of(a.pool.head_dim / 16);
    const int64_t pieces = a.pool.tile_bytes / 16;
    dispatch(dtype, a.pool.code, wide_ok(a.pool, k, v, k_stride, v_stride, dtype), [&](auto t, auto code, auto w) {
        using T = decltype(t);
        constexpr int CODE = decltype(code)::value, V = decltype(w)::value;
        cudaStream_t s = (cudaStream_t)stream;
        if constexpr (V == 16) {    // a tile of up to 4 KiB of 16-bit rows (8 KiB of fp32) stays in registers
            if (pieces <= 64) return store_q8_prefill_kernel<T, CODE, V, 2><<<grid, threads, 0, s>>>(a);
            if (pieces <= 128) return store_q8_prefill_kernel<T, CODE, V, 4><<<grid, threads, 0, s>>>(a);
        }
        store_q8_prefill_kernel<T, CODE, V, 0><<<grid, threads, 0, s>>>(a);
    });
    MKV_LAUNCH_CHECK();
    return MKV_OK;
}

int mkv_store_kv_q8_decode(int device, void *stream, const void *k, const void *v, int64_t k_stride, int64_t v_stride,
                           int dtype, const mkv_pool_q8 *pool, const int32_t *block_table, int64_t table_stride,
                           int num_rows, const int32_t *seq_ids, const int32_t *seq_lens, int batch, int cur_layer) {
    StoreQ8Args a;
    int st = validate_pool_q8(pool, &a.pool);
    if (st) return st;
    if (batch < 0 || table_stride < 1 || num_rows < 0) return MKV_ERR_SHAPE;
    if ((st = check_rows(a.pool, k_stride, v_stride, dtype))) return st;
    if (cur_layer < 0 || cur_layer >= a.pool.num_layers) return MKV_ERR_RANGE;
    if (batch == 0) return MKV_OK;
    if (!k || !v || !block_table || !seq_ids || !seq_lens) return MKV_ERR_NULL;
    a.k = k; a.v = v; a.k_stride = k_stride; a.v_stride = v_stride; a.num_tokens = batch;
    a.block_table = block_table; a.table_cols = table_stride; a.num_rows = num_rows;
    a.seq_ids = seq_ids; a.start_locs = nullptr; a.seq_lens = seq_lens; a.num_seqs = batch; a.cur_layer = cur_layer;
    DeviceGuard guard(device);
    if (guard.err != cudaSuccess) return set_cuda_error(guard.err);
    const dim3 grid((unsigned)batch, blocks_for(2 * a.pool.num_kv_heads, kItemWarps));
    a.vecs_magic = 0;
    dispatch(dtype, a.pool.code, wide_ok(a.pool, k, v, k_stride, v_stride, dtype), [&](auto t, auto code, auto w) {
        store_q8_decode_kernel<decltype(t), decltype(code)::value, decltype(w)::value>
            <<<grid, warps_for(2 * a.pool.num_kv_heads, kItemWarps) * 32, 0, (cudaStream_t)stream>>>(a);
    });
    MKV_LAUNCH_CHECK();
    return MKV_OK;
}

int mkv_load_kv_q8(int device, void *stream, void *k, void *v, int64_t k_stride, int64_t v_stride, int dtype,
                   int64_t num_out_rows, const mkv_pool_q8 *pool, const int32_t *block_table, int64_t table_stride,
                   int num_rows, const int32_t *seq_ids, const int32_t *begins, const int32_t *ends,
                   const int32_t *start_locs, int num_seqs, int max_len, int cur_layer) {
    LoadQ8Args a;
    int st = validate_pool_q8(pool, &a.pool);
    if (st) return st;
    if (num_seqs < 0 || max_len < 0 || table_stride < 1 || num_rows < 0 || num_out_rows < 0) return MKV_ERR_SHAPE;
    if ((st = check_rows(a.pool, k_stride, v_stride, dtype))) return st;
    if (cur_layer < 0 || cur_layer >= a.pool.num_layers) return MKV_ERR_RANGE;
    if (num_seqs == 0 || max_len == 0 || num_out_rows == 0) return MKV_OK;
    if (!k || !v || !block_table || !seq_ids || !begins || !ends || !start_locs) return MKV_ERR_NULL;
    a.k = k; a.v = v; a.k_stride = k_stride; a.v_stride = v_stride; a.num_out_rows = num_out_rows;
    a.block_table = block_table; a.table_cols = table_stride; a.num_rows = num_rows;
    a.seq_ids = seq_ids; a.begins = begins; a.ends = ends; a.start_locs = start_locs;
    a.num_seqs = num_seqs; a.cur_layer = cur_layer;
    DeviceGuard guard(device);
    if (guard.err != cudaSuccess) return set_cuda_error(guard.err);
    const bool wide = wide_ok(a.pool, k, v, k_stride, v_stride, dtype);
    a.vecs_magic = magic_of(a.pool.head_dim / 16);
    // A range that starts inside a block touches one block more.  A page's chunks go to so many blocks that a warp has eight
    // of them (two flights), or four (one) where the ranges are a part of a page each or there would be few blocks otherwise
    // (append and load back of 256 last pages: 10.2 us with four, 12.9 with eight, 13.6 with two; 32 prefixes of up to 2048 tokens:
    // 25, 23, 28 us).
    int sms = 0;
    if ((st = mkv_sm_count(device, &sms))) return st;
    const int64_t pages = num_out_rows / a.pool.block_size + 2 * (int64_t)num_seqs;
    const int64_t chunks = ceil_div64(a.pool.tile_bytes / (wide ? 16 : 1), 32) * 2 * a.pool.num_kv_heads;
    const int64_t rounds = num_out_rows >= (int64_t)num_seqs * a.pool.block_size && chunks * pages >= 8 * (kLoadThreads / 32) * 4ll * sms ? 8 : 4;
    const dim3 grid((unsigned)std::min(ceil_div64(max_len, a.pool.block_size) + 1, table_stride), (unsigned)std::min(num_seqs, 65535),
                    (unsigned)std::max<int64_t>(1, std::min<int64_t>(chunks / (rounds * (kLoadThreads / 32)), 65535)));
    dispatch(dtype, a.pool.code, wide, [&](auto t, auto code, auto w) {
        load_q8_kernel<decltype(t), decltype(code)::value, decltype(w)::value>
            <<<grid, kLoadThreads, 0, (cudaStream_t)stream>>>(a);
    });
    MKV_LAUNCH_CHECK();
    return MKV_OK;
}

}  // extern "C"
