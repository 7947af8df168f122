// Into and out of the 8-bit pool: prefill scatter, decode append, and the gather back to rows of the model's type.
// HBM / latency bound; the number format is kv_q8.cuh's.
#include <string.h>

#include <algorithm>

#include "kv_q8.cuh"

namespace mkv {

int validate_pool_q8(const mkv_pool_q8 *pool, PoolViewQ8 *out) {
    if (!pool) return MKV_ERR_NULL;
    if (pool->num_segments < 1 || pool->num_segments > MKV_MAX_SEGMENTS) return MKV_ERR_SHAPE;
    if (pool->code != MKV_Q8_INT8 && pool->code != MKV_Q8_E4M3) return MKV_ERR_DTYPE;
    if (pool->num_layers < 1 || pool->num_kv_heads < 1 || pool->block_size < 1 || pool->head_dim < 1) return MKV_ERR_SHAPE;
    if ((int64_t)pool->block_size * pool->head_dim > (1 << 24)) return MKV_ERR_SHAPE;
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

// V elements of T at once: as few and as wide loads as the alignment allows.
template <typename T, int V>
struct alignas(sizeof(T) * V) Pack {
    T x[V];
};

template <typename T, int V>
__device__ __forceinline__ void load_pack(const T *src, float (&x)[V]) {
    const Pack<T, V> p = *reinterpret_cast<const Pack<T, V> *>(src);
#pragma unroll
    for (int i = 0; i < V; ++i) x[i] = value_of<T>(p.x[i]);
}

// Largest absolute value, as the bits of an fp32 number: the integer order puts infinity and NaN on top.
template <int V>
__device__ __forceinline__ uint32_t peak_bits(const float (&x)[V], uint32_t peak) {
#pragma unroll
    for (int i = 0; i < V; ++i) peak = max(peak, __float_as_uint(x[i]) & 0x7fffffffu);
    return peak;
}

template <int CODE, int V>
__device__ __forceinline__ void store_codes(uint8_t *dst, const float (&x)[V], float inv) {
    if constexpr (V % 4 == 0) {
        Pack<uint32_t, V / 4> p;
#pragma unroll
        for (int i = 0; i < V / 4; ++i)
            p.x[i] = inv > 0.f ? encode4<CODE>(x[4 * i], x[4 * i + 1], x[4 * i + 2], x[4 * i + 3], inv) : 0u;
        *reinterpret_cast<Pack<uint32_t, V / 4> *>(dst) = p;
    } else {
#pragma unroll
        for (int i = 0; i < V; ++i) dst[i] = inv > 0.f ? encode1<CODE>(x[i], inv) : (uint8_t)0;
    }
}

// ------------------------------------------------------------------ prefill scatter
// One warp per (block, head, K or V): the block's peak, then its codes.  grid = (logical blocks, prompts).
template <typename T, int CODE, int V>
__global__ void store_q8_prefill_kernel(const T *__restrict__ k, const T *__restrict__ v, int64_t k_stride, int64_t v_stride,
                                        int64_t num_tokens, const __grid_constant__ PoolViewQ8 pool,
                                        const int32_t *__restrict__ block_table, int64_t table_stride, int num_rows,
                                        const int32_t *__restrict__ seq_ids, const int32_t *__restrict__ start_locs,
                                        const int32_t *__restrict__ seq_lens, int num_seqs, int cur_layer) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
    const int D = pool.head_dim, bs = pool.block_size, Hkv = pool.num_kv_heads;
    for (int i = blockIdx.y; i < num_seqs; i += gridDim.y) {
        const int row = seq_ids[i];
        const int64_t start = start_locs[i];
        const int64_t len = min((int64_t)seq_lens[i], start < 0 ? 0 : num_tokens - start);
        if ((int64_t)blockIdx.x * bs >= len) continue;
        bool again = false;  // the same sequence further on: that one counts
        for (int j = i + 1 + lane; j < num_seqs; j += 32) again |= seq_ids[j] == row && seq_lens[j] > 0;
        if (__any_sync(0xffffffffu, again)) continue;
        for (int64_t lb = blockIdx.x; lb * bs < len; lb += gridDim.x) {
            int seg = 0;
            const int64_t tile0 = page_of(pool, block_table, table_stride, num_rows, row, (int)min(lb, table_stride), cur_layer, seg);
            if (tile0 < 0) continue;
            const int ntok = (int)min((int64_t)bs, len - lb * bs);
            const int vecs = D / V, total = ntok * vecs;
            for (int item = warp; item < 2 * Hkv; item += warps) {
                const int h = item >> 1, which = item & 1;
                const T *src = (which ? v : k) + (start + lb * bs) * (which ? v_stride : k_stride) + (int64_t)h * D;
                const int64_t stride = which ? v_stride : k_stride;
                uint32_t peak = 0;
                for (int e = lane; e < total; e += 32) {
                    float x[V];
                    load_pack<T, V>(src + (e / vecs) * stride + (e % vecs) * V, x);
                    peak = peak_bits<V>(x, peak);
                }
                peak = __reduce_max_sync(0xffffffffu, peak);
                const float s = scale_of<CODE>(peak), inv = inverse_of(s);
                uint8_t *dst = (which ? pool.v_base[seg] : pool.k_base[seg]) + (tile0 + h) * pool.tile_bytes;
                for (int e = lane; e < total; e += 32) {
                    float x[V];
                    load_pack<T, V>(src + (e / vecs) * stride + (e % vecs) * V, x);
                    store_codes<CODE, V>(dst + (int64_t)e * V, x, inv);
                }
                if (lane == 0) (which ? pool.v_scale[seg] : pool.k_scale[seg])[tile0 + h] = s;
            }
        }
    }
}

// ------------------------------------------------------------------ decode append
// One warp per (sequence, head, K or V): nobody else touches the tile in this launch.
template <typename T, int CODE, int V>
__global__ void store_q8_decode_kernel(const T *__restrict__ k, const T *__restrict__ v, int64_t k_stride, int64_t v_stride,
                                       const __grid_constant__ PoolViewQ8 pool, const int32_t *__restrict__ block_table,
                                       int64_t table_stride, int num_rows, const int32_t *__restrict__ seq_ids,
                                       const int32_t *__restrict__ seq_lens, int batch, int cur_layer) {
    const int lane = threadIdx.x & 31;
    const int64_t wid = ((int64_t)blockIdx.x * blockDim.x + threadIdx.x) >> 5;
    const int D = pool.head_dim, bs = pool.block_size, Hkv = pool.num_kv_heads;
    if (wid >= (int64_t)batch * Hkv * 2) return;
    const int b = (int)(wid / (2 * Hkv)), item = (int)(wid - (int64_t)b * 2 * Hkv), h = item >> 1, which = item & 1;
    const int len = seq_lens[b], row = seq_ids[b];
    bool again = false;
    for (int j = b + 1 + lane; j < batch; j += 32) again |= seq_ids[j] == row && seq_lens[j] > 0;
    if (__any_sync(0xffffffffu, again) || len <= 0) return;
    const int lb = (len - 1) / bs, slot = (len - 1) - lb * bs;
    int seg = 0;
    const int64_t tile0 = page_of(pool, block_table, table_stride, num_rows, row, lb, cur_layer, seg);
    if (tile0 < 0) return;
    const T *src = (which ? v + b * v_stride : k + b * k_stride) + (int64_t)h * D;
    float *scale = (which ? pool.v_scale[seg] : pool.k_scale[seg]) + tile0 + h;
    uint8_t *tile = (which ? pool.v_base[seg] : pool.k_base[seg]) + (tile0 + h) * pool.tile_bytes;
    const float held = *scale;
    uint32_t peak = 0;
    for (int e = lane; e < D / V; e += 32) {
        float x[V];
        load_pack<T, V>(src + e * V, x);
        peak = peak_bits<V>(x, peak);
    }
    peak = __reduce_max_sync(0xffffffffu, peak);
    const float fresh = scale_of<CODE>(peak);
    const float s = slot == 0 ? fresh : larger_scale(held, fresh), inv = inverse_of(s);
    for (int e = lane; e < D / V; e += 32) {
        float x[V];
        load_pack<T, V>(src + e * V, x);
        store_codes<CODE, V>(tile + (int64_t)slot * D + e * V, x, inv);
    }
    if (slot > 0 && s > held) {  // the codes before it to the new scale
        const float ratio = __fmul_rn(held, inv);
        for (int e = lane; e < slot * D / V; e += 32) {
            uint8_t *at = tile + (int64_t)e * V;
            float x[V];
            if constexpr (V % 4 == 0) {
                const Pack<uint32_t, V / 4> p = *reinterpret_cast<const Pack<uint32_t, V / 4> *>(at);
#pragma unroll
                for (int i = 0; i < V / 4; ++i) {
                    const float4 f = decode4<CODE>(p.x[i]);
                    x[4 * i] = f.x; x[4 * i + 1] = f.y; x[4 * i + 2] = f.z; x[4 * i + 3] = f.w;
                }
            } else {
#pragma unroll
                for (int i = 0; i < V; ++i) x[i] = decode1<CODE>(at[i]);
            }
            store_codes<CODE, V>(at, x, ratio);
        }
    }
    if (lane == 0) *scale = s;
}

// ------------------------------------------------------------------ gather
// One warp per (block, head, K or V).  grid = (blocks of the longest range, ranges).
template <typename T, int CODE, int V>
__global__ void load_q8_kernel(T *__restrict__ k, T *__restrict__ v, int64_t k_stride, int64_t v_stride, int64_t num_out_rows,
                               const __grid_constant__ PoolViewQ8 pool, const int32_t *__restrict__ block_table,
                               int64_t table_stride, int num_rows, const int32_t *__restrict__ seq_ids,
                               const int32_t *__restrict__ begins, const int32_t *__restrict__ ends,
                               const int32_t *__restrict__ start_locs, int num_seqs, int cur_layer) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
    const int D = pool.head_dim, bs = pool.block_size, Hkv = pool.num_kv_heads, vecs = D / V;
    for (int i = blockIdx.y; i < num_seqs; i += gridDim.y) {
        const int row = seq_ids[i], begin = max(begins[i], 0);
        const int64_t shift = (int64_t)start_locs[i] - begins[i];  // output row of token t: t + shift
        const int64_t end = min((int64_t)ends[i], num_out_rows - shift);
        for (int64_t lb = begin / bs + blockIdx.x; lb * bs < end; lb += gridDim.x) {
            int seg = 0;
            const int64_t tile0 = page_of(pool, block_table, table_stride, num_rows, row, (int)min(lb, table_stride), cur_layer, seg);
            if (tile0 < 0) continue;
            const int64_t t0 = max((int64_t)begin, lb * bs), t1 = min(end, (lb + 1) * bs);
            const int64_t first = max(t0, -shift);  // a negative start_locs entry reaches no row in front of the output
            const int total = (int)(t1 - first) * vecs;
            for (int item = warp; item < 2 * Hkv; item += warps) {
                const int h = item >> 1, which = item & 1;
                const float s = (which ? pool.v_scale[seg] : pool.k_scale[seg])[tile0 + h];
                const uint8_t *tile = (which ? pool.v_base[seg] : pool.k_base[seg]) + (tile0 + h) * pool.tile_bytes +
                                      (first - lb * bs) * D;
                const int64_t stride = which ? v_stride : k_stride;
                T *dst = (which ? v : k) + (first + shift) * stride + (int64_t)h * D;
                for (int e = lane; e < total; e += 32) {
                    Pack<T, V> out;
                    if constexpr (V % 4 == 0) {
                        const Pack<uint32_t, V / 4> p = *reinterpret_cast<const Pack<uint32_t, V / 4> *>(tile + (int64_t)e * V);
#pragma unroll
                        for (int j = 0; j < V / 4; ++j) {
                            const float4 f = decode4<CODE>(p.x[j]);
                            out.x[4 * j] = rounded<T>(f.x * s);
                            out.x[4 * j + 1] = rounded<T>(f.y * s);
                            out.x[4 * j + 2] = rounded<T>(f.z * s);
                            out.x[4 * j + 3] = rounded<T>(f.w * s);
                        }
                    } else {
#pragma unroll
                        for (int j = 0; j < V; ++j) out.x[j] = rounded<T>(decode1<CODE>(tile[(int64_t)e * V + j]) * s);
                    }
                    *reinterpret_cast<Pack<T, V> *>(dst + (e / vecs) * stride + (e % vecs) * V) = out;
                }
            }
        }
    }
}

// Elements per access: 16 bytes of the model's type where rows, strides and bases allow it, else one element.
static bool wide_ok(const PoolViewQ8 &pv, const void *k, const void *v, int64_t k_stride, int64_t v_stride, int dtype, int *vec) {
    const int w = 16 / dtype_bytes(dtype);
    *vec = w;
    if (pv.head_dim % w != 0 || k_stride % w != 0 || v_stride % w != 0) return false;
    if ((((uintptr_t)k | (uintptr_t)v) & 15) != 0) return false;
    for (int i = 0; i < pv.num_segments; ++i)
        if ((((uintptr_t)pv.k_base[i] | (uintptr_t)pv.v_base[i]) & (w - 1)) != 0) return false;
    return true;
}

// Calls f with (T{}, code tag, vector tag).
template <int N> struct Int { static constexpr int value = N; };
template <typename F>
static void dispatch(int dtype, int code, bool wide, F &&f) {
    auto with_code = [&](auto t, auto w) {
        if (code == MKV_Q8_INT8) {
            if (wide) f(t, Int<MKV_Q8_INT8>{}, w); else f(t, Int<MKV_Q8_INT8>{}, Int<1>{});
        } else {
            if (wide) f(t, Int<MKV_Q8_E4M3>{}, w); else f(t, Int<MKV_Q8_E4M3>{}, Int<1>{});
        }
    };
    if (dtype == MKV_F16) with_code(__half{}, Int<8>{});
    else if (dtype == MKV_BF16) with_code(__nv_bfloat16{}, Int<8>{});
    else with_code(float{}, Int<4>{});
}

static int check_rows(const PoolViewQ8 &pv, int64_t k_stride, int64_t v_stride, int dtype) {
    if (!dtype_ok(dtype)) return MKV_ERR_DTYPE;
    const int64_t row = (int64_t)pv.num_kv_heads * pv.head_dim;
    return k_stride < row || v_stride < row ? MKV_ERR_SHAPE : MKV_OK;
}

}  // namespace mkv

using namespace mkv;

extern "C" {

int mkv_store_kv_q8_prefill(int device, void *stream, const void *k, const void *v, int64_t k_stride, int64_t v_stride,
                            int dtype, int64_t num_tokens, const mkv_pool_q8 *pool, const int32_t *block_table,
                            int64_t table_stride, int num_rows, const int32_t *seq_ids, const int32_t *start_locs,
                            const int32_t *seq_lens, int num_seqs, int max_seq_len, int cur_layer) {
    PoolViewQ8 pv;
    int st = validate_pool_q8(pool, &pv);
    if (st) return st;
    if (num_seqs < 0 || max_seq_len < 0 || table_stride < 1 || num_rows < 0 || num_tokens < 0) return MKV_ERR_SHAPE;
    if ((st = check_rows(pv, k_stride, v_stride, dtype))) return st;
    if (cur_layer < 0 || cur_layer >= pv.num_layers) return MKV_ERR_RANGE;
    if (num_seqs == 0 || max_seq_len == 0) return MKV_OK;
    if (!k || !v || !block_table || !seq_ids || !seq_lens || !start_locs) return MKV_ERR_NULL;
    DeviceGuard guard(device);
    if (guard.err != cudaSuccess) return set_cuda_error(guard.err);
    int vec;
    const bool wide = wide_ok(pv, k, v, k_stride, v_stride, dtype, &vec);
    const dim3 grid((unsigned)ceil_div64(max_seq_len, pv.block_size), (unsigned)std::min(num_seqs, 65535));
    dispatch(dtype, pv.code, wide, [&](auto t, auto code, auto w) {
        using T = decltype(t);
        store_q8_prefill_kernel<T, decltype(code)::value, decltype(w)::value><<<grid, 256, 0, (cudaStream_t)stream>>>(
            (const T *)k, (const T *)v, k_stride, v_stride, num_tokens, pv, block_table, table_stride, num_rows, seq_ids,
            start_locs, seq_lens, num_seqs, cur_layer);
    });
    MKV_LAUNCH_CHECK();
    return MKV_OK;
}

int mkv_store_kv_q8_decode(int device, void *stream, const void *k, const void *v, int64_t k_stride, int64_t v_stride,
                           int dtype, const mkv_pool_q8 *pool, const int32_t *block_table, int64_t table_stride,
                           int num_rows, const int32_t *seq_ids, const int32_t *seq_lens, int batch, int cur_layer) {
    PoolViewQ8 pv;
    int st = validate_pool_q8(pool, &pv);
    if (st) return st;
    if (batch < 0 || table_stride < 1 || num_rows < 0) return MKV_ERR_SHAPE;
    if ((st = check_rows(pv, k_stride, v_stride, dtype))) return st;
    if (cur_layer < 0 || cur_layer >= pv.num_layers) return MKV_ERR_RANGE;
    if (batch == 0) return MKV_OK;
    if (!k || !v || !block_table || !seq_ids || !seq_lens) return MKV_ERR_NULL;
    const int64_t blocks = ceil_div64((int64_t)batch * pv.num_kv_heads * 2, 4);
    if (blocks > 0x7fffffff) return MKV_ERR_SHAPE;
    DeviceGuard guard(device);
    if (guard.err != cudaSuccess) return set_cuda_error(guard.err);
    int vec;
    const bool wide = wide_ok(pv, k, v, k_stride, v_stride, dtype, &vec);
    dispatch(dtype, pv.code, wide, [&](auto t, auto code, auto w) {
        using T = decltype(t);
        store_q8_decode_kernel<T, decltype(code)::value, decltype(w)::value><<<(unsigned)blocks, 128, 0, (cudaStream_t)stream>>>(
            (const T *)k, (const T *)v, k_stride, v_stride, pv, block_table, table_stride, num_rows, seq_ids, seq_lens, batch,
            cur_layer);
    });
    MKV_LAUNCH_CHECK();
    return MKV_OK;
}

int mkv_load_kv_q8(int device, void *stream, void *k, void *v, int64_t k_stride, int64_t v_stride, int dtype,
                   int64_t num_out_rows, const mkv_pool_q8 *pool, const int32_t *block_table, int64_t table_stride,
                   int num_rows, const int32_t *seq_ids, const int32_t *begins, const int32_t *ends,
                   const int32_t *start_locs, int num_seqs, int max_len, int cur_layer) {
    PoolViewQ8 pv;
    int st = validate_pool_q8(pool, &pv);
    if (st) return st;
    if (num_seqs < 0 || max_len < 0 || table_stride < 1 || num_rows < 0 || num_out_rows < 0) return MKV_ERR_SHAPE;
    if ((st = check_rows(pv, k_stride, v_stride, dtype))) return st;
    if (cur_layer < 0 || cur_layer >= pv.num_layers) return MKV_ERR_RANGE;
    if (num_seqs == 0 || max_len == 0 || num_out_rows == 0) return MKV_OK;
    if (!k || !v || !block_table || !seq_ids || !begins || !ends || !start_locs) return MKV_ERR_NULL;
    DeviceGuard guard(device);
    if (guard.err != cudaSuccess) return set_cuda_error(guard.err);
    int vec;
    const bool wide = wide_ok(pv, k, v, k_stride, v_stride, dtype, &vec);
    // a range that starts inside a block touches one block more
    const dim3 grid((unsigned)(ceil_div64(max_len, pv.block_size) + 1), (unsigned)std::min(num_seqs, 65535));
    dispatch(dtype, pv.code, wide, [&](auto t, auto code, auto w) {
        using T = decltype(t);
        load_q8_kernel<T, decltype(code)::value, decltype(w)::value><<<grid, 256, 0, (cudaStream_t)stream>>>(
            (T *)k, (T *)v, k_stride, v_stride, num_out_rows, pv, block_table, table_stride, num_rows, seq_ids, begins, ends,
            start_locs, num_seqs, cur_layer);
    });
    MKV_LAUNCH_CHECK();
    return MKV_OK;
}

}  // extern "C"
