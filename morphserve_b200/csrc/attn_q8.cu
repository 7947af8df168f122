// Decode attention over the 8-bit pool.
#include "kv_q8.cuh"

namespace mkv {

constexpr float kLog2e = 1.4426950408889634f;

// ------------------------------------------------------------------ plain kernel
// One warp per (sequence, query head); lane l holds dims l, l + 32, ...  fp32 throughout.
constexpr int kPlainDims = 16;  // head_dim <= 512

template <typename T, int CODE>
__global__ void attn_q8_plain_kernel(const T *__restrict__ q, int64_t q_stride, T *__restrict__ o,
                                     const __grid_constant__ PoolViewQ8 pool, const int32_t *__restrict__ block_table,
                                     int64_t table_stride, int num_rows, const int32_t *__restrict__ seq_ids,
                                     const int32_t *__restrict__ seq_lens, int batch, int num_q_heads, int cur_layer,
                                     float scale_log2, int *error_flags) {
    const int lane = threadIdx.x & 31;
    const int64_t wid = ((int64_t)blockIdx.x * blockDim.x + threadIdx.x) >> 5;
    if (wid >= (int64_t)batch * num_q_heads) return;
    const int b = (int)(wid / num_q_heads), hq = (int)(wid - (int64_t)b * num_q_heads);
    const int h = hq / (num_q_heads / pool.num_kv_heads);
    const int D = pool.head_dim, bs = pool.block_size;
    const int len = seq_lens[b], row = seq_ids[b];
    if (len <= 0) return;
    float qr[kPlainDims], acc[kPlainDims];
#pragma unroll
    for (int i = 0; i < kPlainDims; ++i) {
        const int d = lane + 32 * i;
        qr[i] = d < D ? value_of<T>(q[b * q_stride + (int64_t)hq * D + d]) : 0.f;
        acc[i] = 0.f;
    }
    float m = -INFINITY, l = 0.f;
    bool bad = row < 0 || row >= num_rows;
    const int nblk = bad ? 0 : (int)min(((int64_t)len + bs - 1) / bs, table_stride);
    bad |= (int64_t)nblk * bs < len;
    for (int jb = 0; jb < nblk; ++jb) {
        const int64_t blk = __ldg(block_table + (int64_t)row * table_stride + jb);
        if (blk < 0 || blk >= pool.total_blocks) {
            bad = true;
            continue;
        }
        int seg;
        int64_t brow;
        locate_block(pool, blk, seg, brow);
        const int64_t tile = tile_index(pool, brow, cur_layer, h);
        const uint8_t *kt = pool.k_base[seg] + tile * pool.tile_bytes, *vt = pool.v_base[seg] + tile * pool.tile_bytes;
        const float ks = pool.k_scale[seg][tile] * scale_log2, vs = pool.v_scale[seg][tile];
        const int ntok = (int)min((int64_t)bs, len - (int64_t)jb * bs);
        for (int tk = 0; tk < ntok; ++tk) {
            float dot = 0.f;
#pragma unroll
            for (int i = 0; i < kPlainDims; ++i) {
                const int d = lane + 32 * i;
                if (d < D) dot += qr[i] * decode1<CODE>(kt[(int64_t)tk * D + d]);
            }
#pragma unroll
            for (int s = 16; s > 0; s >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, s);
            const float sc = dot * ks;
            const float mn = fmaxf(m, sc), base = mn == -INFINITY ? 0.f : mn;  // no finite score yet: all weights are 0
            const float a = exp2f(m - base), w = exp2f(sc - base);
            l = l * a + w;
#pragma unroll
            for (int i = 0; i < kPlainDims; ++i) {
                const int d = lane + 32 * i;
                if (d < D) acc[i] = acc[i] * a + w * (decode1<CODE>(vt[(int64_t)tk * D + d]) * vs);
            }
            m = mn;
        }
    }
    if (bad && lane == 0 && error_flags) atomicOr(error_flags, 1);
#pragma unroll
    for (int i = 0; i < kPlainDims; ++i) {
        const int d = lane + 32 * i;
        if (d < D) o[((int64_t)b * num_q_heads + hq) * D + d] = rounded<T>(acc[i] / l);
    }
}

}  // namespace mkv

using namespace mkv;

extern "C" {

size_t mkv_attn_q8_zero_bytes(int device) {
    (void)device;
    return 256;
}

size_t mkv_attn_q8_workspace_bytes(int device, int batch, int num_q_heads, int num_kv_heads, int head_dim) {
    if (batch < 0 || num_q_heads < 1 || num_kv_heads < 1 || head_dim < 1) return 0;
    return mkv_attn_q8_zero_bytes(device);
}

int mkv_paged_attention_q8(int device, void *stream, const void *q, int64_t q_stride, void *o, int dtype,
                           const mkv_pool_q8 *pool, const int32_t *block_table, int64_t table_stride, int num_rows,
                           const int32_t *seq_ids, const int32_t *seq_lens, int batch, int num_q_heads, int cur_layer,
                           float softmax_scale, int max_seq_len, void *workspace, size_t workspace_bytes) {
    PoolViewQ8 pv;
    int st = validate_pool_q8(pool, &pv);
    if (st) return st;
    if (!dtype_ok(dtype)) return MKV_ERR_DTYPE;
    if (batch < 0 || num_q_heads < 1 || table_stride < 1 || num_rows < 0 || max_seq_len < 0) return MKV_ERR_SHAPE;
    if (num_q_heads % pv.num_kv_heads != 0 || pv.head_dim > 32 * kPlainDims) return MKV_ERR_SHAPE;
    if (q_stride < (int64_t)num_q_heads * pv.head_dim) return MKV_ERR_SHAPE;
    if (cur_layer < 0 || cur_layer >= pv.num_layers) return MKV_ERR_RANGE;
    if (batch == 0) return MKV_OK;
    if (!q || !o || !block_table || !seq_ids || !seq_lens) return MKV_ERR_NULL;
    if (workspace && ((uintptr_t)workspace & 255) != 0) return MKV_ERR_WORKSPACE;
    const int64_t blocks = ceil_div64((int64_t)batch * num_q_heads, 4);
    if (blocks > 0x7fffffff) return MKV_ERR_SHAPE;
    DeviceGuard guard(device);
    if (guard.err != cudaSuccess) return set_cuda_error(guard.err);
    int *flags = workspace && workspace_bytes >= 256 ? (int *)workspace : nullptr;
    const float scale_log2 = softmax_scale * kLog2e;
#define PLAIN(T, CODE)                                                                                                  \
    attn_q8_plain_kernel<T, CODE><<<(unsigned)blocks, 128, 0, (cudaStream_t)stream>>>(                                  \
        (const T *)q, q_stride, (T *)o, pv, block_table, table_stride, num_rows, seq_ids, seq_lens, batch, num_q_heads, \
        cur_layer, scale_log2, flags)
    if (pv.code == MKV_Q8_INT8) {
        if (dtype == MKV_F16) PLAIN(__half, MKV_Q8_INT8);
        else if (dtype == MKV_BF16) PLAIN(__nv_bfloat16, MKV_Q8_INT8);
        else PLAIN(float, MKV_Q8_INT8);
    } else {
        if (dtype == MKV_F16) PLAIN(__half, MKV_Q8_E4M3);
        else if (dtype == MKV_BF16) PLAIN(__nv_bfloat16, MKV_Q8_E4M3);
        else PLAIN(float, MKV_Q8_E4M3);
    }
#undef PLAIN
    MKV_LAUNCH_CHECK();
    return MKV_OK;
}

}  // extern "C"
