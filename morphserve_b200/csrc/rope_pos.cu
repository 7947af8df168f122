// Rotary embedding by position: no tables.  Pair j of token t turns by positions[t] * inv_freq[j].
//
// The angle is formed in 64 bits and reduced to a fraction of a turn there: a position of 10^5..10^6 leaves a 32-bit
// product without correct digits behind the point, while here the reduced angle is good to 2^-24 of half a turn.  One
// thread block computes the sines and cosines of its tokens once, in shared memory, for all heads of q and k; its first
// row loads are in flight meanwhile.  HBM bound: every element is read and written once.
#include "kv_q8.cuh"

namespace mkv {

struct RopePosArgs {
    const void *q, *k;
    void *q_out, *k_out;
    int64_t q_tok, q_head, k_tok, k_head, qo_tok, qo_head, ko_tok, ko_head;  // strides, elements
    const void *positions;
    const double *inv_freq;
    float scale;
    int64_t num_tokens;
    int num_pairs, q_heads, heads, head_dim;
    int pos64;
    int pair_tasks;     // tasks of V pairs in a head
    int tasks;          // ... and those that copy V elements behind the rotated part
    int tokens_per_block;
};

template <typename T, int V>
struct alignas(sizeof(T) * V) RopeVec {
    T x[V];
};

// One task: V pairs of one head (two vectors, read and written once), or V elements that pass through.
template <typename T, int V, bool INTER>
struct RopeTask {
    const T *src;
    T *dst;
    const float2 *turn;  // null: pass through
    int second;          // distance of the second vector
    RopeVec<T, V> a, b;

    __device__ __forceinline__ void load(const RopePosArgs &p, int64_t tok0, int idx, const float2 *turns) {
        const int per_tok = p.heads * p.tasks;
        const int tk = idx / per_tok, rem = idx - tk * per_tok, head = rem / p.tasks, j = rem - head * p.tasks;
        const int64_t tok = tok0 + tk;
        if (head < p.q_heads) {
            src = (const T *)p.q + tok * p.q_tok + head * p.q_head;
            dst = (T *)p.q_out + tok * p.qo_tok + head * p.qo_head;
        } else {
            src = (const T *)p.k + tok * p.k_tok + (head - p.q_heads) * p.k_head;
            dst = (T *)p.k_out + tok * p.ko_tok + (head - p.q_heads) * p.ko_head;
        }
        if (j < p.pair_tasks) {
            turn = turns + tk * p.num_pairs + j * V;
            second = INTER ? V : p.num_pairs;
            const int first = INTER ? 2 * V * j : V * j;
            src += first;
            dst += first;
            b = *reinterpret_cast<const RopeVec<T, V> *>(src + second);
        } else {
            turn = nullptr;
            const int first = 2 * p.num_pairs + (j - p.pair_tasks) * V;
            src += first;
            dst += first;
        }
        a = *reinterpret_cast<const RopeVec<T, V> *>(src);
    }
    __device__ __forceinline__ void finish() {
        if (turn) {
            T x[2 * V];
#pragma unroll
            for (int i = 0; i < V; ++i) {
                x[i] = a.x[i];
                x[V + i] = b.x[i];
            }
#pragma unroll
            for (int i = 0; i < V; ++i) {
                const int m = INTER ? 2 * i : i, n = INTER ? 2 * i + 1 : V + i;
                const float u = value_of<T>(x[m]), w = value_of<T>(x[n]);
                const float2 cs = turn[i];
                x[m] = rounded<T>(u * cs.x - w * cs.y);
                x[n] = rounded<T>(u * cs.y + w * cs.x);
            }
#pragma unroll
            for (int i = 0; i < V; ++i) {
                a.x[i] = x[i];
                b.x[i] = x[V + i];
            }
            *reinterpret_cast<RopeVec<T, V> *>(dst + second) = b;
        }
        *reinterpret_cast<RopeVec<T, V> *>(dst) = a;
    }
};

template <typename T, int V, bool INTER>
__global__ void rope_pos_kernel(const RopePosArgs p) {
    extern __shared__ float2 turns[];  // (cos, sin) * scale of [token of the block][pair]
    const int64_t tok0 = (int64_t)blockIdx.x * p.tokens_per_block;
    const int ntok = (int)min((int64_t)p.tokens_per_block, p.num_tokens - tok0);
    const int total = ntok * p.heads * p.tasks;
    RopeTask<T, V, INTER> t;
    int idx = threadIdx.x;
    if (idx < total) t.load(p, tok0, idx, turns);
    for (int i = threadIdx.x; i < ntok * p.num_pairs; i += blockDim.x) {
        const int tk = i / p.num_pairs, j = i - tk * p.num_pairs;
        const double pos = p.pos64 ? (double)((const int64_t *)p.positions)[tok0 + tk]
                                   : (double)((const int32_t *)p.positions)[tok0 + tk];
        // a radians are a / 2 pi turns; 1 / 2 pi in two parts, so that the fraction keeps its digits however many whole
        // turns go away
        const double a = pos * p.inv_freq[j];
        const double x = fma(a, 0.15915494309189535, -rint(a * 0.15915494309189535)) + a * -9.839338337591243e-18;
        float sn, cs;
        sincospif((float)(2.0 * x), &sn, &cs);
        turns[i] = make_float2(cs * p.scale, sn * p.scale);
    }
    __syncthreads();
    while (idx < total) {
        t.finish();
        idx += blockDim.x;
        if (idx < total) t.load(p, tok0, idx, turns);
    }
}

template <typename T, int V>
static cudaError_t launch_rope_pos(RopePosArgs p, bool interleaved, bool copies, cudaStream_t s) {
    const int rest = p.head_dim - 2 * p.num_pairs;
    p.pair_tasks = p.num_pairs / V;
    p.tasks = p.pair_tasks + (copies ? rest / V : 0);
    const int64_t per_tok = (int64_t)p.heads * p.tasks;
    // whole tokens for each block: at least a block's threads of tasks, as long as the sines fit in 16 KiB
    int n = 1;
    while (n * per_tok < 256 && (n + 1) * p.num_pairs <= 2048) ++n;
    p.tokens_per_block = n;
    const int64_t blocks = ceil_div64(p.num_tokens, n);
    const size_t smem = (size_t)n * p.num_pairs * sizeof(float2);
    if (interleaved)
        rope_pos_kernel<T, V, true><<<(unsigned)blocks, 256, smem, s>>>(p);
    else
        rope_pos_kernel<T, V, false><<<(unsigned)blocks, 256, smem, s>>>(p);
    return cudaGetLastError();
}

}  // namespace mkv

using namespace mkv;

extern "C" int mkv_rotary_positions(int device, void *stream, const void *q, const void *k, void *q_out, void *k_out,
                                    const int64_t *strides, const void *positions, int positions_bytes,
                                    const double *inv_freq, int num_pairs, int interleaved, float attention_scale,
                                    int64_t num_tokens, int num_q_heads, int num_kv_heads, int head_dim, int dtype) {
    if (!dtype_ok(dtype) || (positions_bytes != 4 && positions_bytes != 8)) return MKV_ERR_DTYPE;
    if (num_tokens < 0 || num_tokens > 0x7fffffff || num_q_heads < 0 || num_kv_heads < 0 || num_q_heads + num_kv_heads < 1 ||
        head_dim < 2 || num_pairs < 1 || 2 * num_pairs > head_dim || num_pairs > 2048)
        return MKV_ERR_SHAPE;
    if ((int64_t)(num_q_heads + num_kv_heads) * head_dim > (1 << 26)) return MKV_ERR_SHAPE;
    if (num_tokens == 0) return MKV_OK;
    if (!strides || !positions || !inv_freq) return MKV_ERR_NULL;
    if ((num_q_heads && (!q || !q_out)) || (num_kv_heads && (!k || !k_out))) return MKV_ERR_NULL;
    RopePosArgs p;
    p.q = q; p.k = k; p.q_out = q_out; p.k_out = k_out;
    p.q_tok = strides[0]; p.q_head = strides[1]; p.k_tok = strides[2]; p.k_head = strides[3];
    p.qo_tok = strides[4]; p.qo_head = strides[5]; p.ko_tok = strides[6]; p.ko_head = strides[7];
    p.positions = positions;
    p.inv_freq = inv_freq;
    p.scale = attention_scale;
    p.num_tokens = num_tokens;
    p.num_pairs = num_pairs;
    p.q_heads = num_q_heads;
    p.heads = num_q_heads + num_kv_heads;
    p.head_dim = head_dim;
    p.pos64 = positions_bytes == 8;
    DeviceGuard guard(device);
    if (guard.err != cudaSuccess) return set_cuda_error(guard.err);
    // the widest vector that bases, strides and the split of the head allow (16 bytes at most)
    const bool copies = !(q == q_out && k == k_out) && 2 * num_pairs < head_dim;
    uint64_t elems = (uint64_t)num_pairs;
    if (copies) elems |= (uint64_t)(head_dim - 2 * num_pairs);
    uint64_t bytes = 0;
    for (int i = 0; i < 8; ++i)
        if ((i < 2 || i == 4 || i == 5) ? num_q_heads : num_kv_heads) elems |= (uint64_t)strides[i];
    if (num_q_heads) bytes |= (uint64_t)q | (uint64_t)q_out;
    if (num_kv_heads) bytes |= (uint64_t)k | (uint64_t)k_out;
    const int size = dtype_bytes(dtype);
    int vec = 16 / size;
    while (vec > 1 && ((elems & (vec - 1)) || (bytes & ((uint64_t)vec * size - 1)))) vec >>= 1;
    const bool in = interleaved != 0;
    cudaStream_t s = (cudaStream_t)stream;
    cudaError_t e;
#define ROPE_V(T)                                                              \
    (vec == 8   ? launch_rope_pos<T, 8>(p, in, copies, s)                      \
     : vec == 4 ? launch_rope_pos<T, 4>(p, in, copies, s)                      \
     : vec == 2 ? launch_rope_pos<T, 2>(p, in, copies, s) : launch_rope_pos<T, 1>(p, in, copies, s))
    if (dtype == MKV_F16) e = ROPE_V(__half);
    else if (dtype == MKV_BF16) e = ROPE_V(__nv_bfloat16);
    else e = vec == 4 ? launch_rope_pos<float, 4>(p, in, copies, s)
             : vec == 2 ? launch_rope_pos<float, 2>(p, in, copies, s) : launch_rope_pos<float, 1>(p, in, copies, s);
#undef ROPE_V
    if (e != cudaSuccess) return set_cuda_error(e);
    return MKV_OK;
}
