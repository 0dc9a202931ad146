// attention.hip -- attention of new tokens over a paged fp16 cache.
//
// Token j of a request with n cached and new tokens, m of them new, is at position
// p = n - m + j.  Its output is sum_k w_k v_k / sum_k w_k over the keys k that it sees,
// w_k = exp(s_k - max s), s_k = scale q . k_k, with the maximum and the sums carried
// over the keys in one pass.
#include "common.h"

#include <algorithm>

namespace ds3k {

// The request of row t (below offsets[n_seq]).
__device__ __forceinline__ int request_of(const int32_t *offsets, int n_seq, int t)
{
    int lo = 0, hi = n_seq;
    while (hi - lo > 1) {
        const int mid = (lo + hi) / 2;
        if (offsets[mid] <= t) lo = mid;
        else hi = mid;
    }
    return lo;
}

// One wave a row and q head: a lane takes a key of each 64 for the scores, then
// values of the head for the products.
template <typename T>
__global__ void __launch_bounds__(64) k_attn_rows(AttnArgs p)
{
    __shared__ float q_s[256];
    const int t = blockIdx.x / p.n_head, h = blockIdx.x % p.n_head, g = h / (p.n_head / p.n_head_kv), lane = threadIdx.x;
    if (t >= min(p.offsets[p.n_seq], p.n_tokens)) return;
    const int i = request_of(p.offsets, p.n_seq, t);
    const T *q = (const T *)((const uint8_t *)p.q + (uint64_t)t * p.q_stride) + (int64_t)h * p.head_dim;
    for (int d = lane; d < p.head_dim; d += 64) q_s[d] = (float)q[d];
    __syncthreads();
    const int64_t n = min((int64_t)max(p.lens[i], 0), (int64_t)p.max_blocks << p.log_block);
    const int64_t pos = (int64_t)p.lens[i] - p.offsets[i + 1] + t, last = min(pos, n - 1);
    const int64_t first = p.window ? max(pos - p.window + 1, (int64_t)0) : 0;
    float m = -INFINITY, sum = 0.0f, acc[4] = { 0, 0, 0, 0 };
    for (int64_t k0 = first; k0 <= last; k0 += 64) {
        const int64_t key = k0 + lane;
        int64_t at = -1;                              // the key's row of the cache
        if (key <= last) {
            const int block = p.table[(int64_t)i * p.max_blocks + (key >> p.log_block)];
            if (block >= 0 && block < p.n_blocks)
                at = ((((int64_t)block * p.n_head_kv + g) << p.log_block) + (key & ((1 << p.log_block) - 1))) * p.head_dim;
        }
        float s = -INFINITY;
        if (at >= 0) {
            s = 0.0f;
            for (int d = 0; d < p.head_dim; d++) s += q_s[d] * (float)p.k[at + d];
            s *= p.scale;
        }
        float top = s;
        for (int d = 32; d > 0; d /= 2) top = fmaxf(top, __shfl_xor(top, d));
        const float m2 = fmaxf(m, top);
        if (m2 == -INFINITY) continue;
        const float w = expf(s - m2), keep = expf(m - m2);
        float add = w;
        for (int d = 32; d > 0; d /= 2) add += __shfl_xor(add, d);
        sum = sum * keep + add;
        m = m2;
#pragma unroll
        for (int r = 0; r < 4; r++) acc[r] *= keep;
        for (int j = 0; j < 64; j++) {
            const float wj = __shfl(w, j);
            const int64_t aj = __shfl(at, j);
            if (aj < 0) continue;
#pragma unroll
            for (int r = 0; r < 4; r++)
                if (lane + 64 * r < p.head_dim) acc[r] += wj * (float)p.v[aj + lane + 64 * r];
        }
    }
    T *out = (T *)((uint8_t *)p.out + (uint64_t)t * p.out_stride) + (int64_t)h * p.head_dim;
#pragma unroll
    for (int r = 0; r < 4; r++)
        if (lane + 64 * r < p.head_dim) out[lane + 64 * r] = (T)(sum == 0.0f ? 0.0f : acc[r] / sum);
}

hipError_t launch_attention(const AttnArgs &p, int type, hipStream_t s)
{
    const dim3 grid((unsigned)p.n_tokens * p.n_head);
    if (type == T_F32) hipLaunchKernelGGL(k_attn_rows<float>, grid, 64, 0, s, p);
    else hipLaunchKernelGGL(k_attn_rows<_Float16>, grid, 64, 0, s, p);
    return hipGetLastError();
}

}  // namespace ds3k
