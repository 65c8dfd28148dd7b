// Attention of new tokens over a paged cache of 8-bit keys and values (gfx950).
#include "cache_device.hpp"

namespace q8 {
namespace {

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

// A wave for each token and head: 64 keys at a time, one a lane for the scores; then the values' sums, four
// of them a lane.
template <int DT> __global__ void __launch_bounds__(64) row_kernel(const Attention a) {
    typedef typename Type<DT>::T T;
    __shared__ float q[Q8_MAX_DIM], weight[64];
    const Paged& c = a.at;
    const uint32_t lane = threadIdx.x, head = blockIdx.x % a.heads, token = blockIdx.x / a.heads;
    uint32_t b = 0;
    while (b < c.seqs && c.starts[b + 1] <= (int)token) ++b;
    if (b >= c.seqs || (int)token < c.starts[b]) return;
    const int64_t p = (int64_t)c.lengths[b] - chunk_end(c, b) + token;
    const int64_t last = min(p, (int64_t)c.lengths[b] - 1);
    const int64_t first = a.window ? max((int64_t)0, p - a.window + 1) : 0;
    const T* row = (const T*)a.q + (uint64_t)token * a.ldq + head * c.dim;
    for (uint32_t d = lane; d < Q8_MAX_DIM; d += 64) q[d] = d < c.dim ? Type<DT>::get(row + d) : 0.0f;
    __syncthreads();
    const uint32_t kv = head / a.group;
    float m = -__builtin_huge_valf(), l = 0.0f, o[4] = {};
    for (int64_t j0 = first; j0 <= last; j0 += 64) {
        const int64_t at = j0 + lane <= last ? row_at(c, b, j0 + lane) : -1;
        const int64_t r = at < 0 ? -1 : at + (int64_t)kv * c.page_tokens;
        float t = -__builtin_huge_valf();
        if (r >= 0) {
            float sum = 0.0f;
            for (uint32_t d = 0; d < c.dim; ++d) sum = __builtin_fmaf(q[d], (float)c.k[r * c.pitch + d], sum);
            t = sum * c.k_scale[r] * (a.scale * kLog2e);
        }
        float top = t;
        for (int x = 1; x < 64; x *= 2) top = fmaxf(top, __shfl_xor(top, x));
        const float next = fmaxf(m, top), base = next == -__builtin_huge_valf() ? 0.0f : next;
        const float w = r >= 0 ? __builtin_exp2f(t - base) : 0.0f, down = __builtin_exp2f(m - base);
        float s = w;
        for (int x = 1; x < 64; x *= 2) s += __shfl_xor(s, x);
        l = l * down + s;
        m = next;
        weight[lane] = r >= 0 ? w * c.v_scale[r] : 0.0f;
        __syncthreads();
#pragma unroll
        for (int e = 0; e < 4; ++e) o[e] *= down;
        for (int j = 0; j < 64; ++j) {
            const int64_t rj = __shfl(r, j);
            if (rj < 0) continue;
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (lane + 64 * e < c.dim) o[e] = __builtin_fmaf(weight[j], (float)c.v[rj * c.pitch + lane + 64 * e], o[e]);
        }
        __syncthreads();
    }
    T* out = (T*)a.out + (uint64_t)token * a.ldo + head * c.dim;
#pragma unroll
    for (int e = 0; e < 4; ++e)
        if (lane + 64 * e < c.dim) Type<DT>::put(out + lane + 64 * e, l == 0.0f ? 0.0f : o[e] / l);
    if (a.lse && lane == 0) a.lse[(uint64_t)token * a.heads + head] = l == 0.0f ? -__builtin_huge_valf() : (m + __builtin_log2f(l)) * kLn2;
}

template <int DT> hipError_t attention_any(const Attention& a, hipStream_t s) {
    void* args[] = {const_cast<Attention*>(&a)};
    return hipLaunchKernel(reinterpret_cast<const void*>(&row_kernel<DT>), dim3(a.at.tokens * a.heads), dim3(64), args, 0, s);
}

}  // namespace

hipError_t launch_attention(int dtype, const Attention& a, hipStream_t s) {
    return dtype == Q8_F32 ? attention_any<Q8_F32>(a, s)
                           : dtype == Q8_F16 ? attention_any<Q8_F16>(a, s) : attention_any<Q8_BF16>(a, s);
}

hipError_t prepare_attention() {
    hipFuncAttributes a;
    return hipFuncGetAttributes(&a, reinterpret_cast<const void*>(&row_kernel<Q8_F32>));
}

}  // namespace q8
