// Row kernels of the cache's operators (gfx950): heads turned by positions, keys
// and values to 8 bits into their pages, and back.  All are one pass over their
// data and bounded by memory.
#include "cache_device.hpp"

namespace q8 {
namespace {

constexpr uint32_t kThreads = 256;
// Work-groups that a launch has at most (2^32 work-items are one grid's end); they take their tokens in turn.
constexpr uint32_t kMostGroups = 1u << 20;

// sin and cos of position * freq: the product exact in two doubles, in turns (1 / 2 pi in two doubles), less
// the whole ones and then the nearest quarter, so that what is left, at most an eighth of a turn, is FP32 to
// half a unit however far the position.
__device__ __forceinline__ void angle(int position, float freq, float& c, float& s) {
    constexpr double kTurn = 0.15915494309189535, kTurnLow = -9.839338337591243e-18;
    const double p = (double)position, f = (double)freq;
    const double t = p * f, tl = __builtin_fma(p, f, -t);
    const double u = t * kTurn, ul = __builtin_fma(t, kTurn, -u) + (t * kTurnLow + tl * kTurn);
    const double part = (u - __builtin_rint(u)) + ul;
    const double quarter = __builtin_rint(part * 4.0);
    const float r = (float)(part * 2.0 - quarter * 0.5);      // in half turns, at most a quarter
    const float cr = cospif(r), sr = sinpif(r);
    const int q = (int)quarter & 3;
    c = q == 0 ? cr : q == 1 ? -sr : q == 2 ? -cr : sr;
    s = q == 0 ? sr : q == 1 ? cr : q == 2 ? -sr : -cr;
}

// A work-group turns the heads of `p.step` tokens: sine and cosine once for each token and pair, into LDS, and then
// items of eight pairs (or eight values, of neighbours and of those that stay).  An item's values are
// read and written by one thread, two items' loads before their stores, so y may be x.  (16384 tokens of 40 heads of 128, BF16: two tokens
// a work-group and two items at once 68.5 us, 4.9 TB/s, a large copy's 5.1; eight and four 79.1.  One token: 3.1 us.)
constexpr uint32_t kAngles = 2 * Q8_MAX_DIM / 2;
struct RotaryPlan {
    Rotary p;
    uint32_t step;              // tokens a work-group
    uint32_t turned, items;     // items of a head: with pairs, in all
    Divisor by_items, by_heads, by_pairs;
};

template <int DT, bool NEIGHBOURS> __global__ void __launch_bounds__(kThreads) rotary_kernel(const RotaryPlan a) {
    typedef typename Type<DT>::T T;
    __shared__ float cosine[kAngles], sine[kAngles];
    const Rotary& p = a.p;
    const uint32_t pairs = p.form.pairs;
    for (uint32_t first = blockIdx.x * a.step; first < p.tokens; first += gridDim.x * a.step) {
        const uint32_t tokens = min(a.step, p.tokens - first);
        for (uint32_t i = threadIdx.x; i < tokens * pairs; i += kThreads) {
            const uint32_t token = divide(i, a.by_pairs), j = i - token * pairs;
            float c, s;
            angle(p.positions[(uint64_t)p.form.axis[j] * p.ldp + first + token], p.freq[j], c, s);
            cosine[i] = c;
            sine[i] = p.inverse ? -s : s;
        }
        __syncthreads();
        const uint32_t count = tokens * p.heads * a.items;
        constexpr int AT_ONCE = 2;
        for (uint32_t i0 = threadIdx.x; i0 < count; i0 += kThreads * AT_ONCE) {
            float v[AT_ONCE][2][8];
            uint32_t token[AT_ONCE], item[AT_ONCE], column[AT_ONCE];
#pragma unroll
            for (int n = 0; n < AT_ONCE; ++n) {
                const uint32_t i = i0 + n * kThreads;
                if (i >= count) continue;
                const uint32_t row = divide(i, a.by_items);
                token[n] = divide(row, a.by_heads);
                item[n] = i - row * a.items;
                column[n] = (row - token[n] * p.heads) * p.form.dim;
                const T* x = (const T*)p.x + (uint64_t)(first + token[n]) * p.ldx + column[n];
                if (item[n] >= a.turned) load_part<DT>(x, 2 * pairs + (item[n] - a.turned) * 8, p.form.dim, v[n][0]);
                else if (NEIGHBOURS) load_part<DT>(x, item[n] * 8, 2 * pairs, v[n][0]);
                else {
                    load_part<DT>(x, item[n] * 8, pairs, v[n][0]);
                    load_part<DT>(x + pairs, item[n] * 8, pairs, v[n][1]);
                }
            }
#pragma unroll
            for (int n = 0; n < AT_ONCE; ++n) {
                const uint32_t i = i0 + n * kThreads;
                if (i >= count) continue;
                T* y = (T*)p.y + (uint64_t)(first + token[n]) * p.ldy + column[n];
                if (item[n] >= a.turned) {
                    store_part<DT>(y, 2 * pairs + (item[n] - a.turned) * 8, p.form.dim, v[n][0]);
                } else if (NEIGHBOURS) {
                    float w[8];
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const uint32_t j = token[n] * pairs + min(item[n] * 4 + e, pairs - 1);
                        const float c = cosine[j], s = sine[j], x1 = v[n][0][2 * e], x2 = v[n][0][2 * e + 1];
                        w[2 * e] = x1 * c - x2 * s;
                        w[2 * e + 1] = x2 * c + x1 * s;
                    }
                    store_part<DT>(y, item[n] * 8, 2 * pairs, w);
                } else {
                    float w[2][8];
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        const uint32_t j = token[n] * pairs + min(item[n] * 8 + e, pairs - 1);
                        const float c = cosine[j], s = sine[j], x1 = v[n][0][e], x2 = v[n][1][e];
                        w[0][e] = x1 * c - x2 * s;
                        w[1][e] = x2 * c + x1 * s;
                    }
                    store_part<DT>(y, item[n] * 8, pairs, w[0]);
                    store_part<DT>(y + pairs, item[n] * 8, pairs, w[1]);
                }
            }
        }
        __syncthreads();
    }
}

// Where the tokens first .. first + count of a work-group lie: row of head 0, -1 (a place that is not there) or
// -2 (no chunk's).  The first token's sequence by counting starts, all threads at once; the others' from there on.
__device__ __forceinline__ void find_places(const Paged& c, uint32_t first, uint32_t count, int64_t* place, uint32_t* sum) {
    if (threadIdx.x == 0) *sum = 0;
    __syncthreads();
    uint32_t below = 0;
    for (uint32_t i = threadIdx.x; i < c.seqs; i += kThreads) below += c.starts[i + 1] <= (int)first;
    if (below) atomicAdd(sum, below);
    __syncthreads();
    if (threadIdx.x < count) {
        const int token = (int)(first + threadIdx.x);
        uint32_t b = *sum;
        while (b < c.seqs && c.starts[b + 1] <= token) ++b;
        place[threadIdx.x] = b >= c.seqs || token < c.starts[b]
                                 ? -2 : row_at(c, b, (int64_t)c.lengths[b] - chunk_end(c, b) + token);
    }
    __syncthreads();
}

// Keys and values: G threads a head of eight values each, `step` tokens a work-group.  (16384 tokens of 8 heads of 128, BF16: writing 27.6 us,
// 3.6 TB/s: a thread has one load of 16 bytes on its way, in 16 passes that wait for one another; reading 19.0, 5.3 TB/s; a large copy 5.1.)
constexpr uint32_t kMostStep = 16;
struct CachePlan {
    CacheRows p;
    uint32_t step;
    Divisor by_heads;
};

template <int DT, int G> __global__ void __launch_bounds__(kThreads) cache_write_kernel(const CachePlan a) {
    typedef typename Type<DT>::T T;
    __shared__ int64_t place[kMostStep];
    __shared__ uint32_t sum;
    const Paged& c = a.p.at;
    for (uint32_t first = blockIdx.x * a.step; first < c.tokens; first += gridDim.x * a.step) {
        const uint32_t tokens = min(a.step, c.tokens - first);
        find_places(c, first, tokens, place, &sum);
        const uint32_t lane = threadIdx.x % G, rows = tokens * 2 * c.heads, at = lane * 8;
        for (uint32_t r0 = threadIdx.x / G; r0 < rows; r0 += kThreads / G) {
            const uint32_t half = divide(r0, a.by_heads), head = r0 - half * c.heads, token = half >> 1;
            const bool value = half & 1;
            const int64_t to = place[token];
            if (to < 0) continue;       // the same for the G threads of a row
            const T* x = value ? (const T*)a.p.v + (uint64_t)(first + token) * a.p.ldv + head * c.dim
                               : (const T*)a.p.k + (uint64_t)(first + token) * a.p.ldk + head * c.dim;
            float v[8] = {};
            if (at < c.dim) load_part<DT>(x, at, c.dim, v);
            uint32_t top = 0;
#pragma unroll
            for (int e = 0; e < 8; ++e) top = max(top, magnitude(v[e]));
#pragma unroll
            for (int m = 1; m < G; m *= 2) top = max(top, (uint32_t)__shfl_xor((int)top, m));
            const Scale s = scale_of(top, 1.0f);
            const int64_t row = to + (int64_t)head * c.page_tokens;
            if (lane == 0) (value ? c.v_scale : c.k_scale)[row] = s.s;
            if (at < c.pitch) *reinterpret_cast<u32x2*>((value ? c.v : c.k) + row * c.pitch + at) = bytes8(v, s);
        }
    }
}

template <int DT, int G> __global__ void __launch_bounds__(kThreads) cache_read_kernel(const CachePlan a) {
    typedef typename Type<DT>::T T;
    __shared__ int64_t place[kMostStep];
    __shared__ uint32_t sum;
    const Paged& c = a.p.at;
    for (uint32_t first = blockIdx.x * a.step; first < c.tokens; first += gridDim.x * a.step) {
        const uint32_t tokens = min(a.step, c.tokens - first);
        find_places(c, first, tokens, place, &sum);
        const uint32_t lane = threadIdx.x % G, rows = tokens * 2 * c.heads, at = lane * 8;
        for (uint32_t r0 = threadIdx.x / G; r0 < rows; r0 += kThreads / G) {
            const uint32_t half = divide(r0, a.by_heads), head = r0 - half * c.heads, token = half >> 1;
            const bool value = half & 1;
            const int64_t from = place[token];
            if (from == -2 || at >= c.dim) continue;
            T* y = value ? (T*)a.p.v + (uint64_t)(first + token) * a.p.ldv + head * c.dim
                         : (T*)a.p.k + (uint64_t)(first + token) * a.p.ldk + head * c.dim;
            float v[8] = {};
            if (from >= 0) {
                const int64_t row = from + (int64_t)head * c.page_tokens;
                const float s = (value ? c.v_scale : c.k_scale)[row];
                const u32x2 w = *reinterpret_cast<const u32x2*>((value ? c.v : c.k) + row * c.pitch + at);
#pragma unroll
                for (int e = 0; e < 8; ++e) v[e] = (float)(int8_t)(w[e / 4] >> (8 * (e % 4))) * s;
            }
            store_part<DT>(y, at, c.dim, v);
        }
    }
}

uint32_t groups_for(uint32_t tokens, uint32_t step) {
    const uint64_t g = ceil_div(tokens, step);
    return (uint32_t)(g < kMostGroups ? g : kMostGroups);
}

template <typename P> hipError_t launch(void (*f)(P), uint32_t groups, const P& p, hipStream_t stream) {
    void* args[] = {const_cast<P*>(&p)};
    return hipLaunchKernel(reinterpret_cast<const void*>(f), dim3(groups), dim3(kThreads), args, 0, stream);
}

template <int DT> hipError_t rotary_any(const RotaryPlan& a, hipStream_t s) {
    const uint32_t groups = groups_for(a.p.tokens, a.step);
    return a.p.form.neighbours ? launch(rotary_kernel<DT, true>, groups, a, s) : launch(rotary_kernel<DT, false>, groups, a, s);
}

template <int DT, bool WRITE> hipError_t cache_any(const CacheRows& p, hipStream_t s) {
    const Paged& c = p.at;
    // Tokens a work-group, as many as leave each CU some work-groups (written and read, 8 heads of 128, us): 16384 tokens BF16 51.5 by 16
    // and 56.5 by 8; 4096 16.9 by 4, 18.9 by 2, 21.0 by one; 2048 FP32 13.5, 12.4, 14.5; 1239 of 3 heads of 80 9.6 by 4 and 9.0 by one.
    const uint32_t step = c.tokens >= 8192 ? 16 : c.tokens >= 4096 ? 4 : c.tokens >= 2048 ? 2 : 1;
    const CachePlan a = {p, step, divisor(c.heads)};
    const uint32_t groups = groups_for(c.tokens, step);
    if (c.dim <= 64) return launch(WRITE ? cache_write_kernel<DT, 8> : cache_read_kernel<DT, 8>, groups, a, s);
    if (c.dim <= 128) return launch(WRITE ? cache_write_kernel<DT, 16> : cache_read_kernel<DT, 16>, groups, a, s);
    return launch(WRITE ? cache_write_kernel<DT, 32> : cache_read_kernel<DT, 32>, groups, a, s);
}

}  // namespace

hipError_t launch_rotary(int dtype, const Rotary& p, hipStream_t s) {
    const q8_rotation& f = p.form;
    RotaryPlan a = {};
    a.p = p;
    // 40 heads of 128, BF16: 4096 tokens 15.3 us by two and 17.8 by one, 1024 tokens 7.0 and 6.3
    a.step = p.tokens >= 2048 ? 2 : 1;
    a.turned = (uint32_t)ceil_div(f.neighbours ? 2 * f.pairs : f.pairs, 8);
    a.items = a.turned + (p.y == p.x ? 0 : (uint32_t)ceil_div(f.dim - 2 * f.pairs, 8));
    if (!a.items) return hipSuccess;
    a.by_items = divisor(a.items);
    a.by_heads = divisor(p.heads);
    a.by_pairs = divisor(f.pairs ? f.pairs : 1);
    return dtype == Q8_F32 ? rotary_any<Q8_F32>(a, s) : dtype == Q8_F16 ? rotary_any<Q8_F16>(a, s) : rotary_any<Q8_BF16>(a, s);
}

hipError_t launch_cache_write(int dtype, const CacheRows& p, hipStream_t s) {
    return dtype == Q8_F32 ? cache_any<Q8_F32, true>(p, s)
                           : dtype == Q8_F16 ? cache_any<Q8_F16, true>(p, s) : cache_any<Q8_BF16, true>(p, s);
}

hipError_t launch_cache_read(int dtype, const CacheRows& p, hipStream_t s) {
    return dtype == Q8_F32 ? cache_any<Q8_F32, false>(p, s)
                           : dtype == Q8_F16 ? cache_any<Q8_F16, false>(p, s) : cache_any<Q8_BF16, false>(p, s);
}

hipError_t prepare_cache_rows() {
    hipFuncAttributes a;
    return hipFuncGetAttributes(&a, reinterpret_cast<const void*>(&cache_read_kernel<Q8_F32, 32>));
}

}  // namespace q8
