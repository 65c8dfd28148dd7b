// Attention of many new tokens over the paged cache (gfx950): chunks and prompts.
#include "cache_attention_device.hpp"

namespace q8 {
namespace {

typedef float f32x16 __attribute__((ext_vector_type(16)));

template <bool H> __device__ __forceinline__ void mfma32(u32x4 a, u32x4 b, f32x16& c) {
    if constexpr (H) c = __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
    else c = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

// A work-group of four waves has a tile of 128 RB rows, 32 RB a wave, and takes 64 keys a step: keys and values go from
// memory to registers, and as 16-bit values to LDS while the step before them is computed, which has them once for all rows.
// Keys lie in LDS by rows of a key's values, values by rows of one value's keys, both in pieces of 16 bytes whose place
// in the row is turned by the row's number, so that reads of 16 bytes down a column meet all banks.  The eight keys of a piece
// of the values are those that a lane has of each 16 after the scores (0-3, 8-11 and 4-7, 12-15).
constexpr int kWaves = 4, kThreads = 64 * kWaves;
template <int DT, int DP, int RB> struct Many {
    static constexpr int TERMS = DT == Q8_F32 ? 3 : 1, ROWS = 32 * RB * kWaves;
    static constexpr bool QH = DT == Q8_F16, VH = DT != Q8_F32;
    static constexpr int KEY_LOADS = 64 * (DP / 16) / kThreads;                     // 16 bytes each
    static constexpr int VALUE_UNITS = 8 * (DP / 4);                                // eight keys of four values
    static constexpr int VALUE_LOADS = (VALUE_UNITS + kThreads - 1) / kThreads;
    struct Shared {
        u32x4 k[2][64 * (DP / 8)];
        u32x4 v[2][DP * 8];
        uint64_t offset[kWaves][64];
        float scale[kWaves][128];
    };
};

template <int DT, int DP, int RB> __global__ void __launch_bounds__(kThreads, 1) many_kernel(const AttentionArgs g) {
    typedef Many<DT, DP, RB> F;
    typedef typename Type<DT>::T T;
    constexpr int TERMS = F::TERMS, S = DP / 16, D = DP / 32;
    __shared__ typename F::Shared shared;
    const Attention& a = g.a;
    const Paged& c = a.at;
    const uint32_t kv = blockIdx.x % c.heads, piece = blockIdx.y;
    Place t;
    // the last tiles of a sequence see the most keys and come first
    if (!find_tile(g, g.slots - 1 - blockIdx.x / c.heads, F::ROWS, t)) return;
    const int pieces = max(1, pieces_of(t, g.piece));
    if ((int)piece >= pieces) return;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, n = lane & 31, half = lane >> 5;
    const int begin = t.begin + (int)(piece * g.piece), end = min(t.end, begin + (int)g.piece);

    // this lane's rows, one of each 32; those past the tile's are its last
    int position[RB];
    int64_t oldest[RB];
    Row at[RB];
    bool mine[RB];
#pragma unroll
    for (int b = 0; b < RB; ++b) {
        const int r = wave * 32 * RB + b * 32 + n, rr = min(r, t.rows - 1);
        mine[b] = r < t.rows;
        at[b] = row_of(g, t, kv, rr);
        position[b] = t.at + ((int)at[b].row - t.first);
        oldest[b] = a.window ? (int64_t)position[b] - a.window + 1 : INT32_MIN;
    }
    // of this wave's rows: the first's and the last's position
    const int low = __builtin_amdgcn_readlane(position[0], 0);
    const int high = wave * 32 * RB < t.rows ? __builtin_amdgcn_readlane(position[RB - 1], 31) : -1;     // -1: no rows, nothing to compute
    const int64_t all_from = a.window ? (int64_t)high - a.window + 1 : INT32_MIN, none_to = a.window ? (int64_t)low - a.window + 1 : INT32_MIN;

    u32x4 q[RB][S][TERMS];
#pragma unroll
    for (int b = 0; b < RB; ++b) {
        const T* row = (const T*)a.q + at[b].row * a.ldq + at[b].head * c.dim;
#pragma unroll
        for (int s = 0; s < S; ++s) {
            const uint32_t d = s * 16 + half * 8;
            float v[8] = {};
            if (mine[b] && d < c.dim) load_part<DT>(row, d, c.dim, v);
            terms_of<TERMS, F::QH>(v, q[b][s]);
        }
    }
    const float factor = a.scale * kLog2e;
    float R[RB], l[RB];
    f32x16 o[RB][D];
#pragma unroll
    for (int b = 0; b < RB; ++b) {
        R[b] = kUnset;
        l[b] = 0.0f;
#pragma unroll
        for (int d = 0; d < D; ++d)
#pragma unroll
            for (int i = 0; i < 16; ++i) o[b][d][i] = 0.0f;
    }

    const int64_t head_rows = (int64_t)kv * c.page_tokens, page_rows = (int64_t)c.heads * c.page_tokens;
    auto page_of = [&](int k) __attribute__((always_inline)) {
        return k + lane < end ? page_at(c, t.b, divide((uint32_t)(k + lane), c.page)) : -1;
    };
    uint64_t* offset = shared.offset[wave];
    float* factors = shared.scale[wave];
    u32x4 ks[F::KEY_LOADS];
    uint32_t vs[F::VALUE_LOADS][8];
    float k_scale = 0.0f, v_scale = 0.0f;
    // A step's loads; every wave finds all 64 keys for itself.  Rows of keys that are not there become those of one that
    // is; 0: none is.
    auto load = [&](int k, int page) __attribute__((always_inline)) {
        const uint64_t there = __ballot(page >= 0);
        if (!there) return there;
        const uint32_t key = (uint32_t)(k + lane), slot = key - divide(key, c.page) * c.page_tokens;
        int64_t row = page * page_rows + head_rows + slot;
        const int some = __builtin_ctzll(there);
        const int64_t other = (int64_t)((uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(row >> 32), some) << 32 |
                                        (uint32_t)__builtin_amdgcn_readlane((int)row, some));
        row = page < 0 ? other : row;
        k_scale = c.k_scale[row];
        v_scale = c.v_scale[row];
        offset[lane] = (uint64_t)row * c.pitch;
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int x = 0; x < F::KEY_LOADS; ++x) {
            const int u = tid + x * kThreads, key_of = u / (DP / 16), d = u % (DP / 16) * 16;
            ks[x] = *reinterpret_cast<const u32x4*>(c.k + offset[key_of] + (d < (int)c.pitch ? d : 0));
        }
#pragma unroll
        for (int x = 0; x < F::VALUE_LOADS; ++x) {
            const int u = tid + x * kThreads, part = u / (DP / 4), d = u % (DP / 4) * 4;
            if (F::VALUE_UNITS % kThreads && u >= F::VALUE_UNITS) break;
            const int first = part / 2 * 16 + part % 2 * 4;
#pragma unroll
            for (int e = 0; e < 8; ++e)
                vs[x][e] = *reinterpret_cast<const uint32_t*>(c.v + offset[first + (e >> 2) * 8 + (e & 3)] + (d < (int)c.pitch ? d : 0));
        }
        __builtin_amdgcn_wave_barrier();
        return there;
    };
    auto store = [&](int to) __attribute__((always_inline)) {
#pragma unroll
        for (int x = 0; x < F::KEY_LOADS; ++x) {
            const int u = tid + x * kThreads, key_of = u / (DP / 16), part = u % (DP / 16) * 2;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const u32x2 w0 = four<F::QH>(kept(ks[x][2 * h])), w1 = four<F::QH>(kept(ks[x][2 * h + 1]));
                shared.k[to][key_of * (DP / 8) + ((part + h) ^ (key_of & (DP / 8 < 16 ? 7 : 15)))] = u32x4{w0[0], w0[1], w1[0], w1[1]};
            }
        }
#pragma unroll
        for (int x = 0; x < F::VALUE_LOADS; ++x) {
            const int u = tid + x * kThreads, part = u / (DP / 4), d = u % (DP / 4) * 4;
            if (F::VALUE_UNITS % kThreads && u >= F::VALUE_UNITS) break;
            uint32_t w[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) w[e] = kept(vs[x][e]);
            u32x4 r[4];
            columns<F::VH>(w, r);
#pragma unroll
            for (int j = 0; j < 4; ++j) shared.v[to][(d + j) * 8 + (part ^ ((d + j) & 7))] = r[j];
        }
    };
    // 32 keys from k, the i-th half of a step's
    auto compute = [&](int from, int i, int k, uint32_t there) __attribute__((always_inline)) {
        if (!there || k > high || k + 31 < none_to) return;
        f32x16 score[RB];
#pragma unroll
        for (int b = 0; b < RB; ++b)
#pragma unroll
            for (int e = 0; e < 16; ++e) score[b][e] = 0.0f;
#pragma unroll
        for (int s = 0; s < S; ++s) {
            const int key_of = i * 32 + n;
            const u32x4 w = shared.k[from][key_of * (DP / 8) + ((2 * s + half) ^ (key_of & (DP / 8 < 16 ? 7 : 15)))];
#pragma unroll
            for (int b = 0; b < RB; ++b)
#pragma unroll
                for (int m = 0; m < TERMS; ++m) mfma32<F::QH>(w, q[b][s][m], score[b]);
        }
        float sk[16], sv[16];
#pragma unroll
        for (int e = 0; e < 16; e += 4) {
            const f32x4 x = *reinterpret_cast<const f32x4*>(factors + i * 32 + 2 * e + 4 * half);
            const f32x4 y = *reinterpret_cast<const f32x4*>(factors + 64 + i * 32 + 2 * e + 4 * half);
#pragma unroll
            for (int z = 0; z < 4; ++z) { sk[e + z] = x[z]; sv[e + z] = y[z]; }
        }
        __builtin_amdgcn_sched_barrier(0);
        const bool whole = there == 0xffffffffu && k + 31 <= low && k >= all_from;
        u32x4 weight[RB][2][TERMS];
#pragma unroll
        for (int b = 0; b < RB; ++b) {
            uint32_t seen = 0xffff;
            if (!whole) {
                seen = 0;
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    const int x = (e >> 2) * 8 + half * 4 + (e & 3);
                    const bool on = (there >> x & 1) && k + x <= position[b] && k + x >= oldest[b];
                    seen |= on ? 1u << e : 0u;
                    if (!on) score[b][e] = -__builtin_huge_valf();
                }
            }
            float p[16], w[16], top = 0.0f;
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                p[e] = __builtin_amdgcn_exp2f(__builtin_fmaf(score[b][e], sk[e], -R[b]));
                if (!whole && !(seen >> e & 1)) p[e] = 0.0f;
                w[e] = p[e] * sv[e];
                if (!whole && !(seen >> e & 1)) w[e] = 0.0f;
                top = e ? fmaxf(top, fabsf(w[e])) : fabsf(w[e]);
            }
            if (__any(!(top <= kTop))) {
                float most = kUnset;
#pragma unroll
                for (int e = 0; e < 16; ++e)
                    if (seen >> e & 1)
                        most = fmaxf(most, __builtin_fmaf(score[b][e], sk[e], __builtin_amdgcn_logf(fmaxf(fabsf(sv[e]), 0x1p-100f))));
                most = fmaxf(most, __shfl_xor(most, 32));
                const float next = most > R[b] + kRoom ? most - kRoom : R[b];
                const float down = __builtin_amdgcn_exp2f(R[b] - next);
                R[b] = next;
                l[b] *= down;
#pragma unroll
                for (int d = 0; d < D; ++d) o[b][d] *= down;
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    p[e] = w[e] = 0.0f;
                    if (seen >> e & 1) {
                        p[e] = __builtin_amdgcn_exp2f(__builtin_fmaf(score[b][e], sk[e], -R[b]));
                        w[e] = p[e] * sv[e];
                    }
                }
            }
#pragma unroll
            for (int e = 0; e < 16; ++e) l[b] += p[e];
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const float x[8] = {w[8 * j], w[8 * j + 1], w[8 * j + 2], w[8 * j + 3], w[8 * j + 4], w[8 * j + 5], w[8 * j + 6], w[8 * j + 7]};
                terms_of<TERMS, F::VH>(x, weight[b][j]);
            }
            __builtin_amdgcn_sched_barrier(0);
        }
#pragma unroll
        for (int d = 0; d < D; ++d)
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const int row = d * 32 + n;
                const u32x4 w = shared.v[from][row * 8 + ((i * 4 + j * 2 + half) ^ (row & 7))];
#pragma unroll
                for (int b = 0; b < RB; ++b)
#pragma unroll
                    for (int m = 0; m < TERMS; ++m) mfma32<F::VH>(w, weight[b][j][m], o[b][d]);
            }
    };

    int page = page_of(begin);
    uint64_t there = 0;
    if (begin < end) {
        there = load(begin, page);
        page = page_of(begin + 64);
        if (there) store(0);
    }
    int buffer = 0;
    for (int k = begin; k < end; k += 64, buffer ^= 1) {
        const uint64_t here = there;
        if (here) {
            factors[lane] = k_scale * factor;
            factors[64 + lane] = v_scale;
        }
        __syncthreads();        // this step is in LDS, and the one before is done with its half of it
        const bool more = k + 64 < end;
        if (more) {
            there = load(k + 64, page);
            page = page_of(k + 128);
        }
        __builtin_amdgcn_sched_barrier(0);
        compute(buffer, 0, k, (uint32_t)here);
        __builtin_amdgcn_sched_barrier(0);
        compute(buffer, 1, k + 32, (uint32_t)(here >> 32));
        __builtin_amdgcn_sched_barrier(0);
        if (more && there) store(buffer ^ 1);
    }

    // Rows' results; of pieces their sums, which the work-group that finishes the tile's last piece adds in their order.
#pragma unroll
    for (int b = 0; b < RB; ++b) l[b] += __shfl_xor(l[b], 32);
    const uint64_t stride = (uint64_t)c.tokens * a.heads;
    if (pieces > 1) {
#pragma unroll
        for (int b = 0; b < RB; ++b) {
            if (!mine[b]) continue;
            const uint64_t to = piece * stride + at[b].row * a.heads + at[b].head;
#pragma unroll
            for (int d = 0; d < D; ++d)
#pragma unroll
                for (int i = 0; i < 16; i += 2)
                    publish(g.sums + to * DP + d * 32 + (i >> 2) * 8 + half * 4 + (i & 3), o[b][d][i], o[b][d][i + 1]);
            if (half == 0) publish(g.stats + 2 * to, R[b], l[b]);
        }
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");        // this wave's stores have arrived
        __shared__ int last;
        __syncthreads();
        if (tid == 0) {
            uint32_t* ticket = g.tickets + blockIdx.x;
            last = __hip_atomic_fetch_add(ticket, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == (uint32_t)pieces - 1;
            if (last) __hip_atomic_store(ticket, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        }
        __syncthreads();
        if (!last) return;
#pragma unroll
        for (int b = 0; b < RB; ++b) {
            R[b] = kUnset;
            l[b] = 0.0f;
#pragma unroll
            for (int d = 0; d < D; ++d)
#pragma unroll
                for (int i = 0; i < 16; ++i) o[b][d][i] = 0.0f;
            for (int p = 0; p < pieces; ++p) {
                const uint64_t from = p * stride + at[b].row * a.heads + at[b].head;
                float r, lp;
                published(g.stats + 2 * from, r, lp);
                const float next = fmaxf(R[b], r), down = __builtin_amdgcn_exp2f(R[b] - next), part = __builtin_amdgcn_exp2f(r - next);
                R[b] = next;
                l[b] = l[b] * down + lp * part;
#pragma unroll
                for (int d = 0; d < D; ++d)
#pragma unroll
                    for (int i = 0; i < 16; i += 2) {
                        float x, y;
                        published(g.sums + from * DP + d * 32 + (i >> 2) * 8 + half * 4 + (i & 3), x, y);
                        o[b][d][i] = o[b][d][i] * down + x * part;
                        o[b][d][i + 1] = o[b][d][i + 1] * down + y * part;
                    }
            }
        }
    }
#pragma unroll
    for (int b = 0; b < RB; ++b) {
        if (!mine[b]) continue;
        const float part = l[b] == 0.0f ? 0.0f : 1.0f / l[b];
        T* out = (T*)a.out + at[b].row * a.ldo + at[b].head * c.dim;
#pragma unroll
        for (int d = 0; d < D; ++d)
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const uint32_t x = d * 32 + (i >> 2) * 8 + half * 4 + (i & 3);
                if (x < c.dim) Type<DT>::put(out + x, o[b][d][i] * part);
            }
        if (a.lse && half == 0)
            a.lse[at[b].row * a.heads + at[b].head] = l[b] == 0.0f ? -__builtin_huge_valf() : (R[b] + __builtin_log2f(l[b])) * kLn2;
    }
}

template <int DT, int DP> hipError_t run(const AttentionArgs& g, uint32_t pieces, hipStream_t s) {
    constexpr int RB = many_rows(DT == Q8_F32, DP) / 128;
    void* args[] = {const_cast<AttentionArgs*>(&g)};
    return hipLaunchKernel(reinterpret_cast<const void*>(&many_kernel<DT, DP, RB>), dim3(g.slots * g.a.at.heads, pieces), dim3(kThreads),
                           args, 0, s);
}

}  // namespace

hipError_t launch_many(int dtype, const AttentionArgs& g, uint32_t pieces, hipStream_t s) {
    return for_head(dtype, g.a.at.dim, [&](auto dt, auto dp) { return run<decltype(dt)::value, decltype(dp)::value>(g, pieces, s); });
}

hipError_t prepare_many() {
    hipFuncAttributes a;
    return hipFuncGetAttributes(&a, reinterpret_cast<const void*>(&many_kernel<Q8_F32, 64, 1>));
}

}  // namespace q8
