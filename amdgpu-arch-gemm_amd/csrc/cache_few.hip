// Attention of few new tokens over the paged cache (gfx950): decoding.
#include "cache_attention_device.hpp"

namespace q8 {
namespace {

// Few rows: 16 of a tile, for which memory is what counts.  Each of a work-group's four waves takes 32 keys in
// turn from memory to registers, and their sums meet in LDS at the end.  Of a step's keys, lane l has the
// 16-byte pieces l / 16 of key l % 16 for the scores, and DP / 16 values of eight keys for the second product, those
// whose weights it has.  DP: values of a head, those past dim are 0 in q and left out at the end.
// (32 heads of 128 on 8 of the cache: 64 sequences of up to 8192 keys 134 us, 4.7 TB/s; one of 131072 64, 4.3; one of 4096 13, which
// is latency: launch and tile 5, pages, keys and products 6, the join of 32 pieces 2.)
constexpr int kWaves = 4;
template <int DT, int DP> struct Few {
    static constexpr int TERMS = DT == Q8_F32 ? 3 : 1, BYTES = DP / 16, WORDS = BYTES / 4;
    static constexpr bool QH = DT == Q8_F16, VH = DT != Q8_F32;       // half precision in the products
    static constexpr int PITCH = DP + 4;
    struct Stage {
        uint64_t offset[kWaves][32];
        float scale[kWaves][64];
    };
    struct Sums {
        float o[kWaves][16][PITCH];
        float r[kWaves][16], l[kWaves][16];
    };
    struct Join {
        float o[64 * kWaves * 8 / DP][DP + 4];
        float r[64 * kWaves * 8 / DP], l[64 * kWaves * 8 / DP];
        int last;
    };
    union Shared {
        Stage stage;
        Sums sums;
        Join join;
    };
};

template <int DT, int DP> __global__ void __launch_bounds__(64 * kWaves, DP == 256 ? (DT == Q8_F32 ? 1 : 2) : DT == Q8_F32 ? 2 : DP == 64 ? 4 : 3) few_kernel(const AttentionArgs g) {
    typedef Few<DT, DP> F;
    typedef typename Type<DT>::T T;
    constexpr int TERMS = F::TERMS, S = DP / 64, WORDS = F::WORDS;
    __shared__ typename F::Shared shared;
    __shared__ Far fars[kWaves][16];
    const Attention& a = g.a;
    const Paged& c = a.at;
    const uint32_t kv = blockIdx.x % c.heads, piece = blockIdx.y;
    Place t;
    if (!find_tile(g, blockIdx.x / c.heads, 16, t)) return;
    const int pieces = max(1, pieces_of(t, g.piece));
    if ((int)piece >= pieces) return;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), n = lane & 15, grp = lane >> 4;
    const int begin = t.begin + (int)(piece * g.piece), end = piece_end(t, begin, g.piece);

    // this lane's row of the scores
    const bool mine = n < t.rows;
    const uint32_t token = divide((uint32_t)(t.row + (mine ? n : 0)), g.by_group);
    const uint32_t head = kv * a.group + (uint32_t)(t.row + (mine ? n : 0)) - token * a.group;
    const int position = t.at + (int)token;
    const int64_t oldest = a.window ? (int64_t)position - a.window + 1 : INT32_MIN;
    // keys that every row sees
    const int low = t.at + (int)divide((uint32_t)t.row, g.by_group), high = t.at + (int)divide((uint32_t)(t.row + t.rows - 1), g.by_group);
    const int64_t all_from = a.window ? (int64_t)high - a.window + 1 : INT32_MIN;

    const float factor = a.scale * kLog2e;
    float R = kUnset, l = 0.0f;
    f32x4 o[F::BYTES];
#pragma unroll
    for (int j = 0; j < F::BYTES; ++j) o[j] = f32x4{0, 0, 0, 0};

    const int64_t head_rows = (int64_t)kv * c.page_tokens, page_rows = (int64_t)c.heads * c.page_tokens;
    // What the table says of this lane's key (lane % 32) of the step from key k.  Not looked at before the step's loads: a
    // wait for it would be one for all loads before it.
    const int32_t* pages = c.table + (uint64_t)t.b * c.table_ld;
    auto page_of = [&](int k) __attribute__((always_inline)) { return pages[divide((uint32_t)min(k + (lane & 31), end - 1), c.page)]; };
    // Where the step's keys lie; rows of keys that are not there become those of one that is, and what the padding
    // holds meets zeros of q.
    uint64_t* offset = shared.stage.offset[wave];
    float* factors = shared.stage.scale[wave];
    auto locate = [&](int k, int page, uint32_t& there, float& scale) __attribute__((always_inline)) {
        page = k + (lane & 31) < end && (uint32_t)kept(page) < c.pages ? page : -1;
        there = (uint32_t)__ballot(page >= 0);
        if (!there) return;
        const uint32_t key = (uint32_t)(k + (lane & 31)), slot = key - divide(key, c.page) * c.page_tokens;
        int64_t row = page * page_rows + head_rows + slot;
        const int some = __builtin_ctz(there);
        const int64_t other = (int64_t)((uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(row >> 32), some) << 32 |
                                        (uint32_t)__builtin_amdgcn_readlane((int)row, some));
        row = page < 0 ? other : row;
        scale = (lane < 32 ? c.k_scale : c.v_scale)[row];
        if (lane < 32) offset[lane] = (uint64_t)row * c.pitch;
        __builtin_amdgcn_wave_barrier();
    };
    u32x4 kd[2][S];
    uint32_t vd[8][WORDS];
    auto load_keys = [&]() __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int8_t* base = c.k + offset[i * 16 + n];
#pragma unroll
            for (int s = 0; s < S; ++s) {
                const uint32_t d = s * 64 + grp * 16;
                kd[i][s] = *reinterpret_cast<const u32x4*>(base + (d < c.pitch ? d : 0));
            }
        }
    };
    auto load_values = [&]() __attribute__((always_inline)) {
        const int8_t* base = c.v + (n * F::BYTES < (int)c.pitch ? n * F::BYTES : 0);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const int8_t* from = base + offset[(e >> 2) * 16 + grp * 4 + (e & 3)];
            if constexpr (WORDS == 1) vd[e][0] = *reinterpret_cast<const uint32_t*>(from);
            else if constexpr (WORDS == 2) {
                const u32x2 w = *reinterpret_cast<const u32x2*>(from);
                vd[e][0] = w[0]; vd[e][1] = w[1];
            } else {
                const u32x4 w = *reinterpret_cast<const u32x4*>(from);
#pragma unroll
                for (int m = 0; m < 4; ++m) vd[e][m] = w[m];
            }
        }
        __builtin_amdgcn_wave_barrier();
    };

    // One step's loads ahead: the next keys' once the scores are taken from these, the next values' once these are
    // multiplied, into the same registers; and the pages of the step after are asked for before them.
    constexpr int STRIDE = 32 * kWaves;
    int k0 = begin + wave * 32, page = -1;
    uint32_t there = 0;
    float scale = 0.0f;
    if (k0 < end) {
        page = page_of(k0);
        locate(k0, page, there, scale);
        if (k0 + STRIDE < end) page = page_of(k0 + STRIDE);
        if (there) {
            load_keys();
            load_values();
        }
    }
    u32x4 q[S][2][TERMS];
    {
        const T* row = (const T*)a.q + (uint64_t)(t.first + (int)token) * a.ldq + head * c.dim;
#pragma unroll
        for (int s = 0; s < S; ++s)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const uint32_t d = s * 64 + grp * 16 + h * 8;
                float v[8];
                query<DT>(row, d, c.dim, v);
                terms_of<TERMS, F::QH>(v, q[s][h]);
            }
    }
    while (k0 < end) {
        const uint32_t here = there;
        const float s_here = scale;
        const bool more = k0 + STRIDE < end;
        f32x4 score[2] = {f32x4{0, 0, 0, 0}, f32x4{0, 0, 0, 0}};
        if (here) {
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int s = 0; s < S; ++s) {
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const u32x2 w0 = four<F::QH>(kept(kd[i][s][2 * h])), w1 = four<F::QH>(kept(kd[i][s][2 * h + 1]));
                        const u32x4 w = {w0[0], w0[1], w1[0], w1[1]};
#pragma unroll
                        for (int m = 0; m < TERMS; ++m) mfma16<F::QH>(w, q[s][h][m], score[i]);
                    }
                    if (!F::QH) __builtin_amdgcn_sched_barrier(0);
                }
            factors[lane] = lane < 32 ? s_here * factor : s_here;
        }
        __builtin_amdgcn_sched_barrier(0);
        if (more) {
            locate(k0 + STRIDE, page, there, scale);
            page = k0 + 2 * STRIDE < end ? page_of(k0 + 2 * STRIDE) : -1;
            if (there) load_keys();
        }
        __builtin_amdgcn_sched_barrier(0);
        if (here) {
            float sk[8], sv[8], w[8];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const f32x4 ks = *reinterpret_cast<const f32x4*>(factors + i * 16 + grp * 4);
                const f32x4 vs = *reinterpret_cast<const f32x4*>(factors + 32 + i * 16 + grp * 4);
#pragma unroll
                for (int e = 0; e < 4; ++e) { sk[4 * i + e] = ks[e]; sv[4 * i + e] = vs[e]; }
            }
            __builtin_amdgcn_wave_barrier();
            // keys that this row sees, if not all do
            uint32_t seen = 0xff;
            const bool whole = here == 0xffffffffu && k0 + 31 <= low && k0 >= all_from;
            if (!whole) {
                seen = 0;
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const int k = (e >> 2) * 16 + grp * 4 + (e & 3);
                    const bool on = (here >> k & 1) && k0 + k <= position && k0 + k >= oldest;
                    seen |= on ? 1u << e : 0u;
                    if (!on) { score[e >> 2][e & 3] = -__builtin_huge_valf(); sk[e] = 1.0f; sv[e] = 0.0f; }
                }
            }
            float top, sum;
            auto weigh = [&](auto exponent_of) __attribute__((always_inline)) {
                float p[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    p[e] = __builtin_amdgcn_exp2f(exponent_of(score[e >> 2][e & 3], sk[e]));
                    w[e] = p[e] * sv[e];
                }
                if (!whole) {
#pragma unroll
                    for (int e = 0; e < 8; ++e)
                        if (!(seen >> e & 1)) p[e] = w[e] = 0.0f;
                }
                sum = l;
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    sum += p[e];
                    top = e ? fmaxf(top, fabsf(w[e])) : fabsf(w[e]);
                }
            };
            auto less_R = [&](float t, float k) __attribute__((always_inline)) { return __builtin_fmaf(t, k, -R); };
            weigh(less_R);
            // (a product with a scale of 0 may be no number, which fmaxf passes over; the exponential then is infinite)
            if (__any(!(top <= kTop) || !(sum <= kMostSum))) {
                Reference r(R, &fars[wave][kept((uint32_t)n)]);
                const float down = moved<16>(r, l, kRoom, [&](auto each) __attribute__((always_inline)) {
                    const uint32_t mask = kept(seen);
#pragma unroll
                    for (int e = 0; e < 8; ++e) each(mask >> e & 1, score[e >> 2][e & 3], sk[e], sv[e]);
                });
                R = r.R;
                r.keep(&fars[wave][kept((uint32_t)n)]);
                l *= down;
#pragma unroll
                for (int j = 0; j < F::BYTES; ++j) o[j] *= down;
                if (__builtin_expect(__any(r.is_far()), 0)) {
                    const Reference wide(R, &fars[wave][kept((uint32_t)n)]);
                    weigh([&](float t, float k) __attribute__((always_inline)) { return exponent(wide, t, k); });
                } else {
                    weigh(less_R);
                }
            }
            l = sum;
            u32x4 weight[TERMS];
            terms_of<TERMS, F::VH>(w, weight);
            auto multiply = [&](auto word) __attribute__((always_inline)) {
                constexpr int W = decltype(word)::value;
                uint32_t v[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) v[e] = kept(vd[e][W]);
                u32x4 vj[4];
                columns<F::VH>(v, vj);
#pragma unroll
                for (int j = 0; j < 4; ++j)
#pragma unroll
                    for (int m = 0; m < TERMS; ++m) mfma16<F::VH>(vj[j], weight[m], o[4 * W + j]);
                __builtin_amdgcn_sched_barrier(0);
            };
            multiply(Int<0>{});
            if constexpr (WORDS > 1) multiply(Int<1>{});
            if constexpr (WORDS > 2) {
                multiply(Int<2>{});
                multiply(Int<3>{});
            }
        }
        if (more && there) load_values();
        __builtin_amdgcn_sched_barrier(0);
        k0 += STRIDE;
    }
    // the waves' sums: each lane has values 8 (4 grp + i) .. of row n (DP 128), and of l what its keys had
    l += __shfl_xor(l, 16);
    l += __shfl_xor(l, 32);
    const float up = without_rest(Reference(R, &fars[wave][n]), R, l);
#pragma unroll
    for (int j = 0; j < F::BYTES; ++j) o[j] *= up;
    __syncthreads();        // every wave is done with its stage
    typename F::Sums& sums = shared.sums;
    if (grp == 0) { sums.r[wave][n] = R; sums.l[wave][n] = l; }
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < F::BYTES; j += 4)
            *reinterpret_cast<f32x4*>(&sums.o[wave][n][(4 * grp + i) * F::BYTES + j]) = f32x4{o[j][i], o[j + 1][i], o[j + 2][i], o[j + 3][i]};
    __syncthreads();
    // a row's result
    auto finish = [&](int r, int d, float most, float total, float (&v)[8]) __attribute__((always_inline)) {
        const Row at = row_of(g, t, kv, r);
        const float part = total == 0.0f ? 0.0f : 1.0f / total;
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] *= part;
        if (d < (int)c.dim) store_part<DT>((T*)a.out + at.row * a.ldo + at.head * c.dim, d, c.dim, v);
        if (a.lse && d == 0)
            a.lse[at.row * a.heads + at.head] = total == 0.0f ? -__builtin_huge_valf() : (most + __builtin_log2f(total)) * kLn2;
    };
    constexpr int ACROSS = DP / 8, LANES = 64 * kWaves / ACROSS;      // threads of a row's values, rows of threads
    const int d = threadIdx.x % ACROSS * 8, part = threadIdx.x / ACROSS;
    for (int r = part; r < t.rows; r += LANES) {
        float most = kUnset, total = 0.0f, v[8] = {};
#pragma unroll
        for (int w = 0; w < kWaves; ++w) most = fmaxf(most, sums.r[w][r]);
#pragma unroll
        for (int w = 0; w < kWaves; ++w) {
            const float down = __builtin_amdgcn_exp2f(sums.r[w][r] - most);
            total = __builtin_fmaf(sums.l[w][r], down, total);
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = __builtin_fmaf(sums.o[w][r][d + e], down, v[e]);
        }
        if (pieces > 1) {
            const Row at = row_of(g, t, kv, r);
            const uint64_t to = ((uint64_t)piece * c.tokens + at.row) * a.heads + at.head;
            const float down = settle(most, total);
#pragma unroll
            for (int e = 0; e < 8; e += 2) publish(g.sums + to * DP + d + e, v[e] * down, v[e + 1] * down);
            if (d == 0) publish(g.stats + 2 * to, most, total);
        } else {
            finish(r, d, most, total, v);
        }
    }
    if (pieces == 1) return;

    // The work-group that finishes a tile's last piece adds them, in the pieces' order whichever it is.
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");        // this wave's stores have arrived
    __syncthreads();
    if (threadIdx.x == 0) {
        uint32_t* ticket = g.tickets + blockIdx.x;
        const bool last = __hip_atomic_fetch_add(ticket, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == (uint32_t)pieces - 1;
        if (last) __hip_atomic_store(ticket, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        shared.join.last = last;
    }
    __syncthreads();
    if (!shared.join.last) return;
    // rows and slices of the pieces over the rows of threads; slices meet in LDS
    int held = 1;
    while (held < t.rows && held < LANES) held *= 2;
    const int slices = LANES / held, slice = part / held;
    const uint64_t stride = (uint64_t)c.tokens * a.heads;
    for (int r0 = 0; r0 < t.rows; r0 += held) {
        const int r = r0 + part % held;
        float most = kUnset, total = 0.0f, v[8] = {};
        if (r < t.rows) {
            const Row at = row_of(g, t, kv, r);
            const uint64_t first = at.row * a.heads + at.head;
            constexpr int AHEAD = 4;
            for (int p0 = slice; p0 < pieces; p0 += slices * AHEAD) {
                float o[AHEAD][8], rp[AHEAD], lp[AHEAD];
#pragma unroll
                for (int i = 0; i < AHEAD; ++i) {
                    const uint64_t from = first + (uint64_t)min(p0 + i * slices, pieces - 1) * stride;
                    published(g.stats + 2 * from, rp[i], lp[i]);
#pragma unroll
                    for (int e = 0; e < 8; e += 2) published(g.sums + from * DP + d + e, o[i][e], o[i][e + 1]);
                }
#pragma unroll
                for (int i = 0; i < AHEAD; ++i) {
                    if (p0 + i * slices >= pieces) continue;
                    add_part(most, total, v, rp[i], lp[i], o[i]);
                }
            }
        }
        __syncthreads();
        shared.join.r[part] = most;
        shared.join.l[part] = total;
        *reinterpret_cast<f32x4*>(&shared.join.o[part][d]) = f32x4{v[0], v[1], v[2], v[3]};
        *reinterpret_cast<f32x4*>(&shared.join.o[part][d + 4]) = f32x4{v[4], v[5], v[6], v[7]};
        __syncthreads();
        if (slice == 0 && r < t.rows) {
            for (int x = 1; x < slices; ++x) {
                const int from = x * held + part;
                float o[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) o[e] = shared.join.o[from][d + e];
                add_part(most, total, v, shared.join.r[from], shared.join.l[from], o);
            }
            finish(r, d, most, total, v);
        }
    }
}

template <int DT, int DP> hipError_t run(const AttentionArgs& g, uint32_t pieces, hipStream_t s) {
    void* args[] = {const_cast<AttentionArgs*>(&g)};
    return hipLaunchKernel(reinterpret_cast<const void*>(&few_kernel<DT, DP>), dim3(g.slots * g.a.at.heads, pieces), dim3(64 * kWaves),
                           args, 0, s);
}

}  // namespace

hipError_t launch_few(int dtype, const AttentionArgs& g, uint32_t pieces, hipStream_t s) {
    return for_head(dtype, g.a.at.dim, [&](auto dt, auto dp) { return run<decltype(dt)::value, decltype(dp)::value>(g, pieces, s); });
}

hipError_t prepare_few() {
    hipFuncAttributes a;
    return hipFuncGetAttributes(&a, reinterpret_cast<const void*>(&few_kernel<Q8_F32, 64>));
}

}  // namespace q8
